"""The global gradient norm and clipping (gcodec.clip) on the GPU, against the
formulas in 64 bits.

Tolerances.  u(t) = eps / 2 is a rounding to type t, relative to the value.
  norm   a sum of 64-bit terms (each off by 2^-53 at most, the sum of n < 2^33 of
         them in a tree by less than 64 * 2^-53), then one rounding to float32:
         2^-24 (1 + 2^-20)
  clip   c rounds once to float32 (2^-24), the product once (2^-24), the result
         once to its type: (1 + 2^-24)^2 (1 + u) - 1 < (2^-23 + u)(1 + 2^-6); for
         a float32 result the product is the result: 2^-23 (1 + 2^-6).  Below the
         normal range a rounding is off by half the smallest subnormal, absolutely.
  decode a value rounds 4 times before c: k = RN(norm / s), alpha to float32, RN(k Q),
         RN(. alpha); a norm of such values is off by as much and rounds once
         itself (5 times 2^-24), and c takes the norm's 4 (8 more for a result)."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # collected on CPU, skipped there
    pytest.skip("no GPU", allow_module_level=True)

import gcodec  # noqa: E402
from gcodec import codec, shapes  # noqa: E402

DEV = torch.device("cuda", 0)
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF = math.inf

RAGGED = [0, 1, 3, 4, 5, 17, 1000, 0, 4099, 70_001, 2, 250_000, 7, 0, 64, 65]
LISTS = {
    "one": [1],
    "only empty": [0, 0],
    "empty ends": [0, 2047, 0],
    "a tile": [2048],
    "past a tile": [2049],
    "vector ends": [255, 256, 257, 511, 512, 513, 7, 8, 9],
    "ragged": RAGGED,
    "one block's": [32_767, 2],
    "tiny, past the LDS table": [i % 8 for i in range(1500)],
    "only empty, past the LDS table": [0] * 1100,
    "many, past the LDS table": [1500 + i % 9 for i in range(1100)],
    "small": [83 + 7 * (i % 5) for i in range(120)],
    "small among large": [300_000] + [40] * 300 + [70_001, 0, 5],
    "several blocks": [1_000_003, 12, 2_000_001],
}
UNIT = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}


def types_of(kind, count):
    return {"fp32": [F32] * count, "fp16": [F16] * count, "bf16": [BF16] * count,
            "mixed": [(F32, BF16, F16)[i % 3] for i in range(count)]}[kind]


def carve(sizes, types, seed, scale=1.0, misalign=True):
    """Tensors cut from one buffer a type at element offsets of every alignment, with a guard of 7.0 between them."""
    rng = np.random.default_rng(seed)
    out = []
    for s, t in zip(sizes, types):
        gap = int(rng.integers(1, 16)) if misalign else 16
        buf = torch.full((gap + s + 16,), 7.0, dtype=t, device=DEV)
        v = buf[gap:gap + s]
        v.copy_(torch.from_numpy((rng.standard_normal(s) * scale * 2.0 ** rng.integers(-3, 4)).astype(np.float32)))
        out.append((buf, gap, v))
    return out


def views(carved):
    return [v for _, _, v in carved]


def guards_hold(carved):
    for buf, gap, v in carved:
        assert bool((buf[:gap] == 7).all()) and bool((buf[gap + v.numel():] == 7).all())


def f64(ts):
    return [t.detach().cpu().double().numpy().reshape(-1) for t in ts]


def norm64(xs, p):
    """The formula in 64 bits, exactly rounded sums."""
    x = np.abs(np.concatenate(xs)) if xs else np.zeros(0)
    if x.size == 0:
        return 0.0
    if p == INF:
        return float(x.max())
    if not np.isfinite(x).all():
        return float("nan") if np.isnan(x).any() else INF
    return math.fsum(x) if p == 1 else math.sqrt(math.fsum(x * x))


def coef64(n, max_norm):
    q = max_norm / (n + 1e-6)
    return 1.0 if q > 1.0 else q


def close_norm(got, want, roundings=1):
    got = float(got)
    if math.isnan(want) or math.isinf(want):
        assert math.isnan(got) == math.isnan(want) and (math.isnan(want) or got == want)
    else:
        assert abs(got - want) <= roundings * 2.0 ** -24 * (1 + 2.0 ** -6) * want, (got, want)


def close_values(got, want, extra=0):
    """got tensors of their types against 64-bit values; `extra` more float32 roundings"""
    for g, w in zip(got, want):
        u = UNIT[g.dtype]
        rel = ((2 + extra) * 2.0 ** -24 + (u if g.dtype != F32 else 0.0)) * (1 + 2.0 ** -6)
        tol = rel * np.abs(w) + TINY[g.dtype] * 0.5 + (1 + extra) * 2.0 ** -150
        err = np.abs(g.detach().cpu().double().numpy().reshape(-1) - w)
        assert (err <= tol).all(), (g.dtype, g.shape, float((err - tol).max()))


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("p", [1, 2, INF])
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16", "mixed"])
@pytest.mark.parametrize("name", list(LISTS))
def test_norm(name, kind, p):
    sizes = LISTS[name]
    ts = views(carve(sizes, types_of(kind, len(sizes)), seed=len(sizes)))
    xs = f64(ts)
    close_norm(gcodec.grad_norm(ts, p), norm64(xs, p))
    total, each = gcodec.grad_norm(gcodec.Grads(ts), p, per_tensor=True)
    close_norm(total, norm64(xs, p))
    assert each.shape == (len(sizes),) and each.dtype == F32
    for e, x in zip(each.tolist(), xs):
        close_norm(e, norm64([x], p))


@pytest.mark.parametrize("p", [1, 2, INF])
@pytest.mark.parametrize("scale", [1e-30, 1e-42, 1e30])
def test_norm_of_extreme_gradients(scale, p):
    """Squares that float32 cannot hold, and subnormal elements."""
    ts = views(carve([5000, 33, 1], [F32] * 3, seed=3, scale=scale))
    want = norm64(f64(ts), p)
    got = float(gcodec.grad_norm(ts, p))
    assert abs(got - want) <= 2.0 ** -24 * (1 + 2.0 ** -6) * want + 2.0 ** -150


@pytest.mark.parametrize("p", [1, 2, INF])
@pytest.mark.parametrize("bad", [INF, -INF, math.nan])
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
def test_norm_carries_infinities_and_nan(kind, bad, p):
    ts = views(carve([3000, 70, 9], types_of(kind, 3), seed=5))
    ts[1][69] = bad
    total, each = gcodec.grad_norm(ts, p, per_tensor=True)
    want = math.nan if math.isnan(bad) else INF
    close_norm(total, want)
    close_norm(each[1], want)
    assert math.isfinite(each[0]) and math.isfinite(each[2])
    ts[0][0] = math.nan  # a NaN is above an infinity
    close_norm(gcodec.grad_norm(ts, p), math.nan)
    with pytest.raises(RuntimeError, match="not finite"):
        gcodec.grad_norm(ts, p, error_if_nonfinite=True)


def test_norm_repeats_bit_for_bit():
    ts = views(carve([3_000_001, 5, 40_000], [F32, BF16, F16], seed=8))
    g = gcodec.Grads(ts)
    first = gcodec.grad_norm(g, 2, per_tensor=True)
    for _ in range(5):
        again = gcodec.grad_norm(ts, 2, per_tensor=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_norm_past_32_bit_offsets():
    """2^32 + 70,001 elements, two tensors: the far end counts and is clipped, the rest stays."""
    n = 2 ** 32 + 65_536
    a, b = torch.zeros(n, dtype=BF16, device=DEV), torch.zeros(4465, dtype=BF16, device=DEV)
    a[-1], a[2 ** 32 + 1], a[3], b[-1] = 3.0, 4.0, 12.0, 84.0
    assert float(gcodec.grad_norm([a, b], 2)) == 85.0  # sqrt(9 + 16 + 144 + 7056)
    assert float(gcodec.grad_norm([a, b], INF)) == 84.0
    total, each = gcodec.grad_norm([a, b], 1, per_tensor=True)
    assert float(total) == 103.0 and each.tolist() == [19.0, 84.0]
    w, v = torch.nn.Parameter(a), torch.nn.Parameter(b)  # the gradient is the parameter itself: in place
    w.grad, v.grad = w.data, v.data
    gcodec.clip_grad_norm_([w, v], 42.5)
    assert [float(x) for x in (a[-1], a[2 ** 32 + 1], a[3], b[-1])] == [1.5, 2.0, 6.0, 42.0]
    assert int(torch.count_nonzero(a)) == 3 and int(torch.count_nonzero(b)) == 1


# ---------------------------------------------------------------------------
# clip
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("factor", [0.37, 3.0])
@pytest.mark.parametrize("p", [1, 2, INF])
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16", "mixed"])
@pytest.mark.parametrize("name", list(LISTS))
def test_clip_list_to_list(name, kind, p, factor):
    sizes = LISTS[name]
    types = types_of(kind, len(sizes))
    src, dst = carve(sizes, types, seed=11), carve(sizes, types[1:] + types[:1], seed=12)
    xs = f64(views(src))
    n = norm64(xs, p)
    m = factor * n if n else 1.0
    version = views(dst)[0]._version
    total = gcodec.clip_grads(views(src), views(dst), m, p)
    close_norm(total, n)
    close_values(views(dst), [x * coef64(n, m) for x in xs])
    guards_hold(dst)
    assert views(dst)[0]._version > version  # autograd sees the write
    for x, t in zip(xs, views(src)):
        assert np.array_equal(x, t.cpu().double().numpy())  # read only


@pytest.mark.parametrize("p", [1, 2, INF])
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16", "mixed"])
@pytest.mark.parametrize("name", ["one", "ragged", "tiny, past the LDS table", "several blocks"])
def test_clip_in_place(name, kind, p):
    sizes = LISTS[name]
    grads = carve(sizes, types_of(kind, len(sizes)), seed=21)
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in views(grads)]
    params.insert(1, torch.nn.Parameter(torch.zeros(3, device=DEV)))  # without a gradient
    for q, g in zip(params[:1] + params[2:], views(grads)):
        q.grad = g
    xs = f64(views(grads))
    n = norm64(xs, p)
    before = [g.clone() for g in views(grads)]
    version = views(grads)[0]._version
    close_norm(gcodec.clip_grad_norm_(params, 2 * n + 1, p), n)  # under the limit: nothing changes
    for a, b in zip(before, views(grads)):
        assert torch.equal(a, b)
    close_norm(gcodec.clip_grad_norm_(iter(params), 0.4 * n, p), n)
    close_values(views(grads), [x * coef64(n, 0.4 * n) for x in xs])
    guards_hold(grads)
    assert views(grads)[0]._version > version  # autograd sees the write


def test_clip_agrees_with_the_trainer_call():
    """torch.nn.utils.clip_grad_norm_ on float32: its norm is a float32 sum, here within 2^-16 of ours."""
    grads = views(carve(shapes.vgg16_sizes()[:20], [F32] * 20, seed=31, scale=1e-2))
    mine = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    ref = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for a, b, g in zip(mine, ref, grads):
        a.grad, b.grad = g.clone(), g.clone()
    na, nb = gcodec.clip_grad_norm_(mine, 1.0), torch.nn.utils.clip_grad_norm_(ref, 1.0)
    assert na.shape == nb.shape and na.dtype == nb.dtype
    torch.testing.assert_close(na, nb, rtol=2.0 ** -16, atol=0)
    for a, b in zip(mine, ref):
        torch.testing.assert_close(a.grad, b.grad, rtol=2.0 ** -15, atol=0)


@pytest.mark.parametrize("max_norm", [0.0, INF, 1.0])
@pytest.mark.parametrize("bad", [None, INF, -INF, math.nan])
def test_clip_limits_and_nonfinite_gradients(bad, max_norm):
    """max_norm 0 clears, infinity leaves; an infinite norm gives c = 0 (NaN where the gradient is infinite, 0
    elsewhere), a NaN or infinity over infinity NaN everywhere: the formula's own values."""
    ts = views(carve([300, 5000], [F32, BF16], seed=41))
    if bad is not None:
        ts[0][7] = bad
    xs = f64(ts)
    n = norm64(xs, 2)
    with np.errstate(invalid="ignore", divide="ignore"):
        c = np.float64(max_norm) / (np.float64(n) + 1e-6)
        c = 1.0 if c > 1.0 else c
        want = [x * c for x in xs]
    outs = [torch.full_like(t, 5.0) for t in ts]
    close_norm(gcodec.clip_grads(ts, outs, max_norm), n)
    for o, w in zip(outs, want):
        g = o.cpu().double().numpy()
        assert np.array_equal(np.isnan(g), np.isnan(w))
        ok = ~np.isnan(w)
        assert (np.abs(g[ok] - w[ok]) <= (2.0 ** -23 + UNIT[o.dtype]) * 1.02 * np.abs(w[ok])).all()
    if bad is not None:
        params = [torch.nn.Parameter(torch.zeros_like(t)) for t in ts]
        for q, t in zip(params, ts):
            q.grad = t
        with pytest.raises(RuntimeError, match="not finite"):
            gcodec.clip_grad_norm_(params, max_norm, error_if_nonfinite=True)
        for x, t in zip(xs, ts):
            assert np.array_equal(x, t.cpu().double().numpy(), equal_nan=True)  # raised before anything was written


def test_clip_partly_in_place_and_dense_orders():
    a, b = views(carve([1000, 300], [F32, BF16], seed=51))
    out = torch.zeros(300, device=DEV)
    xs = f64([a, b])
    n = norm64(xs, 2)
    gcodec.clip_grads([a, b], [a, out], 0.5 * n)  # the first onto itself, the second elsewhere
    close_values([a, out], [x * coef64(n, 0.5 * n) for x in xs])
    w = torch.nn.Parameter(torch.randn(8, 6, 5, 4, device=DEV).to(memory_format=torch.channels_last))
    w.grad = torch.randn(8, 6, 5, 4, device=DEV).to(memory_format=torch.channels_last)
    assert not w.grad.is_contiguous()
    x = w.grad.cpu().double().numpy()
    n = norm64([x.reshape(-1)], 2)
    close_norm(gcodec.grad_norm([w.grad]), n)
    gcodec.clip_grad_norm_(w, 0.5 * n)  # one parameter, not a list
    close_values([w.grad.contiguous()], [(x * coef64(n, 0.5 * n)).reshape(-1)])


def test_refusals():
    x = torch.ones(8, 8, device=DEV)
    y = torch.ones(64, device=DEV)
    E = gcodec.GCodecError
    for bad in ([x[:, :4]], [x.t()], [x.double()], [x.to(torch.int32)], [x.cpu()], [x, x.cpu()], [x.to_sparse()], []):
        with pytest.raises(E):
            gcodec.Grads(bad)
    with pytest.raises(E, match="not dense"):
        gcodec.grad_norm([x[:, :4]])
    with pytest.raises(E, match="not dense"):
        gcodec.grad_norm([y[:1].expand(4)])
    with pytest.raises(E, match="share memory"):
        gcodec.clip_grads([y, y], [y, y], 1.0)
    with pytest.raises(E, match="shares memory"):
        gcodec.clip_grads([y[:32]], [y[16:48]], 1.0)
    with pytest.raises(E, match="sizes"):
        gcodec.clip_grads([x, y], [y[:63], torch.empty(65, device=DEV)], 1.0)
    with pytest.raises(E, match="tensors into"):
        gcodec.clip_grads([x, y], [torch.empty_like(y)], 1.0)
    with pytest.raises(E, match="flat"):
        gcodec.flatten_clip([y], 1.0, flat=torch.empty(63, device=DEV))
    with pytest.raises(E, match="float32"):
        gcodec.flatten_clip([y], 1.0, flat=torch.empty(64, device=DEV, dtype=F16))
    with pytest.raises(E, match="flat bucket"):
        gcodec.flatten_clip([y], 1.0, flat=y)
    words = torch.zeros(codec.qsgd_layout(64, 4).plane_words, dtype=torch.int32, device=DEV)
    one = torch.ones(1, device=DEV)
    for w, kw, msg in [(words[:4], {}, "needed"), (words.float(), {}, "int32"), (words.cpu(), {}, "GPU only"),
                       (words, dict(lanes=codec.qsgd_layout(63, 4)), "n=63"), (words, dict(lanes=codec.qsgd_layout(64, 2)), "lanes")]:
        with pytest.raises(E, match=msg):
            gcodec.qsgd_decode_clip(w, one, 4, [torch.empty(64, device=DEV)], 1.0, **kw)
    with pytest.raises(E, match="empty norm"):
        gcodec.qsgd_decode_clip(words, one[:0], 4, [torch.empty(64, device=DEV)], 1.0)


# ---------------------------------------------------------------------------
# flatten
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("factor", [0.37, 3.0])
@pytest.mark.parametrize("p", [1, 2, INF])
@pytest.mark.parametrize("kind", ["fp32", "bf16", "mixed"])
@pytest.mark.parametrize("name", list(LISTS))
def test_flatten(name, kind, p, factor):
    sizes = LISTS[name]
    ts = views(carve(sizes, types_of(kind, len(sizes)), seed=61))
    xs = f64(ts)
    n = norm64(xs, p)
    m = factor * n if n else 1.0
    store = torch.full((sum(sizes) + 9,), 7.0, device=DEV)
    out = store[5:5 + sum(sizes)]
    flat, peak, total = gcodec.flatten_clip(ts, m, p, flat=out)
    assert flat.data_ptr() == out.data_ptr() and peak.shape == (1,)
    close_norm(total, n)
    close_values([flat], [np.concatenate(xs) * coef64(n, m)])
    assert bool((store[:5] == 7).all()) and bool((store[5 + sum(sizes):] == 7).all())
    assert float(peak) == (float(flat.abs().max()) if flat.numel() else 0.0)  # the codec's max-norm, exactly


@pytest.mark.parametrize("bad", [INF, math.nan])
def test_flatten_nonfinite(bad):
    ts = views(carve([100, 3000], [F32, BF16], seed=62))
    ts[1][8] = bad
    flat, peak, total = gcodec.flatten_clip(ts, 1.0)
    assert math.isnan(float(peak)) and math.isnan(float(flat.abs().max()))
    close_norm(total, bad)


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------
def packed(n, bits, world, seed, norm=0.02):
    """Words of random levels summed over `world` ranks, by the codec's own packer."""
    rng = np.random.default_rng(seed)
    s = (1 << bits) - 1
    q = np.zeros(n, dtype=np.int64)
    for _ in range(world):
        q += np.clip(np.rint(rng.standard_normal(n) * s / 4), -s, s).astype(np.int64)
    if n:
        q[0] = world * s
    lanes = codec.qsgd_layout(n, bits, world)
    words = torch.zeros(lanes.plane_words, dtype=torch.int64, device=DEV)
    lane = torch.from_numpy(q + world * s).to(DEV)
    for k in range(lanes.per_word):
        part = lane[k * lanes.plane_words:(k + 1) * lanes.plane_words]
        words[:part.numel()] += part << (k * lanes.bits)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    return words, q, torch.tensor([norm], dtype=F32, device=DEV)


@pytest.mark.parametrize("factor", [0.37, 3.0])
@pytest.mark.parametrize("bits,world,p", [(1, 1, 2), (2, 1, 1), (4, 1, 2), (4, 1, INF), (4, 3, 2), (8, 8, 2), (8, 1, 1),
                                          (12, 2, 2), (16, 8, 2), (20, 1, 1), (24, 1, INF)])
@pytest.mark.parametrize("name,kind", [("one", "fp32"), ("empty ends", "bf16"), ("ragged", "mixed"), ("ragged", "fp32"),
                                       ("tiny, past the LDS table", "fp16"), ("several blocks", "bf16"),
                                       ("many, past the LDS table", "mixed"), ("small among large", "mixed")])
def test_decode(name, kind, bits, world, p, factor):
    sizes = LISTS[name]
    n = sum(sizes)
    words, q, norm = packed(n, bits, world, seed=bits)
    dst = carve(sizes, types_of(kind, len(sizes)), seed=71)
    flat = q * (float(norm) / ((1 << bits) - 1) / world)
    parts = np.split(flat, np.cumsum(sizes)[:-1])
    want = norm64([flat], p)
    m = factor * want
    total = gcodec.qsgd_decode_clip(words, norm, bits, views(dst), m, p, world=world, alpha=1.0 / world)
    close_norm(total, want, roundings=5)
    close_values(views(dst), [x * coef64(want, m) for x in parts], extra=8)
    guards_hold(dst)


@pytest.mark.parametrize("bits,world", [(2, 1), (4, 3), (8, 8), (16, 1)])
def test_decode_unclipped_is_the_decode(bits, world):
    """Under the limit the values are qsgd_decode_segments' own, bit for bit."""
    ts = views(carve(RAGGED, [F32] * len(RAGGED), seed=81))
    us = views(carve(RAGGED, [F32] * len(RAGGED), seed=82))
    words, _, norm = packed(sum(RAGGED), bits, world, seed=9)
    codec.qsgd_decode_segments(words, norm, bits, codec.Segments(ts), world, 1.0 / world)
    gcodec.qsgd_decode_clip(words, norm, bits, us, INF, world=world, alpha=1.0 / world)
    for a, b in zip(ts, us):
        assert torch.equal(a.view(torch.int32), b.view(torch.int32))


@pytest.mark.parametrize("p", [1, 2, INF])
@pytest.mark.parametrize("norm", [0.0, 1e-44, 1e-20, 3e38, INF, math.nan])
def test_decode_extreme_norms(norm, p):
    """The norm is that of the decoded values also where they leave the normal range or are not finite."""
    words, q, nt = packed(5000, 4, 2, seed=3, norm=norm)
    plain = [torch.empty(5000, device=DEV)]
    codec.qsgd_decode_segments(words, nt, 4, codec.Segments(plain), 2, 1.0)  # alpha 1: W max-norms may pass float32
    xs = f64(plain)
    want = norm64(xs, p)
    out = [torch.empty(5000, device=DEV)]
    total = gcodec.qsgd_decode_clip(words, nt, 4, out, 1.0, p, world=2, alpha=1.0)
    if want > 3.4028235e38:
        want = INF
    if math.isfinite(want):
        assert abs(float(total) - want) <= 2.0 ** -22 * want + 2.0 ** -150
    else:
        close_norm(total, want)
    with np.errstate(invalid="ignore", divide="ignore"):
        w64 = norm64(xs, p)
        w = xs[0] * coef64(w64, 1.0)
    g = out[0].cpu().double().numpy()
    assert np.array_equal(np.isnan(g), np.isnan(w))
    ok = ~np.isnan(w)
    assert (np.abs(g[ok] - w[ok]) <= 2.0 ** -22 * np.abs(w[ok]) + 2.0 ** -149).all()


# ---------------------------------------------------------------------------
# together, streams, graphs
# ---------------------------------------------------------------------------
def test_a_step_with_all_of_them():
    """Local clipping into the codec, and the reduced gradient clipped as it is decoded (one rank)."""
    sizes = [27, 64, 0, 1000, 3, 4099, 10, 70_001]
    ts = views(carve(sizes, types_of("mixed", len(sizes)), seed=91, scale=0.01))
    outs = carve(sizes, types_of("mixed", len(sizes)), seed=92)
    xs = f64(ts)
    flat, peak, total = gcodec.flatten_clip(ts, 0.5)
    close_norm(total, norm64(xs, 2))
    words = codec.qsgd_encode(flat, peak, 8, gcodec.Generator(5, "philox").reserve(flat.numel()))
    dense = codec.qsgd_decode(words, flat.numel(), peak, 8)
    n = gcodec.qsgd_decode_clip(words, peak, 8, views(outs), 0.3)
    want = dense.cpu().double().numpy()
    close_norm(n, norm64([want], 2), roundings=4)
    c = coef64(norm64([want], 2), 0.3)
    close_values(views(outs), [x * c for x in np.split(want, np.cumsum(sizes)[:-1])], extra=1)
    after = gcodec.grad_norm(views(outs))
    assert abs(float(after) - 0.3) < 0.3 * 2.0 ** -7  # what was stored has the limit's norm, to bf16's rounding


def test_two_streams_at_once():
    a = views(carve([2_000_001, 17], [F32, BF16], seed=101))
    b = views(carve([1_500_000, 999], [BF16, F32], seed=102))
    ga, gb = gcodec.Grads(a), gcodec.Grads(b)
    wa, wb = gcodec.grad_norm(ga), gcodec.grad_norm(gb)
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        with torch.cuda.stream(sa):
            got.append((gcodec.grad_norm(ga), wa))
        with torch.cuda.stream(sb):
            got.append((gcodec.grad_norm(gb), wb))
            got.append((gcodec.grad_norm(ga), wa))  # one table on two streams
    torch.cuda.synchronize()
    for x, w in got:
        assert torch.equal(x, w)


def test_captured_and_replayed():
    """Two graphs, lists and tables, replayed between eager calls with new gradients each time."""
    src, dst = carve(RAGGED, types_of("mixed", len(RAGGED)), seed=111), carve(RAGGED, [F32] * len(RAGGED), seed=112)
    s, d = views(src), views(dst)
    gs, gd = gcodec.Grads(s), gcodec.Grads(d)
    gcodec.clip_grads(gs, gd, 1.0)
    torch.cuda.synchronize()
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        n1 = gcodec.clip_grads(gs, gd, 1.0)
        with pytest.raises(gcodec.GCodecError, match="capture"):
            gcodec.Grads(s)
    with torch.cuda.graph(two):
        flat, peak, n2 = gcodec.flatten_clip(s, 2.0)
        n3, each = gcodec.grad_norm(s, 1, per_tensor=True)
    for step in range(4):
        with torch.no_grad():
            for t in s:
                t.mul_(-1.5)
        xs = f64(s)
        two.replay()
        one.replay()
        close_norm(gcodec.grad_norm(s, INF), norm64(xs, INF))  # eager work between the replays
        torch.cuda.synchronize()
        n = norm64(xs, 2)
        close_norm(n1, n)
        close_norm(n2, n)
        close_norm(n3, norm64(xs, 1))
        close_values(d, [x * coef64(n, 1.0) for x in xs])
        close_values([flat], [np.concatenate(xs) * coef64(n, 2.0)])
        assert float(peak) == float(flat.abs().max())
        for e, x in zip(each.tolist(), xs):
            close_norm(e, norm64([x], 1))


def test_table_keeps_its_memory():
    """A table made of tensors that are dropped still reads their memory, not a later tensor's."""
    t = torch.full((1 << 20,), 2.0, device=DEV)
    g = gcodec.Grads([t])
    del t
    other = [torch.full((1 << 20,), 9.0, device=DEV) for _ in range(4)]
    assert float(gcodec.grad_norm(g, INF)) == 2.0
    del other


# ---------------------------------------------------------------------------
# the reducers' options (one rank)
# ---------------------------------------------------------------------------
REDUCERS = [
    ("QSGDMaxNormReducer", dict(quantization_level=4)),
    ("QSGDMaxNormTwoScaleReducer", dict(lower_quantization_level=2, higher_quantization_level=4)),
    ("QSGDMaxNormMultiScaleReducer", dict(quantization_levels=[2, 4, 6])),
    ("GlobalRandKMaxNormReducer", dict(K=1000, quantization_level=4)),
    ("GlobalRandKMaxNormTwoScaleReducer", dict(K=1000, lower_quantization_level=2, higher_quantization_level=4)),
]
STEP = [27, 64, 0, 1000, 3, 4099, 10, 70_001]


def reducer(name, kw, **more):
    return getattr(gcodec, name)(DEV, generator=gcodec.Generator(5, "philox"), **kw, **more)


@pytest.mark.parametrize("name,kw", REDUCERS)
def test_reducer_clips_what_it_writes(name, kw):
    """max_grad_norm: the unclipped step's gradients, clipped; under the limit the same bits."""
    ts = views(carve(STEP, [F32] * len(STEP), seed=121, scale=0.01))
    plain, clipped, loose = ([torch.full_like(t, 9.0) for t in ts] for _ in range(3))
    bits = reducer(name, kw).reduce(ts, plain)
    r = reducer(name, kw, max_grad_norm=0.05)
    assert r.grad_norm is None
    assert r.reduce(ts, clipped) == bits
    xs = f64(plain)
    n = norm64(xs, 2)
    assert n > 0.05
    close_norm(r.grad_norm, n, roundings=5)
    close_values(clipped, [x * coef64(n, 0.05) for x in xs], extra=8)
    reducer(name, kw, max_grad_norm=2 * n).reduce(ts, loose)
    for a, b in zip(plain, loose):
        assert torch.equal(a.view(torch.int32), b.view(torch.int32))


@pytest.mark.parametrize("name,kw", REDUCERS)
def test_reducer_clips_what_it_sends(name, kw):
    """local_max_norm: the bits of a step on gradients that clip_grads had clipped before."""
    ts = views(carve(STEP, [F32] * len(STEP), seed=131, scale=0.01))
    before = [torch.empty_like(t) for t in ts]
    n = gcodec.clip_grads(ts, before, 0.05)
    want, got = ([torch.full_like(t, 9.0) for t in ts] for _ in range(2))
    bits = reducer(name, kw).reduce(before, want)
    r = reducer(name, kw, local_max_norm=0.05)
    assert r.reduce(ts, got) == bits and torch.equal(r.local_grad_norm, n)
    for a, b in zip(want, got):
        assert torch.equal(a.view(torch.int32), b.view(torch.int32))


@pytest.mark.parametrize("name,kw", REDUCERS[:3])
def test_reducer_on_bfloat16_gradients(name, kw):
    """Both options take gradients of the smaller types (the codec itself is float32)."""
    types = types_of("mixed", len(STEP))
    ts, outs = views(carve(STEP, types, seed=141, scale=0.01)), views(carve(STEP, types, seed=142))
    f = [t.float() for t in ts]
    want = [torch.empty_like(t) for t in f]
    reducer(name, kw, local_max_norm=0.5).reduce(f, want)
    r = reducer(name, kw, local_max_norm=0.5, max_grad_norm=math.inf)
    r.reduce(ts, outs)
    close_norm(r.local_grad_norm, norm64(f64(ts), 2))
    for a, b in zip(want, outs):
        assert torch.equal(a.to(b.dtype), b)


def test_reducer_step_captured_and_replayed():
    """Local clipping, codec and clipped decode in one graph (Philox draws at a fixed offset)."""
    ts, outs = views(carve(STEP, [F32] * len(STEP), seed=151, scale=0.01)), views(carve(STEP, [F32] * len(STEP), seed=152))
    gi, go = gcodec.Grads(ts), gcodec.Grads(outs)
    rng = gcodec.Generator(5, "philox").reserve(sum(STEP))

    def step():
        flat, peak, total = gcodec.flatten_clip(gi, 0.5)
        words = codec.qsgd_encode(flat, peak, 8, rng)
        return gcodec.qsgd_decode_clip(words, peak, 8, go, 0.3), total

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        n, total = step()
    for _ in range(4):
        with torch.no_grad():
            for t in ts:
                t.mul_(1.7)
        g.replay()
        torch.cuda.synchronize()
        got, first = [o.clone() for o in outs], (float(n), float(total))
        en, et = step()  # eager, on the same inputs
        assert first == (float(en), float(et))
        for a, b in zip(got, outs):
            assert torch.equal(a, b)


def test_ranks_clip_their_shards_by_the_whole():
    import os
    import tempfile

    import torch.multiprocessing as mp

    import _clip_workers as W

    with tempfile.TemporaryDirectory() as td:
        mp.spawn(W.clip_shards, args=(2, os.path.join(td, "init"), td), nprocs=2, join=True)
        r = [dict(np.load(os.path.join(td, f"r{k}.npz"), allow_pickle=False)) for k in range(2)]
    parts = [[s.double().numpy() for s in W.shards(k, 2)] for k in range(2)]
    for p in (1.0, 2.0, INF):
        n = norm64(parts[0] + parts[1], p)
        for k in range(2):
            close_norm(r[k][f"norm/{p}"], n)
            close_norm(r[k][f"clip/{p}"], n)
            close_values([torch.from_numpy(r[k][f"grads/{p}"])], [np.concatenate(parts[k]) * coef64(n, 0.75)])
    for k in range(2):
        assert float(r[k]["alone"]) == 6.0 and np.isnan(r[k]["nan"]).all()


def test_checked_calls_clip_alike():
    """error_if_nonfinite takes the norm in a call of its own: the same bits follow."""
    ts = views(carve(RAGGED, types_of("mixed", len(RAGGED)), seed=161))
    a, b = ([torch.zeros_like(t) for t in ts] for _ in range(2))
    na = gcodec.clip_grads(ts, a, 1.0)
    nb = gcodec.clip_grads(ts, b, 1.0, error_if_nonfinite=True)
    assert torch.equal(na, nb) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_lists_on_another_stream():
    """Lists made, used and dropped on a stream of their own, over and over."""
    s = torch.cuda.Stream()
    want = None
    with torch.cuda.stream(s):
        for _ in range(30):
            ts = [torch.full((5000 + i,), 0.5, device=DEV, dtype=(F32, BF16)[i % 2]) for i in range(40)]
            got = gcodec.clip_grads(ts, ts, 1.0)
            flat, peak, after = gcodec.flatten_clip(ts, 10.0)
            res = torch.stack([got, after, peak[0]])
            want = res if want is None else want
            del ts, flat
            assert torch.equal(res, want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [8_193, 1_100_000, 9_000_001, 30_000_001, 70_000_003])
def test_each_norm_over_the_tile_sizes(n, dtype):
    """Ones: every sum is a whole number, whatever tile and slots a list of n elements is given."""
    ts = [torch.ones(n, dtype=dtype, device=DEV), torch.ones(5, dtype=dtype, device=DEV), torch.ones(n // 3, dtype=dtype, device=DEV)]
    m = [t.numel() for t in ts]
    total, each = gcodec.grad_norm(ts, 1, per_tensor=True)
    assert float(total) == float(np.float32(sum(m))) and each.tolist() == [float(np.float32(k)) for k in m]
    total, each = gcodec.grad_norm(ts, 2, per_tensor=True)
    assert float(total) == float(np.float32(math.sqrt(sum(m))))
    assert each.tolist() == [float(np.float32(math.sqrt(k))) for k in m]
    for t in ts:
        t[-1] = 3.0
    total, each = gcodec.grad_norm(ts, INF, per_tensor=True)
    assert float(total) == 3.0 and each.tolist() == [3.0] * 3


@pytest.mark.parametrize("p", [1, 2, INF])
def test_short_lists_touch_no_workspace(p):
    """gc_grad_workspace_size is 0 for them: a pointer that is passed all the same is left alone."""
    from gcodec import _lib

    lib = _lib.load()
    ts = views(carve([1000, 3], [F32, BF16], seed=171))
    g = gcodec.Grads(ts)
    assert lib.gc_grad_workspace_size(g.n, g.count, 0) == 0
    ws, norm = torch.full((64,), 7, dtype=torch.int64, device=DEV), torch.zeros((), device=DEV)
    code = _lib.GC_NORM_INF if p == INF else p
    st = torch.cuda.current_stream().cuda_stream
    assert lib.gc_grad_norm(g._ref, code, None, norm.data_ptr(), None, ws.data_ptr(), st) == 0
    close_norm(norm, norm64(f64(ts), p))
    outs = [torch.empty_like(t) for t in ts]
    o = gcodec.Grads(outs)
    assert lib.gc_grad_clip(g._ref, o._ref, code, 0.5, None, norm.data_ptr(), ws.data_ptr(), st) == 0
    flat, peak = torch.empty(g.n, device=DEV), torch.zeros(1, device=DEV)
    assert lib.gc_grad_flatten_clip(g._ref, flat.data_ptr(), code, 0.5, peak.data_ptr(), norm.data_ptr(),
                                    ws.data_ptr(), st) == 0
    assert bool((ws == 7).all())


def test_every_write_is_told_to_autograd():
    """Lists, tables of tensors and the bucket: a tensor saved for a backward is not changed unnoticed."""
    sizes = [5000, 0, 33]
    src = views(carve(sizes, [F32, BF16, F16], seed=181))
    words, _, scale = packed(sum(sizes), 4, 1, seed=3)
    read = [t._version for t in src]
    for make in (list, gcodec.Grads):
        for write in (lambda o: gcodec.clip_grads(src, make(o), 1.0), lambda o: gcodec.clip_grads(make(src), make(o), 1.0),
                      lambda o: gcodec.qsgd_decode_clip(words, scale, 4, make(o), 1.0),
                      lambda o: (lambda g: gcodec.clip_grads(g, g, 0.5))(make(o))):
            outs = [torch.ones(s, device=DEV) for s in sizes]
            w = torch.full((sizes[0],), 2.0, device=DEV, requires_grad=True)
            y = (w * outs[0]).sum()  # keeps outs[0]
            before = [o._version for o in outs]
            write(outs)
            assert all(o._version > v for o, v in zip(outs, before))
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()
    flat = torch.zeros(sum(sizes), device=DEV)
    view, before = flat[3:9], flat._version
    gcodec.flatten_clip(gcodec.Grads(src), 1.0, flat=flat)
    assert flat._version > before and view._version == flat._version
    assert [t._version for t in src] == read  # reading is none


def test_a_call_that_writes_nothing_tells_autograd_nothing():
    """Refused, or raised by error_if_nonfinite ahead of the write."""
    src = views(carve([5000, 33], [F32, BF16], seed=182))
    outs, y = [torch.ones(5000, device=DEV), torch.ones(33, device=DEV)], torch.ones(5033, device=DEV)
    words, _, scale = packed(5033, 4, 1, seed=3)
    before = [o._version for o in outs + [y]]
    E = gcodec.GCodecError
    for make in (list, gcodec.Grads):
        with pytest.raises(E, match="sizes"):
            gcodec.clip_grads([y[:5001], y[5001:]], make(outs), 1.0)
        with pytest.raises(E, match="tensors into"):
            gcodec.clip_grads([y], make(outs), 1.0)
        with pytest.raises(E, match="needed"):
            gcodec.qsgd_decode_clip(words[:8], scale, 4, make(outs), 1.0)
        with pytest.raises(E, match="lanes"):
            gcodec.qsgd_decode_clip(words, scale, 4, make(outs), 1.0, lanes=codec.qsgd_layout(5033, 2))
    with pytest.raises(E, match="flat bucket"):
        gcodec.flatten_clip([y], 1.0, flat=y)
    src[0][9] = math.nan
    for make in (list, gcodec.Grads):
        with pytest.raises(RuntimeError, match="not finite"):
            gcodec.clip_grads(src, make(outs), 1.0, error_if_nonfinite=True)
    assert [o._version for o in outs + [y]] == before
    assert all(bool((o == 1).all()) for o in outs)


def test_dropped_table_holds_its_memory_for_the_stream():
    """A table that was the last to hold its tensors, used on a side stream and dropped while that stream still
    waits: the tensors' memory is not given out again before the stream has run."""
    side, n = torch.cuda.Stream(), 1 << 20
    for write in (False, True):
        src, out = [torch.full((n,), 2.0, device=DEV)], [torch.zeros(n, device=DEV)]
        gi, go = gcodec.Grads(src), gcodec.Grads(out)
        held = {t.data_ptr() for t in (src + out if write else src)}
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)  # 0.01 s at least
            norm = gcodec.clip_grads(gi, go, INF) if write else gcodec.grad_norm(gi, INF)
        del src, gi
        if write:
            del out, go
        assert not side.query()
        later = [torch.full((n,), 9.0, device=DEV) for _ in range(4)]  # on the current stream, ahead of the side's work
        assert not held & {t.data_ptr() for t in later}
        torch.cuda.synchronize()
        # clip_grads takes the 2-norm: 2^20 twos have 2 * 2^10
        assert float(norm) == (2048.0 if write else 2.0) and all(bool((t == 9).all()) for t in later)


def test_copy_on_write_tensors_are_written_alone():
    """A lazy clone shares its source's memory until one of the two is written."""
    n = 5000
    words, _, scale = packed(n, 4, 1, seed=3)
    for make in (list, gcodec.Grads):
        for write in (lambda o: gcodec.clip_grads([torch.full((n,), 3.0, device=DEV)], make(o), 1.0),
                      lambda o: gcodec.qsgd_decode_clip(words, scale, 4, make(o), 1.0),
                      lambda o: (lambda g: gcodec.clip_grads(g, g, 0.5))(make(o))):
            a = torch.full((n,), 2.0, device=DEV)
            b = torch._lazy_clone(a)
            write([b])
            assert bool((a == 2).all()) and not bool((b == 2).any())
    w, a = torch.nn.Parameter(torch.zeros(n, device=DEV)), torch.full((n,), 2.0, device=DEV)
    w.grad = torch._lazy_clone(a)
    gcodec.clip_grad_norm_([w], 1.0)
    assert bool((a == 2).all()) and not bool((w.grad == 2).any())
    flat = torch._lazy_clone(a)
    gcodec.flatten_clip([torch.full((n,), 3.0, device=DEV)], 1.0, flat=flat)
    assert bool((a == 2).all()) and not bool((flat == 2).any())
    # partly in place: the clone is both an input and its own output
    b, c = torch._lazy_clone(a), torch.empty(7, device=DEV)
    gcodec.clip_grads([b, torch.ones(7, device=DEV)], [b, c], 1.0)
    assert bool((a == 2).all())
    norm = math.sqrt(4.0 * n + 7)
    close_values([b, c], [np.full(n, 2.0 * coef64(norm, 1.0)), np.full(7, coef64(norm, 1.0))])
    b = torch._lazy_clone(a)  # a read one is left as it is
    assert float(gcodec.grad_norm([b], INF)) == 2.0 and torch._C._is_cow_tensor(b)


@pytest.mark.parametrize("name,kw", REDUCERS)
def test_reducer_options_take_any_strides(name, kw):
    """channels_last, transposed and sliced gradients, as without the options; outputs also of wider types
    and on the host."""
    shapes_ = [(8, 6, 5, 4), (64,), (30, 40), (0, 3), (7, 9)]
    rng = np.random.default_rng(191)
    plain = [torch.from_numpy(rng.standard_normal(s).astype(np.float32) * 0.01).to(DEV) for s in shapes_]

    def odd(ts):
        return [ts[0].contiguous(memory_format=torch.channels_last), ts[1], ts[2].t().contiguous().t(), ts[3],
                torch.cat([ts[4], ts[4]], 1)[:, :9]]

    def outs():
        ones = odd([torch.full(s, 9.0, device=DEV) for s in shapes_])
        ones[1] = ones[1].double()
        if not name.startswith("GlobalRandK"):  # whose setgrad adds in place, on the GPU only
            ones[4] = ones[4].cpu()
        return ones

    ins = odd(plain)
    assert [t.is_contiguous() for t in ins] == [False, True, False, True, False]
    want = outs()
    bits = reducer(name, kw).reduce(ins, want)
    same = [torch.full_like(t, 9.0) for t in plain]
    reducer(name, kw).reduce(plain, same)
    for a, b in zip(want, same):
        assert torch.equal(a.to(DEV, F32), b)
    n = norm64(f64(same), 2)
    got = outs()
    r = reducer(name, kw, local_max_norm=INF, max_grad_norm=2 * n)  # under both limits: the same bits
    assert r.reduce(ins, got) == bits
    close_norm(r.local_grad_norm, norm64(f64(plain), 2))
    close_norm(r.grad_norm, n, roundings=5)
    for a, b in zip(got, want):
        assert a.stride() == b.stride() and torch.equal(a, b)
    got = outs()
    r = reducer(name, kw, max_grad_norm=0.5 * n)
    r.reduce(ins, got)
    # a clipped value is a float32's before it is any wider type's
    close_values([t.to(DEV, F32) for t in got], [x * coef64(n, 0.5 * n) for x in f64(same)], extra=8)
    before = [torch.empty_like(t) for t in plain]
    gcodec.clip_grads(plain, before, 0.05)
    reducer(name, kw).reduce(before, same)
    reducer(name, kw, local_max_norm=0.05).reduce(ins, got)
    for a, b in zip(got, same):
        assert torch.equal(a.to(DEV, F32), b)


@pytest.mark.parametrize("shape,perm", [((3, 4, 5), (0, 1, 2)), ((3, 4, 5), (2, 0, 1)), ((2, 3, 4, 5), (0, 2, 3, 1)),
                                        ((1, 4, 1), (2, 1, 0)), ((4, 1, 6), (1, 2, 0)), ((0, 3), (1, 0)), ((6000, 7), (1, 0))])
def test_dense_orders_of_gradients(shape, perm):
    """Any order of the dimensions, with sizes of one and none: the norm and the clip in place take them all."""
    rng = np.random.default_rng(201)
    for t in (F32, BF16, F16):
        w = torch.nn.Parameter(torch.zeros(shape, dtype=t, device=DEV).permute(perm))
        g = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(DEV, t).permute(perm)
        w.grad = g
        x = g.cpu().double().numpy().copy()
        n = norm64([x.reshape(-1)], 2)
        close_norm(gcodec.grad_norm([g]), n)
        close_norm(gcodec.clip_grad_norm_([w], 0.3), n)
        assert w.grad.stride() == g.stride() and w.grad.data_ptr() == g.data_ptr()
        close_values([w.grad.contiguous()], [x.reshape(-1) * coef64(n, 0.3)])
    # one tensor's rows, columns or repetitions are not dense
    for bad in (torch.zeros(4, 6, device=DEV)[:, :3], torch.zeros(4, 1, device=DEV).expand(4, 5), torch.zeros(9, device=DEV)[::2]):
        with pytest.raises(gcodec.GCodecError, match="not dense"):
            gcodec.grad_norm([bad])


# ---------------------------------------------------------------------------
# lists as large as a model's, checked on the device
# ---------------------------------------------------------------------------
LARGE = {  # odd sizes and ends; more work than one round of the launch, more bytes than the cache in front of the memory
    "few": [100_000_003, 0, 17, 60_000_000, 5001],
    "few and 1200 small": [30_000_001, *(1 + i % 9 for i in range(600)), 90_000_007, *(i % 700 for i in range(600)), 40_000_005],
    "large, then a run of ones": [25_000_001] + [1 + i % 3 for i in range(2500)],
}


def guarded(sizes, dtype):
    """Tensors at odd offsets of one buffer with 7.0 between them; the buffer and a mask of what lies between."""
    buf = torch.full((sum(sizes) + 3 * len(sizes) + 8,), 7.0, dtype=dtype, device=DEV)
    between = torch.ones(buf.numel(), dtype=torch.bool, device=DEV)
    at, out = 1, []
    for s in sizes:
        out.append(buf[at:at + s])
        between[at:at + s] = False
        at += s + 3
    return out, buf, between


def close_on_device(got, want, extra=0):
    """close_values for tensors end to end, a part at a time"""
    u, rel = UNIT[got.dtype], (2 + extra) * 2.0 ** -24 * (1 + 2.0 ** -6)
    rel += u * (1 + 2.0 ** -6) if got.dtype != F32 else 0.0
    for g, w in zip(got.split(1 << 26), want.split(1 << 26)):
        err = (g.double() - w).abs_()
        tol = w.abs().mul_(rel).add_(TINY[got.dtype] * 0.5 + (1 + extra) * 2.0 ** -150)
        assert bool((err <= tol).all())


def norm_on_device(x, p):
    """in 64 bits; its sums are within 2^-40 of the exact ones (a tree of n < 2^28 terms)"""
    if p == INF:
        return float(x.abs().max())
    return math.sqrt(float(x.square().sum())) if p == 2 else float(x.abs().sum())


@pytest.mark.parametrize("p", [1, 2, INF])
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("name", list(LARGE))
def test_large_lists(name, kind, p):
    """Norms, list to list, in place and into the bucket."""
    sizes = LARGE[name]
    src, _, _ = guarded(sizes, kind)
    gen = torch.Generator(device=DEV).manual_seed(7)
    for i, t in enumerate(src):
        if t.numel():
            t.copy_(torch.randn(t.numel(), generator=gen, device=DEV) * 2.0 ** (i % 5 - 2))
    x = torch.cat(src).double()
    n = norm_on_device(x, p)
    c = coef64(n, 0.3 * n)
    total, each = gcodec.grad_norm(src, p, per_tensor=True)
    close_norm(total, n)
    mine = each.tolist()
    at = 0
    for k, s in enumerate(sizes):
        if s > 1000 or k % 97 == 0:
            close_norm(mine[k], norm_on_device(x[at:at + s], p) if s else 0.0)
        at += s
    outs, buf, between = guarded(sizes, BF16)
    close_norm(gcodec.clip_grads(src, outs, 0.3 * n, p), n)
    x.mul_(c)
    close_on_device(torch.cat(outs), x)
    assert bool((buf[between] == 7).all())
    del outs, buf, between
    flat, peak, total = gcodec.flatten_clip(src, 0.3 * n, p)
    close_norm(total, n)
    close_on_device(flat, x)
    assert float(peak) == float(flat.abs().max())
    del flat
    table = gcodec.Grads(src)
    close_norm(gcodec.clip_grads(table, table, 0.3 * n, p), n)
    close_on_device(torch.cat(src), x)


@pytest.mark.parametrize("p", [1, 2, INF])
@pytest.mark.parametrize("name,kind,bits,world", [("few", BF16, 8, 8), ("few and 1200 small", BF16, 8, 8),
                                                  ("few and 1200 small", F32, 4, 1), ("few", F32, 16, 1),
                                                  ("large, then a run of ones", F32, 4, 3)])
def test_decode_of_large_lists(name, kind, bits, world, p):
    sizes = LARGE[name]
    n, s = sum(sizes), (1 << bits) - 1
    # every place has its own level: a product with an odd number, folded into -world s .. world s
    i = torch.arange(n, dtype=torch.int64, device=DEV)
    q = ((i * 2_654_435_761 + 12_345) >> 7) % (2 * world * s + 1) - world * s
    del i
    lanes = codec.qsgd_layout(n, bits, world)
    words = torch.zeros(lanes.plane_words, dtype=torch.int64, device=DEV)
    for k in range(lanes.per_word):
        part = q[k * lanes.plane_words:(k + 1) * lanes.plane_words]
        words[:part.numel()] += (part + world * s) << (k * lanes.bits)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    norm = torch.tensor([0.02], dtype=F32, device=DEV)
    x = q.double().mul_(float(norm) / s / world)
    del q
    want = norm_on_device(x, p)
    outs, buf, between = guarded(sizes, kind)
    total = gcodec.qsgd_decode_clip(words, norm, bits, outs, 0.37 * want, p, world=world, alpha=1.0 / world)
    close_norm(total, want, roundings=5)
    close_on_device(torch.cat(outs), x.mul_(coef64(want, 0.37 * want)), extra=8)
    assert bool((buf[between] == 7).all())


# ---------------------------------------------------------------------------
# calls that the documentation allows
# ---------------------------------------------------------------------------
def test_the_trainer_call_captured_and_replayed():
    """clip_grad_norm_ in a graph: replays above and under the limit, eager calls between them."""
    grads = carve(RAGGED, types_of("mixed", len(RAGGED)), seed=211)
    params = [torch.nn.Parameter(torch.zeros_like(v)) for v in views(grads)]
    for w, v in zip(params, views(grads)):
        w.grad = v
    clean = [v.clone() for v in views(grads)]
    limit = 0.5 * norm64(f64(clean), 2)
    gcodec.clip_grad_norm_(params, limit)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = gcodec.clip_grad_norm_(params, limit)
    for factor in (1.0, 0.25, 4.0, 0.5, 1.0):
        for v, c in zip(views(grads), clean):
            v.copy_(c * factor)
        xs = f64(views(grads))
        want = norm64(xs, 2)
        graph.replay()
        close_norm(gcodec.grad_norm(clean), norm64(f64(clean), 2))
        torch.cuda.synchronize()
        close_norm(n, want)
        close_values(views(grads), [x * coef64(want, limit) for x in xs])
        guards_hold(grads)


def test_two_threads_at_once():
    """One table and lists of each thread's own, on streams of their own."""
    import threading

    shared = views(carve([1_000_003, 12, 50_000], [F32, BF16, F16], seed=221))
    table, want = gcodec.Grads(shared), norm64(f64(shared), 2)
    torch.cuda.synchronize()
    wrong = []

    def work(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                own = views(carve([70_001, 5, 9000 + seed], [F32, F16, BF16], seed=seed))
                xs = f64(own)
                n = norm64(xs, 2)
                for _ in range(20):
                    a = gcodec.grad_norm(table)
                    outs = [torch.empty_like(t) for t in own]
                    b = gcodec.clip_grads(own, outs, 0.5 * n)
                    with pytest.raises(gcodec.GCodecError, match=("share memory", "sizes", "tensors into")[seed - 1]):
                        gcodec.clip_grads(own, (own[:1] * 3, own[::-1], own[:2])[seed - 1], 1.0)  # each its own message
                    torch.cuda.current_stream().synchronize()
                    close_norm(a, want)
                    close_norm(b, n)
                    close_values(outs, [x * coef64(n, 0.5 * n) for x in xs])
        except BaseException as e:  # noqa: BLE001 - handed to the test's thread
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in (1, 2, 3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if wrong:
        raise wrong[0]


@pytest.mark.parametrize("p", [1, 2, INF])
def test_a_tensor_read_twice(p):
    """A list that is only read may hold a tensor twice, or parts that overlap: each counts."""
    y = views(carve([9000], [F32], seed=231))[0]
    ts = [y, y, y[5:7000], y[:0]]
    xs = f64(ts)
    n = norm64(xs, p)
    total, each = gcodec.grad_norm(ts, p, per_tensor=True)
    close_norm(total, n)
    for e, x in zip(each.tolist(), xs):
        close_norm(e, norm64([x], p))
    flat, peak, total = gcodec.flatten_clip(gcodec.Grads(ts), 0.5 * n, p)
    close_norm(total, n)
    close_values([flat], [np.concatenate(xs) * coef64(n, 0.5 * n)])
    outs = [torch.empty_like(t) for t in ts]
    gcodec.clip_grads(ts, outs, 0.5 * n, p)
    close_values(outs, [x * coef64(n, 0.5 * n) for x in xs])


@pytest.mark.parametrize("count", [1, 3, 1100])
def test_decode_of_no_elements(count):
    outs = [torch.empty(0, device=DEV) for _ in range(count)]
    words = torch.empty(0, dtype=torch.int32, device=DEV)
    for scale in (0.02, 0.0, INF, math.nan):
        norm = torch.tensor([scale], device=DEV)
        for p in (1, 2, INF):
            assert float(gcodec.qsgd_decode_clip(words, norm, 4, outs, 1.0, p)) == 0.0


@pytest.mark.parametrize("p", [1, 2, INF])
@pytest.mark.parametrize("bits,world", [(24, 128), (24, 8), (17, 16_000), (1, 2_000_000_000)])
def test_decode_of_the_widest_lanes(bits, world, p):
    """Lanes of up to 32 bits, whose sums pass 31: the values are qsgd_decode's, bit for bit."""
    sizes = [5000, 0, 33, 4001]
    n, s = sum(sizes), (1 << bits) - 1
    lanes = codec.qsgd_layout(n, bits, world)
    assert lanes.per_word == 1 and lanes.bits >= 28
    rng = np.random.default_rng(241)
    q = rng.integers(-world * s, world * s + 1, n)
    q[:3] = world * s, -world * s, 0
    words = torch.zeros(lanes.plane_words, dtype=torch.int64, device=DEV)
    words[:n] = torch.from_numpy(q + world * s).to(DEV)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    norm = torch.tensor([0.02], device=DEV)
    dense = codec.qsgd_decode(words, n, norm, bits, world, alpha=1.0 / world)
    outs = views(carve(sizes, [F32] * len(sizes), seed=242))
    total = gcodec.qsgd_decode_clip(words, norm, bits, outs, INF, p, world=world, alpha=1.0 / world)
    assert torch.equal(torch.cat(outs).view(torch.int32), dense.view(torch.int32))
    want = norm64(f64([dense]), p)
    close_norm(total, want)
    # the integers' own: RN(norm / s), RN of the integer to float32, two products, alpha: five roundings, and the norm's
    close_norm(total, norm64([q * (float(norm) / s / world)], p), roundings=6)
    gcodec.qsgd_decode_clip(words, norm, bits, outs, 0.5 * want, p, world=world, alpha=1.0 / world)
    close_values([torch.cat(outs)], [dense.cpu().double().numpy() * coef64(want, 0.5 * want)])


def test_decode_takes_the_scale_in_any_form():
    words, q, norm = packed(5000, 4, 1, seed=251, norm=0.25)
    want, got = ([torch.empty(5000, device=DEV)] for _ in range(2))
    gcodec.qsgd_decode_clip(words, norm, 4, want, 1.0)
    for form in (0.25, norm.double(), norm.cpu(), norm.reshape(()), torch.tensor([0.25, 9.0], device=DEV)[:1],
                 torch.tensor([[0.25, 9.0]], device=DEV, dtype=torch.float64)):
        got[0].fill_(9.0)
        gcodec.qsgd_decode_clip(words, form, 4, got, 1.0)
        assert torch.equal(want[0], got[0])


def test_a_workspace_of_no_bytes_shares_no_memory():
    """A short list's workspace may point anywhere, also into the bucket."""
    from gcodec import _lib

    lib = _lib.load()
    ts = views(carve([1000, 3], [F32, BF16], seed=261))
    g, want = gcodec.Grads(ts), gcodec.flatten_clip(ts, 0.5)
    flat, peak, norm = torch.empty(g.n, device=DEV), torch.zeros(1, device=DEV), torch.zeros((), device=DEV)
    assert lib.gc_grad_flatten_clip(g._ref, flat.data_ptr(), 2, 0.5, peak.data_ptr(), norm.data_ptr(),
                                    flat.data_ptr() + 64, torch.cuda.current_stream().cuda_stream) == 0, _lib.last_error()
    assert torch.equal(flat, want[0]) and torch.equal(peak, want[1]) and torch.equal(norm, want[2])
