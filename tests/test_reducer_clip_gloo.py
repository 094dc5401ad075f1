"""The reducers' clipping options across ranks (gloo, CPU, W = 2) with the oracle
codec and clip operators written from the formulas in 64 bits: every rank clips
the averaged gradient by the same norm, and each its own by its own."""
import os
import sys
import tempfile
import types

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import torch.distributed as dist  # noqa: E402
import torch.multiprocessing as mp  # noqa: E402

HERE = os.path.dirname(os.path.abspath(__file__))
if HERE not in sys.path:
    sys.path.insert(0, HERE)
SIZES = [27, 0, 640, 1000, 3]


def _clip_ops(oc):
    """gcodec.clip's operators that the reducers call, on CPU tensors."""

    def scale(xs, max_norm):
        n = float(np.sqrt(sum(float((x.double() ** 2).sum()) for x in xs)))
        return np.float32(min(1.0, max_norm / (n + 1e-6))), torch.tensor(n, dtype=torch.float32)

    def clip_grads(grads, out, max_norm):
        c, n = scale(grads, max_norm)
        for g, o in zip(grads, out):
            o.copy_(g * c)
        return n

    def flatten_clip(grads, max_norm):
        c, n = scale(grads, max_norm)
        flat = torch.cat([g.reshape(-1) for g in grads]) * c
        return flat, flat.abs().max().reshape(1), n

    def qsgd_decode_clip(words, norm, bits, grads, max_norm, world=1, alpha=1.0):
        n = sum(g.numel() for g in grads)
        dec = oc.qsgd_decode(words, n, norm, bits, world, alpha)
        for g, x in zip(grads, torch.split(dec, [g.numel() for g in grads])):
            g.copy_(x.view_as(g))
        return clip_grads(grads, grads, max_norm)

    return types.SimpleNamespace(clip_grads=clip_grads, flatten_clip=flatten_clip, qsgd_decode_clip=qsgd_decode_clip)


def _codec():
    import oracle_codec as oc

    c = types.SimpleNamespace(**{k: getattr(oc, k) for k in dir(oc) if not k.startswith("__")})
    c.clip = _clip_ops(oc)
    return c


def _grads(rank):
    g = torch.Generator().manual_seed(7 + rank)
    return [torch.randn(s, generator=g) * 0.1 * (1 + rank) for s in SIZES]


def _worker(rank, world, init, out):
    import gcodec
    from _gloo_workers import make_reducer

    dist.init_process_group("gloo", init_method=f"file://{init}", rank=rank, world_size=world)
    res = {}
    for name in ("qsgd", "ts", "ms", "randk", "randk_ts"):
        for tag, kw in (("plain", {}), ("out", dict(max_grad_norm=0.5)), ("in", dict(local_max_norm=0.5))):
            red = make_reducer(name, codec=_codec(), generator=gcodec.Generator(3 + rank, "philox"), **kw)
            outs = [torch.full((s,), 9.0) for s in SIZES]
            red.reduce(_grads(rank), outs)
            res[f"{name}/{tag}"] = torch.cat(outs).numpy()
            if tag == "out":
                res[f"{name}/norm"] = red.grad_norm.numpy()
            if tag == "in":
                res[f"{name}/local"] = red.local_grad_norm.numpy()
        # the step on gradients that were clipped by hand
        red = make_reducer(name, codec=_codec(), generator=gcodec.Generator(3 + rank, "philox"))
        gs = _grads(rank)
        _codec().clip.clip_grads(gs, gs, 0.5)
        outs = [torch.full((s,), 9.0) for s in SIZES]
        red.reduce(gs, outs)
        res[f"{name}/hand"] = torch.cat(outs).numpy()
    np.savez(os.path.join(out, f"r{rank}.npz"), **res)
    dist.destroy_process_group()


def test_ranks_clip_alike():
    with tempfile.TemporaryDirectory() as td:
        mp.spawn(_worker, args=(2, os.path.join(td, "init"), td), nprocs=2, join=True)
        r = [dict(np.load(os.path.join(td, f"r{k}.npz"), allow_pickle=False)) for k in range(2)]
    for name in ("qsgd", "ts", "ms", "randk", "randk_ts"):
        for k in range(2):
            plain, out = r[k][f"{name}/plain"].astype(np.float64), r[k][f"{name}/out"].astype(np.float64)
            n = np.sqrt((plain ** 2).sum())
            assert n > 0.5
            # the norm rounds once, c once, the product once
            assert abs(float(r[k][f"{name}/norm"]) - n) <= 2.0 ** -23 * n
            want = plain * (0.5 / (n + 1e-6))
            assert (np.abs(out - want) <= 2.0 ** -22 * np.abs(want)).all()
            assert r[k][f"{name}/in"].tobytes() == r[k][f"{name}/hand"].tobytes()
            own = np.sqrt(sum((g.double() ** 2).sum().item() for g in _grads(k)))
            assert abs(float(r[k][f"{name}/local"]) - own) <= 2.0 ** -23 * own
        if not name.startswith("randk"):  # GlobalRandK leaves each rank its own unselected coordinates
            assert r[0][f"{name}/out"].tobytes() == r[1][f"{name}/out"].tobytes()


def test_a_codec_without_clip_operators_is_refused():
    import oracle_codec

    from gcodec import reducer as R

    for kw in (dict(max_grad_norm=1.0), dict(local_max_norm=1.0)):
        with pytest.raises(ValueError, match="clip operators"):
            R.QSGDMaxNormReducer(torch.device("cpu"), None, quantization_level=4, codec=oracle_codec, **kw)


@pytest.mark.parametrize("option", ["max_grad_norm", "local_max_norm"])
@pytest.mark.parametrize("bad", [-1.0, float("nan"), float("-inf"), "1", [1.0]])
def test_a_limit_is_checked_when_the_reducer_is_made(option, bad):
    """Not in the step, behind its collectives and its writes to grad_out."""
    from _gloo_workers import make_reducer

    from gcodec import GCodecError

    for name in ("qsgd", "ts", "ms", "randk", "randk_ts"):
        with pytest.raises(GCodecError, match=option):
            make_reducer(name, codec=_codec(), **{option: bad})
    for good in (0, 0.5, float("inf"), np.float32(2.0), None):
        make_reducer("qsgd", codec=_codec(), **{option: good})
