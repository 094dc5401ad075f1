#!/usr/bin/env python
"""Headline benchmark: QSGD-MaxNorm 4-bit encode+pack of a device-resident
100M-fp32 gradient bucket (BASELINE.json metric / configs[1]).

One step = the encode of one rank's bucket exactly as the data-parallel
reducer runs it: local max-norm (HIP) -> all_reduce MAX of the 4-byte norm
(RCCL, N > 1 only) -> fused quantize + stochastic round + carry-free pack
(HIP, Philox draws).  value = grad floats encoded by ALL ranks per second
(weak scaling: every rank owns a full bucket).

Also reported (not part of `value`): per-kernel HIP-event times and the
roofline of the dominant kernel (k_qsgd_encode), the decode, the full
encode -> RCCL all_reduce(SUM, packed words) -> decode path, the
reference-parity (torch MT19937) encode, and the CPU oracle on the host
cores (rank 0, N = 1).

    python bench.py [--gpus N --steps K --warmup W]
    torchrun --nproc-per-node N bench.py --gpus N ...
"""
from __future__ import annotations

import argparse
import json
import os
import sys
import time

ROOT = os.path.dirname(os.path.abspath(__file__))
for _p in (ROOT, os.path.join(ROOT, "gradient-compression_amd")):
    if _p not in sys.path:
        sys.path.insert(0, _p)

HBM_PEAK_GBS = 8000.0  # MI355X HBM3E spec (MI355X_MICROARCH.md)
# VALU issue ceiling: 256 CUs x 4 SIMD16 = one wave64 VALU instruction per cycle per CU
# at the 2.4 GHz peak clock (measured 0.85-1.07 per cycle per CU for the encode's
# instruction mix, tools/valu_rates.hip, profiles/r01m_valu_rates.log)
VALU_PEAK_WAVE_INSTR_S = 256 * 2.4e9


def _args():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--warmup", type=int, default=20)
    ap.add_argument("--settle", type=float, default=0.5,
                    help="seconds of untimed steps before the W warmup steps: MI355X clocks ramp over ~0.1-0.3 s "
                         "of sustained load (profiles/r01h_*: 181 us/step after 5 steps, 163 us after 1000)")
    ap.add_argument("--n", "--numel", dest="n", type=int, default=100_000_000,
                    help="bucket elements per rank (--numel under torchrun, whose parser takes --n as ambiguous)")
    ap.add_argument("--bits", type=int, default=4)
    ap.add_argument("--cpu-seconds", type=float, default=10.0, help="CPU-oracle sample budget (0 = skip)")
    ap.add_argument("--no-extras", action="store_true", help="skip every leg after the headline (= --legs none)")
    ap.add_argument("--legs", default="all",
                    help="comma list of the legs after the headline: " + ",".join(LEGS) + " (or all / none)")
    ap.add_argument("--n5", type=int, default=1_000_000_000, help="config 5 bucket elements per rank")
    a = ap.parse_args()
    want = "none" if a.no_extras else a.legs
    a.legs = (set(LEGS) if want == "all" else set() if want == "none" else
              {s.strip() for s in want.split(",") if s.strip()})
    bad = a.legs - set(LEGS)
    if bad:
        ap.error(f"unknown legs {sorted(bad)}; known: {','.join(LEGS)}")
    return a


# the legs after the headline, in the order they run (none of them is `value`)
LEGS = ("decode", "reduce", "torch", "pcie", "config3", "epilogue", "config4", "config5", "packers")


_HOLD_MS_PER_MCYCLE = []


def _gpu_hold(torch, ms):
    """Keep the current stream busy for about `ms` (torch.cuda._sleep, calibrated
    once), so launches issued meanwhile queue up and then run back to back."""
    if not hasattr(torch.cuda, "_sleep"):
        return False
    if not _HOLD_MS_PER_MCYCLE:
        s, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        s.record()
        torch.cuda._sleep(1_000_000)
        e.record()
        e.synchronize()
        _HOLD_MS_PER_MCYCLE.append(max(s.elapsed_time(e), 1e-3))
    torch.cuda._sleep(int(min(ms, 500.0) / _HOLD_MS_PER_MCYCLE[0] * 1e6))
    return True


def _events(torch, fn, reps):
    """mean ms of fn() over reps, one HIP event pair on the current stream around
    the whole loop.  The loop is queued behind a GPU hold sized from the host's
    issue rate, so short kernels (config 3/4: 4-40 us against 10-50 us of
    Python per call) run back to back and the events time the GPU, not the
    host's issue gaps; for long kernels the hold changes nothing."""
    t0 = time.perf_counter()
    for _ in range(2):
        fn()
    issue_ms = (time.perf_counter() - t0) / 2 * 1e3
    torch.cuda.synchronize()
    _gpu_hold(torch, 1.5 * issue_ms * reps + 0.5)
    s, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    s.record()
    for _ in range(reps):
        fn()
    e.record()
    e.synchronize()
    return s.elapsed_time(e) / reps


def _traffic(kernel: str, n: int, bits: int):
    """HBM bytes per launch of `kernel` from the committed PMC profile
    (profiles/pmc_traffic.json: rocprofv3 --pmc FETCH_SIZE / WRITE_SIZE passes
    over this same workload, collected by tools/gpu.sh pmc on an earlier run)
    -> (bytes, source) or (None, None).  Not measured by this run: PMC
    counters need their own rocprofv3 pass."""
    p = os.path.join(ROOT, "profiles", "pmc_traffic.json")
    try:
        with open(p) as f:
            d = json.load(f)
        k = d["kernels"][kernel]
        if d.get("n") == n and d.get("bits") == bits:
            return k["hbm_bytes_per_launch"], f"profiles/pmc_traffic.json (rocprofv3 --pmc, tag {d.get('tag')})"
    except Exception:
        pass
    return None, None


def _valu_insts(kernel: str):
    """VALU wave-instructions per launch of `kernel` from the committed SQ
    counter pass (profiles/pmc_sq.json: rocprofv3 --pmc SQ_INSTS_VALU over
    tools/prof_kernels.py, whose config-3 legs are the TS (2,4) ResNet50 bucket
    at W = 1) -> (count, source) or (None, None)."""
    try:
        with open(os.path.join(ROOT, "profiles", "pmc_sq.json")) as f:
            d = json.load(f)
        return d["kernels"][kernel]["SQ_INSTS_VALU"], f"profiles/pmc_sq.json (rocprofv3 --pmc, tag {d.get('tag')})"
    except Exception:
        return None, None


def _pg_evidence(torch, dist, dev, local: int, sum_bytes: int) -> dict:
    """What the process group itself reports at N > 1 (not the launcher's env):
    its size and backend, the RCCL version, and every rank's (rank, local rank,
    device, PCI bus id) gathered over the group."""
    props = torch.cuda.get_device_properties(dev)
    bus = "%04x:%02x:%02x" % (getattr(props, "pci_domain_id", 0), getattr(props, "pci_bus_id", 0),
                              getattr(props, "pci_device_id", 0))
    mine = {"rank": dist.get_rank(), "local_rank": local, "device": str(dev), "pci_bus_id": bus,
            "name": props.name}
    ranks = [None] * dist.get_world_size()
    dist.all_gather_object(ranks, mine)
    try:
        ver = ".".join(str(v) for v in torch.cuda.nccl.version())
    except Exception as e:  # noqa: BLE001 — report, never fail the bench
        ver = f"unavailable: {type(e).__name__}"
    return {"world_size": dist.get_world_size(), "backend": dist.get_backend(), "rccl_version": ver,
            "ranks": ranks, "distinct_devices": len({(r["pci_bus_id"], r["device"]) for r in ranks}),
            "bytes_per_rccl_sum": sum_bytes}


def cpu_baseline(n: int, bits: int, budget_s: float):
    """The CPU oracle (oracle/gcodec_oracle.c) running the reference's CPU
    algorithm on the same 100M-element bucket: max-norm, one MT19937 draw per
    element in element order (torch.bernoulli's serial stream, compressors.py:310),
    quantize, pack.  The draws are generated serially, as torch does; the
    max-norm and the quantize + pack run on `threads` host threads (torch runs
    its elementwise CPU ops on its intra-op pool): OMP_NUM_THREADS if set (the
    GPU box sets it to its per-GPU CPU share), else every CPU of the process."""
    import numpy as np

    from oracle import oracle as O

    threads = int(os.environ.get("OMP_NUM_THREADS") or 0) or len(os.sched_getaffinity(0))
    x = O.gen_input(n, seed=42)
    done, t_tot, passes, t_mt = 0, 0.0, 0, 0.0
    while t_tot < budget_s or passes == 0:
        t0 = time.perf_counter()
        norm = O.absmax_par(x, threads)
        mt = O.MT19937(42 + passes)
        t1 = time.perf_counter()
        draws = mt.draws(n)
        t_mt += time.perf_counter() - t1
        O.qsgd_encode_par(x, norm, bits, 1, O.stream_rng(draws), threads)
        t_tot += time.perf_counter() - t0
        done += n
        passes += 1
        del draws
    del x
    np.random.default_rng(0)
    return {"value": done / t_tot, "unit": "grad-floats/s", "cores": threads, "kind": "port",
            "mt19937_share": t_mt / t_tot,
            "sample": f"{passes} full encode pass(es) of the {n}-fp32 bucket (absmax + serial MT19937 draws + "
                      f"quantize + pack, {bits}-bit), {t_tot:.1f} s; absmax and quantize+pack on {threads} host "
                      f"threads, the draws serial ({100 * t_mt / t_tot:.0f}% of the time)"}


def pcie_inclusive(torch, codec, gen, x, n, bits, world, lanes, K):
    """Host-to-host rates (never `value`): pinned host x -> H2D -> absmax +
    encode -> D2H packed words, and H2D words -> decode -> D2H floats.
    serial_*: one bucket at a time on one stream (latency).  *_ms: buckets
    back to back with the copies on their own streams and double-buffered
    device/host buffers, so bucket t's D2H runs while bucket t+1's H2D is on
    the link (PCIe is full duplex) and the kernels hide under the copies: the
    per-bucket cost is then the larger copy, not the sum."""
    M = lanes.plane_words
    dev = x.device
    xh = torch.empty(n, dtype=torch.float32, pin_memory=True)
    xh.copy_(x)
    wh = [torch.empty(M, dtype=torch.int32, pin_memory=True) for _ in range(2)]
    dh = [torch.empty(n, dtype=torch.float32, pin_memory=True) for _ in range(2)]
    xd = [torch.empty_like(x) for _ in range(2)]
    wd = [torch.empty(M, dtype=torch.int32, device=dev) for _ in range(2)]
    nd = [torch.empty(1, dtype=torch.float32, device=dev) for _ in range(2)]
    comp = torch.cuda.current_stream(dev)
    up, down = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    ev = {k: [torch.cuda.Event() for _ in range(2)] for k in ("in", "kern", "out")}

    def encode_bucket(t):
        b = t & 1
        with torch.cuda.stream(up):
            up.wait_event(ev["kern"][b])  # the encode that last read xd[b] is done
            xd[b].copy_(xh, non_blocking=True)
            ev["in"][b].record(up)
        comp.wait_event(ev["in"][b])
        comp.wait_event(ev["out"][b])  # wd[b] has left for the host
        codec.absmax(xd[b], out=nd[b])
        codec.qsgd_encode(xd[b], nd[b], bits, gen.reserve(n), world, out=wd[b], lanes=lanes)
        ev["kern"][b].record(comp)
        with torch.cuda.stream(down):
            down.wait_event(ev["kern"][b])
            wh[b].copy_(wd[b], non_blocking=True)
            ev["out"][b].record(down)

    def decode_bucket(t):
        b = t & 1
        with torch.cuda.stream(up):
            up.wait_event(ev["kern"][b])
            wd[b].copy_(wh[b], non_blocking=True)
            ev["in"][b].record(up)
        comp.wait_event(ev["in"][b])
        comp.wait_event(ev["out"][b])  # xd[b] (the floats) has left for the host
        codec.qsgd_decode(wd[b], n, nd[b], bits, world, 1.0 / world, out=xd[b], lanes=lanes)
        ev["kern"][b].record(comp)
        with torch.cuda.stream(down):
            down.wait_event(ev["kern"][b])
            dh[b].copy_(xd[b], non_blocking=True)
            ev["out"][b].record(down)

    def serial_encode():
        xd[0].copy_(xh, non_blocking=True)
        codec.absmax(xd[0], out=nd[0])
        codec.qsgd_encode(xd[0], nd[0], bits, gen.reserve(n), world, out=wd[0], lanes=lanes)
        wh[0].copy_(wd[0], non_blocking=True)

    def serial_decode():
        wd[0].copy_(wh[0], non_blocking=True)
        codec.qsgd_decode(wd[0], n, nd[0], bits, world, 1.0 / world, out=xd[0], lanes=lanes)
        dh[0].copy_(xd[0], non_blocking=True)

    def wall_ms(fn, k):
        for e in ev.values():
            for i in range(2):
                e[i].record(comp)
        fn(0)
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        for t in range(1, k + 1):
            fn(t)
        torch.cuda.synchronize()
        return (time.perf_counter() - t0) / k * 1e3

    pk = max(6, K // 2)
    enc_ms = wall_ms(encode_bucket, pk)
    dec_ms = wall_ms(decode_bucket, pk)
    ser_e = _events(torch, serial_encode, max(3, K // 4))
    ser_d = _events(torch, serial_decode, max(3, K // 4))
    # the link alone: the same H2D / D2H copies with no kernels
    h2d_ms = _events(torch, lambda: xd[0].copy_(xh, non_blocking=True), 3)
    d2h_ms = _events(torch, lambda: dh[0].copy_(xd[0], non_blocking=True), 3)
    res = {"encode_grad_floats_per_s": n / (enc_ms * 1e-3), "encode_ms": enc_ms,
           "decode_grad_floats_per_s": n / (dec_ms * 1e-3), "decode_ms": dec_ms,
           "serial_encode_ms": ser_e, "serial_decode_ms": ser_d,
           "h2d_gbs": 4 * n / (h2d_ms * 1e-3) / 1e9, "d2h_gbs": 4 * n / (d2h_ms * 1e-3) / 1e9,
           "note": "pinned host buffers, hipMemcpyAsync.  *_ms: buckets back to back, H2D / kernels / D2H on "
                   "three streams with double buffers (bucket t's D2H under bucket t+1's H2D); serial_*: "
                   "one bucket at a time on one stream"}
    del xh, wh, dh, xd, wd
    return res


def other_configs(torch, dist, gcodec, codec, dev, world, rank, K, legs, n5):
    """BASELINE.json configs 3-5 and the fused epilogue (parity cases; not the
    headline `value`), the ones named in `legs`."""
    res = {}
    reps = max(20, K)

    def sync_ms(fn, reps=reps):
        for _ in range(2):
            fn()
        torch.cuda.synchronize()
        if world > 1:
            dist.barrier()
        t0 = time.perf_counter()
        for _ in range(reps):
            fn()
        torch.cuda.synchronize()
        if world > 1:
            dist.barrier()
        el = time.perf_counter() - t0
        if world > 1:
            t = torch.tensor([el], dtype=torch.float64, device=dev)
            dist.all_reduce(t, op=dist.ReduceOp.MAX)
            el = t.item()
        return el / reps * 1e3

    if legs & {"config3", "epilogue"}:
        res.update(_config3_epilogue(torch, dist, gcodec, codec, dev, world, rank, sync_ms, reps, legs))
    if "config4" in legs:
        res.update(_config4(torch, dist, gcodec, codec, dev, world, rank, sync_ms, reps))
    if "config5" in legs:
        res.update(_config5(torch, dist, gcodec, codec, dev, world, sync_ms, n5))
    torch.cuda.empty_cache()
    return res


def _config3_epilogue(torch, dist, gcodec, codec, dev, world, rank, sync_ms, reps, legs):
    from gcodec import shapes
    res = {}
    g = torch.Generator(device=dev).manual_seed(11 + rank)
    gen = gcodec.Generator(5 + rank, "philox")
    if "config3" not in legs:
        return _epilogue(torch, gcodec, codec, dev, world, g, gen, sync_ms, res)
    # config 3: two-scale "4+2" on a ResNet50-sized bucket (MultiScale levels [2, 4])
    n3 = 23_520_842
    x3 = torch.randn(n3, device=dev, generator=g).mul_(0.01)
    for tag, ms in (("twoscale_2_4", gcodec.QSGDMaxNormTwoScaleCompressor(dev, 2, 4, generator=gen)),
                    ("multiscale_2_4", gcodec.QSGDMaxNormMultiScaleCompressor(dev, [2, 4], generator=gen)),
                    ("twoscale_2_4_q_cache",
                     gcodec.QSGDMaxNormTwoScaleCompressor(dev, 2, 4, generator=gen, q_cache=True)),
                    # the (4, 8) pair of the reference's logged runs; 8 bits take the
                    # generic kernels (the fast path needs every level <= 7 bits)
                    ("twoscale_4_8", gcodec.QSGDMaxNormTwoScaleCompressor(dev, 4, 8, generator=gen)),
                    ("twoscale_4_8_q_cache",
                     gcodec.QSGDMaxNormTwoScaleCompressor(dev, 4, 8, generator=gen, q_cache=True))):
        nrm = torch.empty(1, device=dev)
        holder = {}

        one_pass = world == 1 and not ms.q_cache  # W = 1: mask + select in one pass (gc_ms_encode_w1)

        def ms_step():
            codec.absmax(x3, out=nrm)
            if world > 1:
                dist.all_reduce(nrm, op=dist.ReduceOp.MAX)
            both = ms.encode_w1(nrm, x3) if one_pass else None
            if both is not None:
                m, w = both
            else:
                m = ms.encode_mask(nrm, x3, world)
                if world > 1:
                    dist.all_reduce(m)
                w = ms.encode(nrm, x3, m, world)
                if world > 1:
                    dist.all_reduce(w)
            holder["d"] = ms.decode(nrm, w, m, n3, world, 1.0 / world)

        t = sync_ms(ms_step)
        # per kernel (HIP events, W = this rank's lane sizing), algorithmic bytes per
        # mask 4n + mask words (+ q cache cells), select 4n + mask + words
        # (from the cache: cells + mask + words), decode words + mask + 4n
        lvls = ms._packed_levels()
        ql, ml = codec.ms_layouts(n3, lvls, world)
        mwords = codec.mask_words_total(ml, lvls)
        m_ = ms.encode_mask(nrm, x3, world)
        cached = ms._cache_key is not None
        cell = codec.ms_cache_bytes(n3, lvls) * n3 if cached else 0
        w_ = ms.encode(nrm, x3, m_, world)
        d_ = torch.empty(n3, device=dev)
        kt = {
            "absmax": (_events(torch, lambda: codec.absmax(x3, out=nrm), reps), 4 * n3),
            **({"mask_select_one_pass": (_events(torch, lambda: ms.encode_w1(nrm, x3), reps),
                                         4 * n3 + 4 * mwords + 4 * ql.plane_words)} if one_pass else {}),
            "mask_encode": (_events(torch, lambda: ms.encode_mask(nrm, x3, world), reps), 4 * n3 + 4 * mwords + cell),
            "select_encode": (_events(torch, lambda: ms.encode(nrm, x3, m_, world), reps),
                              (cell if cached else 4 * n3) + 4 * mwords + 4 * ql.plane_words),
            "decode": (_events(torch, lambda: ms.decode(nrm, w_, m_, n3, world, 1.0 / world, out=d_), reps),
                       4 * n3 + 4 * mwords + 4 * ql.plane_words),
        }
        kernels = {k: {"us": ms_ * 1e3, "gbs": b / (ms_ * 1e-3) / 1e9,
                       "frac_hbm_peak": b / (ms_ * 1e-3) / 1e9 / HBM_PEAK_GBS} for k, (ms_, b) in kt.items()}
        if tag == "twoscale_2_4" and world == 1:
            # the multi-scale kernels issue Philox + rounding work, not bytes: their
            # roofline is VALU issue (the SQ pass ran this same workload)
            for k, sq in (("mask_select_one_pass", "k_ms_fused_w1"), ("mask_encode", "k_ms_mask_fast"),
                          ("select_encode", "k_ms_select_fast"), ("decode", "k_ms_decode_fast")):
                ins, src = _valu_insts(sq)
                if k in kernels and ins:
                    kernels[k]["valu"] = {"kernel": sq, "wave_instr_per_launch": ins, "source": src,
                                          "per_element": 64 * ins / n3,
                                          "frac_valu_issue_peak": ins / (kernels[k]["us"] * 1e-6) / VALU_PEAK_WAVE_INSTR_S}
        res[f"config3_{tag}"] = {
            "n": n3, "ms_per_step": t, "grad_floats_per_s": world * n3 / (t * 1e-3), "q_cache": cached,
            "step": ("absmax, mask+select encode in one pass (W = 1), decode" if one_pass else
                     "absmax, MAX, mask encode, SUM(mask lanes), select encode, SUM(words), decode"),
            "two_pass_kernels": "mask_encode / select_encode are the W > 1 passes, timed for reference",
            "kernels": kernels}
        del m_, w_, d_
    del x3
    if "epilogue" in legs:
        _epilogue(torch, gcodec, codec, dev, world, g, gen, sync_ms, res)
    return res


def _epilogue(torch, gcodec, codec, dev, world, g, gen, sync_ms, res):
    """fused TensorBuffer / setgrad on the ResNet50 list (161 tensors)."""
    from gcodec import shapes
    sizes = shapes.resnet50_sizes()
    base = torch.randn(sum(sizes) + 4 * len(sizes), device=dev, generator=g).mul_(0.01)
    grads, pos = [], 0
    for sz in sizes:
        grads.append(base[pos:pos + sz])
        pos += sz + (sz % 4 == 0) * 4  # keep most tensors 16-byte aligned like separate allocations
    segs = codec.Segments(grads)
    ln3 = codec.qsgd_layout(segs.n, 4, world)
    nrm = torch.empty(1, device=dev)
    flat = torch.empty(segs.n, device=dev)
    w3 = torch.empty(ln3.plane_words, dtype=torch.int32, device=dev)
    codec.qsgd_encode(torch.cat(grads), nrm, 4, gen.reserve(segs.n), world, out=w3, lanes=ln3)
    ep = {"tensors": len(sizes), "n": segs.n}
    ep["unfused_flatten_norm_ms"] = sync_ms(lambda: codec.absmax(torch.cat(grads), out=nrm))
    ep["fused_flatten_norm_ms"] = sync_ms(lambda: codec.segments_flatten_absmax(segs, flat, nrm))

    def unfused_setgrad():
        d = codec.qsgd_decode(w3, segs.n, nrm, 4, world, 1.0 / world, out=flat, lanes=ln3)
        torch._foreach_copy_(grads, list(torch.split(d, sizes)))

    ep["unfused_decode_setgrad_ms"] = sync_ms(unfused_setgrad)
    ep["fused_decode_setgrad_ms"] = sync_ms(
        lambda: codec.qsgd_decode_segments(w3, nrm, 4, segs, world, 1.0 / world, lanes=ln3))
    for fused in (False, True):
        red = gcodec.QSGDMaxNormReducer(dev, quantization_level=4, generator=gen, fused=fused)
        ep[f"reducer_step_ms_{'fused' if fused else 'unfused'}"] = sync_ms(lambda: red.reduce(grads, grads))
    res["epilogue_resnet50_qsgd4"] = ep
    del base, grads, segs, flat
    return res


def _config4(torch, dist, gcodec, codec, dev, world, rank, sync_ms, reps):
    from gcodec import shapes
    res = {}
    gen = gcodec.Generator(5 + rank, "philox")
    # config 4: GRandK K=10000, 4-bit, VGG16-sized bucket: gather -> encode -> RCCL -> decode/scatter.
    # codec.RandKStep: pointers and structs resolved once, one ctypes call per launch.  W = 1: gather +
    # max-norm + encode in one launch (gc_randk_encode_w1), then the decode-scatter; W > 1: gather + local
    # norm, MAX, dense encode of the gathered subset, SUM, decode-scatter
    n4, K4 = 14_728_266, 10_000
    g = torch.Generator(device=dev).manual_seed(12 + rank)
    x4 = torch.randn(n4, device=dev, generator=g).mul_(0.01)
    idx = torch.randperm(n4, generator=torch.Generator().manual_seed(42))[:K4].to(dev)
    rk = codec.RandKStep(x4, K4, 4, gen, world)

    def rk_step():
        if rk.fused:
            w, nrm = rk.encode(idx)
        else:
            _, nrm = rk.gather(idx)
            dist.all_reduce(nrm, op=dist.ReduceOp.MAX)
            w = rk.encode_gathered()
            dist.all_reduce(w)
        rk.decode(w, idx, x4, 1.0 / world)

    t = sync_ms(rk_step, reps=max(200, reps))
    kr = max(200, reps)
    if rk.fused:
        kt4 = {"gather_absmax_encode (one launch)": _events(torch, lambda: rk.encode(idx), kr)}
    else:
        kt4 = {"gather_absmax": _events(torch, lambda: rk.gather(idx), kr),
               "encode_gathered": _events(torch, rk.encode_gathered, kr)}
    kt4["decode_scatter"] = _events(torch, lambda: rk.decode(rk.words, idx, x4, 1.0 / world), kr)
    # the previous round's three-launch form (gather-absmax, gather-encode, decode-scatter), for comparison
    nrm4 = torch.empty(1, device=dev)
    comp = gcodec.GlobalRandKMaxNormCompressor(dev, 4, generator=gen)

    def rk_step_3():
        codec.absmax(x4, idx=idx, out=nrm4)
        if world > 1:
            dist.all_reduce(nrm4, op=dist.ReduceOp.MAX)
        w = comp.encode(nrm4, x4, world, idx=idx)
        if world > 1:
            dist.all_reduce(w)
        comp.decode(nrm4, w, K4, world, 1.0 / world, idx=idx, out=x4)

    t3 = sync_ms(rk_step_3, reps=max(200, reps))
    # the reducer step itself (reducer.py:697-766) on the VGG16 tensor list: flatten
    # (+ norm) -> device index pop -> encode -> SUM -> decode-scatter -> setgrad (x1/W
    # of all n coordinates: the reference keeps the local gradient of the rest)
    sizes4 = shapes.vgg16_sizes()
    gin4 = list(torch.split(x4, sizes4))
    gout4 = [torch.empty_like(t_) for t_ in gin4]
    red4 = gcodec.GlobalRandKMaxNormReducer(dev, seed=42, K=K4, quantization_level=4, generator=gen)
    t_red = sync_ms(lambda: red4.reduce(gin4, gout4), reps=max(200, reps))
    segs_in, segs_out = codec.Segments(gin4), codec.Segments(gout4)
    rgen = gcodec.Generator(3, "philox")
    if codec.randk_fused_ok(K4, 4, world):
        red_kernels = {"gather_absmax_encode_from_tensors": _events(
            torch, lambda: codec.randk_encode_w1_segments(segs_in, idx, 4, rgen.reserve(K4)), 50)}
    else:
        red_kernels = {"gather_absmax_from_tensors": _events(
            torch, lambda: codec.randk_gather_absmax_segments(segs_in, idx), 50)}
    red_kernels["setgrad_tensor_to_tensor"] = _events(
        torch, lambda: codec.segments_copy(segs_in, segs_out, 1.0 / world), 50)
    red_kernels["decode_scatter_into_tensors"] = _events(
        torch, lambda: codec.qsgd_decode_scatter_segments(rk.words, idx, rk.norm, 4, segs_out, world, 1.0 / world),
        50)
    del gin4, gout4, red4, segs_in, segs_out
    gpu_us = sum(kt4.values()) * 1e3
    res["config4_grandk_k10000"] = {
        "n": n4, "K": K4, "us_per_step": t * 1e3, "us_per_step_three_launch_codec_calls": t3 * 1e3,
        "reducer_us_per_step": t_red * 1e3,
        "reducer_kernels_us": {k: v * 1e3 for k, v in red_kernels.items()},
        "reducer_step": "GlobalRandKMaxNormReducer.reduce(54 VGG16 tensors), no flat bucket: device index pop "
                        "(one permutation upload per refill), gather + norm + encode read from the tensors, "
                        "setgrad of all n tensor to tensor (x 1/W), decode-scatter into grad_out",
        "step": ("gather+absmax+encode (1 launch), decode-scatter" if rk.fused else
                 "gather+absmax, MAX, encode(gathered), SUM(words), decode-scatter"),
        "kernels_us": {k: v * 1e3 for k, v in kt4.items()},
        "bound": ("kernel latency (the step's launches sum to %.1f us of the %.1f us step)" % (gpu_us, t * 1e3)
                  if gpu_us > 0.8 * t * 1e3 else
                  "host issue (launches sum to %.1f us of the %.1f us step)" % (gpu_us, t * 1e3))}
    if world == 1:
        # the same step captured once in a HIP graph and replayed: the C ABI enqueues on
        # the caller's stream with no allocation or host sync, so the launches capture
        # as-is; a replay reuses the captured draw offset (timing only)
        try:
            graph = torch.cuda.CUDAGraph()
            side = torch.cuda.Stream(dev)
            side.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(side):
                rk_step()
            torch.cuda.current_stream(dev).wait_stream(side)
            with torch.cuda.graph(graph):
                rk_step()
            res["config4_grandk_k10000"]["hipgraph_us_per_step"] = _events(torch, graph.replay, max(200, reps)) * 1e3
        except Exception as e:  # capture unsupported on this runtime: report, do not fail the bench
            res["config4_grandk_k10000"]["hipgraph_us_per_step"] = f"capture failed: {type(e).__name__}: {e}"
    del x4
    return res


def _config5(torch, dist, gcodec, codec, dev, world, sync_ms, n5):
    """config 5: 1B fp32, 8-bit, chunked encode | RCCL SUM | decode on separate
    streams.  N > 1: one extra traced call records, from HIP events, whether
    chunk c's decode started (and finished) before chunk c+1's SUM ended."""
    res = {}
    gen = gcodec.Generator(17, "philox")
    try:
        x5 = torch.empty(n5, device=dev).normal_(0, 0.01)
        out5 = torch.empty_like(x5)
        pipe = gcodec.ChunkedQSGDAllReduce(n5, 8, dev, chunks=8, generator=gen)
        t = sync_ms(lambda: pipe(x5, out5), reps=3)
        ln = codec.qsgd_layout(n5, 8, world)
        r = {"n": n5, "chunks": 8, "ms_per_step": t, "grad_floats_per_s": world * n5 / (t * 1e-3),
             "lane_bits": ln.bits, "packed_bytes_per_rank": 4 * ln.plane_words,
             "reference_wire_bytes_per_rank": 4 * n5}
        if world > 1:
            tr = pipe.trace(x5, out5)
            r["overlap"] = tr
        res["config5_1b_8bit_chunked"] = r
        del pipe
        if world == 1:
            # config 5's own lane width on one GPU: lanes sized for W = 8 (12-bit, 2 per word),
            # no collective; the full-bucket encode / decode kernels timed with HIP events
            pipe8 = gcodec.ChunkedQSGDAllReduce(n5, 8, dev, chunks=8, generator=gen, world=8, collective=False)
            t8 = sync_ms(lambda: pipe8(x5, out5), reps=3)
            del pipe8
            l8 = codec.qsgd_layout(n5, 8, 8)
            w8 = torch.empty(l8.plane_words, dtype=torch.int32, device=dev)
            nrm5 = codec.absmax(x5)
            ms_e = _events(torch, lambda: codec.qsgd_encode(x5, nrm5, 8, gen.reserve(n5), 8, out=w8, lanes=l8), 5)
            ms_d = _events(torch, lambda: codec.qsgd_decode(w8, n5, nrm5, 8, 8, 1.0 / 8, out=out5, lanes=l8), 5)
            eb = 4 * n5 + 4 * l8.plane_words

            def kr(ms):
                gbs = eb / (ms * 1e-3) / 1e9
                return {"us": ms * 1e3, "algorithmic_bytes": eb, "gbs": gbs, "frac_hbm_peak": gbs / HBM_PEAK_GBS}

            res["config5_1b_8bit_w8_lanes"] = {
                "n": n5, "chunks": 8, "world_lanes": 8, "lane_bits": l8.bits, "lanes_per_word": l8.per_word,
                "packed_bytes_per_rank": 4 * l8.plane_words, "reference_wire_bytes_per_rank": 4 * n5,
                "ms_per_step_chunked_no_collective": t8, "grad_floats_per_s": n5 / (t8 * 1e-3),
                "k_qsgd_encode": kr(ms_e), "k_qsgd_decode": kr(ms_d),
                "note": "the W = 8 layout of config 5 (compressors.py:294-297, reducer.py:498-554 at b = 8) on one "
                        "GPU: the same kernels an 8-GPU rank runs, without the SUM"}
            del w8
    except torch.cuda.OutOfMemoryError:
        res["config5_1b_8bit_chunked"] = {"skipped": "out of device memory"}
    torch.cuda.empty_cache()
    return res


def _timed_steps(torch, dist, fn, k, world, dev) -> float:
    """Seconds for k calls of fn, barrier + synchronize on both sides, MAX over ranks."""
    for _ in range(2):
        fn()
    torch.cuda.synchronize()
    if world > 1:
        dist.barrier()
    t0 = time.perf_counter()
    for _ in range(k):
        fn()
    torch.cuda.synchronize()
    if world > 1:
        dist.barrier()
    el = time.perf_counter() - t0
    if world > 1:
        t = torch.tensor([el], dtype=torch.float64, device=dev)
        dist.all_reduce(t, op=dist.ReduceOp.MAX)
        el = t.item()
    return el


def reduce_legs(torch, dist, codec, step, words, dec, norm, n, bits, world, lanes, K, dev) -> dict:
    x_of = lambda f: f.x  # noqa: E731 — the headline bucket and encode, carried on step()
    enc_of = lambda f: f.encode  # noqa: E731
    """The full DP path: absmax -> MAX -> encode -> all_reduce(SUM packed words)
    -> decode + 1/W; at N >= 4 (even) also through gcodec.NodeTopology as two
    'nodes' of N/2 ranks, with the flat and hierarchical sums compared."""
    res = {}

    def path():
        step()
        if world > 1:
            dist.all_reduce(words)
        codec.qsgd_decode(words, n, norm, bits, world, 1.0 / world, out=dec, lanes=lanes)

    pel = _timed_steps(torch, dist, path, K, world, dev)
    rp = {"grad_floats_per_s": world * n * K / pel, "ms_per_step": pel / K * 1e3,
          "packed_bytes_per_rank": 4 * lanes.plane_words,
          "steps": "absmax, all_reduce MAX, encode, all_reduce SUM (RCCL), decode + 1/W"}
    # per phase, from HIP events on the codec's (torch's current) stream: an
    # event after each phase of one path() call; RCCL runs on its own stream and
    # the current stream waits for it, so the event after a collective marks its
    # completion as the next phase sees it.  Median of 5 traced calls, MAX over ranks.
    names = ("absmax", "max", "encode", "sum", "decode")
    traced = []
    for _ in range(5):
        ev = [torch.cuda.Event(enable_timing=True) for _ in range(6)]
        torch.cuda.synchronize()
        if world > 1:
            dist.barrier()
        ev[0].record()
        codec.absmax(x_of(step), out=norm)
        ev[1].record()
        if world > 1:
            dist.all_reduce(norm, op=dist.ReduceOp.MAX)
        ev[2].record()
        enc_of(step)()
        ev[3].record()
        if world > 1:
            dist.all_reduce(words)
        ev[4].record()
        codec.qsgd_decode(words, n, norm, bits, world, 1.0 / world, out=dec, lanes=lanes)
        ev[5].record()
        torch.cuda.synchronize()
        traced.append([ev[i].elapsed_time(ev[i + 1]) for i in range(5)])
    ph = torch.tensor([sorted(c)[2] for c in zip(*traced)], dtype=torch.float64, device=dev)
    if world > 1:
        dist.all_reduce(ph, op=dist.ReduceOp.MAX)
    rp["phase_ms"] = dict(zip(names, ph.tolist()))
    rp["phase_method"] = ("HIP events between the phases of one call on the current stream (median of 5 calls, "
                          "MAX over ranks); the untraced path above is what ms_per_step measures")
    if world > 1:
        # the packed SUM alone, and the reference's NoneAllReducer (reducer.py:140-170): an
        # fp32 all_reduce of the same bucket, both timed as K barrier-bracketed calls, MAX over ranks
        busf = 2.0 * (world - 1) / world
        t_sum = _timed_steps(torch, dist, lambda: dist.all_reduce(words), K, world, dev) / K
        pb = 4 * lanes.plane_words
        xf = x_of(step).clone()
        t_f32 = _timed_steps(torch, dist, lambda: dist.all_reduce(xf), K, world, dev) / K
        del xf
        rp["sum_packed"] = {"ms": t_sum * 1e3, "bytes_per_rank": pb, "algbw_gbs": pb / t_sum / 1e9,
                            "busbw_gbs": busf * pb / t_sum / 1e9}
        rp["sum_fp32_reference"] = {"ms": t_f32 * 1e3, "bytes_per_rank": 4 * n, "algbw_gbs": 4 * n / t_f32 / 1e9,
                                    "busbw_gbs": busf * 4 * n / t_f32 / 1e9,
                                    "reference": "NoneAllReducer, reducer.py:140-170 (fp32 all_reduce of the bucket)"}
        rp["sum_fp32_over_packed"] = t_f32 / t_sum
        rp["wire_bytes_fp32_over_packed"] = 4 * n / pb
        rp["busbw_note"] = ("busbw = 2(N-1)/N x bytes / t (ring all-reduce); MI355X xGMI: 7 links x ~153 GB/s per "
                            "GPU, one ring uses one link each way")
    rp["rng"] = "philox (the headline's explicit Generator; torch mode is timed in torch_parity_mode)"
    res["reduce_path"] = rp
    if world >= 4 and world % 2 == 0:
        # intra reduce-scatter, "inter-node" all-reduce of 1/L of the words, intra
        # all-gather: the multi-node code path on one node
        try:
            from gcodec.topology import NodeTopology
            topo = NodeTopology(world // 2)

            def hpath():
                step()
                topo.all_reduce(words)
                codec.qsgd_decode(words, n, norm, bits, world, 1.0 / world, out=dec, lanes=lanes)

            hel = _timed_steps(torch, dist, hpath, K, world, dev)
            step()  # flat vs hierarchical sum of the same encoded words
            a = words.clone()
            dist.all_reduce(a)
            b = words.clone()
            topo.all_reduce(b)
            ok = torch.tensor([int(torch.equal(a, b))], device=dev)
            dist.all_reduce(ok, op=dist.ReduceOp.MIN)  # every rank's sums agree
            res["reduce_path_2x_nodes"] = {"ms_per_step": hel / K * 1e3, "local_size": world // 2,
                                           "bit_identical_to_flat": bool(ok.item())}
        except Exception as e:  # noqa: BLE001 — report, never fail the headline bench
            res["reduce_path_2x_nodes"] = f"failed: {type(e).__name__}: {e}"
    return res


def torch_mode_leg(torch, np, gcodec, codec, x, n, bits, words, lanes, dev, pgen_philox) -> dict:
    """Reference-parity mode (compressors.py:310 under torch.manual_seed): the
    torch CPU generator's MT19937 stream made on the GPU (jumped parallel
    generators on two side streams), then the encode from those draws; torch's
    generator state advances exactly as the reference's would.  Timed three
    ways against the Philox path in the same harness (W = 1 lanes):
    encode only (norm fixed), absmax + encode per call (what a reducer does),
    and a training cadence (each call behind a few ms of unrelated GPU work,
    the backward, so the speculation has time to run ahead)."""
    from gcodec import compressors as gcomp

    pgen = gcodec.Generator(0, "torch")
    torch.manual_seed(42)
    nm = codec.absmax(x)
    pgen.reserve(n)  # warm: builds the jump table once per process
    codec.qsgd_encode_torch(x, nm, bits, 1, out=words, lanes=lanes)
    fmt = gcomp.TORCH_DRAW_FORMAT  # the draw format the compressors' packed encode asks for

    def enc_fmt(f):
        codec.qsgd_encode(x, nm, bits, pgen.reserve(n, fmt=f), 1, out=words, lanes=lanes)

    def enc_torch():  # the product's form (QSGDMaxNormCompressor.encode in torch mode)
        enc_fmt(fmt)

    def step_torch():
        codec.absmax(x, out=nm)
        enc_torch()

    def enc_philox():
        codec.qsgd_encode(x, nm, bits, pgen_philox.reserve(n), 1, out=words, lanes=lanes)

    def step_philox():
        codec.absmax(x, out=nm)
        enc_philox()

    def per_call_ms(fn, reps=20, runs=3):
        for _ in range(8):  # warm: both end-state jump polynomials of this count, the speculation started
            fn()
        torch.cuda.synchronize()
        best = []
        for _ in range(runs):  # the fastest of `runs` timed loops
            t0 = time.perf_counter()
            for _ in range(reps):
                fn()
            torch.cuda.synchronize()
            best.append((time.perf_counter() - t0) / reps * 1e3)
        return min(best), best

    codec.mt_stats(reset=True)
    enc_ms, enc_runs = per_call_ms(enc_torch)
    held = codec.mt_reserved_bytes(dev)  # what the speculation holds while calls repeat
    plan = codec._mt_plan(n, fmt, True)
    other_fmts = {}
    for f in ("plain", "split16", "packed24"):
        if f != fmt:
            codec.mt_release(dev)
            other_fmts[f] = per_call_ms(lambda: enc_fmt(f))[0]
    codec.mt_release(dev)
    stp_ms, stp_runs = per_call_ms(step_torch)
    enc_px, _ = per_call_ms(enc_philox)
    stp_px, _ = per_call_ms(step_philox)
    t0 = time.perf_counter()
    for _ in range(20):  # fused: the generator kernel quantizes with its own draws, then the lane pack
        codec.qsgd_encode_torch(x, nm, bits, 1, out=words, lanes=lanes)
    torch.cuda.synchronize()
    t_fused = (time.perf_counter() - t0) / 20 * 1e3

    # training cadence: a stand-in backward (bf16 GEMMs, ~3 ms) between calls
    a = torch.randn(8192, 8192, device=dev, dtype=torch.bfloat16)
    c = torch.empty_like(a)

    def backward():
        for _ in range(3):
            torch.mm(a, a, out=c)

    bw_ms, _ = per_call_ms(backward, reps=10)
    cad_torch, _ = per_call_ms(lambda: (backward(), step_torch()), reps=10)
    cad_px, _ = per_call_ms(lambda: (backward(), step_philox()), reps=10)
    del a, c
    paths = codec.mt_stats(reset=True)

    st = codec.mt19937_seed_state(42)
    sd = torch.from_numpy(st.view(np.int32)).to(dev)
    draws = torch.empty(n, dtype=torch.int32, device=dev)
    ms_gen = _events(torch, lambda: codec.mt19937_generate(sd, n, out=draws), 3)
    ms_ser = _events(torch, lambda: codec.mt19937_generate(sd, 10_000_000, out=draws, parallel=False), 1)
    del draws
    return {
        "n": n,
        "encode_only": {"ms_per_call": enc_ms, "grad_floats_per_s": n / (enc_ms * 1e-3), "runs_ms": enc_runs,
                        "draws": fmt, "other_draw_formats_ms_per_call": other_fmts,
                        "philox_ms_per_call": enc_px, "frac_of_philox_rate": enc_px / enc_ms},
        "speculation": {"held_device_bytes": held, "budget_bytes": codec.MT_SPECULATE_BUDGET,
                        "calls_per_run": plan[0], "calls_ahead": plan[1],
                        "bytes_per_call": codec.mt_format_bytes(n, fmt),
                        "reserve_paths": paths,
                        "note": "device memory the torch-mode speculation holds between calls "
                                "(codec.mt_reserved_bytes: queued draws, workspaces, tables); reserve_paths = "
                                "codec.mt_stats() over this leg's torch-mode calls (queued = served from the "
                                "speculative queue, fresh_* = made on demand, and why)"},
        "absmax_plus_encode": {"ms_per_call": stp_ms, "grad_floats_per_s": n / (stp_ms * 1e-3), "runs_ms": stp_runs,
                               "philox_ms_per_call": stp_px, "frac_of_philox_rate": stp_px / stp_ms},
        "training_cadence": {"backward_standin_ms": bw_ms, "torch_added_ms_per_call": cad_torch - bw_ms,
                             "philox_added_ms_per_call": cad_px - bw_ms,
                             "note": "each step = 3 bf16 8192^3 GEMMs (the stand-in backward) then absmax + "
                                     "encode; added = step - GEMMs alone (the side-stream draws run during "
                                     "the GEMMs and share the chip with them)"},
        "fused_generator_quantize_ms_per_call": t_fused,
        "mt19937_parallel_ms": ms_gen, "mt19937_parallel_draws_per_s": n / (ms_gen * 1e-3),
        "mt19937_serial_draws_per_s": 10_000_000 / (ms_ser * 1e-3),
        "note": "torch-CPU-generator (MT19937) draws, bit-exact with compressors.py: jump-ahead parallel "
                "generators on two side streams (phase 1 = sequence + jumps + a jump straight to "
                "the end state, phase 2 = the generators) -> encode from the draws on the caller's stream; "
                "torch's state is written back every call (host sync) as soon as phase 1 is done; back to back, "
                "the next same-size call's run is enqueued behind this one and used only if torch's generator "
                "is untouched.  The headline (Philox) step is absmax + encode: compare absmax_plus_encode."}


def packers_leg(torch, gcodec, codec, dev, gen, rank) -> dict:
    """The literal drop-in packers on the ResNet50 bucket (23,520,842 elements,
    4-bit sign + xi of the QSGDBP call site, compressors.py:338-378): device
    greedy 4-mode pack / unpack (Extension CPU/bitpacking.cpp:16-55) and byte
    pack / unpack (Extension CPU BP/bytepacking.cpp:6-64), each timed as queued
    launches with HIP events; algorithmic bytes = what the call must read +
    write.  Plus the QSGDBPCompressor.compress / decompress calls end to end
    (they synchronise: word counts go to the host)."""
    n = 23_520_842
    g = torch.Generator(device=dev).manual_seed(21 + rank)
    x = torch.randn(n, device=dev, generator=g).mul_(0.01)
    nm = codec.absmax(x)
    xi, sg = codec.qsgd_quantize_split(x, nm, 4, gen.reserve(n))
    res = {"n": n, "bits": 4}

    def row(us, nbytes, **kw):
        gbs = nbytes / (us * 1e-6) / 1e9
        return {"us": us, "algorithmic_bytes": nbytes, "gbs": gbs, "frac_hbm_peak": gbs / HBM_PEAK_GBS, **kw}

    pk = gcodec.codec.Greedy4Device(n, dev)
    for name, src in (("xi", xi), ("sign", sg)):
        pk.pack(src)
        nw = pk.result()
        w = pk.words[:nw].clone()
        us_p = _events(torch, lambda: pk.pack(src), 20) * 1e3
        pk.unpack(w)
        cnt = pk.unpack_result()
        ok = bool(torch.equal(pk.values[:n], src))
        us_u = _events(torch, lambda: pk.unpack(w), 20) * 1e3
        res[f"greedy4_pack_{name}"] = row(us_p, 4 * n + 4 * nw, words=nw)
        res[f"greedy4_unpack_{name}"] = row(us_u, 4 * nw + 4 * cnt, values=cnt, round_trip_exact=ok)
    q8 = codec.qsgd_quantize(x, nm, 4, gen.reserve(n))
    bw = codec.bytepack8(q8)
    us_bp = _events(torch, lambda: codec.bytepack8(q8), 20) * 1e3
    us_bu = _events(torch, lambda: codec.byteunpack8(bw), 20) * 1e3
    res["bytepack8_int8"] = row(us_bp, n + 8 * bw.numel())
    res["byteunpack8"] = row(us_bu, 8 * bw.numel() + 8 * bw.numel())
    comp = gcodec.QSGDBPCompressor(dev, 4, generator=gen)
    c = comp.compress(x)
    t0 = time.perf_counter()
    for _ in range(10):
        c = comp.compress(x)
    torch.cuda.synchronize()
    t_c = (time.perf_counter() - t0) / 10 * 1e3
    comp.decompress(c[0], c[1], c[2], n)  # warm: the unpack buffers' first allocation
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(10):
        comp.decompress(c[0], c[1], c[2], n)
    torch.cuda.synchronize()
    t_d = (time.perf_counter() - t0) / 10 * 1e3
    res["qsgdbp_compress_ms"] = t_c
    res["qsgdbp_decompress_ms"] = t_d
    res["qsgdbp_note"] = ("compress = absmax + quantize_split + 2 device greedy4 packs + 2 host syncs (both word "
                          "counts in one read, then the norm); decompress = 2 device greedy4 unpacks (1 host sync: "
                          "both value counts) + the fused combine (gc_qsgdbp_decode); the reference packs on the "
                          "host at 0.56 M elem/s (BASELINE.md)")
    del x, xi, sg, q8, bw, pk
    return res


def _free_port() -> int:
    import socket

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def launch_ranks(n: int) -> int:
    """`python bench.py --gpus N` (N > 1) without a launcher: start N ranks
    as ONE child `python -m torch.distributed.run` (one process per GPU,
    rendezvous on 127.0.0.1), before this process has touched the GPU, and
    return the child's exit code.  Never an exec: the child is a separate
    process, this one only forwards its output (rank 0's JSON line included)."""
    import subprocess

    # torchrun's own parser would take a bare "--n" as an abbreviation of its options
    fwd = ["--numel" if a == "--n" else ("--numel=" + a[4:] if a.startswith("--n=") else a) for a in sys.argv[1:]]
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", str(n),
           "--master-addr", "127.0.0.1", "--master-port", str(_free_port()),
           os.path.abspath(__file__), *fwd]
    print(f"bench.py: --gpus {n} without WORLD_SIZE: launching {n} ranks ({' '.join(cmd[1:5])} ...)",
          file=sys.stderr, flush=True)
    env = dict(os.environ, GC_BENCH_LAUNCHED="1")
    return subprocess.run(cmd, env=env).returncode


def main():
    args = _args()
    if args.gpus < 1:
        print(f"bench.py: --gpus {args.gpus} must be >= 1", file=sys.stderr)
        return 2
    if args.gpus > 1 and "WORLD_SIZE" not in os.environ:
        if os.environ.get("GC_BENCH_LAUNCHED"):  # the child launcher did not set it: never recurse
            print("bench.py: launched ranks have no WORLD_SIZE", file=sys.stderr)
            return 2
        return launch_ranks(args.gpus)
    world = int(os.environ.get("WORLD_SIZE", "1"))
    if world != args.gpus:
        print(f"bench.py: --gpus {args.gpus} but WORLD_SIZE={world}: the launcher and the flag disagree",
              file=sys.stderr)
        return 2

    import numpy as np
    import torch
    import torch.distributed as dist

    import gcodec
    from gcodec import codec

    rank = int(os.environ.get("RANK", "0"))
    local = int(os.environ.get("LOCAL_RANK", "0"))
    # GC_BENCH_BACKEND=gloo: rehearsal of the N>1 control flow on a 1-GPU box
    # (ranks share the card, collectives go through gloo; not a perf number)
    backend = os.environ.get("GC_BENCH_BACKEND", "nccl")
    if backend != "nccl":
        local %= max(torch.cuda.device_count(), 1)
    elif world > 1 and torch.cuda.device_count() < world:  # device_count does not initialise the GPU
        print(f"bench.py: {world} ranks over RCCL need {world} GPUs, {torch.cuda.device_count()} visible",
              file=sys.stderr)
        return 2
    torch.cuda.set_device(local)
    dev = torch.device("cuda", local)
    if world > 1:
        if backend == "nccl":
            dist.init_process_group("nccl", device_id=dev)
        else:
            dist.init_process_group(backend)
    n, bits, K, Wm = args.n, args.bits, args.steps, args.warmup

    g = torch.Generator(device=dev).manual_seed(1234 + rank)
    x = torch.randn(n, device=dev, generator=g, dtype=torch.float32).mul_(0.01)
    gen = gcodec.Generator(42 + rank, "philox")
    lanes = codec.qsgd_layout(n, bits, world)
    M = lanes.plane_words
    words = torch.empty(M, dtype=torch.int32, device=dev)
    norm = torch.empty(1, dtype=torch.float32, device=dev)

    def norm_step():
        codec.absmax(x, out=norm)
        if world > 1:
            dist.all_reduce(norm, op=dist.ReduceOp.MAX)

    def encode_step():
        codec.qsgd_encode(x, norm, bits, gen.reserve(n), world, out=words, lanes=lanes)

    def step():
        norm_step()
        encode_step()

    step.x, step.encode = x, encode_step  # for reduce_legs' per-phase trace

    norms = (norm, torch.empty_like(norm))

    def run_steps(k, buckets=None):
        """k whole steps over `buckets` ((x, words, lanes) triples, cycled; the
        headline bucket by default).  N > 1: software-pipelined over consecutive
        buckets, as a bucketed DDP backward issues them: bucket t's max-norm and
        its async all_reduce(MAX) are enqueued before bucket t-1's encode, so the
        RCCL latency of the 4-byte MAX runs beside an encode instead of between
        the two kernels.  Every bucket still runs absmax -> MAX -> encode with its
        own global norm (two norm buffers; the encode waits on its bucket's MAX
        work only).  The last bucket's encode is issued before returning, so k
        steps are complete when the caller synchronises."""
        if world == 1 and buckets is None:
            for _ in range(k):
                step()
            return
        bks = buckets or [(x, words, lanes)]
        pend = None
        for t in range(k):
            xb, wb, lb = bks[t % len(bks)]
            nb = norms[t & 1]
            codec.absmax(xb, out=nb)
            work = dist.all_reduce(nb, op=dist.ReduceOp.MAX, async_op=True) if world > 1 else None
            if pend is not None:
                _encode_pending(pend)
            pend = (xb, wb, lb, nb, work)
        if pend is not None:
            _encode_pending(pend)

    def _encode_pending(p):
        px, pw, pl, pn, pwork = p
        if pwork is not None:
            pwork.wait()  # the current stream waits on this bucket's MAX (no host block on RCCL)
        codec.qsgd_encode(px, pn, bits, gen.reserve(px.numel()), world, out=pw, lanes=pl)

    # clock settle (untimed), then the W warmup steps
    settle_steps = 0
    t_settle = time.perf_counter()
    while args.settle > 0:
        run_steps(20)
        settle_steps += 20
        torch.cuda.synchronize()
        done = torch.tensor([float(time.perf_counter() - t_settle >= args.settle)], device=dev)
        if world > 1:  # every rank runs the same number of steps (each step holds collectives)
            dist.all_reduce(done, op=dist.ReduceOp.MAX)
        if done.item() > 0:
            break
    run_steps(Wm)
    torch.cuda.synchronize()
    if world > 1:
        dist.barrier()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    run_steps(K)
    torch.cuda.synchronize()
    if world > 1:
        dist.barrier()
    el = time.perf_counter() - t0
    if world > 1:
        t = torch.tensor([el], dtype=torch.float64, device=dev)
        dist.all_reduce(t, op=dist.ReduceOp.MAX)
        el = t.item()
    ms_step = el / K * 1e3
    value = world * n * K / el

    # the pipelined issue order against the plain one on two different buckets
    # (two slices of x with different norms, same draws): the packed words must
    # be bit-identical, so no bucket ever encodes with another bucket's norm
    m = max(1, min(n // 2, 1 << 22))
    lm = codec.qsgd_layout(m, bits, world)
    xa, xb = x[:m], x[m:2 * m]
    wp = [torch.empty(lm.plane_words, dtype=torch.int32, device=dev) for _ in range(4)]
    off = gen.offset
    run_steps(3, [(xa, wp[0], lm), (xb, wp[1], lm)])  # a, b, a: wp[0] ends with the third bucket
    gen.offset = off
    for xs, ws in ((xa, wp[2]), (xb, wp[3]), (xa, wp[2])):
        codec.absmax(xs, out=norm)
        if world > 1:
            dist.all_reduce(norm, op=dist.ReduceOp.MAX)
        codec.qsgd_encode(xs, norm, bits, gen.reserve(m), world, out=ws, lanes=lm)
    torch.cuda.synchronize()
    pipe_ok = bool(torch.equal(wp[0], wp[2]) and torch.equal(wp[1], wp[3]))
    del wp

    # ---- per-kernel HIP-event timing (roofline.achieved), on the stream the
    # codec launches on (torch's current stream), one event pair per loop (an
    # event pair per launch inflated the kernel times by ~13 % at the driver's
    # 20 steps).  The encode is timed as it runs IN the step: the
    # local step loop (absmax -> encode with the global norm) minus the
    # absmax-only loop.  In the step the encode follows a full read of x by the
    # absmax and finds its tail in the 256 MB Infinity Cache; back to back
    # (encode_isolated) it does not, and takes ~8 % longer.  So absmax +
    # encode = the step's GPU time, which the timed step's wall clock bounds.
    reps = max(K, 200)
    nrm_scratch = torch.empty_like(norm)
    torch.cuda.synchronize()
    if world > 1:
        codec.absmax(x, out=norm)
        dist.all_reduce(norm, op=dist.ReduceOp.MAX)  # the encode's global norm, held fixed
    ms_absmax = _events(torch, lambda: codec.absmax(x, out=nrm_scratch), reps)

    def step_local():  # absmax -> encode, the MAX left out (N > 1: the encode keeps the global norm)
        codec.absmax(x, out=nrm_scratch if world > 1 else norm)
        encode_step()

    ms_step_events = _events(torch, step_local, reps)
    ms_absmax2 = _events(torch, lambda: codec.absmax(x, out=nrm_scratch), reps)
    ms_absmax = 0.5 * (ms_absmax + ms_absmax2)  # bracketing the step loop (clock drift)
    # N = 1: the timed loop holds nothing but absmax -> encode, so the step's own
    # clock bounds their sum too; the smaller of the two step measurements is the
    # one with less clock drift / host jitter in it (they differ by ~1 %)
    ms_step_gpu = min(ms_step_events, ms_step) if world == 1 else ms_step_events
    ms_encode = ms_step_gpu - ms_absmax
    ms_encode_iso = _events(torch, encode_step, reps)
    enc_bytes = 4 * n + 4 * M  # read x once, write the packed words
    achieved = enc_bytes / (ms_encode * 1e-3) / 1e9
    step_bytes = 8 * n + 4 * M  # + the max-norm read of x

    out = {
        "metric": "grad-floats/sec encode+pack (device-resident), 100M fp32 bucket; % HBM peak",
        "value": value,
        "unit": "grad-floats/s",
        "n_gpus": world,
        "steps": K,
        "warmup": Wm,
        "ms_per_step": ms_step,
        "higher_is_better": True,
        "scaling": "weak",
        "vs_baseline": None,
        "dtype": "f32->u32 (int lanes)",
        "data": "synthetic N(0, 0.01) fp32 bucket generated on device; Philox4x32-10 draws",
        "config": {"workload": f"QSGD-MN {bits}-bit encode+pack, {n} fp32 per rank, W={world} carry-free "
                               f"{lanes.bits}-bit lanes x{lanes.per_word}/word",
                   "global_batch": n * world, "parallelism": f"dp{world}",
                   "step": "absmax -> all_reduce(MAX) if N>1 -> quantize+round+pack",
                   "pipelining": ("bucket t's absmax + async RCCL MAX enqueued before bucket t-1's encode "
                                  "(double-buffered norm)" if world > 1 else None)},
        "clock_settle": {"seconds": args.settle, "steps": settle_steps},
        "pipelined_issue_bit_identical": pipe_ok,
        "collectives": backend if world > 1 else None,
        "pct_hbm_peak_step": 100.0 * step_bytes * K / el / 1e9 / HBM_PEAK_GBS,
        "roofline": {"bound": "hbm", "kernel": "k_qsgd_encode", "achieved": achieved, "peak": HBM_PEAK_GBS,
                     "unit": "GB/s", "frac": achieved / HBM_PEAK_GBS,
                     "traffic": _traffic("k_qsgd_encode", n, bits)[0],
                     "traffic_source": _traffic("k_qsgd_encode", n, bits)[1],
                     "bytes_per_launch": enc_bytes, "ms_per_launch": ms_encode},
        "kernels_ms": {"k_absmax": ms_absmax, "k_qsgd_encode": ms_encode},
        "kernel_timing": {"method": f"HIP event pairs around {reps}-launch loops on the codec's stream: "
                                    "k_absmax = absmax-only loop (before and after), k_qsgd_encode = "
                                    "(absmax -> encode) step time - absmax loop, i.e. the encode as it runs in "
                                    "the step; step time = min(step event loop, timed step) at N = 1 (the timed "
                                    "loop is the same two launches), the event loop at N > 1",
                          "step_events_ms": ms_step_events,
                          "k_qsgd_encode_isolated_ms": ms_encode_iso,
                          "absmax_plus_encode_ms": ms_absmax + ms_encode,
                          "fits_timed_step": ms_absmax + ms_encode <= ms_step},
    }
    if world > 1:
        out["process_group"] = _pg_evidence(torch, dist, dev, local, 4 * M)

    legs = args.legs
    dec = torch.empty(n, dtype=torch.float32, device=dev) if legs & {"decode", "reduce"} else None
    if "decode" in legs:
        # decode of the (W-summed) words, 1/W folded in
        ms_dec = _events(torch, lambda: codec.qsgd_decode(words, n, norm, bits, world, 1.0 / world, out=dec,
                                                           lanes=lanes), reps)
        out["kernels_ms"]["k_qsgd_decode"] = ms_dec
        out["decode_gbs"] = (4 * M + 4 * n) / (ms_dec * 1e-3) / 1e9

        # achievable-bandwidth reference: a STREAM-style device copy of
        # the bucket (read 4n + write 4n) through the runtime's own copy kernel
        ms_copy = _events(torch, lambda: dec.copy_(x), reps)
        copy_gbs = 8 * n / (ms_copy * 1e-3) / 1e9
        out["roofline"]["achievable_copy_gbs"] = copy_gbs
        out["roofline"]["frac_of_copy"] = out["roofline"]["achieved"] / copy_gbs
    if "reduce" in legs:
        out.update(reduce_legs(torch, dist, codec, step, words, dec, norm, n, bits, world, lanes, K, dev))
    del dec
    if "torch" in legs:
        out["torch_parity_mode"] = torch_mode_leg(torch, np, gcodec, codec, x, n, bits, words, lanes, dev, gen)
    if "pcie" in legs:
        # PCIe-inclusive: the reference's path starts and ends in host memory
        out["pcie_inclusive"] = pcie_inclusive(torch, codec, gen, x, n, bits, world, lanes, K)
    cfg = other_configs(torch, dist, gcodec, codec, dev, world, rank, K, legs, args.n5)
    if cfg:
        cfg["rng"] = ("philox (explicit Generator(seed, 'philox') in every config leg; the package default, "
                      "torch mode, is the reference-identical stream timed in torch_parity_mode)")
        out["configs"] = cfg
    if "packers" in legs:
        out["packers"] = packers_leg(torch, gcodec, codec, dev, gen, rank)

    if rank == 0 and world == 1 and args.cpu_seconds > 0:
        out["cpu_baseline"] = cpu_baseline(n, bits, args.cpu_seconds)

    if rank == 0:
        print(json.dumps(out), flush=True)
    if world > 1:
        dist.barrier()
        dist.destroy_process_group()


if __name__ == "__main__":
    sys.exit(main() or 0)
