"""The gradient table and the refusals of the clipping entry points, on the CPU:
every call here is turned down (or planned) by the host before any launch."""
import ctypes as C
import math
import os
import subprocess
import sys

import numpy as np
import pytest

from gcodec import _lib, clip

torch = pytest.importorskip("torch")

F32, F16, BF16 = _lib.GC_F32, _lib.GC_F16, _lib.GC_BF16


class Table:
    """A planned table over made-up addresses; `rec` stands for the device copy, which is never read here."""

    def __init__(self, sizes, ptrs, types):
        c = len(sizes)
        self.sizes = np.array(sizes, dtype=np.uint64)
        self.ptrs = np.array(ptrs, dtype=np.uint64)
        self.types = np.array(types, dtype=np.uint32)
        self.host = np.zeros(2 * (c + 1), dtype=np.uint64)
        self.order = np.zeros(max(c, 1), dtype=np.uint32)
        self.s = _lib.gc_grads()
        self.rc = _lib.load().gc_grads_plan(self.sizes.ctypes.data, self.ptrs.ctypes.data, self.types.ctypes.data, c,
                                            self.host.ctypes.data, self.order.ctypes.data, C.byref(self.s))
        self.s.rec = 0x1000

    @property
    def ref(self):
        return C.byref(self.s)


def err():
    return _lib.last_error()


def test_plan_lays_the_tensors_end_to_end():
    t = Table([3, 0, 5, 8], [0x4000, 0, 0x2000, 0x3000], [F32, F32, BF16, F16])
    assert t.rc == 0 and t.s.n == 16 and t.s.count == 4 and t.s.flags == 0
    assert t.host[1::2].tolist() == [0, 3, 3, 8, 16]
    assert [int(v) >> 56 for v in t.host[0::2]] == [0, 0, 2, 1, 0]
    assert [int(v) & ((1 << 56) - 1) for v in t.host[0::2]] == [0x4000, 0, 0x2000, 0x3000, 0]
    assert t.order.tolist() == [2, 3, 0, 1]  # by address, the empty one last


@pytest.mark.parametrize("sizes,ptrs,types,overlap", [
    ([4, 4], [0x1000, 0x1010], [F32, F32], False),  # touching
    ([4, 4], [0x1000, 0x100c], [F32, F32], True),   # the last element is the next one's first
    ([4, 4], [0x1000, 0x1000], [F32, F32], True),   # the same tensor twice
    ([9, 1, 1], [0x1000, 0x1002, 0x2000], [F16, BF16, F32], True),
    ([0, 4], [0x1000, 0x1000], [F32, F32], False),  # an empty tensor covers nothing
    ([64, 1, 1], [0x1000, 0x1004, 0x1200], [F32, F32, F32], True),  # inside another
])
def test_plan_finds_shared_memory(sizes, ptrs, types, overlap):
    t = Table(sizes, ptrs, types)
    assert t.rc == 0 and bool(t.s.flags & _lib.GC_GRADS_OVERLAP) == overlap


@pytest.mark.parametrize("sizes,ptrs,types,msg", [
    ([4], [0x1002], [F32], "aligned"),
    ([4], [0x1001], [BF16], "aligned"),
    ([4], [0], [F32], "no data pointer"),
    ([4], [0x1000], [_lib.GC_I32], "float32"),
    ([1 << 52], [0x1000], [F32], "overflow"),
])
def test_plan_refuses(sizes, ptrs, types, msg):
    t = Table(sizes, ptrs, types)
    assert t.rc == _lib.GC_EINVAL and msg in err()


WS, NORM = 0x100000, 0x200000


def clip_call(src, dst, p=2, max_norm=1.0, total=None, norm=NORM, ws=WS):
    return _lib.load().gc_grad_clip(src.ref, dst.ref, p, max_norm, total, norm, ws, None)


def test_clip_refuses_what_would_race_or_misread():
    a = Table([4, 8], [0x1000, 0x2000], [F32, F16])
    big = Table([9000], [0x80000], [F32])
    for bad, msg in [
        (Table([4], [0x3000], [F32]), "tensors into"),
        (Table([4, 9], [0x3000, 0x4000], [F32, F16]), "sizes"),
        (Table([4, 8], [0x3000, 0x3008], [F32, F16]), "share memory"),          # outputs overlap each other
        (Table([4, 8], [0x1004, 0x4000], [F32, F16]), "shares memory"),         # shifted onto its input
        (Table([4, 8], [0x2000, 0x4000], [F32, F16]), "shares memory"),         # onto another tensor's input
        (Table([4, 8], [0x1000, 0x2000], [F32, BF16]), "shares memory"),        # its own input under another type
    ]:
        assert clip_call(a, bad) == _lib.GC_EINVAL and msg in err(), err()
    twice = Table([4, 4], [0x1000, 0x1000], [F32, F32])
    assert clip_call(twice, twice) == _lib.GC_EINVAL and "share memory" in err()
    assert clip_call(big, big, ws=None) == _lib.GC_EINVAL and "workspace" in err()
    assert clip_call(a, a, ws=WS + 4) == _lib.GC_EINVAL and "workspace" in err()
    assert clip_call(a, a, p=3) == _lib.GC_EINVAL and "GC_NORM_INF" in err()
    for m in (-1.0, math.nan, -math.inf):
        assert clip_call(a, a, max_norm=m) == _lib.GC_EINVAL and "max_norm" in err()
    a.s.rec = None
    assert clip_call(a, a) == _lib.GC_EINVAL and "device" in err()


def test_norm_and_flatten_refuse():
    lib = _lib.load()
    a = Table([4, 8], [0x1000, 0x2000], [F32, F16])
    assert lib.gc_grad_norm(a.ref, 7, None, NORM, None, WS, None) == _lib.GC_EINVAL
    assert lib.gc_grad_norm(a.ref, 2, None, NORM, NORM, None, None) == _lib.GC_EINVAL and "workspace" in err()
    assert lib.gc_grad_norm(a.ref, 2, None, NORM, None, WS + 4, None) == _lib.GC_EINVAL and "workspace" in err()
    assert lib.gc_grad_workspace_size(12, 2, 0) == 0 < lib.gc_grad_workspace_size(12, 2, 1)
    assert lib.gc_grad_workspace_size(12, 1100, 0) > 0 and lib.gc_grad_workspace_size(9000, 1, 0) > 0
    assert lib.gc_grad_norm(None, 2, None, NORM, None, WS, None) == _lib.GC_EINVAL
    assert lib.gc_grad_norm_root(None, 2, NORM, None) == _lib.GC_EINVAL
    flat = lib.gc_grad_flatten_clip
    assert flat(a.ref, 0x3000, 2, 1.0, None, NORM, WS, None) == _lib.GC_EINVAL
    assert flat(a.ref, None, 2, 1.0, NORM, NORM, WS, None) == _lib.GC_EINVAL
    assert flat(a.ref, 0x3002, 2, 1.0, NORM, NORM, WS, None) == _lib.GC_EINVAL
    assert flat(a.ref, 0x3000, 2, -1.0, NORM, NORM, WS, None) == _lib.GC_EINVAL
    assert flat(a.ref, 0x1fe0, 2, 1.0, NORM, NORM, WS, None) == _lib.GC_EINVAL and "flat bucket" in err()


def test_decode_refuses():
    lib = _lib.load()
    a = Table([4, 8], [0x1000, 0x2000], [F32, F16])

    def call(g, n=12, bits=4, ln=None, words=0x8000, norm=0x9000, p=2, m=1.0, out=NORM, ws=WS):
        if ln is None:
            ln = _lib.gc_lanes()
            assert lib.gc_qsgd_layout(n, bits, 1, C.byref(ln)) == 0
        return lib.gc_qsgd_decode_clip(words, n, norm, bits, C.byref(ln), 1.0, g.ref, p, m, out, ws, None)

    for kw in (dict(n=13), dict(words=None), dict(words=0x8004), dict(norm=None), dict(out=None), dict(ws=WS + 4),
               dict(p=5), dict(m=math.nan), dict(words=0x2000), dict(norm=0x1004)):
        assert call(a, **kw) == _lib.GC_EINVAL, kw
    other = _lib.gc_lanes()
    assert lib.gc_qsgd_layout(12, 8, 1, C.byref(other)) == 0
    assert call(a, ln=other) == _lib.GC_EINVAL and "gc_qsgd_layout" in err()
    twice = Table([6, 6], [0x1000, 0x1000], [F32, F32])
    assert call(twice) == _lib.GC_EINVAL and "share memory" in err()


def test_what_a_call_writes_beside_the_tensors_stands_alone():
    """Blocks that are done write the norm while others still read: it shares memory with nothing the call uses."""
    lib = _lib.load()
    n = 20_000  # two launches
    a, b = Table([n, 8], [0x40000, 0x2000], [F32, F16]), Table([n, 8], [0x80000, 0x3000], [F32, F16])
    ln = _lib.gc_lanes()
    assert lib.gc_qsgd_layout(n + 8, 4, 1, C.byref(ln)) == 0
    words, scale = 0x300000, 0x9000

    def decode(out, norm=scale, ws=WS):
        return lib.gc_qsgd_decode_clip(words, n + 8, norm, 4, C.byref(ln), 1.0, b.ref, 2, 1.0, out, ws, None)

    for rc, msg in [
        (lambda: decode(scale), "share memory"),                          # the scale that every block reads
        (lambda: decode(words + 4 * ln.plane_words - 4), "share memory"),  # the last word
        (lambda: decode(0x80000 + 4 * n - 4), "output tensor 0"),
        (lambda: decode(0x3000), "output tensor 1"),
        (lambda: decode(WS), "share memory"),
        (lambda: decode(NORM, norm=WS + 8), "share memory"),
        (lambda: decode(NORM, ws=words), "share memory"),
        (lambda: decode(NORM, ws=0x80000), "output tensor 0"),
        (lambda: clip_call(a, b, norm=0x40000), "input tensor 0"),
        (lambda: clip_call(a, b, norm=0x2008), "input tensor 1"),
        (lambda: clip_call(a, b, norm=0x80004), "output tensor 0"),
        (lambda: clip_call(a, a, norm=0x40004), "tensor 0"),
        (lambda: clip_call(a, b, norm=WS + 16), "share memory"),
        (lambda: clip_call(a, b, total=NORM, norm=NORM + 4), "share memory"),
        (lambda: clip_call(a, b, total=0x80000), "output tensor 0"),
        (lambda: clip_call(a, b, ws=0x40000), "input tensor 0"),
        (lambda: lib.gc_grad_flatten_clip(a.ref, 0x400000, 2, 1.0, NORM, NORM, WS, None), "share memory"),
        (lambda: lib.gc_grad_flatten_clip(a.ref, 0x400000, 2, 1.0, 0x400010, NORM, WS, None), "share memory"),
        (lambda: lib.gc_grad_flatten_clip(a.ref, 0x400000, 2, 1.0, NORM, 0x40010, WS, None), "input tensor 0"),
        (lambda: lib.gc_grad_flatten_clip(a.ref, 0x400000, 2, 1.0, NORM, NORM + 4, 0x400000, None), "share memory"),
        (lambda: lib.gc_grad_norm(a.ref, 2, NORM, NORM, None, WS, None), "share memory"),
        (lambda: lib.gc_grad_norm(a.ref, 2, None, NORM, NORM - 4, WS, None), "share memory"),
        (lambda: lib.gc_grad_norm(a.ref, 2, None, NORM, WS + 6144, WS, None), "share memory"),
        (lambda: lib.gc_grad_norm(a.ref, 2, None, 0x40000, None, WS, None), "input tensor 0"),
    ]:
        assert rc() == _lib.GC_EINVAL and msg in err(), err()
    twice = Table([n, n, 4], [0x40000, 0x40100, 0x1000], [F32, F32, F32])  # a list that is only read may overlap itself
    for at, tensor in ((0x1008, 2), (0x40000, 0), (0x40100 + 4 * n - 4, 1)):
        assert lib.gc_grad_norm(twice.ref, 2, None, at, None, WS, None) == _lib.GC_EINVAL
        assert f"input tensor {tensor}" in err(), err()


def test_python_refusals():
    x = torch.ones(4)
    with pytest.raises(_lib.GCodecError, match="no CPU fallback"):
        clip.grad_norm([x])
    for bad in (3, 0.5, -1, 0, float("nan")):
        with pytest.raises(_lib.GCodecError, match="norm_type"):
            clip.grad_norm([x], bad)
    for bad in (-1.0, float("nan"), "1", None, torch.ones(1)):
        with pytest.raises(_lib.GCodecError, match="max_norm"):
            clip.clip_grad_norm_([x], bad)
    with pytest.raises(_lib.GCodecError, match="empty"):
        clip.grad_norm([])
    with pytest.raises(_lib.GCodecError, match="dense tensor"):
        clip.grad_norm([1.0])
    assert clip.clip_grad_norm_([torch.nn.Parameter(x)], 1.0).item() == 0.0  # no gradients
    assert clip.clip_grad_norm_([], 1.0).item() == 0.0


WORKER = r"""
import math, sys
sys.path[:0] = [sys.argv[3], sys.argv[4]]
import torch, torch.distributed as dist
from gcodec import clip, _lib
rank, port = int(sys.argv[1]), sys.argv[2]
dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=2)
def t(v): return torch.tensor(v, dtype=torch.float64)
assert clip._sum_ranks(t([3.0, 5.0][rank]), 2, dist.group.WORLD).item() == 8.0
assert clip._sum_ranks(t([3.0, 5.0][rank]), 1, dist.group.WORLD).item() == 8.0
assert clip._sum_ranks(t([7.5, 5.0][rank]), _lib.GC_NORM_INF, dist.group.WORLD).item() == 7.5
assert math.isnan(clip._sum_ranks(t([math.nan, math.inf][rank]), _lib.GC_NORM_INF, dist.group.WORLD).item())
assert math.isnan(clip._sum_ranks(t([1.0, math.nan][rank]), 2, dist.group.WORLD).item())
assert clip._sum_ranks(t([math.inf, 0.0][rank]), _lib.GC_NORM_INF, dist.group.WORLD).item() == math.inf
dist.destroy_process_group()
"""


def test_ranks_join_their_totals():
    import socket

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = str(s.getsockname()[1])
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    args = [port, root, os.path.join(root, "gradient-compression_amd")]
    ps = [subprocess.Popen([sys.executable, "-c", WORKER, str(r)] + args) for r in range(2)]
    assert [p.wait(timeout=120) for p in ps] == [0, 0]


def test_the_trainer_call_keeps_its_arguments():
    """torch.nn.utils.clip_grad_norm_'s own, in its order; foreach chooses between torch's two ways, here one."""
    import inspect

    theirs = list(inspect.signature(torch.nn.utils.clip_grad_norm_).parameters)
    mine = inspect.signature(clip.clip_grad_norm_).parameters
    assert list(mine)[:len(theirs)] == theirs
    assert mine["group"].kind is inspect.Parameter.KEYWORD_ONLY
    w = torch.nn.Parameter(torch.ones(4))
    for foreach in (None, True, False):
        assert clip.clip_grad_norm_([w], 1.0, 2.0, False, foreach).item() == 0.0
        assert clip.clip_grad_norm_([w], 1.0, foreach=foreach).item() == 0.0
    with pytest.raises(_lib.GCodecError, match="foreach"):
        clip.clip_grad_norm_([w], 1.0, 2.0, False, object())  # a group is given by name
