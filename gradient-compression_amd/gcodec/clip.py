"""The global norm of a model's gradients and clipping by it.

    N = (sum |x|^p)^(1/p) over every element of every gradient, p = 1, 2 or infinity
    c = min(1, max_norm / (N + 1e-6)),  gradient = RN_type(gradient * c)

    grad_norm(grads)                       N (and the norm of each tensor)
    clip_grad_norm_(parameters, max_norm)  in place; the call of torch.nn.utils.clip_grad_norm_
    clip_grads(grads, out, max_norm)       from one list into another (the reducers' grad_in -> grad_out)
    flatten_clip(grads, max_norm)          into the float32 bucket that the codec encodes, with its max-norm
    qsgd_decode_clip(words, ...)           packed words, summed over the ranks, into the gradients

Gradients are float32, float16 or bfloat16, mixed as they come, on one GPU;
norms are float32 scalars on that GPU, so nothing waits for the device (but
error_if_nonfinite=True reads the norm back).  The sums are held in 64 bits and
added in a fixed order: equal gradients give equal bits on every call.  No
operator here is differentiable: the gradients are taken as numbers.

Where ranks hold different shards of one gradient (tensor parallelism, sharded
data parallelism), `group=` adds the ranks' sums, so that every rank clips by
the norm of the whole.  Every element must then live on one rank only.

Every function takes a list of tensors or a Grads, the table of such a list.
A list's table is made in each call (its records travel in kernel arguments);
a program whose gradients stay where they are keeps a Grads instead.  Calls on
different streams share nothing, and a captured call owns its workspace.
"""
from __future__ import annotations

import ctypes as C
import math
import numbers

import numpy as np
import torch
import torch.distributed as dist

from . import _lib
from ._lib import check
from .codec import _dev, _f32, _p, _stream, norm_tensor, qsgd_layout

_TYPE = {torch.float32: _lib.GC_F32, torch.float16: _lib.GC_F16, torch.bfloat16: _lib.GC_BF16}


def _refuse(msg: str):
    raise _lib.GCodecError(_lib.GC_EINVAL, msg)


def _norm_code(norm_type) -> int:
    p = float(norm_type)
    if p == math.inf:
        return _lib.GC_NORM_INF
    if p not in (1.0, 2.0):
        _refuse(f"norm_type must be 1, 2 or inf, got {norm_type}")
    return int(p)


def _limit(max_norm) -> float:
    if not isinstance(max_norm, numbers.Real) or not float(max_norm) >= 0.0:
        _refuse(f"max_norm must be a number at or above 0, got {max_norm!r}")
    return float(max_norm)


class _on:
    """Makes `device` the current one for a launch, where it is not already."""

    def __init__(self, device):
        self._ctx = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self._ctx is not None:
            self._ctx.__enter__()

    def __exit__(self, *exc):
        if self._ctx is not None:
            self._ctx.__exit__(*exc)


def _dense(t: torch.Tensor) -> bool:
    """Whether the tensor fills its range of memory once, in any order of its dimensions."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for sz, st in zip(t.shape, t.stride()) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


class Grads:
    """The table of a list of gradient tensors: contiguous float32, float16 and
    bfloat16 tensors of any sizes on one GPU, addressed as one sequence of
    elements.  Made once for tensors that stay where they are (the reducers'
    buffers, the views of a flat bucket, gradients that are zeroed instead of
    dropped) and reused; usable on every stream from then on, but not made
    under graph capture.

    It keeps the tensors' memory alive, not their shapes or later replacements:
    a gradient that is replaced by another tensor needs another table, and a
    storage that is resized under a table must not be used through it."""

    def __init__(self, tensors):
        tensors = list(tensors)
        self._build(tensors)
        if torch.cuda.is_current_stream_capturing():
            _refuse("Grads: made under graph capture; make the table before it")
        rec = torch.from_numpy(self._host.view(np.int64))
        self._rec = rec.to(self.device)  # complete when this returns, whatever stream reads it
        self._home = torch.cuda.current_stream(self.device)
        self.struct.rec = self._rec.data_ptr()
        self._keep = [t.untyped_storage() for t in tensors]

    @classmethod
    def _of_call(cls, tensors, ordered=True):
        """The table of a list for the length of one call, filled on the current stream."""
        self = cls.__new__(cls)
        self._build(tensors, ordered)
        self._rec = torch.empty(self._host.size, dtype=torch.int64, device=self.device)
        with _on(self.device):
            check(_lib.load().gc_grads_fill(C.byref(self.struct), _p(self._rec), _stream(self.device)), "gc_grads_fill")
        self._home = None
        self.struct.rec = self._rec.data_ptr()
        return self

    def _build(self, tensors, ordered=True):
        """ordered: element i of a tensor is its i-th in row-major order (else any dense order does)"""
        if not tensors:
            _refuse("Grads: empty tensor list")
        for t in tensors:
            if not isinstance(t, torch.Tensor) or t.layout != torch.strided:
                _refuse(f"Grads: not a dense tensor ({type(t).__name__})")
        self.device = dev = _dev(tensors[0])
        if len(set(map(torch.Tensor.get_device, tensors))) != 1:
            _refuse("Grads: the tensors are on different devices")
        types = list(map(_TYPE.get, [t.dtype for t in tensors]))
        if None in types:
            _refuse(f"Grads: {tensors[types.index(None)].dtype} is not float32, float16 or bfloat16")
        if not all(map(torch.Tensor.is_contiguous, tensors)):
            bad = [i for i, t in enumerate(tensors) if not (t.is_contiguous() if ordered else _dense(t))]
            if bad:
                t = tensors[bad[0]]
                _refuse(f"Grads: tensor {bad[0]} is not {'contiguous' if ordered else 'dense'} (shape {tuple(t.shape)}, "
                        f"strides {t.stride()})")
        lib = _lib.load()
        self.count = count = len(tensors)
        sizes = np.fromiter(map(torch.Tensor.numel, tensors), dtype=np.uint64, count=count)
        ptrs = np.fromiter(map(torch.Tensor.data_ptr, tensors), dtype=np.uint64, count=count)
        kinds = np.fromiter(types, dtype=np.uint32, count=count)
        self._host = np.empty(2 * (count + 1), dtype=np.uint64)
        self._order = np.empty(count, dtype=np.uint32)
        self.struct = _lib.gc_grads()
        check(lib.gc_grads_plan(sizes.ctypes.data, ptrs.ctypes.data, kinds.ctypes.data, count, self._host.ctypes.data,
                                self._order.ctypes.data, C.byref(self.struct)), "gc_grads_plan")
        self.n = int(self.struct.n)

    def _use(self):
        """Tells the allocator of a stream other than the one the table was made on."""
        if self._home is not None and not torch.cuda.is_current_stream_capturing():
            now = torch.cuda.current_stream(self.device)
            if now != self._home:
                self._rec.record_stream(now)
        return C.byref(self.struct)


def _table(grads, ordered=True) -> Grads:
    if isinstance(grads, Grads):
        return grads
    if isinstance(grads, torch.Tensor):
        grads = [grads]
    return Grads._of_call(list(grads), ordered)


def _workspace(g: Grads, each: bool = False) -> torch.Tensor:
    size = _lib.load().gc_grad_workspace_size(g.n, g.count, int(each))
    return torch.empty(size, dtype=torch.uint8, device=g.device)


def _scalar(g: Grads, dtype=torch.float32) -> torch.Tensor:
    return torch.empty((), dtype=dtype, device=g.device)


def _sum_ranks(total: torch.Tensor, code: int, group) -> torch.Tensor:
    """The ranks' totals as one: their sum, or for p = infinity their maximum.
    The maximum is taken of the bits, which order non-negative numbers as
    their values and put a NaN above them all."""
    word = total.view(torch.int64) if code == _lib.GC_NORM_INF else total
    op = dist.ReduceOp.MAX if code == _lib.GC_NORM_INF else dist.ReduceOp.SUM
    if total.is_cuda and dist.get_backend(group) == "gloo":  # gloo is given host memory only
        host = word.cpu()
        dist.all_reduce(host, op=op, group=group)
        word.copy_(host)
    else:
        dist.all_reduce(word, op=op, group=group)
    return total


def _finite(norm: torch.Tensor, what: str):
    if not bool(torch.isfinite(norm)):
        raise RuntimeError(f"{what}: the total norm of the gradients is {float(norm)}, which is not finite")


@torch.no_grad()
def grad_norm(grads, norm_type: float = 2.0, per_tensor: bool = False, error_if_nonfinite: bool = False, group=None):
    """The norm of all gradients together, a float32 scalar tensor; with
    per_tensor=True (norm, norms), `norms` a float32 tensor of each tensor's own
    (with a group: of this rank's part).  No gradients at all have norm 0."""
    code = _norm_code(norm_type)
    g = _table(grads, ordered=False)
    lib = _lib.load()
    with _on(g.device):
        norm = _scalar(g)
        each = torch.empty(g.count, dtype=torch.float32, device=g.device) if per_tensor else None
        total = _scalar(g, torch.float64) if group is not None else None
        check(lib.gc_grad_norm(g._use(), code, _p(total), _p(norm), _p(each), _p(_workspace(g, per_tensor)),
                               _stream(g.device)), "gc_grad_norm")
        if group is not None:
            _sum_ranks(total, code, group)
            check(lib.gc_grad_norm_root(_p(total), code, _p(norm), _stream(g.device)), "gc_grad_norm_root")
    if error_if_nonfinite:
        _finite(norm, "grad_norm")
    return (norm, each) if per_tensor else norm


def _clip(src: Grads, dst: Grads, max_norm: float, code: int, error_if_nonfinite: bool, group, what: str):
    lib = _lib.load()
    if src.device != dst.device:
        _refuse(f"{what}: gradients on {src.device}, outputs on {dst.device}")
    with _on(src.device):
        norm = _scalar(src)
        total = None
        if group is not None or error_if_nonfinite:
            total = _scalar(src, torch.float64)
            check(lib.gc_grad_norm(src._use(), code, _p(total), None, None, _p(_workspace(src)), _stream(src.device)),
                  "gc_grad_norm")
            if group is not None:
                _sum_ranks(total, code, group)
            if error_if_nonfinite:  # before anything is written
                check(lib.gc_grad_norm_root(_p(total), code, _p(norm), _stream(src.device)), "gc_grad_norm_root")
                _finite(norm, what)
        check(lib.gc_grad_clip(src._use(), dst._use(), code, max_norm, _p(total), _p(norm), _p(_workspace(src)),
                               _stream(src.device)), "gc_grad_clip")
    return norm


@torch.no_grad()
def clip_grads(grads, out, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False, group=None):
    """out[i] = grads[i] * min(1, max_norm / (norm + 1e-6)), two lists of the same
    tensor sizes (their types may differ); -> the norm before clipping.  A
    tensor may be clipped onto itself; apart from that the tensors of `out`
    share no memory with each other or with `grads`."""
    max_norm, code = _limit(max_norm), _norm_code(norm_type)
    src = _table(grads)
    dst = src if out is grads else _table(out)
    return _clip(src, dst, max_norm, code, error_if_nonfinite, group, "clip_grads")


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False, group=None):
    """Clips the gradients of `parameters` in place; -> their norm before it (a
    float32 scalar tensor, 0 without any gradient).  As
    torch.nn.utils.clip_grad_norm_, with the norm held in 64 bits."""
    max_norm, code = _limit(max_norm), _norm_code(norm_type)
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [g for g in (p.grad for p in parameters) if g is not None]
    if not grads:
        dev = parameters[0].device if parameters else None
        norm = torch.zeros((), dtype=torch.float64, device=dev)
        if group is not None:  # the other ranks wait for this one's share
            if dev is None and dist.get_backend(group) != "gloo":
                norm = norm.cuda()
            _sum_ranks(norm, code, group)
        norm = (norm.sqrt() if code == 2 else norm).float()
        if error_if_nonfinite:
            _finite(norm, "clip_grad_norm_")
        return norm
    src = _table(grads, ordered=False)
    norm = _clip(src, src, max_norm, code, error_if_nonfinite, group, "clip_grad_norm_")
    torch.autograd.graph.increment_version([g for g in grads if not g.is_inference()])
    return norm


@torch.no_grad()
def flatten_clip(grads, max_norm: float, norm_type: float = 2.0, flat=None):
    """-> (flat, peak, norm): the clipped gradients end to end in one float32
    bucket, its max-norm (as segments_flatten_absmax: what qsgd_encode scales
    by), and the gradients' norm before clipping."""
    max_norm, code = _limit(max_norm), _norm_code(norm_type)
    g = _table(grads)
    with _on(g.device):
        if flat is None:
            flat = torch.empty(g.n, dtype=torch.float32, device=g.device)
        elif flat.device != g.device or flat.numel() != g.n or not flat.is_contiguous():
            _refuse(f"flatten_clip: flat must be contiguous, {g.n} elements on {g.device}")
        peak = torch.empty(1, dtype=torch.float32, device=g.device)
        norm = _scalar(g)
        check(_lib.load().gc_grad_flatten_clip(g._use(), _p(_f32(flat, "flatten_clip")), code, max_norm, _p(peak),
                                               _p(norm), _p(_workspace(g)), _stream(g.device)), "gc_grad_flatten_clip")
    return flat, peak, norm


@torch.no_grad()
def qsgd_decode_clip(words, norm, bits: int, grads, max_norm: float, norm_type: float = 2.0, world: int = 1,
                     alpha: float = 1.0, lanes=None):
    """qsgd_decode of the packed words (summed over `world` ranks) times alpha into
    the gradient tensors, clipped by the norm of all of them; -> that norm
    before clipping.  The unclipped gradients are never stored."""
    max_norm, code = _limit(max_norm), _norm_code(norm_type)
    dev = _dev(words)
    g = _table(grads)
    if dev != g.device:
        _refuse(f"qsgd_decode_clip: words on {dev}, gradients on {g.device}")
    if words.dtype != torch.int32 or not words.is_contiguous():
        _refuse("qsgd_decode_clip: words must be contiguous int32")
    lanes = lanes or qsgd_layout(g.n, bits, world)
    if words.numel() < lanes.plane_words:
        _refuse(f"qsgd_decode_clip: {words.numel()} words, {lanes.plane_words} needed")
    with _on(dev):
        nt = norm_tensor(norm, dev)
        if nt.numel() < 1:
            _refuse("qsgd_decode_clip: empty norm")
        out = _scalar(g)
        check(_lib.load().gc_qsgd_decode_clip(_p(words), g.n, _p(nt), int(bits), C.byref(lanes), float(alpha), g._use(),
                                              code, max_norm, _p(out), _p(_workspace(g)), _stream(dev)),
              "gc_qsgd_decode_clip")
    return out
