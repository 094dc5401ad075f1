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

import torch
import torch.distributed as dist

from . import _lib
from .codec import _dev, _raw_stream, norm_tensor, qsgd_layout

_DEVICES = {}  # index -> torch.device


def _refuse(msg: str):
    raise _lib.GCodecError(_lib.GC_EINVAL, msg)


def _norm_code(norm_type) -> int:
    p = float(norm_type)
    if p == 2.0:
        return 2
    if p == math.inf:
        return _lib.GC_NORM_INF
    if p != 1.0:
        _refuse(f"norm_type must be 1, 2 or inf, got {norm_type}")
    return 1


def _limit(max_norm, name: str = "max_norm") -> float:
    if not isinstance(max_norm, numbers.Real) or not float(max_norm) >= 0.0:
        _refuse(f"{name} must be a number at or above 0, got {max_norm!r}")
    return float(max_norm)


def _call(name: str, device, *args):
    """One entry point on `device` and its current stream (the last argument)."""
    fn = getattr(_lib.load(), name)
    index = device.index
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc < 0:
        raise _lib.GCodecError(rc, f"{name}: {_lib.last_error()}")


def _at(t):
    return None if t is None else t.data_ptr()


def _on_gpu(t: torch.Tensor) -> torch.device:
    """t's device, always with its index."""
    dev = _dev(t)
    return dev if dev.index is not None else torch.device("cuda", torch.cuda.current_device())


class Grads:
    """The table of a list of gradient tensors: contiguous float32, float16 and
    bfloat16 tensors of any sizes on one GPU, addressed as one sequence of
    elements.  Made once for tensors that stay where they are (the reducers'
    buffers, the views of a flat bucket, gradients that are zeroed instead of
    dropped) and reused; usable on every stream from then on, but not made
    under graph capture.

    It keeps the tensors' memory alive, not their shapes or later replacements:
    a gradient that is replaced by another tensor needs another table, and a
    storage that is resized under a table must not be used through it.  A
    captured call needs its table for as long as the graph is replayed.  A
    write through a table counts as an in-place change of the tensors it was
    made of, as a write to a list does."""

    def __init__(self, tensors):
        tensors = list(tensors)
        if not self._build(tensors, written=True):
            _refuse("Grads: empty tensor list")
        if torch.cuda.is_current_stream_capturing():
            _refuse("Grads: made under graph capture; make the table before it")
        rec = torch.frombuffer(bytearray(self._host), dtype=torch.int64)
        self._rec = rec.to(self.device)  # complete when this returns, whatever stream reads it
        self._streams = set()  # those that the allocator was told of
        self.struct.rec = self._rec.data_ptr()
        self._tensors = [t.detach() for t in tensors]  # their memory and their version counters

    @classmethod
    def _of_call(cls, tensors, of_grads=False, ordered=True, written=False):
        """The table of a list (of_grads: of the list's gradients; None if there are none) for the length of
        one call, filled on the current stream."""
        self = cls.__new__(cls)
        if not self._build(tensors, of_grads, ordered, written):
            return None
        self._tensors = tensors
        self._rec = torch.empty(len(self._host) // 8, dtype=torch.int64, device=self.device)
        self._streams = None
        self.struct.rec = rec = self._rec.data_ptr()
        _call("gc_grads_fill", self.device, self._ref, rec)
        return self

    def _build(self, tensors, of_grads=False, ordered=True, written=False) -> bool:
        """ordered: element i of a tensor is its i-th in row-major order (else any dense order does)
        written: the tensors may be written, or are kept (a copy-on-write one gets its own memory)"""
        lib, self._lists = _lib.load(), _lib.tensor_list()
        self.struct = _lib.gc_grads()
        self._ref = C.byref(self.struct)
        self._of_grads = of_grads
        try:
            got = self._lists.gather(tensors, of_grads, ordered, written,
                                     C.cast(lib.gc_grads_plan, C.c_void_p).value, C.addressof(self.struct))
        except LookupError as e:
            raise _lib.GCodecError(_lib.GC_ENODEV, f"gcodec runs on the GPU only: {e}; there is no CPU fallback") from None
        except ValueError as e:
            _refuse(f"Grads: {e}")
        except RuntimeError as e:
            _refuse(f"Grads: {e}: {_lib.last_error()}")
        if got is None:
            return False
        index, self._host, self._order = got  # the struct points into these
        _lib.require_device(index)
        self._index = index
        self.device = _DEVICES.get(index)
        if self.device is None:
            self.device = _DEVICES[index] = torch.device("cuda", index)
        self.count, self.n = self.struct.count, self.struct.n
        self._ws = lib.gc_grad_workspace_size(self.n, self.count, 0)
        return True

    def _use(self):
        """The table for a launch.  A kept table may be the last to hold its tensors and be dropped while a kernel
        runs on a stream other than theirs: the allocator is told, once for each stream, and gives their memory
        out again only behind that stream's work."""
        if self._streams is not None and (raw := _raw_stream(self._index)) not in self._streams:
            if not torch.cuda.is_current_stream_capturing():
                stream = torch.cuda.current_stream(self.device)
                for t in (self._rec, *self._tensors):
                    t.record_stream(stream)
                self._streams.add(raw)
        return self._ref

    def _written(self):
        """Tells autograd of a write to the tensors, once the launch is made."""
        self._lists.written(self._tensors, self._of_grads)

    def _workspace(self, each: bool = False):
        """A call's workspace, or None where it needs none."""
        size = _lib.load().gc_grad_workspace_size(self.n, self.count, 1) if each else self._ws
        return torch.empty(size, dtype=torch.uint8, device=self.device) if size else None

    def _scalar(self, dtype=torch.float32) -> torch.Tensor:
        return torch.empty((), dtype=dtype, device=self.device)


def _table(grads, ordered=True, written=False) -> Grads:
    """The table of a list (written: whose tensors this call writes)."""
    if isinstance(grads, Grads):
        return grads
    if isinstance(grads, torch.Tensor):
        grads = [grads]
    elif not isinstance(grads, (list, tuple)):
        grads = list(grads)
    g = Grads._of_call(grads, False, ordered, written)
    if g is None:
        _refuse("Grads: empty tensor list")
    return g


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


def _norm_into(g: Grads, code: int, norm, each=None, total=None):
    ws = g._workspace(each is not None)
    _call("gc_grad_norm", g.device, g._use(), code, _at(total), _at(norm), _at(each), _at(ws))


def grad_norm(grads, norm_type: float = 2.0, per_tensor: bool = False, error_if_nonfinite: bool = False, group=None):
    """The norm of all gradients together, a float32 scalar tensor; with
    per_tensor=True (norm, norms), `norms` a float32 tensor of each tensor's own
    (with a group: of this rank's part).  Empty tensors have norm 0; a list of no
    tensors, which names no device, is refused."""
    code = _norm_code(norm_type)
    g = _table(grads, ordered=False)
    norm = g._scalar()
    each = torch.empty(g.count, dtype=torch.float32, device=g.device) if per_tensor else None
    total = g._scalar(torch.float64) if group is not None else None
    _norm_into(g, code, norm, each, total)
    if group is not None:
        _sum_ranks(total, code, group)
        _call("gc_grad_norm_root", g.device, total.data_ptr(), code, norm.data_ptr())
    if error_if_nonfinite:
        _finite(norm, "grad_norm")
    return (norm, each) if per_tensor else norm


def _clip(src: Grads, dst: Grads, max_norm: float, code: int, error_if_nonfinite: bool, group, what: str):
    if src.device != dst.device:
        _refuse(f"{what}: gradients on {src.device}, outputs on {dst.device}")
    norm = src._scalar()
    total = None
    if group is not None or error_if_nonfinite:
        total = src._scalar(torch.float64)
        _norm_into(src, code, None, total=total)
        if group is not None:
            _sum_ranks(total, code, group)
        if error_if_nonfinite:  # before anything is written
            _call("gc_grad_norm_root", src.device, total.data_ptr(), code, norm.data_ptr())
            _finite(norm, what)
    ws = src._workspace()
    _call("gc_grad_clip", src.device, src._use(), dst._use(), code, max_norm,
          _at(total), norm.data_ptr(), _at(ws))
    dst._written()
    return norm


def clip_grads(grads, out, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False, group=None):
    """out[i] = grads[i] * min(1, max_norm / (norm + 1e-6)), two lists of the same
    tensor sizes (their types may differ); -> the norm before clipping.  A
    tensor may be clipped onto itself; apart from that the tensors of `out`
    share no memory with each other or with `grads`."""
    max_norm, code = _limit(max_norm), _norm_code(norm_type)
    dst = _table(out, written=True)  # ahead of src: a tensor in both has its own memory by then
    src = dst if out is grads else _table(grads)
    return _clip(src, dst, max_norm, code, error_if_nonfinite, group, "clip_grads")


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False,
                    foreach=None, *, group=None):
    """Clips the gradients of `parameters` in place; -> their norm before it (a
    float32 scalar tensor, 0 without any gradient).  As
    torch.nn.utils.clip_grad_norm_, with the norm held in 64 bits; `foreach`,
    which picks one of torch's two implementations, changes nothing here."""
    max_norm, code = _limit(max_norm), _norm_code(norm_type)
    if foreach not in (None, True, False):
        _refuse(f"foreach must be None, True or False, got {foreach!r} (group= is given by name)")
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    src = Grads._of_call(parameters, True, False, True)
    if src is None:
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
    return _clip(src, src, max_norm, code, error_if_nonfinite, group, "clip_grad_norm_")


def flatten_clip(grads, max_norm: float, norm_type: float = 2.0, flat=None):
    """-> (flat, peak, norm): the clipped gradients end to end in one float32
    bucket, its max-norm (as segments_flatten_absmax: what qsgd_encode scales
    by), and the gradients' norm before clipping."""
    max_norm, code = _limit(max_norm), _norm_code(norm_type)
    g = _table(grads)
    given = flat is not None
    if not given:
        flat = torch.empty(g.n, dtype=torch.float32, device=g.device)
    elif flat.device != g.device or flat.dtype != torch.float32 or flat.numel() != g.n or not flat.is_contiguous():
        _refuse(f"flatten_clip: flat must be contiguous float32, {g.n} elements on {g.device}")
    peak = torch.empty(1, dtype=torch.float32, device=g.device)
    norm = g._scalar()
    ws = g._workspace()
    _call("gc_grad_flatten_clip", g.device, g._use(), flat.data_ptr(), code, max_norm, peak.data_ptr(), norm.data_ptr(),
          _at(ws))
    if given:
        _lib.tensor_list().written([flat], False)
    return flat, peak, norm


def qsgd_decode_clip(words, norm, bits: int, grads, max_norm: float, norm_type: float = 2.0, world: int = 1,
                     alpha: float = 1.0, lanes=None):
    """qsgd_decode of the packed words (summed over `world` ranks) times alpha into
    the gradient tensors, clipped by the norm of all of them; -> that norm
    before clipping.  The unclipped gradients are never stored.  lanes: the
    words' layout, number of ranks included, where it is not that of
    qsgd_layout(n, bits, world)."""
    max_norm, code = _limit(max_norm), _norm_code(norm_type)
    dev = _on_gpu(words)
    g = _table(grads, written=True)
    if dev != g.device:
        _refuse(f"qsgd_decode_clip: words on {dev}, gradients on {g.device}")
    if words.dtype != torch.int32 or not words.is_contiguous():
        _refuse("qsgd_decode_clip: words must be contiguous int32")
    lanes = lanes or qsgd_layout(g.n, bits, world)
    if words.numel() < lanes.plane_words:
        _refuse(f"qsgd_decode_clip: {words.numel()} words, {lanes.plane_words} needed")
    nt = norm_tensor(norm, dev)
    if nt.numel() < 1:
        _refuse("qsgd_decode_clip: empty norm")
    out = g._scalar()
    ws = g._workspace()
    _call("gc_qsgd_decode_clip", dev, words.data_ptr(), g.n, nt.data_ptr(), int(bits), C.byref(lanes), float(alpha),
          g._use(), code, max_norm, out.data_ptr(), _at(ws))
    g._written()
    return out
