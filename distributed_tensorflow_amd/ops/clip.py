"""Global gradient norm and clipping by it (``tf.global_norm`` / ``tf.clip_by_global_norm``) over a list of tensors.

    plan = GlobalNormClip(grads)                   # in place; out=[...] writes clipped copies instead
    norm = plan.norm()                             # fp32 scalar on the device: sqrt(sum of all squares)
    grads, norm = plan.clip(clip_norm)             # g * clip_norm / max(norm, clip_norm), norm before clipping

The plan is made once for tensors that stay where they are (gradient arenas, as everywhere in this package) and holds
nothing but a table of their addresses and shapes in device memory; each call computes the norm anew from the values that
the tensors then have.  A tensor whose memory is replaced (a gradient that is made anew each step) needs a new plan, which
costs a copy to the device and a wait for it and cannot be made while a stream is captured.  Launches go to the current
stream of the tensors' device: the table is only read, the workspace of a call comes from PyTorch's allocator on that
stream, so calls on different streams and in different graphs share nothing that is written.  A plan may be dropped while
its calls still run on any stream; one whose call was captured into a HIP graph has to outlive the graph and its replays.
As in TensorFlow, a norm that is not finite (a value that is not, in some tensor) makes every clipped value NaN.  Norm and
factor are 64-bit numbers: a list of finite values whose norm is beyond fp32 is clipped all the same, though the norm that
is returned, an fp32 scalar, is then infinity.  Autograd does not record the calls: tensors that require gradients are taken
under ``torch.no_grad()`` only.
Kernels: csrc/kernels/clip.hip.
"""
from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Sequence, Tuple

import torch

from . import native
from .native import check, no_autograd, on_device, ptr

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class ClipSpan(ctypes.Structure):
    """Mirror of ``struct DtfClipSpan`` (csrc/kernels/api.h)."""

    _fields_ = [("inp", ctypes.c_void_p), ("out", ctypes.c_void_p), ("n", ctypes.c_long), ("in_pitch", ctypes.c_long),
                ("out_pitch", ctypes.c_long), ("cols", ctypes.c_int), ("dtype", ctypes.c_int)]


def _layout(t: torch.Tensor, o: torch.Tensor) -> Tuple[int, int, int]:
    """(cols, pitch of t, pitch of o) that walk all elements of t and, in the same order, of o: cols == 0 when both are
    contiguous runs, else rows of ``cols`` elements.  ValueError where more than one stride is left, or where elements
    of a tensor share memory."""
    dims = sorted((st, so, n) for n, st, so in zip(t.shape, t.stride(), o.stride()) if n != 1)
    shared = f"elements of a tensor of shape {tuple(t.shape)} with strides {t.stride()} (output {o.stride()}) share memory"
    if any(st == 0 or so == 0 for st, so, _ in dims):
        raise ValueError(shared)
    runs: List[List[int]] = []          # [length, stride in t, stride in o], innermost first; neighbours merged
    for st, so, n in dims:
        if runs and st == runs[-1][1] * runs[-1][0] and so == runs[-1][2] * runs[-1][0]:
            runs[-1][0] *= n
        else:
            runs.append([n, st, so])
    if not runs:
        return 0, 0, 0
    if len(runs) == 1 and runs[0][1] == runs[0][2] == 1:
        return 0, 0, 0
    if runs[0][1] != 1 or runs[0][2] != 1:
        runs.insert(0, [1, 1, 1])       # elements apart from each other: rows of one
    if len(runs) > 2:
        raise ValueError(f"a tensor of shape {tuple(t.shape)} with strides {t.stride()} (output {o.stride()}) is neither "
                         "dense nor made of equally spaced rows")
    (cols, _, _), (rows, pt, po) = runs
    if pt < cols or po < cols:
        raise ValueError(shared)
    if cols >= 1 << 31:
        raise ValueError("rows of 2^31 elements and more are not supported in strided tensors")
    return cols, pt, po


class _Extent:
    """The bytes that a span touches, for the overlap checks: [lo, hi), or every pitch-th row of them."""

    def __init__(self, addr: int, size: int, n: int, cols: int, pitch: int):
        rows = 1 if cols == 0 else n // cols
        self.lo, self.row, self.pitch = addr, (n if cols == 0 else cols) * size, pitch * size
        self.hi = addr + (rows - 1) * self.pitch + self.row
        self.key = (addr, size, n, cols, pitch)

    def meets(self, other: "_Extent") -> bool:
        if self.hi <= other.lo or other.hi <= self.lo:
            return False
        if self.pitch and self.pitch == other.pitch:        # column blocks of one matrix
            d = (other.lo - self.lo) % self.pitch
            return d < self.row or d + other.row > self.pitch
        return True


def _check_writes(reads: Sequence[Tuple[int, _Extent]], writes: Sequence[Tuple[int, _Extent]], what: str):
    """No memory that is written may be written or read through another tensor of the list (a tensor may be its own
    output).  Sorted by address; a later start is compared with what has not ended before it."""
    live: List[Tuple[int, _Extent, bool]] = []
    for i, e, w in sorted([(i, e, False) for i, e in reads] + [(i, e, True) for i, e in writes], key=lambda x: x[1].lo):
        live = [x for x in live if x[1].hi > e.lo]
        for j, x, xw in live:
            if (w or xw) and x.meets(e) and not (i == j and w != xw and x.key == e.key):
                raise ValueError(what)
        live.append((i, e, w))


class GlobalNormClip:
    """Norm of, and clipping over, a fixed list of fp32 / bf16 / fp16 tensors of one GPU.

    tensors: any shapes, mixed types, empty ones allowed; each dense in memory or made of equally spaced rows (a slice
    of a matrix).  out: where the clipped values go, tensors of the same shapes and types; None clips in place (and then
    a norm within the limit leaves every value untouched, without a pass over them)."""

    _requires: Sequence[torch.Tensor] = ()      # a tensor that requires gradients, where there is one
    _written: Sequence[torch.Tensor] = ()       # whose version counters a clipping call raises: views of one tensor share theirs

    def __init__(self, tensors: Sequence[torch.Tensor], out: Optional[Sequence[torch.Tensor]] = None):
        tensors = list(tensors)
        if not tensors:
            raise ValueError("no tensors")
        for t in tensors:
            if not isinstance(t, torch.Tensor) or t.layout != torch.strided:
                raise TypeError(f"strided tensors expected, got {type(t).__name__}")
            if t.dtype not in _DTYPES:
                raise TypeError(f"fp32, bf16 or fp16 tensors expected, got {t.dtype}")
        outs = tensors if out is None else list(out)
        if len(outs) != len(tensors):
            raise ValueError(f"{len(tensors)} tensors but {len(outs)} outputs")
        for t, o in zip(tensors, outs):
            if not isinstance(o, torch.Tensor) or o.layout != torch.strided or o.dtype != t.dtype or o.shape != t.shape:
                raise ValueError("every output needs the shape and type of its tensor")
        no_autograd(tensors + outs)
        self._requires = [t for t in tensors + outs if t.requires_grad][:1]
        self.device = tensors[0].device
        spans = (ClipSpan * len(tensors))()
        ins, writes = [], []
        for k, (s, t, o) in enumerate(zip(spans, tensors, outs)):
            s.dtype, s.n = _DTYPES[t.dtype], t.numel()
            if t.numel() == 0:
                continue
            s.cols, s.in_pitch, s.out_pitch = _layout(t, o)
            s.inp, s.out = t.data_ptr(), o.data_ptr()
            ins.append((k, _Extent(s.inp, t.element_size(), s.n, s.cols, s.in_pitch)))
            writes.append((k, _Extent(s.out, t.element_size(), s.n, s.cols, s.out_pitch)))
        # The norm of a list may count a tensor twice; clipped values need memory of their own.
        self._clip_error: Optional[str] = None
        if out is not None:
            _check_writes(ins, writes, "an output shares memory with another output or tensor")
        else:
            try:
                _check_writes([], writes, "tensors that share memory cannot be clipped in place")
            except ValueError as e:
                self._clip_error = str(e)
        for t in tensors + outs:
            if t.device != self.device:
                raise ValueError(f"tensors on {self.device} and {t.device}")
        if self.device.type != "cuda":
            raise ValueError(f"GPU tensors expected, got {self.device} (ops.reference.clip_by_global_norm runs on the CPU)")
        self.lib = native.load()
        kept = [t.detach() for t in tensors] + [o.detach() for o in outs]            # the memory stays allocated
        self.out = list(outs)
        in_place = ctypes.c_int()
        chunks = int(self.lib.dtf_clip_table(len(tensors), spans, None, 0, ctypes.byref(in_place)))
        check(min(chunks, 0), "clip_table")
        host = torch.empty((max(chunks, 1), 64), dtype=torch.uint8)
        check(min(int(self.lib.dtf_clip_table(len(tensors), spans, ptr(host), chunks, None)), 0), "clip_table")
        self.table = host.to(self.device)                # 64 bytes per chunk, the same for every call
        # every other stream may read the table from here on: the copy is done
        torch.cuda.current_stream(self.device).synchronize()
        self._memory = [self.table] + list({t.untyped_storage().data_ptr(): t for t in kept if t.numel()}.values())
        self._keep, self._streams = kept, set()
        self._written = list({id(b): b for b in (o._base if o._is_view() else o for o in outs)}.values())
        self._used_on(torch.cuda.current_stream(self.device).cuda_stream)
        self.chunks, self._in_place = chunks, in_place.value
        self.slots = int(self.lib.dtf_clip_partials(chunks))    # fp64 words of a call's workspace

    def _buffers(self):
        dev = self.device
        return torch.empty(self.slots, dtype=torch.float64, device=dev), torch.empty((), dtype=torch.float32, device=dev)

    def _used_on(self, stream: int):
        """Called on the current stream, whose handle is ``stream``.  The allocator hands out the memory of a dropped plan (its
        table, and tensors that nobody else keeps) as soon as the streams recorded for it have done what they were given
        until then, so every stream that a call goes to is recorded, once."""
        if stream in self._streams or torch.cuda.is_current_stream_capturing():
            return
        now = torch.cuda.current_stream(self.device)
        for t in self._memory:
            t.record_stream(now)
        self._streams.add(stream)

    def norm(self, scale: float = 1.0) -> torch.Tensor:
        """``scale`` * norm of all tensors, an fp32 scalar on the device (infinity from 3.4e38 on)."""
        scale = _scale(scale)
        if self._requires:
            no_autograd(self._requires)
        with on_device(self.device) as stream:
            self._used_on(stream)
            part, norm = self._buffers()
            check(self.lib.dtf_global_norm(ptr(self.table), self.chunks, ptr(part), self.slots, scale, None, None, 0, 0.0,
                                           ptr(norm), stream), "global_norm")
        return norm

    def clip(self, clip_norm: float, scale: float = 1.0) -> Tuple[List[torch.Tensor], torch.Tensor]:
        """Multiplies every value with ``scale`` (a mean over ranks, a loss scale taken back) and then so that the norm of
        all of them is at most ``clip_norm``.  Returns the outputs and the norm (of the scaled values) before clipping."""
        scale, clip_norm = _scale(scale), float(clip_norm)
        if not (clip_norm > 0.0 and math.isfinite(clip_norm)):
            raise ValueError(f"clip_norm must be positive and finite, got {clip_norm}")
        if self._clip_error:
            raise ValueError(self._clip_error)
        if self._requires:
            no_autograd(self._requires)
        with on_device(self.device) as stream:
            self._used_on(stream)
            part, norm = self._buffers()
            check(self.lib.dtf_clip_by_global_norm(ptr(self.table), self.chunks, self._in_place, ptr(part), self.slots, scale,
                                                   clip_norm, ptr(norm), stream), "clip_by_global_norm")
        torch.autograd.graph.increment_version(self._written)
        return list(self.out), norm


def _scale(scale: float) -> float:
    scale = float(scale)
    if not (scale >= 0.0 and math.isfinite(scale)):
        raise ValueError(f"scale must be finite and not negative, got {scale}")
    return scale
