"""Classifier head with many classes: softmax cross-entropy of ``h @ wT.T (+ bias)`` and its gradient, without logits.

    loss_rows, lse = vocab_head_fwd(h, wT, labels, bias)
    dh, dwT, dbias = vocab_head_bwd(h, wT, labels, lse, bias, grad_scale=1.0 / n)

The ten-class head of the engine keeps a row's logits in registers; here the classes may be a vocabulary.  Conventions are
the engine's: rows of hidden units ``h`` [n, hidden], the weight transposed ``wT`` [classes, hidden], int32 labels, the
per-row loss and everything that is summed in fp32; both operands bf16 (gradients of them bf16 as well, ``dwT`` on request
fp32) or both fp32 (every product to within 2^-21, on average 2^-23, from three bf16 parts of each value on the bf16 matrix
cores; where a factor is below 2e-34, up to 2^-133 of the other is lost as well; infinite values make NaN).  Rows of ``h``
and ``wT`` may be further apart than they are long.  Copied once per call are rows of ``h`` that do not start on 16 bytes, and
rows of ``wT`` that do not start on 4 bytes or leave a gap behind a broken 16 bytes (bf16: an odd number of hidden units).

A row whose label is ``ignore_label`` has loss 0 and takes no part in any gradient, whatever its hidden units hold
(padding); any other label outside the classes makes its loss, and with it every gradient it enters, NaN, as
``tf.nn.sparse_softmax_cross_entropy_with_logits`` does on a GPU.  A class can be masked by a bias of -inf; an infinite
weight makes NaN, of its own class or of the one before it.

The backward pass computes the logits again, one piece of the classes at a time: its workspace holds the gradient of the
piece's logits in the operands' type (at most 2^27 values, or 1024 classes of very many rows; bf16 drops up to 2^-8 of a value
there, unless ``keep_rounding`` asks for two bf16 values), a copy of ``h`` without its ignored rows, fp32 sums of ``dh`` where
there are several pieces or the classes are cut among workgroups, and the copies above.  Calls launch on the current stream of
the operands' device, take their workspace from PyTorch's allocator on that stream and keep nothing, so they can be captured
into HIP graphs and run on several streams at once.  Autograd does not record them: operands that require gradients are taken
under ``torch.no_grad()`` only.
Kernels: csrc/kernels/vocab_head.hip.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import native
from .native import check, no_autograd, on_device, ptr

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_MAX_ROW = 1 << 20          # rows, hidden units and row strides of one call


def _rows(t: torch.Tensor, name: str, rows: int, cols: int) -> int:
    """Row stride (elements) of a matrix with contiguous rows."""
    ld, inner = t.stride()
    if inner != 1 and cols > 1:
        raise ValueError(f"{name} must be a matrix with contiguous rows, got shape {tuple(t.shape)}, strides {t.stride()}")
    if rows <= 1:
        ld = cols               # the stride of a single row says nothing
    if ld < cols:
        raise ValueError(f"rows of {name} share memory (strides {t.stride()})")
    if ld > _MAX_ROW:
        raise ValueError(f"rows of {name} may be at most {_MAX_ROW} elements long and apart, got {ld}")
    return ld


def _vector(t: Optional[torch.Tensor], name: str, n: int, dtype: torch.dtype, device: torch.device):
    if t is None:
        return
    if t.dtype != dtype or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} vector of {n} elements, got {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the hidden rows on {device}")


def _check(h, wT, labels, bias, ignore_label, *others) -> Tuple[int, int, int, int, int]:
    dtype, dev = h.dtype, h.device
    if dtype not in _DTYPES or wT.dtype != dtype:
        raise TypeError(f"h and wT must both be bf16 or both fp32, got {dtype} and {wT.dtype}")
    for t, name in ((h, "h"), (wT, "wT")):
        if t.dim() != 2:
            raise ValueError(f"{name} must be a matrix with contiguous rows, got shape {tuple(t.shape)}")
    (n, hidden), (classes, width) = h.shape, wT.shape
    ldh, ldw = _rows(h, "h", n, hidden), _rows(wT, "wT", classes, width)
    if width != hidden:
        raise ValueError(f"h has {hidden} hidden units, wT {width}")
    if hidden < 1 or not 1 <= classes < 1 << 30:
        raise ValueError(f"at least one hidden unit and 1 to 2^30 - 1 classes expected, got wT {tuple(wT.shape)}")
    if n > _MAX_ROW:
        raise ValueError(f"at most {_MAX_ROW} rows per call, got {n}")
    if wT.device != dev:
        raise ValueError(f"wT is on {wT.device}, the hidden rows on {dev}")
    _vector(labels, "labels", n, torch.int32, dev)
    _vector(bias, "bias", classes, torch.float32, dev)
    if not -(1 << 31) <= ignore_label < 1 << 31:
        raise ValueError(f"ignore_label must be an int32, got {ignore_label}")
    no_autograd((h, wT, bias) + others)
    if dev.type != "cuda":
        raise ValueError(f"GPU tensors expected, got {dev} (ops.reference.softmax_cross_entropy_with_logits runs on the CPU)")
    return n, hidden, classes, ldh, ldw


def vocab_head_fwd(h: torch.Tensor, wT: torch.Tensor, labels: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                   ignore_label: int = -1) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss_rows, lse), fp32 [n]: per-row cross-entropy and the logarithm of the sum of exponentials of the logits (what the
    backward pass needs)."""
    n, hidden, classes, ldh, ldw = _check(h, wT, labels, bias, ignore_label)
    loss, lse = torch.empty((2, n), dtype=torch.float32, device=h.device)
    if n == 0:
        return loss, lse
    lib, dt = native.load(), _DTYPES[h.dtype]
    with on_device(h.device) as stream:
        need = lib.dtf_vocab_head_workspace(dt, 0, ptr(h), ldh, ptr(wT), ldw, n, hidden, classes, int(bias is not None), 0)
        check(min(need, 0), "vocab_head_workspace")
        ws = torch.empty(need, dtype=torch.uint8, device=h.device)
        check(lib.dtf_vocab_head_fwd(dt, ptr(h), ldh, ptr(wT), ldw, ptr(bias), ptr(labels), n, hidden, classes, ignore_label,
                                     ptr(loss), ptr(lse), ptr(ws), need, stream), "vocab_head_fwd")
    return loss, lse


def _span(t: torch.Tensor) -> Tuple[int, int]:
    last = sum((s - 1) * st for s, st in zip(t.shape, t.stride())) if t.numel() else -1
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def vocab_head_bwd(h: torch.Tensor, wT: torch.Tensor, labels: torch.Tensor, lse: torch.Tensor,
                   bias: Optional[torch.Tensor] = None, *, grad_scale: float = 1.0, row_scale: Optional[torch.Tensor] = None,
                   ignore_label: int = -1, need_dh: bool = True, need_dwT: bool = True, dh: Optional[torch.Tensor] = None,
                   dwT: Optional[torch.Tensor] = None, dbias: Optional[torch.Tensor] = None, piece: int = 0,
                   keep_rounding: bool = False):
    """(dh, dwT, dbias) of sum_i grad_scale * row_scale[i] * loss_rows[i]; dbias is None without a bias, dh / dwT where they
    are not wanted.  ``row_scale``: fp32 [n], the upstream gradient of the loss rows (default: ones).  ``dh`` / ``dwT`` /
    ``dbias``: where to write (contiguous, 16-byte aligned; ``dwT`` in the operands' type or fp32), e.g. views of a gradient
    arena.  ``piece``: classes per piece (rounded up to 256; 0: chosen from n).  ``keep_rounding``: bf16 operands keep what
    rounding drops of the logits' gradient for any number of rows, not up to 32 only; dh and dwT then take two products each (1.6
    to 1.75 times the time of a large backward pass) and are as exact as if it had stayed in fp32."""
    n, hidden, classes, ldh, ldw = _check(h, wT, labels, bias, ignore_label, lse, row_scale, dh, dwT, dbias)
    _vector(lse, "lse", n, torch.float32, h.device)
    _vector(row_scale, "row_scale", n, torch.float32, h.device)
    if lse is None:
        raise ValueError("lse is missing: it is the second result of vocab_head_fwd")
    if not 0 <= piece <= _MAX_ROW:
        raise ValueError(f"piece must lie between 0 and {_MAX_ROW}, got {piece}")
    if dbias is not None and bias is None:
        raise ValueError("dbias without a bias")
    reads = [t for t in (h, wT, labels, lse, bias, row_scale) if t is not None]
    for t, name, shape, types in ((dh, "dh", (n, hidden), (h.dtype,)), (dwT, "dwT", (classes, hidden), (h.dtype, torch.float32)),
                                  (dbias, "dbias", (classes,), (torch.float32,))):
        if t is None:
            continue
        if t.shape != shape or t.dtype not in types or not t.is_contiguous() or t.device != h.device or t.data_ptr() % 16:
            raise ValueError(f"{name} must be a contiguous, 16-byte aligned {' or '.join(map(str, types))} tensor of shape {shape} "
                             f"on {h.device}")
        a, b = _span(t)
        for other in reads:
            c, d = _span(other)
            if a < d and c < b:
                raise ValueError(f"{name} shares memory with an operand or another output")
        reads.append(t)
    given = [t for t in (dh, dwT, dbias) if t is not None]
    dev = h.device
    if dh is None and need_dh:
        dh = torch.empty((n, hidden), dtype=h.dtype, device=dev)
    if dwT is None and need_dwT:
        dwT = torch.empty((classes, hidden), dtype=h.dtype, device=dev)
    if dbias is None and bias is not None:
        dbias = torch.empty(classes, dtype=torch.float32, device=dev)
    if n == 0:
        for t in (dwT, dbias):
            if t is not None:
                t.zero_()
        return dh, dwT, dbias
    if given:
        torch.autograd.graph.increment_version(given)       # written in place
    lib, dt = native.load(), _DTYPES[h.dtype]
    with on_device(dev) as stream:
        need = lib.dtf_vocab_head_workspace(dt, 2 if keep_rounding else 1, ptr(h), ldh, ptr(wT), ldw, n, hidden, classes, int(dbias is not None), piece)
        check(min(need, 0), "vocab_head_workspace")
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        check(lib.dtf_vocab_head_bwd(dt, ptr(h), ldh, ptr(wT), ldw, ptr(bias), ptr(labels), ptr(lse), ptr(row_scale),
                                     float(grad_scale), n, hidden, classes, ignore_label, piece, int(keep_rounding), ptr(dh),
                                     ptr(dwT), int(dwT is not None and dwT.dtype == torch.float32), ptr(dbias), ptr(ws), need,
                                     stream),
              "vocab_head_bwd")
    return dh, dwT, dbias
