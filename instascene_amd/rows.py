"""Operators on the rows of a ``[P,F]`` table beside ``row_normalize`` / ``gather_rows``: the root-mean-square norm with the residual's
addition (:func:`rms_norm`, with its backward pass), the same with an output in 8 bits (:func:`rms_norm_quantized`), and a table kept in
8 bits (:class:`QuantizedRows`: written as a whole, by range or by index, read back likewise).  The kernels are ``iso_rms_norm_*``
and ``iso_rows8_*`` (include/instascene_ops.h); every call runs on the current stream of its tensors' device, allocates from torch and
synchronises nothing, so it can be captured into a graph."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _hot
from ._lib import check, lib

ROW_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
CODE_TYPES = {torch.int8: 1, torch.float8_e4m3fn: 2}
SCAN_MAX = 256          # ISO_ROWS8_SCAN: up to here a written row looks for a later one of the same index itself
_MAX_WIDTH = 1 << 24


def _p(t):
    return None if t is None else t.data_ptr()


def _rows2d(t: torch.Tensor) -> torch.Tensor:
    """``t`` as ``[rows, F]`` with the columns of a row next to each other (a copy only where they are not)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _check_rows(what: str, x: torch.Tensor):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError(f"{what}: needs CUDA tensors (the HIP library is the only backend)")
    if x.dtype not in ROW_TYPES:
        raise TypeError(f"{what}: float32, bfloat16 or float16, not {x.dtype}")
    if x.dim() < 1 or not (1 <= x.shape[-1] <= _MAX_WIDTH):
        raise ValueError(f"{what}: rows of 1 to 2^24 columns, not a tensor of shape {tuple(x.shape)}")


def _check_norm(what, x, weight, eps, residual):
    _check_rows(what, x)
    if not float(eps) > 0.0:
        raise ValueError(f"{what}: eps must be positive")
    if weight is not None:
        if weight.device != x.device or weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
            raise ValueError(f"{what}: weight must be [{x.shape[-1]}] on {x.device}, not {tuple(weight.shape)} on {weight.device}")
        if weight.dtype != torch.float32 and weight.dtype != x.dtype:
            raise TypeError(f"{what}: weight must be float32 or {x.dtype}, not {weight.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"{what}: residual must be a {x.dtype} {tuple(x.shape)} on {x.device} like x")


def _check_group(what, width, group) -> int:
    if group is None or group == width:
        return width
    if group not in (32, 64, 128) or width % group:
        raise ValueError(f"{what}: groups of 32, 64 or 128 columns that divide the row, or None for one per row: not {group} of {width}")
    return int(group)


def _forward(x, weight, eps, residual, want_rstd):
    x2, r2 = _rows2d(x), None if residual is None else _rows2d(residual)
    n, F = x2.shape
    dev = x.device
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    s = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=dev)
    rstd = torch.empty(n, dtype=torch.float32, device=dev) if want_rstd else None
    w = None if weight is None else weight.contiguous()
    with _hot.on_device(dev):
        check(lib().iso_rms_norm_forward(ROW_TYPES[x.dtype], n, F, _p(x2), x2.stride(0), _p(r2), 0 if r2 is None else r2.stride(0),
                                         _p(w), int(w is not None and w.dtype == torch.float32), float(eps), _p(y), _p(s), _p(rstd),
                                         _hot.raw_stream(dev)), "iso_rms_norm_forward")
    return y, s, rstd


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        y, s, rstd = _forward(x, weight, eps, residual, True)
        # float32: s is x + residual exactly as the norm took it.  16 bits: s was rounded once more on its way out, and the gradient
        # of the weight would carry that (2^-9 of every term): x and the residual are read again instead
        if s is None or x.dtype == torch.float32:
            ctx.save_for_backward(x if s is None else s, None, weight, rstd)
        else:
            ctx.save_for_backward(x, residual, weight, rstd)
        ctx.set_materialize_grads(False)
        return y if s is None else (y, s)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gs=None):
        x, residual, weight, rstd = ctx.saved_tensors
        need_x, need_w, _, need_r = ctx.needs_input_grad
        if gy is None:                                    # only the sum was used: its gradient passes through
            return (gs if need_x else None), None, None, (gs if need_r else None)
        L, dev = lib(), x.device
        x2, g2 = _rows2d(x), _rows2d(gy)
        r2 = None if residual is None else _rows2d(residual)
        q2 = None if gs is None else _rows2d(gs)
        n, F = x2.shape
        kind = ROW_TYPES[x.dtype]
        ds = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x or need_r else None
        dw = scratch = w = None
        nbytes = 0
        if weight is not None:
            w = weight.contiguous()
            if need_w:
                dw = torch.empty(F, dtype=weight.dtype, device=dev) if n else torch.zeros(F, dtype=weight.dtype, device=dev)
                nbytes = L.iso_rms_norm_scratch_bytes(kind, n, F)
                scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        if ds is None and dw is None:
            return None, None, None, None
        with _hot.on_device(dev):
            check(L.iso_rms_norm_backward(kind, n, F, _p(x2), x2.stride(0), _p(r2), 0 if r2 is None else r2.stride(0), _p(w),
                                          int(w is not None and w.dtype == torch.float32), _p(rstd), _p(g2), g2.stride(0), _p(q2), 0 if q2 is None else q2.stride(0), _p(ds), _p(dw), _p(scratch), nbytes,
                                          _hot.raw_stream(dev)), "iso_rms_norm_backward")
        return (ds if need_x else None), dw, None, (ds if need_r else None)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6, residual: Optional[torch.Tensor] = None):
    """``y = s / sqrt(mean(s^2) + eps) * weight`` over the last dimension, ``s = x + residual``; returns ``y``, or ``(y, s)`` with a
    residual.  float32, bfloat16 or float16, rows of any width and stride; everything between input and output is held in 32 bits
    (the sum of squares in 64), ``y`` and ``s`` are rounded once.  ``weight`` is float32 or of x's type.  Differentiable in ``x``,
    ``weight`` and ``residual``."""
    _check_norm("rms_norm", x, weight, eps, residual)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _RmsNorm.apply(x, weight, eps, residual)
    y, s, _ = _forward(x, weight, eps, residual, False)
    return y if s is None else (y, s)


def rms_norm_quantized(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
                       dtype: torch.dtype = torch.float8_e4m3fn, group: Optional[int] = None):
    """:func:`rms_norm` of ``[rows, F]`` with the output in 8 bits: a :class:`QuantizedRows`, or ``(rows, s)`` with a residual.  Not
    differentiable: inputs that require a gradient are refused unless gradients are disabled."""
    what = "rms_norm_quantized"
    _check_norm(what, x, weight, eps, residual)
    if x.dim() != 2:
        raise ValueError(f"{what}: x must be [rows, F]")
    if dtype not in CODE_TYPES:
        raise TypeError(f"{what}: dtype must be torch.int8 or torch.float8_e4m3fn, not {dtype}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")
    n, F = x.shape
    G = _check_group(what, F, group)
    x2, r2 = _rows2d(x), None if residual is None else _rows2d(residual)
    w = None if weight is None else weight.contiguous()
    dev = x.device
    out = QuantizedRows._of(torch.empty((n, F), dtype=dtype, device=dev), torch.empty((n, F // G), dtype=torch.float32, device=dev))
    s = None if residual is None else torch.empty((n, F), dtype=x.dtype, device=dev)
    with _hot.on_device(dev):
        check(lib().iso_rms_norm_quant(ROW_TYPES[x.dtype], CODE_TYPES[dtype], n, F, G, _p(x2), x2.stride(0), _p(r2),
                                       0 if r2 is None else r2.stride(0), _p(w), int(w is not None and w.dtype == torch.float32),
                                       float(eps), _p(out.codes), _p(out.scales), _p(s), _hot.raw_stream(dev)), "iso_rms_norm_quant")
    return out if s is None else (out, s)


class QuantizedRows:
    """A table of ``rows`` rows of ``width`` columns in 8 bits: ``codes [rows, width]`` (int8 or float8_e4m3fn) and one float32 scale per
    row, or per ``group`` (32, 64, 128) of its columns: ``scales [rows, width / group]``; a value is code * scale.  A new table holds
    zeros.  A group whose largest magnitude is below 2^-116 is stored as zeros; one that holds an infinity or NaN reads back as NaN.

    A trained feature table takes a quarter of its bytes this way; :func:`~instascene_amd.contrastive.gather_rows` and ``render()`` read
    it in the place of a float table.  Nothing here carries a gradient."""

    def __init__(self, rows: int, width: int, dtype: torch.dtype = torch.float8_e4m3fn, group: Optional[int] = None, device="cuda"):
        what = "QuantizedRows"
        dev = torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError(f"{what}: needs a CUDA device (the HIP library is the only backend)")
        if dtype not in CODE_TYPES:
            raise TypeError(f"{what}: dtype must be torch.int8 or torch.float8_e4m3fn, not {dtype}")
        if rows < 0 or not (1 <= width <= _MAX_WIDTH):
            raise ValueError(f"{what}: needs rows >= 0 and 1 <= width <= 2^24")
        G = _check_group(what, width, group)
        self.codes = torch.zeros((rows, width), dtype=torch.uint8, device=dev).view(dtype)
        self.scales = torch.zeros((rows, width // G), dtype=torch.float32, device=dev)
        self._owner = torch.full((rows,), -1, dtype=torch.int32, device=dev)

    @classmethod
    def _of(cls, codes, scales):
        """The table on existing tensors (no copy)."""
        t = cls.__new__(cls)
        t.codes, t.scales, t._owner = codes, scales, None
        return t

    @classmethod
    def from_rows(cls, x: torch.Tensor, dtype: torch.dtype = torch.float8_e4m3fn, group: Optional[int] = None) -> "QuantizedRows":
        _check_rows("QuantizedRows.from_rows", x)
        if x.dim() != 2:
            raise ValueError("QuantizedRows.from_rows: x must be [rows, width]")
        if dtype not in CODE_TYPES:
            raise TypeError(f"QuantizedRows.from_rows: dtype must be torch.int8 or torch.float8_e4m3fn, not {dtype}")
        G = _check_group("QuantizedRows.from_rows", x.shape[1], group)
        t = cls._of(torch.empty(x.shape, dtype=dtype, device=x.device),
                    torch.empty((x.shape[0], x.shape[1] // G), dtype=torch.float32, device=x.device))
        return t.write(x)

    shape = property(lambda s: s.codes.shape)
    dtype = property(lambda s: s.codes.dtype)
    device = property(lambda s: s.codes.device)
    group = property(lambda s: s.codes.shape[1] // s.scales.shape[1])
    nbytes = property(lambda s: s.codes.nbytes + s.scales.nbytes)

    def __len__(self):
        return self.codes.shape[0]

    def _index(self, what, index, n=None):
        if index.dim() != 1 or index.dtype not in (torch.int64, torch.int32) or index.device != self.codes.device:
            raise ValueError(f"{what}: index must be a 1-D int64 or int32 tensor on {self.codes.device}")
        if n is not None and index.shape[0] != n:
            raise ValueError(f"{what}: {index.shape[0]} indices for {n} rows")
        return index.contiguous()

    def write(self, rows: torch.Tensor, index=None) -> "QuantizedRows":
        """Quantise ``rows [n, width]`` into the table: all of it (``index`` None, n = rows of the table), rows ``[index, index + n)`` (an
        int), or row ``index[i]`` for every i (an int64 or int32 tensor): of equal indices the last is kept, and an index outside the
        table - the padding of a batch - writes nothing.  Other rows stay as they are."""
        what = "QuantizedRows.write"
        P, F = self.codes.shape
        _check_rows(what, rows)
        if rows.dim() != 2 or rows.shape[1] != F or rows.device != self.codes.device:
            raise ValueError(f"{what}: rows must be [n, {F}] on {self.codes.device}, not {tuple(rows.shape)} on {rows.device}")
        r2 = _rows2d(rows)
        n = r2.shape[0]
        first, ix, owner = 0, None, None
        if index is None:
            if n != P:
                raise ValueError(f"{what}: {n} rows for a table of {P}; give an index")
        elif isinstance(index, int):
            first = index
            if first < 0 or first + n > P:
                raise ValueError(f"{what}: rows [{first}, {first + n}) of a table of {P}")
        else:
            ix = self._index(what, index, n)
            if n > SCAN_MAX:
                if self._owner is None:
                    if torch.cuda.is_current_stream_capturing():
                        raise RuntimeError(f"{what}: the first write of more than {SCAN_MAX} indices to this table makes a helper table and "
                                           "cannot be captured: write once before the capture")
                    self._owner = torch.full((P,), -1, dtype=torch.int32, device=self.codes.device)
                owner = self._owner
        with _hot.on_device(self.codes.device):
            check(lib().iso_rows8_write(ROW_TYPES[rows.dtype], CODE_TYPES[self.codes.dtype], n, F, F // self.scales.shape[1], P, _p(r2),
                                        r2.stride(0), first, _p(ix), int(ix is not None and ix.dtype == torch.int64), _p(owner),
                                        _p(self.codes), _p(self.scales), _hot.raw_stream(self.codes.device)), "iso_rows8_write")
        torch.autograd.graph.increment_version((self.codes, self.scales))         # the kernel wrote through raw pointers
        return self

    def read(self, index=None, out_dtype: torch.dtype = torch.float32, norm_eps: Optional[float] = None) -> torch.Tensor:
        """The values of the whole table (``index`` None), of a ``slice`` of its rows, or of row ``index[i]`` for every i (an index
        outside the table: zeros) as ``[n, width]`` of ``out_dtype``.  ``norm_eps``: every row divided by (its 2-norm + norm_eps) on the
        way - ``row_normalize`` of what is read."""
        what = "QuantizedRows.read"
        if out_dtype not in ROW_TYPES:
            raise TypeError(f"{what}: out_dtype must be float32, bfloat16 or float16, not {out_dtype}")
        if norm_eps is not None and not float(norm_eps) >= 0.0:
            raise ValueError(f"{what}: norm_eps must not be negative")
        P, F = self.codes.shape
        first, ix, n = 0, None, P
        if isinstance(index, slice):
            first, stop, step = index.indices(P)
            if step != 1:
                raise ValueError(f"{what}: a slice of step 1, not {step}")
            n = max(0, stop - first)
            first = first if n else 0
        elif index is not None:
            ix = self._index(what, index)
            n = ix.shape[0]
        dev = self.codes.device
        out = torch.empty((n, F), dtype=out_dtype, device=dev)
        with _hot.on_device(dev):
            check(lib().iso_rows8_read(ROW_TYPES[out_dtype], CODE_TYPES[self.codes.dtype], n, F, F // self.scales.shape[1], P, _p(self.codes),
                                       _p(self.scales), first, _p(ix), int(ix is not None and ix.dtype == torch.int64),
                                       int(norm_eps is not None), float(norm_eps or 0.0), _p(out), _hot.raw_stream(dev)), "iso_rows8_read")
        return out

    def state_dict(self):
        return {"codes": self.codes, "scales": self.scales}

    def load_state_dict(self, sd):
        codes, scales = sd["codes"], sd["scales"]
        if codes.shape != self.codes.shape or codes.dtype != self.codes.dtype or scales.shape != self.scales.shape:
            raise ValueError("QuantizedRows.load_state_dict: a table of another shape, type or group")
        self.codes.view(torch.uint8).copy_(codes.view(torch.uint8))
        self.scales.copy_(scales)
