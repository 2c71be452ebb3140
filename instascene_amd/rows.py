"""Operators on the rows of a ``[P,F]`` table beside ``row_normalize`` / ``gather_rows``: the root-mean-square norm with the residual's
addition (:func:`rms_norm`, with its backward pass), the same with an output in 8 bits (:func:`rms_norm_quantized`), and a table kept in
8 bits (:class:`QuantizedRows`: written as a whole, by range or by index, read back likewise).  The kernels are ``iso_rms_norm_*``
and ``iso_rows8_*`` (include/instascene_ops.h); every call runs on the current stream of its tensors' device, allocates from torch and
synchronises nothing (but see :meth:`QuantizedRows.write`), so it can be captured into a graph."""
from __future__ import annotations

import functools
import operator
from typing import Optional

import torch

SCAN_MAX = 256          # ISO_ROWS8_SCAN: up to here a written row looks for a later one of the same index itself
_MAX_WIDTH = 1 << 24
CODE_TYPES = (torch.int8, torch.float8_e4m3fn)


@functools.lru_cache(maxsize=None)
def _ext():
    """The compiled host side (csrc_torch/isr_torch_rows.cpp): checks, allocation, the autograd node, the launches.  No fallback.  (It is
    linked to the library beside it: an A/B build named by ISR_LIB_PATH does not reach these operators.)"""
    from . import _lib
    _lib.lib()              # torch's HIP runtime first, then the library: one runtime in the process
    try:
        from . import _C_hip
    except ImportError as e:
        raise RuntimeError(f"instascene_amd.rows: the compiled extension instascene_amd/_C_hip.so does not load ({e}). Build it with "
                           "`python -c 'import __graft_entry__ as g; g.build()'`.") from e
    return _C_hip


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6, residual: Optional[torch.Tensor] = None):
    """``y = s / sqrt(mean(s^2) + eps) * weight`` over the last dimension, ``s = x + residual``; returns ``y``, or ``(y, s)`` with a
    residual.  float32, bfloat16 or float16, rows of any width and stride; everything between input and output is held in 32 bits
    (the sum of squares too, formed again in 64 where it leaves [1e-30, 1e37] and always for rows beyond the registers), ``y`` and ``s`` are
    rounded once.  ``weight`` is float32 or of x's type.  Differentiable in ``x``,
    ``weight`` and ``residual``."""
    y, s = _ext().rms_norm(x, weight, eps, residual)
    return y if s is None else (y, s)


def rms_norm_quantized(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
                       dtype: torch.dtype = torch.float8_e4m3fn, group: Optional[int] = None):
    """:func:`rms_norm` of ``[rows, F]`` with the output in 8 bits: a :class:`QuantizedRows`, or ``(rows, s)`` with a residual.  The codes are
    those of ``s * weight``: a group of which that stays below 2^-116 everywhere is stored as zeros.  Not differentiable: inputs that require a gradient are refused unless gradients are disabled."""
    codes, scales, s = _ext().rms_norm_quantized(x, weight, eps, residual, dtype, group)
    out = QuantizedRows._of(codes, scales)
    return out if s is None else (out, s)


class QuantizedRows:
    """A table of ``rows`` rows of ``width`` columns in 8 bits: ``codes [rows, width]`` (int8 or float8_e4m3fn) and one float32 scale per
    row, or per ``group`` (32, 64, 128) of its columns: ``scales [rows, width / group]``; a value is code * scale.  A new table holds
    zeros.  A group whose largest magnitude is below 2^-116 is stored as zeros; one that holds an infinity or NaN reads back as NaN.

    A trained feature table takes a quarter of its bytes this way; :func:`~instascene_amd.contrastive.gather_rows` and ``render()`` read
    it in the place of a float table.  Nothing here carries a gradient."""

    def __init__(self, rows: int, width: int, dtype: torch.dtype = torch.float8_e4m3fn, group: Optional[int] = None, device="cuda"):
        self._allocate(rows, width, dtype, group, torch.device(device))
        self.codes.view(torch.uint8).zero_()
        self.scales.zero_()
        self._owner = torch.full((rows,), -1, dtype=torch.int32, device=self.codes.device)

    def _allocate(self, rows, width, dtype, group, dev):
        what = "QuantizedRows"
        if dev.type != "cuda":
            raise RuntimeError(f"{what}: needs a CUDA device (the HIP library is the only backend)")
        if dtype not in CODE_TYPES:
            raise TypeError(f"{what}: dtype must be torch.int8 or torch.float8_e4m3fn, not {dtype}")
        if rows < 0 or not (1 <= width <= _MAX_WIDTH):
            raise ValueError(f"{what}: needs rows >= 0 and 1 <= width <= 2^24")
        G = width if group is None else int(group)
        if G != width and (G not in (32, 64, 128) or width % G):
            raise ValueError(f"{what}: groups of 32, 64 or 128 columns that divide the row, or None for one per row: not {group} of {width}")
        self.codes = torch.empty((rows, width), dtype=dtype, device=dev)
        self.scales = torch.empty((rows, width // G), dtype=torch.float32, device=dev)
        self._owner = None      # [rows] -1s: which of equal indices is kept, for writes of many indices (iso_rows8_write)

    @classmethod
    def _of(cls, codes, scales):
        """The table on existing tensors (no copy)."""
        t = cls.__new__(cls)
        t.codes, t.scales, t._owner = codes, scales, None
        return t

    @classmethod
    def from_rows(cls, x: torch.Tensor, dtype: torch.dtype = torch.float8_e4m3fn, group: Optional[int] = None) -> "QuantizedRows":
        """A table of the rows of ``x [rows, width]``."""
        if x.dim() != 2:
            raise ValueError("QuantizedRows.from_rows: x must be [rows, width]")
        t = cls.__new__(cls)
        t._allocate(x.shape[0], x.shape[1], dtype, group, x.device)
        return t.write(x)

    shape = property(lambda s: s.codes.shape)
    dtype = property(lambda s: s.codes.dtype)
    device = property(lambda s: s.codes.device)
    group = property(lambda s: s.codes.shape[1] // s.scales.shape[1])
    nbytes = property(lambda s: s.codes.nbytes + s.scales.nbytes)

    def __len__(self):
        return self.codes.shape[0]

    def write(self, rows: torch.Tensor, index=None) -> "QuantizedRows":
        """Quantise ``rows [n, width]`` into the table: all of it (``index`` None, n = rows of the table), rows ``[index, index + n)`` (an
        int), or row ``index[i]`` for every i (an int64 or int32 tensor): of equal indices the last is kept, and an index outside the
        table - the padding of a batch - writes nothing.  Other rows stay as they are.  Two streams may write disjoint rows at once.  The
        first write of more than 256 indices to a table of ``from_rows`` / ``rms_norm_quantized`` makes a helper table ``[rows]`` and waits
        for it: the one synchronisation of this class."""
        what = "QuantizedRows.write"
        P = self.codes.shape[0]
        first, ix = 0, None
        if index is None:
            if rows.shape[0] != P:
                raise ValueError(f"{what}: {rows.shape[0]} rows for a table of {P}; give an index")
        elif not isinstance(index, torch.Tensor):
            first = operator.index(index)
        else:
            ix = index
            if self._owner is None and ix.numel() > SCAN_MAX:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError(f"{what}: the first write of more than {SCAN_MAX} indices to this table makes a helper table and "
                                       "cannot be captured: write once before the capture")
                owner = torch.full((P,), -1, dtype=torch.int32, device=self.codes.device)
                # once per table: from here on any stream may write, also one that waits for nothing this stream has done
                torch.cuda.current_stream(owner.device).synchronize()
                self._owner = owner
        _ext().rows8_write(self.codes, self.scales, self._owner, rows, ix, first)
        return self

    def read(self, index=None, out_dtype: torch.dtype = torch.float32, norm_eps: Optional[float] = None) -> torch.Tensor:
        """The values of the whole table (``index`` None), of a ``slice`` of its rows, or of row ``index[i]`` for every i (an index
        outside the table: zeros) as ``[n, width]`` of ``out_dtype``.  ``norm_eps``: every row divided by (its 2-norm + norm_eps) on the
        way - ``row_normalize`` of what is read."""
        P = self.codes.shape[0]
        first, ix, n = 0, None, P
        if isinstance(index, slice):
            first, stop, step = index.indices(P)
            if step != 1:
                raise ValueError(f"QuantizedRows.read: a slice of step 1, not {step}")
            n = max(0, stop - first)
            first = first if n else 0
        elif index is not None:
            ix = index
        return _ext().rows8_read(self.codes, self.scales, ix, first, n, out_dtype, norm_eps)

    def record_stream(self, stream) -> None:
        """``torch.Tensor.record_stream`` for all of the table's memory, the helper table included: needed where the table is used on another
        stream than the one it was made on and may be dropped before that stream is done."""
        for t in (self.codes, self.scales, self._owner):
            if t is not None:
                t.record_stream(stream)

    def state_dict(self):
        return {"codes": self.codes, "scales": self.scales}

    def load_state_dict(self, sd):
        codes, scales = sd["codes"], sd["scales"]
        if codes.shape != self.codes.shape or codes.dtype != self.codes.dtype or scales.shape != self.scales.shape:
            raise ValueError("QuantizedRows.load_state_dict: a table of another shape, type or group")
        self.codes.view(torch.uint8).copy_(codes.view(torch.uint8))
        self.scales.copy_(scales)
