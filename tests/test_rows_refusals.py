"""What the row and gradient operators refuse, without a GPU: the Python entries refuse host tensors, the C entries refuse bad
arguments before anything is launched."""
import ctypes

import pytest
import torch

from instascene_amd import _lib
from instascene_amd.optim import clip_grads_, grad_norm
from instascene_amd.rows import SCAN_MAX, QuantizedRows, rms_norm, rms_norm_quantized

EINVAL = -1


def test_host_tensors_are_refused():
    x = torch.ones(2, 4)
    for call in (lambda: rms_norm(x), lambda: rms_norm_quantized(x), lambda: QuantizedRows(2, 4, device="cpu"),
                 lambda: QuantizedRows.from_rows(x), lambda: grad_norm([x]), lambda: clip_grads_([x], 1.0)):
        with pytest.raises(RuntimeError):
            call()
    assert float(grad_norm([])) == 0.0


def _message(rc):
    assert rc != 0
    return _lib.lib().isr_last_error().decode()


def test_c_entries_refuse_bad_arguments():
    L, one = _lib.lib(), ctypes.c_void_p(64)        # never read: every call is refused first
    fwd = lambda type=0, rows=1, F=4, x=one, y=one, eps=1e-6: L.iso_rms_norm_forward(type, rows, F, x, F, None, 0, None, 0, eps, y, None, None, None)
    assert "type" in _message(fwd(type=3)) and "F" in _message(fwd(F=0)) and "F" in _message(fwd(F=(1 << 24) + 1))
    assert "rows" in _message(fwd(rows=-1)) and "null" in _message(fwd(x=None)) and "eps" in _message(fwd(eps=0.0)) and "eps" in _message(fwd(eps=float("nan")))
    assert fwd(rows=0) == 0
    quant = lambda code=1, F=64, group=64: L.iso_rms_norm_quant(0, code, 1, F, group, one, F, None, 0, None, 0, 1e-6, None, None, None, None)
    assert "code" in _message(quant(code=3)) and "group" in _message(quant(group=16)) and "group" in _message(quant(F=96, group=64)) and "null" in _message(quant())
    back = lambda scratch=0, dw=one: L.iso_rms_norm_backward(0, 8, 4, one, 4, None, 0, None, 0, one, one, 4, None, 0, None, dw, one, scratch, None)
    assert "scratch" in _message(back()) and "null" in _message(back(dw=None))
    assert L.iso_rms_norm_scratch_bytes(0, 8, 4) > 0 and L.iso_rms_norm_scratch_bytes(0, 0, 4) == 0
    write = lambda n=2, P=4, first=0, index=None, owner=None: L.iso_rows8_write(0, 1, n, 4, 4, P, one, 4, first, index, 1, owner, one, one, None)
    assert "table of 4" in _message(write(first=3)) and "table" in _message(write(first=-1)) and "owner" in _message(write(n=SCAN_MAX + 1, index=one))
    assert write(n=0) == 0
    read = lambda n=2, P=4, first=0, out=one: L.iso_rows8_read(0, 1, n, 4, 4, P, one, one, first, None, 1, 0, 0.0, out, None)
    assert "table" in _message(read(first=3)) and "null" in _message(read(out=None)) and read(n=0) == 0


def test_the_gradient_entry_refuses_bad_lists():
    L, one = _lib.lib(), ctypes.c_void_p(64)

    def norm(ptrs, sizes, types, kind=2, max_norm=1.0, clip=0, scratch=1 << 20, out=one):
        n = len(ptrs)
        return L.iso_grad_norm(n, (ctypes.c_void_p * max(n, 1))(*ptrs), (ctypes.c_longlong * max(n, 1))(*sizes), (ctypes.c_int * max(n, 1))(*types),
                               kind, max_norm, clip, out, one, scratch, None)

    assert "norm type" in _message(norm([64], [1], [0], kind=3)) and "null" in _message(norm([None], [1], [0]))
    assert "type 5" in _message(norm([64], [1], [5])) and "size -1" in _message(norm([64], [-1], [0]))
    assert "max_norm" in _message(norm([64], [1], [0], max_norm=-1.0, clip=1)) and "max_norm" in _message(norm([64], [1], [0], max_norm=float("nan"), clip=1))
    assert "scratch" in _message(norm([64], [1], [0], scratch=8)) and "null" in _message(norm([64], [1], [0], out=None))
    # 4 floats at 64 and 2 halves at 78: one byte of overlap; a long list takes the other branch
    assert "share memory" in _message(norm([64, 78], [4, 2], [0, 2], clip=1))
    many = [4096 * (i + 1) for i in range(100)]
    assert "share memory" in _message(norm(many + [many[50] + 8], [8] * 101, [0] * 101, clip=1))
