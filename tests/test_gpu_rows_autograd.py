"""rms_norm in programs: gradients that two leaves share, the same leaf twice, clipping behind a backward pass, inference mode."""
import pytest
import torch

from instascene_amd.optim import clip_grad_norm_, grad_norm
from instascene_amd.rows import QuantizedRows, rms_norm, rms_norm_quantized
from test_gpu_rows import BF16, F32, half, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("use", ["both", "y", "s"])
def test_gradients_of_two_leaves_are_two_tensors(dtype, use):
    """x and the residual have the same gradient: their .grad fields do not share memory, so clipping takes them."""
    a, b = (make((40, 96), dtype, k).requires_grad_(True) for k in (1, 2))
    y, s = rms_norm(a, residual=b)
    out = {"both": lambda: (y.float() * 0.5 + s.float()).square().sum(), "y": lambda: y.float().square().sum(), "s": lambda: s.float().square().sum()}[use]()
    out.backward()
    assert torch.equal(a.grad, b.grad) and a.grad.untyped_storage().data_ptr() != b.grad.untyped_storage().data_ptr()
    before = a.grad.clone()
    norm = clip_grad_norm_([a, b], 0.25 * float(grad_norm([a.grad, b.grad])))
    factor = 0.25 * float(norm) / (float(norm) + 1e-6)
    for leaf in (a, b):
        want = before.double() * factor
        assert bool(((leaf.grad.double() - want).abs() <= want.abs() * (half(dtype) + 8 * 2.0 ** -24) + 2.0 ** -140).all())


def test_the_same_leaf_twice():
    a = make((33, 70), F32, 1).requires_grad_(True)
    y, s = rms_norm(a, residual=a)
    gy, gs = make((33, 70), F32, 2), make((33, 70), F32, 3)
    torch.autograd.backward((y, s), (gy, gs))
    lone, other = a.detach().clone().requires_grad_(True), a.detach().clone()
    y2, s2 = rms_norm(lone, residual=other)
    torch.autograd.backward((y2, s2), (gy, gs))
    assert torch.equal(a.grad, 2 * lone.grad)               # (a power of two: exact)


def test_inference_mode():
    with torch.inference_mode():
        x, w = make((300, 64), BF16, 1), torch.nn.Parameter(torch.ones(64, device="cuda"))
        y, s = rms_norm(x, w, residual=x)
        q, _ = rms_norm_quantized(x, w, residual=x, group=32)
        t = QuantizedRows(300, 64)
        t.write(y, torch.arange(300, device="cuda"))
        t.write(y[:2], torch.tensor([5, 5], device="cuda"))
        got = t.read(slice(5, 6))
    assert torch.equal(y, rms_norm(x.clone(), w.detach(), residual=x.clone())[0])
    assert torch.equal(got, QuantizedRows.from_rows(y[1:2].clone()).read())
    assert q.codes.shape == (300, 64)


def test_views_that_negate_their_memory():
    """The imaginary part of a conjugate is a view whose memory holds the negative of its values (here one column wide, and as torch makes
    such a view of any tensor)."""
    c = torch.view_as_complex(make((50, 1, 2), F32, 1))
    x = torch.imag(torch.conj(c))
    assert x.is_neg() and torch.equal(x, -c.imag)
    assert torch.equal(rms_norm(x), rms_norm(x.clone())) and torch.equal(QuantizedRows.from_rows(x).read(), QuantizedRows.from_rows(x.clone()).read())
    x, r, w, gy = (torch._neg_view(t) for t in (make((9, 40), F32, 2), make((9, 40), F32, 3), make((40,), F32, 4), make((9, 40), F32, 5)))
    for a, b in zip(rms_norm(x, w, residual=r), rms_norm(x.clone(), w.clone(), residual=r.clone())):
        assert torch.equal(a, b)
    a, b = (rms_norm_quantized(t[0], t[1], dtype=torch.int8) for t in ((x, w), (x.clone(), w.clone())))
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    leaf, gain = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    for one, other in zip(torch.autograd.grad(rms_norm(leaf, gain), (leaf, gain), gy), torch.autograd.grad(rms_norm(leaf, gain), (leaf, gain), gy.clone())):
        assert torch.equal(one, other)
