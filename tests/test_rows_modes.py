"""Tracing and forward-mode differentiation: the row and gradient operators refuse both (their kernels are not recorded and carry no tangent),
where an output without its values or its tangent would come back otherwise.  The refusal comes before every other check, so that most of it
shows without a GPU."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from instascene_amd.optim import clip_grads_, grad_norm
from instascene_amd.rows import QuantizedRows, rms_norm, rms_norm_quantized

CALLS = {"rms_norm": lambda t: rms_norm(t), "rms_norm_quantized": lambda t: rms_norm_quantized(t).scales, "grad_norm": lambda t: grad_norm([t]),
         "clip_grads_": lambda t: clip_grads_([t], 1.0)}


def refuses(call, x):
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, (x,))
    for mode in ("real", "symbolic"):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(call, tracing_mode=mode)(x)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):       # (no_grad does not turn tangents off)
            call(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("name", CALLS)
def test_traces_and_tangents_are_refused(name):
    refuses(CALLS[name], torch.ones(3, 8))
    w = torch.ones(8)
    if name.startswith("rms"):
        entry = rms_norm if name == "rms_norm" else rms_norm_quantized
        with forward_ad.dual_level():
            for kw in ({"weight": forward_ad.make_dual(w, w)}, {"residual": forward_ad.make_dual(torch.ones(3, 8), torch.ones(3, 8))}):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    entry(torch.ones(3, 8), **kw)


@pytest.mark.gpu
def test_on_the_device():
    x = torch.ones(3, 8, device="cuda")
    for call in CALLS.values():
        refuses(call, x)
        call(x.clone())                                     # and the plain call still runs, also behind a refused one
    refuses(lambda t: rms_norm(t, residual=x)[1], x)
    table = QuantizedRows(3, 8)
    refuses(lambda t: table.write(t).scales, x)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda t: table.read(t), (torch.zeros(2, dtype=torch.int64, device="cuda"),))
    assert bool((table.read() == 0).all())
    # a tangent that reaches the backward pass alone
    leaf = x.clone().requires_grad_(True)
    y, s = rms_norm(leaf, residual=x)
    with forward_ad.dual_level():
        for pair in ((forward_ad.make_dual(x, x), x), (x, forward_ad.make_dual(x, x))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad((y, s), leaf, pair, retain_graph=True)
    assert torch.isfinite(torch.autograd.grad((y, s), leaf, (x, x))[0]).all()
    # inside vmap torch itself refuses
    with pytest.raises(RuntimeError):
        torch.func.vmap(rms_norm)(x[None])
