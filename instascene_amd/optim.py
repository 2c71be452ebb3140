"""``GaussianAdam`` - the optimiser of the reference's ``train.py`` loop (``torch.optim.Adam(l, lr=0.0, eps=1e-15)`` over the
six parameter groups of ``GaussianModel.training_setup``, scene/gaussian_model.py:206-253; stepped at train.py:153-156) as ONE
kernel per iteration (``iso_gaussian_adam_step``, csrc/iso_optim.hip) that also

* applies the chain rule from the gradients of the ACTIVATED tensors the rasterizer consumed - ``exp(_scaling)``,
  ``sigmoid(_opacity)``, ``normalize(_rotation)``, ``cat(_features_dc, _features_rest)`` (the model's getters,
  scene/gaussian_model.py:109-138) - to the raw parameters, and
* emits those activations of the updated parameters for the next forward.

The activations are handed to ``render()`` as autograd LEAVES (``begin()``), so a step is: ``begin()`` -> ``render`` ->
loss -> ``backward()`` -> ``step()``.  Arithmetic and semantics are dense ``torch.optim.Adam``'s (a Gaussian that was not
visible still decays its moments and moves by its momentum); ``tests/test_gpu_harness.py`` pins it against torch's
optimiser.  Row edits by the density control (clone / split / prune) are not supported here: ``RgbTrainer(densify=...)``
keeps ``torch.optim.Adam``.

Beside it, for any list of gradients: their global norm (:func:`grad_norm`) and clipping (:func:`clip_grads_`,
:func:`clip_grad_norm_`) in one pass over all tensors each (``iso_grad_norm``, csrc/iso_gradnorm.hip).
"""
from __future__ import annotations

import ctypes
from typing import Dict, Iterable, Optional, Sequence

import torch

from . import _hot
from ._lib import check, lib
from .rows import _ext

GROUPS = ("xyz", "f_dc", "f_rest", "opacity", "scaling", "rotation")
_ATTR = {"xyz": "_xyz", "f_dc": "_features_dc", "f_rest": "_features_rest", "opacity": "_opacity", "scaling": "_scaling",
         "rotation": "_rotation"}


def _table(tensors):
    arr = (ctypes.c_void_p * 6)()
    for i, t in enumerate(tensors):
        arr[i] = None if t is None else t.data_ptr()
    return arr


class GaussianAdam:
    def __init__(self, model, lrs: Dict[str, float], betas=(0.9, 0.999), eps: float = 1e-15):
        self.model = model
        self.betas, self.eps = betas, float(eps)
        # torch-style groups, so that a learning-rate schedule (GaussianModel.update_learning_rate sets the "xyz" group's
        # lr every iteration, scene/gaussian_model.py:255-262) works unchanged
        self.param_groups = [{"params": [getattr(model, _ATTR[g])], "lr": float(lrs[g]), "name": g} for g in GROUPS]
        for g in self.param_groups:
            p = g["params"][0]
            if not p.is_cuda or p.dtype != torch.float32 or not p.is_contiguous():
                raise ValueError("GaussianAdam needs contiguous float32 CUDA parameters")
        self.exp_avg = {g: torch.zeros_like(getattr(model, _ATTR[g])) for g in GROUPS}
        self.exp_avg_sq = {g: torch.zeros_like(getattr(model, _ATTR[g])) for g in GROUPS}
        self.step_count = 0
        self.last_grad_norm = None      # of the last step with max_grad_norm: a float32 scalar on the device
        self._acts = None               # activations of the current parameters, written by the last step
        self.leaves = None

    # -- activations --------------------------------------------------------------------------------------------------
    def _params(self):
        return [getattr(self.model, _ATTR[g]) for g in GROUPS]

    def _clip_coef(self, grads, max_grad_norm: float):
        """``min(1, max_grad_norm / (norm + 1e-6))`` of the raw parameters' gradients (``iso_gaussian_grad_norm``: this optimiser's chain rule on
        the way), on the device; the norm goes to ``last_grad_norm``."""
        ps = self._params()
        dev = ps[0].device
        g = [None if t is None else t.contiguous().float() for t in grads]
        L = lib()
        nbytes = L.iso_grad_norm_scratch_bytes(1, None)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        out = torch.empty(2, dtype=torch.float32, device=dev)
        p = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())
        with _hot.on_device(dev):
            check(L.iso_gaussian_grad_norm(ps[0].shape[0], 1 + ps[2].shape[1], _table([t.data for t in ps]), p(g[0]), p(g[1]), p(g[2]), p(g[3]),
                                           p(g[4]), float(max_grad_norm), p(out), p(scratch), nbytes, _hot.stream_ptr(dev)), "iso_gaussian_grad_norm")
        self.last_grad_norm = out[0]
        return out[1:2]

    def _launch(self, grads, want_acts: bool, coef=None):
        ps = self._params()
        P = ps[0].shape[0]
        M = 1 + ps[2].shape[1]
        dev = ps[0].device
        acts = None
        if want_acts:
            new = lambda *s: torch.empty(s, dtype=torch.float32, device=dev)
            acts = (new(P, M, 3), new(P, 1), new(P, 2), new(P, 4))
        lr = (ctypes.c_double * 6)(*[float(g["lr"]) for g in self.param_groups])
        p = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())
        g = [None if t is None else t.contiguous().float() for t in grads]
        with _hot.on_device(dev):
            check(lib().iso_gaussian_adam_step_clipped(
                P, M, _table([t.data for t in ps]), _table([self.exp_avg[k] for k in GROUPS]),
                _table([self.exp_avg_sq[k] for k in GROUPS]), lr, float(self.betas[0]), float(self.betas[1]), self.eps,
                max(1, self.step_count), p(g[0]), p(g[1]), p(g[2]), p(g[3]), p(g[4]),
                *(p(a) for a in (acts if acts is not None else (None,) * 4)), p(coef),
                _hot.stream_ptr(dev)), "iso_gaussian_adam_step")
        return acts

    def begin(self):
        """The activated tensors of the current parameters as leaves that require grad:
        ``dict(xyz, shs, opacity, scaling, rotation)`` - what the model's getters return during the step."""
        versions = tuple(p._version for p in self._params())
        if self._acts is None or self._acts[0] != versions:
            self._acts = (versions, self._launch((None,) * 5, want_acts=True))     # no gradient: only the activations are written
        shs, opa, scale, rot = self._acts[1]
        mk = lambda t: t.detach().requires_grad_(True)
        self.leaves = dict(xyz=self.model._xyz, shs=mk(shs), opacity=mk(opa), scaling=mk(scale), rotation=mk(rot))
        return self.leaves

    def leaf_grads(self):
        """The five gradient tensors of the leaves (None where nothing arrived) - what a data-parallel trainer sums."""
        lv = self.leaves
        return [lv["xyz"].grad, lv["shs"].grad, lv["opacity"].grad, lv["scaling"].grad, lv["rotation"].grad]

    def step(self, grads=None, max_grad_norm: Optional[float] = None):
        """Chain rule + Adam + the next activations from the leaves' gradients (or ``grads``, e.g. their sum over ranks).
        ``max_grad_norm``: the gradients of the six raw parameters clipped to this global norm, as ``clip_grad_norm_`` in front of
        ``torch.optim.Adam`` would - the factor is applied inside the step's kernel; their norm is then in ``last_grad_norm``."""
        if self.leaves is None:
            raise RuntimeError("GaussianAdam.step: begin() was not called")
        grads = self.leaf_grads() if grads is None else grads
        coef = None if max_grad_norm is None else self._clip_coef(grads, check_max_norm("GaussianAdam.step", max_grad_norm))
        self.step_count += 1
        acts = self._launch(grads, want_acts=True, coef=coef)
        ps = self._params()
        for prm in ps:
            torch.autograd.graph.increment_version(prm)         # the kernel wrote through raw pointers
        self._acts = (tuple(prm._version for prm in ps), acts)
        self.leaves = None

    def zero_grad(self, set_to_none: bool = True):
        for prm in self._params():
            if set_to_none:
                prm.grad = None
            elif prm.grad is not None:
                prm.grad.zero_()

    # -- torch-compatible state (checkpoints: train.py:157-159 saves optimizer.state_dict()) -------------------------------
    def state_dict(self):
        return {"state": {i: {"step": torch.tensor(float(self.step_count)), "exp_avg": self.exp_avg[g],
                              "exp_avg_sq": self.exp_avg_sq[g]} for i, g in enumerate(GROUPS)},
                "param_groups": [{"lr": pg["lr"], "name": pg["name"], "betas": self.betas, "eps": self.eps, "params": [i]}
                                 for i, pg in enumerate(self.param_groups)]}

    def load_state_dict(self, sd):
        by_name = {pg["name"]: pg for pg in sd["param_groups"]}
        for i, g in enumerate(GROUPS):
            pg = by_name[g]
            st = sd["state"].get(pg["params"][0])
            self.param_groups[i]["lr"] = float(pg["lr"])
            if st is not None:
                self.exp_avg[g].copy_(st["exp_avg"])
                self.exp_avg_sq[g].copy_(st["exp_avg_sq"])
                self.step_count = int(float(st["step"]))
        self._acts = None


# -- the global norm of many gradients, and clipping ----------------------------------------------------------------------------
def check_max_norm(what: str, max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"{what}: the largest norm must not be negative, is {max_norm}")
    return max_norm


def norm_and_coef(tensors: Sequence[torch.Tensor], max_norm: float):
    """``(norm, coef)`` of gradients that an optimiser kernel will scale itself (``FeatureAdam``): one-element views of one tensor;
    ``coef = min(1, max_norm / (norm + 1e-6))``.  Nothing is written to the gradients."""
    out = _ext().grad_norm_coef(list(tensors), 2.0, max_norm)
    return out[0], out[1:2]


def grad_norm(tensors: Iterable[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The norm (2, 1 or inf) of all elements of ``tensors`` together, as a float32 scalar on their device; nothing is synchronised.
    float32, bfloat16 and float16 may be mixed; sums are held in 64 bits.  No tensors: 0."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    return _ext().grad_norm(tensors, norm_type, 0.0, False)


def clip_grads_(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scale ``grads`` in place by ``min(1, max_norm / (norm + 1e-6))`` and return their norm before it: what
    ``torch.nn.utils.clip_grad_norm_`` does, on a list of gradients.  The factor stays on the device; gradients that need no clipping are
    read once and not written.  Two of them may not share memory.  ``error_if_nonfinite`` reads the norm back (a synchronisation) and
    raises before anything is scaled."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    max_norm = check_max_norm("clip_grads_", max_norm)
    if not grads:
        return torch.tensor(0.0)
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"clip_grads_: the norm of order {norm_type} of the gradients is {float(norm)}; nothing was clipped")
    return _ext().grad_norm(grads, norm_type, max_norm, True)


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """:func:`clip_grads_` on the ``.grad`` of ``parameters`` (those that have one)."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    return clip_grads_([p.grad for p in parameters if p.grad is not None], max_norm, norm_type, error_if_nonfinite)
