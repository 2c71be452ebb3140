"""Gradients that share memory are refused by clipping whatever their strides (an element of two of them would count twice in the norm), and
views that interleave without sharing are clipped."""
import math
import random

import pytest
import torch

from instascene_amd._lib import IsrError
from instascene_amd.optim import clip_grads_, grad_norm

pytestmark = pytest.mark.gpu


def refused(tensors, storage):
    before = storage.clone()
    with pytest.raises(IsrError, match="share memory"):
        clip_grads_(tensors, 1e-3)
    assert torch.equal(storage, before)


def values(rows, columns):
    """float32 whose halves are ordinary numbers in bfloat16 too (the views in another type read them)."""
    g = torch.Generator(device="cuda").manual_seed(11)
    return torch.randn(rows, 2 * columns, generator=g, device="cuda").bfloat16().view(torch.float32)


def test_columns_that_overlap():
    s = values(50, 8)
    refused([s[:, :5], s[:, 3:]], s)
    refused([s[:, 2:5], s], s)
    refused([s, s[:, 2:5]], s)
    refused([s[::2], s[::3]], s)
    refused([s[:, :5], torch.ones(3, device="cuda"), s[7:9, 4]], s)
    refused([s.T[1:4], s[40]], s)
    refused([s.view(torch.bfloat16)[:, 3:4], s[:, 1:2]], s)                 # the same bytes in another type
    refused([s.reshape(-1).unfold(0, 3, 1)], s)                             # one tensor onto itself
    refused([s.reshape(-1).as_strided((4, 5), (3, 2))], s)


def test_columns_that_interleave_are_clipped():
    s = values(50, 8)
    for views in (lambda t: [t[:, :5], t[:, 5:]], lambda t: [t[:, ::2], t[:, 1::2]], lambda t: [t[::2], t[1::2]],
                  lambda t: [t[:, 0], t[3, 1:], t[4:9, 2:7]], lambda t: [t.view(torch.bfloat16)[:, 2:4], t[:, :1], t[:, 2:]],
                  lambda t: [t.reshape(-1).as_strided((3, 2), (2, 3))]):    # elements 0 2 4 3 5 7: interleaved with itself
        t = s.clone()
        want = math.sqrt(sum(float(v.double().square().sum()) for v in views(s)))
        clipped = [v.double() * (0.5 * want / (want + 1e-6)) for v in views(s)]
        norm = clip_grads_(views(t), 0.5 * want)
        assert abs(float(norm) - want) <= 2 * 2.0 ** -24 * want             # one root in 64 bits, one rounding
        for v, w in zip(views(t), clipped):
            # the factor 4 u, the product u, one rounding to the type
            assert bool(((v.double() - w).abs() <= w.abs() * (6 * 2.0 ** -24 + torch.finfo(v.dtype).eps / 2)).all())


def test_against_every_element_counted():
    """Random strides: refused exactly where the sets of elements meet."""
    r, n = random.Random(5), 400
    s = torch.zeros(n, device="cuda")
    where = torch.arange(n)
    seen = [0, 0]
    for k in range(600):
        views = []
        for _ in range(2):
            dims = r.choice((1, 2, 3))
            while True:
                size, stride, at = [r.choice((1, 2, 3, 5)) for _ in range(dims)], [r.choice((1, 2, 3, 7, 8, 20, 60)) for _ in range(dims)], r.randrange(n)
                if at + sum((a - 1) * b for a, b in zip(size, stride)) < n:
                    break
            views.append((size, stride, at))
        sets = [where.as_strided(*v).reshape(-1).tolist() for v in views]
        shared = len(set(sets[0] + sets[1])) < len(sets[0] + sets[1])
        seen[shared] += 1
        tensors = [s.as_strided(*v) for v in views]
        if shared:
            with pytest.raises(IsrError, match="share memory"):
                clip_grads_(tensors, 1.0)
        else:
            clip_grads_(tensors, 1.0)
        grad_norm(tensors)                                  # reading twice is fine
    assert min(seen) > 100, seen
