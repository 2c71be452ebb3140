"""Finite rows near the largest float32, whose products with the gain lie beyond it: the quantised norm keeps them (its result is finite).

u = 2^-24.  Codes are those of the products rounded to 24 bits (the kernel's own rounding), taken at a smaller exponent.  Scales: top / Q, rstd
(below the normal numbers here, at least 2^-128 with a half step of 2^-150: 4 u; the sum in 64 bits adds u, the root's float u) and one rounding:
within the 20 u of ordinary rows.  Likewise the normalised read of such a row: the inverse of its length is kept to 24 bits."""
import pytest
import torch

from instascene_amd.rows import QuantizedRows, rms_norm, rms_norm_quantized
from test_gpu_rows import BF16, E4M3, F16, F32, Q, U, check, encode_reference, make, norm_reference

pytestmark = pytest.mark.gpu

# narrower than a vector, a wave and less (one or two vectors per thread), several waves, beyond the registers; per row and in groups
SHAPES = [(3, 3, None), (90, 3, None), (90, 5, None), (7, 64, 32), (300, 192, 64), (33, 1023, None), (5, 4096, 128), (1100, 300, None), (2, 16512, 128), (2, 33001, None),
          (3, 40960, 32)]


@pytest.mark.parametrize("code", [torch.int8, E4M3])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,width,group", SHAPES)
def test_products_beyond_the_largest_float(code, dtype, rows, width, group):
    print(f"case {code} {dtype} {rows} {width} {group}", flush=True)
    G = group or width
    x = make((rows, width), F32, 1).clamp(-3, 3)
    if dtype == F16:                                        # the gain carries the size
        w = 1e37 * (1.5 + make((width,), F32, 3).clamp(-1, 1))
        x = x * 1e4
    else:
        w = 1.5 + make((width,), F32, 3).clamp(-1, 1)
        x = x * 1.1e38
        x[1::3] *= 1e-20                                    # rows of ordinary size between them
        x[2::3, : width // 2] *= 1e-30                      # and groups
    x = x.to(dtype)
    q = rms_norm_quantized(x, w, 1e-6, dtype=code, group=group)
    s, rstd, y = norm_reference(x, w, 1e-6, None)
    t = (s * w.double() * 2.0 ** -40).float()               # one rounding to 24 bits; the codes do not depend on the power of two
    big = (s * w.double()).abs().reshape(rows, -1, G).amax(2) >= 2.0 ** 128
    assert rows * width < 50 or (bool(big.any()) and (dtype == F16 or not bool(big.all())))      # (nine numbers may have none)
    want, top = encode_reference(t, code, G)
    assert torch.equal(q.codes.double(), want)
    scales = top * 2.0 ** 40 * rstd / Q[code]
    check(q.scales, scales, scales * 20 * U, "scales")
    # what the codes stand for is the row that rms_norm gives
    step = 0.5 / 127 if code == torch.int8 else 2.0 ** -4
    largest = y.abs().reshape(rows, -1, G).amax(2, keepdim=True).expand(rows, width // G, G).reshape(rows, width)
    tol = largest * (step + 40 * U) if code == torch.int8 else y.abs() * step + largest * (2.0 ** -10 / 448 + 40 * U)
    got = q.codes.double().reshape(rows, -1, G) * q.scales.double()[:, :, None]
    check(got.reshape(rows, width), y, tol, "values")
    if dtype == F32:
        check(rms_norm(x, w, 1e-6), y, y.abs() * 24 * U, "the plain norm")


@pytest.mark.parametrize("code", [torch.int8, E4M3])
@pytest.mark.parametrize("width,group", [(5, None), (64, 32), (1024, None), (16512, 128), (33001, None)])
def test_real_infinities_still_read_back_as_nan(code, width, group):
    x = torch.ones(4, width, device="cuda")
    x[0, 3], x[1, 3] = float("inf"), float("nan")
    x[2] = 3e38
    w = torch.full((width,), 2.0, device="cuda")
    q = rms_norm_quantized(x, w, 1e-6, dtype=code, group=group)
    G = group or width
    assert bool(torch.isnan(q.scales[0, 0])) and bool((q.scales[0, 1:] == 0).all()) and bool(torch.isnan(q.scales[1]).all())
    assert bool((q.read()[2:] - 2.0).abs().max() <= 1e-5)
    assert q.codes.double()[0, :G].abs().max() == 0


@pytest.mark.parametrize("code", [torch.int8, E4M3])
def test_a_sum_beyond_the_largest_float_is_an_infinity(code):
    x = torch.full((2, 64), 3e38, device="cuda")
    q, s = rms_norm_quantized(x, residual=x, dtype=code, group=32)
    assert bool(torch.isinf(s).all()) and bool(torch.isnan(q.scales).all())
    t = QuantizedRows.from_rows(s, dtype=code)
    assert bool(torch.isnan(t.read()).all())


@pytest.mark.parametrize("code", [torch.int8, E4M3])
@pytest.mark.parametrize("width,group", [(3, None), (64, 32), (129, None), (1024, 128), (4096, None), (20000, None), (36864, 64)])
def test_normalised_read_of_rows_near_the_largest_float(code, width, group):
    print(f"case {code} {width} {group}", flush=True)
    x = make((6, width), F32, 1).clamp(-3, 3) * 1.1e38
    x[1], x[2] = 3.4e38, x[2] * 1e-30
    x[3, width // 2:] *= 1e-25                              # groups of ordinary size beside large ones
    x[4] = 0.0
    t = QuantizedRows.from_rows(x, dtype=code, group=group)
    v = t.read().double()
    for eps in (1e-6, 0.0, 1e38):
        rows = [0, 1, 2, 3, 5] if eps == 0.0 else list(range(6))             # (a zero row has no direction)
        want = v / (v.norm(dim=1, keepdim=True) + float(torch.tensor(eps)))
        for out in (F32, BF16):
            got = t.read(out_dtype=out, norm_eps=eps)
            check(got[rows], want[rows], want[rows].abs() * ((2.0 ** -8 if out == BF16 else U) + 20 * U) + 2.0 ** -149, "normalised")
    zeros = t.read(slice(4, 5), norm_eps=1e-40)              # (an eps below the normal numbers)
    assert bool((zeros == 0).all()) and bool(torch.isnan(t.read(slice(4, 5), norm_eps=0.0)).all())
