"""The launch rules of the row operators that only many rows or many bytes reach, against the definitions in 64 bits: several passes of the
backward kernel's row loop, rows laid over fewer threads than a wave has lanes for them, two vectors per thread with several rows per
workgroup, and streams past the caches.

Tolerances as in test_gpu_rows.py (u = 2^-24).  The sum of a row in the backward pass: two vectors per thread, 3 additions over a vector, 6 over a
wave, 16 over its waves: 27, so 96 u in place of 88 there.  dw: a chain of a thread's passes, 6 additions over the rows of a wave, 3 over the
waves, 64 partials per slice and 32 slices: below passes + 105 u of the magnitudes, and 20 u per term."""
import pytest
import torch

from instascene_amd.rows import QuantizedRows, rms_norm, rms_norm_quantized
from test_gpu_rows import BF16, E4M3, F16, F32, Q, U, check, encode_reference, floor_of, half, make, norm_reference

pytestmark = pytest.mark.gpu


def forward_and_backward(rows, width, dtype, residual, passes):
    print(f"case {rows} {width} {dtype} {residual}", flush=True)
    eps = 1e-5
    x = make((rows, width), dtype, 1).requires_grad_(True)
    r = make((rows, width), dtype, 2, 3.0).requires_grad_(True) if residual else None
    w = (1.0 + 0.5 * make((width,), F32, 3)).requires_grad_(True)
    gy, gs = make((rows, width), dtype, 4), make((rows, width), dtype, 5) if residual else None
    got = rms_norm(x, w, eps, residual=r)
    y, s = got if residual else (got, None)
    dx, dw = torch.autograd.grad((y, s) if residual else y, (x, w), (gy, gs) if residual else gy)
    with torch.no_grad():
        s64, rstd, y64 = norm_reference(x, w, eps, r)
        check(y, y64, y64.abs() * (half(dtype) + 20 * U) + floor_of(dtype), "y")
        if residual:
            check(s, s64, s64.abs() * (half(dtype) + U) + floor_of(dtype), "s")
        del y64, y, s
        h = s64 * rstd
        del s64
        gw = gy.double() * w.double()
        mean = (gw * h).mean(dim=1, keepdim=True)
        ds = rstd * (gw - h * mean) + (gs.double() if residual else 0.0)
        noise = U * rstd * (22 * gw.abs() + 96 * h.abs() * (gw * h).abs().mean(dim=1, keepdim=True)) + (2 * U * gs.double().abs() if residual else 0.0)
        check(dx, ds, noise + ds.abs() * half(dtype) + floor_of(dtype), "dx")
        del noise, ds, gw
        h *= gy.double()
        check(dw, h.sum(dim=0), h.abs().sum(dim=0) * (passes + 125) * U + h.sum(dim=0).abs() * U, "dw")


# rows, width, type, passes of the row loop (workgroups: 2048 at most, 512 for rows from 2048 columns on)
LOOPS = [
    (150_001, 32, F32, 3),          # 8 threads a row, 32 rows a workgroup; the last pass partly filled
    (60_001, 61, F32, 2),           # 16 threads, a last vector that sticks out
    (40_001, 121, BF16, 2),
    (20_001, 300, F32, 3),          # 64 threads with two vectors, 4 rows a workgroup
    (20_001, 600, F16, 3),
    (9_001, 2_401, F16, 18),        # 3 waves, one row a workgroup
    (2_500, 1_021, F32, 3),         # 2 waves
    (1_100, 4_100, F32, 3),         # 9 waves: the form that loads a row anew
    (1_100, 8_192, F32, 3),         # 16 waves
    (1_100, 8_200, BF16, 3),
    (1_100, 4_099, F32, 3),
    (1_100, 8_203, F16, 3),
    (1_100_001, 3, F32, 3),         # narrower than a vector
    (1_100_001, 5, BF16, 3),
]


@pytest.mark.parametrize("rows,width,dtype,passes", LOOPS)
@pytest.mark.parametrize("residual", [False, True])
def test_several_rows_per_thread(rows, width, dtype, passes, residual):
    forward_and_backward(rows, width, dtype, residual, passes)


def test_each_row_of_a_loop_is_its_own():
    """A row's gradient does not depend on the rows that its threads took before it."""
    for rows, width, dtype in ((150_001, 32, F32), (20_001, 300, F32), (1_100, 4_100, F32), (1_100, 8_200, BF16)):
        x, r, w = make((rows, width), dtype, 1), make((rows, width), dtype, 2), 1.0 + 0.1 * make((width,), F32, 3)
        gy, gs = make((rows, width), dtype, 4), make((rows, width), dtype, 5)

        def ds(part):
            leaf = x[part].clone().requires_grad_(True)
            y, s = rms_norm(leaf, w, residual=r[part])
            return torch.autograd.grad((y, s), leaf, (gy[part], gs[part]))[0]

        whole = ds(slice(None))
        n = 1030 if width < 4000 else 300               # (few enough for one pass, enough for the same threads per row)
        for at in (0, rows // 2, rows - n):
            assert torch.equal(whole[at:at + n], ds(slice(at, at + n))), (rows, width, at)


# 64 MB and more per stream
STREAMS = [(600_001, 32, F32, 10), (280_001, 61, F32, 9), (56_001, 300, F32, 7), (17_000, 1_021, F32, 17), (4_200, 4_096, F32, 9), (4_200, 4_100, F32, 9),
           (2_100, 8_192, F32, 5), (530_001, 64, BF16, 9), (4_200, 8_200, BF16, 9), (4_200, 8_192, F16, 9), (4_200, 4_101, F32, 9), (4_200, 8_203, BF16, 9)]


@pytest.mark.parametrize("rows,width,dtype,passes", STREAMS)
@pytest.mark.parametrize("residual", [False, True])
def test_backward_past_the_caches(rows, width, dtype, passes, residual):
    assert rows * width * torch.finfo(dtype).bits // 8 >= 64 << 20
    forward_and_backward(rows, width, dtype, residual, passes)


def sample(rows):
    if rows < 1000:
        return torch.arange(rows, device="cuda")
    return torch.cat((torch.arange(500), torch.randint(0, rows, (3000,), generator=torch.Generator().manual_seed(7)), torch.arange(rows - 500, rows))).cuda()


# (rows, width, group, type): narrowed to half the threads with both vectors of a thread, a group as wide as the row's threads and not; several
# waves; four and eight vectors per thread; from 128 MB on past the caches
TABLES = [(600_001, 64, 32, F32), (600_001, 64, None, F32), (300_001, 192, 64, F32), (300_001, 200, None, F32), (540_001, 63, None, F32), (270_001, 128, 64, F32),
          (600_001, 64, 32, BF16), (1_100_000, 64, 32, BF16), (600_001, 96, 32, F16), (1_060_001, 65, None, BF16), (1_100, 260, None, F32), (1_100, 512, 128, F32),
          (140_001, 256, 128, F32), (2_100, 1000, None, BF16), (17_000, 4_096, 128, BF16), (16_500, 4_099, None, BF16), (7_000, 5_000, None, F32),
          (7_000, 5_001, None, F32), (3_600, 9_600, 64, F32), (3_600, 9_601, None, F32), (4_200, 16_512, 128, BF16), (12_000_001, 3, None, F32),
          (1_200_001, 32, None, F32), (9_000_000, 4, None, F32), (70_001, 61, None, F32), (80_001, 121, None, BF16), (6, 5_000, None, F32), (6, 5_001, None, F32),
          (6, 4_992, 64, F32), (6, 9_600, 64, F32), (6, 9_601, None, F32), (6, 10_001, None, BF16), (6, 9_984, 64, BF16), (6, 20_001, None, F16),
          (6, 19_968, 64, F16)]


@pytest.mark.parametrize("code", [torch.int8, E4M3])
@pytest.mark.parametrize("rows,width,group,dtype", TABLES)
def test_tables_of_many_rows(code, rows, width, group, dtype):
    print(f"case {code} {rows} {width} {group} {dtype}", flush=True)
    G = group or width
    x = make((rows, width), dtype, 1, 5.0)
    t = QuantizedRows.from_rows(x, dtype=code, group=group)
    at = sample(rows)
    want, top = encode_reference(x[at].float(), code, G)
    assert torch.equal(t.codes.view(torch.uint8)[at].view(code).double(), want)
    assert torch.equal(t.scales[at], (top / Q[code]).float())
    few = 900                                               # every row: the bits of a call of few rows, whose launch rule is another
    step = max(1, rows // 40)
    for k in range(0, rows - few, step):
        part = QuantizedRows.from_rows(x[k:k + few], dtype=code, group=group)
        assert torch.equal(t.codes[k:k + few].view(torch.uint8), part.codes.view(torch.uint8)) and torch.equal(t.scales[k:k + few], part.scales)
    v = (t.codes.float().reshape(rows, -1, G) * t.scales[:, :, None]).reshape(rows, width)
    for out in {F32, dtype}:
        assert torch.equal(t.read(out_dtype=out), v.to(out))
    n64 = v.double()
    n64 /= n64.norm(dim=1, keepdim=True) + 1e-6
    check(t.read(norm_eps=1e-6), n64, n64.abs() * (half(F32) + 20 * U) + floor_of(F32), "normalised")
    # the quantised norm: the same codes without a gain, scales with rstd; with a gain on the sample
    q = rms_norm_quantized(x, eps=1e-6, dtype=code, group=group)
    assert torch.equal(q.codes.view(torch.uint8), t.codes.view(torch.uint8))
    rstd = 1.0 / torch.sqrt(x.double().square().mean(1, keepdim=True) + 1e-6)
    check(q.scales, t.scales.double() * rstd, t.scales.double() * rstd * 20 * U, "scales")
    w = 1.0 + 0.3 * make((width,), F32, 3)
    q, s = rms_norm_quantized(x, w, 1e-6, residual=x, dtype=code, group=group)
    want, _ = encode_reference((x[at].float() + x[at].float()) * w, code, G)
    assert torch.equal(q.codes.view(torch.uint8)[at].view(code).double(), want)
    assert torch.equal(s, (x.float() + x.float()).to(dtype))
