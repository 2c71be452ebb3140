"""Row operators on the GPU against their definitions in 64 bits: the root-mean-square norm (forward, backward, 8-bit output) and the
8-bit row table.

Tolerances count roundings: u = 2^-24 is half a step of float32, half(T) half a step of the output's type.  A sum of squares goes through at
most 8 additions per thread, 3 over a vector, 6 over a wave and 8 over its waves: 25 u, and 2 u for s = x + residual; the mean and + eps add
2 u, and the root halves them: 14.5 u.  v_rsq_f32 adds 2 u, s itself u, two products 2 u: below 20 u of |y|, then one rounding to T."""
import math

import pytest
import torch

from instascene_amd.contrastive import gather_rows, row_normalize
from instascene_amd.rows import SCAN_MAX, QuantizedRows, rms_norm, rms_norm_quantized

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E4M3 = torch.float8_e4m3fn
Q = {torch.int8: 127.0, E4M3: 448.0}


def half(t):
    return torch.finfo(t).eps / 2


def floor_of(t):
    """Half the spacing of the type's smallest values."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def make(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def check(got, want, tol, name):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {bad.numel()}, worst {float((got.double() - want).abs()[bad].max())}"


# one column to long rows: below / at / above a vector, a wave, a workgroup, the registers (16 384 float32, 32 768 of 16 bits)
WIDTHS = [1, 3, 4, 8, 31, 32, 63, 64, 65, 255, 256, 1021, 1024, 2048, 2052, 2943, 4096, 4097, 6000, 8192, 8200, 9001, 16384, 16385, 33000]


def norm_reference(x, w, eps, r):
    s = x.double() if r is None else x.double() + r.double()
    rstd = 1.0 / torch.sqrt((s * s).mean(dim=1, keepdim=True) + eps)
    return s, rstd, s * rstd * (1.0 if w is None else w.double())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("rows,residual,gain", [(1, False, None), (5, True, F32), (67, True, "own")])
def test_rms_norm_forward_and_backward(dtype, width, rows, residual, gain):
    print(f"case {dtype} {width} {rows} {residual} {gain}", flush=True)
    eps = 1e-5
    x = make((rows, width), dtype, 1).requires_grad_(True)
    r = make((rows, width), dtype, 2, 3.0).requires_grad_(True) if residual else None
    w = None if gain is None else (1.0 + 0.5 * make((width,), F32, 3)).to(dtype if gain == "own" else gain).requires_grad_(True)
    got = rms_norm(x, w, eps, residual=r)
    y, s = got if residual else (got, None)
    with torch.no_grad():
        s64, rstd, y64 = norm_reference(x, w, eps, r)
        assert y.dtype == dtype and y.shape == x.shape
        check(y, y64, y64.abs() * (half(dtype) + 20 * U) + floor_of(dtype), "y")
        if residual:
            check(s, s64, s64.abs() * (half(dtype) + U) + floor_of(dtype), "s")
    gy, gs = make((rows, width), dtype, 4), make((rows, width), dtype, 5) if residual else None
    inputs = [t for t in (x, r, w) if t is not None]
    grads = torch.autograd.grad((y, s) if residual else y, inputs, (gy, gs) if residual else gy)
    grads = dict(zip([n for n, t in (("x", x), ("r", r), ("w", w)) if t is not None], grads))
    with torch.no_grad():
        h = s64 * rstd
        gw = gy.double() * (1.0 if w is None else w.double())
        mean = (gw * h).mean(dim=1, keepdim=True)
        ds = rstd * (gw - h * mean) + (gs.double() if residual else 0.0)
        # rstd is within 17 u, h within 19 u (below).  First term: rstd, gy w, the product, the difference, + gs: 21 u.  Second: rstd, h, and the
        # mean of gy w h (gy w: u, h: 19 u, a chain of 25 additions, 2 for the division): 17 + 19 + 47 + 4 = 87 u of the magnitudes
        noise = U * rstd * (22 * gw.abs() + 88 * h.abs() * (gw * h).abs().mean(dim=1, keepdim=True)) + (2 * U * gs.double().abs() if residual else 0.0)
        check(grads["x"], ds, noise + ds.abs() * half(dtype) + floor_of(dtype), "dx")
        if residual:
            check(grads["r"], ds, noise + ds.abs() * half(dtype) + floor_of(dtype), "dr")
        if w is not None:
            dw, size = (gy.double() * h).sum(dim=0), (gy.double() * h).abs().sum(dim=0)
            # every term 20 u (h, the product); a sum of n terms in any order n u of the magnitudes
            check(grads["w"], dw, size * (rows + 20) * U + dw.abs() * half(w.dtype) + floor_of(w.dtype), "dw")


def test_rms_norm_gradient_against_differences():
    """Central differences of the 64-bit definition along random directions."""
    x, r, w = make((9, 40), F32, 1), make((9, 40), F32, 2), 1.0 + 0.1 * make((40,), F32, 3)
    gy, gs = make((9, 40), F32, 4), make((9, 40), F32, 5)
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, s = rms_norm(leaves[0], leaves[2], 1e-6, residual=leaves[1])
    grads = torch.autograd.grad((y, s), leaves, (gy, gs))

    def value(a, b, c):
        s64, _, y64 = norm_reference(a, c, 1e-6, b)
        return float((y64 * gy.double()).sum() + (s64 * gs.double()).sum())

    base = [t.double() for t in (x, r, w)]
    for k in range(3):
        d = make(base[k].shape, F32, 10 + k).double()
        step = 1e-5
        up, down = list(base), list(base)
        up[k], down[k] = base[k] + step * d, base[k] - step * d
        slope = (value(*up) - value(*down)) / (2 * step)
        assert abs(float((grads[k].double() * d).sum()) - slope) <= 1e-5 * max(1.0, abs(slope))


def test_rms_norm_backward_long_sums_and_partial_gradients():
    """Many rows (several per thread), gradients of single inputs, of the sum alone, of the output alone."""
    x, r = make((30001, 32), F32, 1).requires_grad_(True), make((30001, 32), F32, 2)
    w = torch.ones(32, device="cuda").requires_grad_(True)
    gy = make((30001, 32), F32, 3)
    y, s = rms_norm(x, w, 1e-6, residual=r)
    dw, = torch.autograd.grad(y, w, gy, retain_graph=True)
    dx, = torch.autograd.grad(y, x, gy, retain_graph=True)
    both = torch.autograd.grad(y, (x, w), gy)
    assert torch.equal(dw, both[1]) and torch.equal(dx, both[0])
    s64, rstd, _ = norm_reference(x.detach(), None, 1e-6, r)
    h = s64 * rstd
    check(dw, (gy.double() * h).sum(0), (gy.double() * h).abs().sum(0) * 512 * U, "dw")   # <= 30001 / 2048 / 32 + 4 + 2048 / 8 + 8 terms in turn
    y, s = rms_norm(x, w, 1e-6, residual=r)
    assert torch.equal(torch.autograd.grad(s, x, gy)[0], gy)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width", [3, 100, 4100, 20003])
def test_rms_norm_gradients_of_one_input_at_a_time(dtype, width):
    """Each gradient alone has the bits it has beside the others; an expanded incoming gradient; 64 rows per partial sum and more."""
    x, r, w = make((150, width), dtype, 1), make((150, width), dtype, 2), 1.0 + 0.1 * make((width,), F32, 3)
    gy = make((150, width), dtype, 4)

    def grads(*wanted):
        leaves = [t.clone().requires_grad_(k in wanted) for k, t in enumerate((x, r, w))]
        y, _ = rms_norm(leaves[0], leaves[2], 1e-6, residual=leaves[1])
        return dict(zip(wanted, torch.autograd.grad(y, [leaves[k] for k in wanted], gy)))

    whole = grads(0, 1, 2)
    assert torch.equal(whole[0], whole[1])
    for k in range(3):
        assert torch.equal(grads(k)[k], whole[k])
    leaf = x.clone().requires_grad_(True)
    rms_norm(leaf, w).sum().backward()                      # (a gradient of one element, expanded)
    again, = torch.autograd.grad(rms_norm(leaf, w), leaf, torch.ones_like(x))
    assert torch.equal(leaf.grad, again)
    for incoming in (gy, gy.clone().requires_grad_(True)):
        g, = torch.autograd.grad(rms_norm(leaf, w), leaf, incoming, create_graph=True)
        assert torch.equal(g, torch.autograd.grad(rms_norm(leaf, w), leaf, gy)[0])
        with pytest.raises(RuntimeError, match="backward pass"):
            g.sum().backward()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rms_norm_strides_views_and_shared_inputs(dtype):
    base = make((40, 3, 130), dtype, 1)
    x = base[:, 1, 1:128]                                  # rows 390 apart, starting at an odd element
    assert not x.is_contiguous()
    assert torch.equal(rms_norm(x), rms_norm(x.contiguous()))
    assert torch.equal(rms_norm(x, residual=x)[1], (x.float() + x.float()).to(dtype))
    t = make((127, 40), dtype, 2).T                        # columns are not next to each other
    assert torch.equal(rms_norm(t), rms_norm(t.contiguous()))
    assert torch.equal(rms_norm(base), rms_norm(base.reshape(-1, 130)).reshape(base.shape))
    one = make((1, 130), dtype, 3).requires_grad_(True)    # a row shared by all
    wide = one.expand(40, 130)
    gy = make((40, 130), dtype, 4)
    dx, = torch.autograd.grad(rms_norm(wide), one, gy)
    assert dx.shape == one.shape
    flat = one.detach().double().repeat(40, 1).requires_grad_(True)
    y64 = flat / torch.sqrt((flat * flat).mean(1, keepdim=True) + 1e-6)
    want = torch.autograd.grad(y64, flat, gy.double())[0]
    # 40 gradients, each rounded to T, summed by torch to T
    check(dx[0], want.sum(0), want.abs().sum(0) * 4 * half(dtype) + 1e-4 * half(dtype) + 40 * 60 * U, "dx of a shared row")
    # strided incoming gradients, incl. an expanded one
    leaf = make((40, 130), dtype, 5).requires_grad_(True)
    a = torch.autograd.grad(rms_norm(leaf), leaf, gy[:1].expand(40, 130))[0]
    b = torch.autograd.grad(rms_norm(leaf), leaf, gy[:1].repeat(40, 1))[0]
    assert torch.equal(a, b)


def test_rms_norm_empty_extreme_and_non_finite_rows():
    assert rms_norm(torch.empty(0, 7, device="cuda")).shape == (0, 7)
    w = torch.ones(7, device="cuda", requires_grad=True)
    x0 = torch.empty(0, 7, device="cuda", requires_grad=True)
    dx, dw = torch.autograd.grad(rms_norm(x0, w), (x0, w), torch.empty(0, 7, device="cuda"))
    assert dx.shape == (0, 7) and torch.equal(dw, torch.zeros(7, device="cuda"))
    for dtype in (F32, BF16):
        big = torch.finfo(dtype).max
        x = torch.tensor([[big, -big, big, -big], [-big, 1.0, 0.0, 0.0], [0.0] * 4, [1e-30, 0, 0, 0]], device="cuda").to(dtype)
        y = rms_norm(x, eps=1e-6).double()
        want = norm_reference(x, None, 1e-6, None)[2]
        check(y, want, want.abs() * (half(dtype) + 20 * U) + floor_of(dtype), "extreme rows")
    x = torch.ones(3, 300, device="cuda")
    x[0, 7], x[1, 9] = float("inf"), float("nan")
    y = rms_norm(x)
    assert bool(torch.isnan(y[0, 7])) and bool((y[0, :7] == 0).all()) and bool(torch.isnan(y[1]).all()) and bool((y[2] - 1).abs().max() < 1e-6)


# ---- 8 bits ------------------------------------------------------------------------------------------------------------------------
def nearest_code(value, dtype):
    """The value of the 8-bit type next to ``value`` (float64), ties to even."""
    if dtype == torch.int8:
        return value.round()
    _, e = torch.frexp(value.cpu())
    unit = torch.ldexp(torch.ones((), dtype=torch.float64), e.clamp(min=-5) - 4).to(value.device)       # (powers of two: exact on the CPU)
    return (value / unit).round() * unit


def encode_reference(t, dtype, group):
    """Values of the codes and top of every group of float32 rows ``t``; the quotient t Q / top in 64 bits (a tie comes out as a tie)."""
    n, F = t.shape
    v = t.double().reshape(n, F // group, group)
    top = v.abs().amax(dim=2, keepdim=True)
    dead = top < 2.0 ** -116
    codes = nearest_code(v * Q[dtype] / torch.where(dead, torch.ones_like(top), top), dtype)
    return torch.where(dead, torch.zeros_like(codes), codes).reshape(n, F), torch.where(dead, torch.zeros_like(top), top).squeeze(2)


@pytest.mark.parametrize("code", [torch.int8, E4M3])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,width,group", [(1, 32, None), (3, 5, None), (7, 64, 32), (33, 1023, None), (5, 4096, 128), (300, 192, 64), (2, 16512, 128), (2, 33001, None), (3, 40960, 32)])
def test_rms_norm_quantized(code, dtype, rows, width, group):
    print(f"case {code} {dtype} {rows} {width} {group}", flush=True)
    x, r = make((rows, width), dtype, 1), make((rows, width), dtype, 2)
    w = 1.0 + 0.3 * make((width,), F32, 3)
    q, s = rms_norm_quantized(x, w, 1e-6, residual=r, dtype=code, group=group)
    assert torch.equal(s, (x.float() + r.float()).to(dtype))
    t = (x.float() + r.float()) * w                          # the kernel's own two roundings: the codes are then exact
    want, top = encode_reference(t, code, group or width)
    assert torch.equal(q.codes.double(), want)
    _, rstd, _ = norm_reference(x, w, 1e-6, r)
    scales = top * rstd / Q[code]
    check(q.scales, scales, scales * 20 * U, "scales")
    assert q.group == (group or width) and len(q) == rows
    # without gain and residual the same codes as the rows' own
    plain = rms_norm_quantized(x, dtype=code, group=group)
    assert torch.equal(plain.codes.double(), encode_reference(x.float(), code, group or width)[0])


@pytest.mark.parametrize("code", [torch.int8, E4M3])
def test_codes_of_ties_and_borders(code):
    """Quotients on the border between two codes, one float32 step to either side, all codes, zeros, the smallest group."""
    q = Q[code]
    every = torch.arange(-127, 128, device="cuda").double() if code == torch.int8 else \
        torch.arange(0, 0x7f, device="cuda", dtype=torch.uint8).view(E4M3).double()
    ties = ((every[1:] + every[:-1]) / 2)
    for top in (q, 1.0, 3.7e-3, 1.1754944e-35, 2.9e38):
        v = torch.cat((every, ties)) * (top / q)
        v = torch.cat((v, torch.nextafter(v.float(), torch.full_like(v, 1e38).float()).double(),
                       torch.nextafter(v.float(), torch.full_like(v, -1e38).float()).double())).float()
        v = v[v.abs() <= top]
        v = torch.cat((v, torch.tensor([top], device="cuda", dtype=F32)))
        t = QuantizedRows.from_rows(v[None], dtype=code)
        want, tops = encode_reference(v[None], code, v.numel())
        assert torch.equal(t.codes.double(), want), top
        assert torch.equal(t.scales, (tops / q).float())         # (in 64 bits: torch divides by a scalar with its reciprocal)


def test_table_groups_that_cannot_be_scaled():
    x = torch.zeros(5, 64, device="cuda")
    x[1, 3], x[2, 40], x[3, 5], x[4, 0] = float("inf"), float("nan"), 1e-36, -float("inf")
    x[1:5, 50] = 1.0
    for code in (torch.int8, E4M3):
        t = QuantizedRows.from_rows(x, dtype=code, group=32)
        v = t.read()
        assert bool((v[0] == 0).all()) and bool((v[3, :32] == 0).all()) and float(v[3, 50]) == 1.0
        assert bool(torch.isnan(v[1, :32]).all()) and float(v[1, 50]) == 1.0
        assert bool((v[2, :32] == 0).all()) and bool(torch.isnan(v[2, 32:]).all())
        assert bool(torch.isnan(v[4, :32]).all())


@pytest.mark.parametrize("code", [torch.int8, E4M3])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width,group", [(1, None), (7, None), (32, None), (32, 32), (64, 32), (129, None), (1024, 128), (20000, None), (36864, 64)])
def test_table_whole(code, dtype, width, group):
    print(f"case {code} {dtype} {width} {group}", flush=True)
    x = make((53, width), dtype, 1, 5.0)
    t = QuantizedRows(53, width, dtype=code, group=group)
    assert bool((t.read() == 0).all())
    t.write(x)
    want, top = encode_reference(x.float(), code, group or width)
    assert torch.equal(t.codes.double(), want)
    assert torch.equal(t.scales, (top / Q[code]).float())
    v = (t.codes.float().reshape(53, -1, group or width) * t.scales[:, :, None]).reshape(53, width)
    for out in (F32, BF16, F16):
        assert torch.equal(t.read(out_dtype=out), v.to(out))
        n64 = v.double() / (v.double().norm(dim=1, keepdim=True) + 1e-6)
        # half of the sum's 25 u, the root (2 u), + eps (u), the reciprocal (2 u), the product (u)
        check(t.read(out_dtype=out, norm_eps=1e-6), n64, n64.abs() * (half(out) + 20 * U) + floor_of(out), "normalised")


@pytest.mark.parametrize("n", [1, 2, 37, SCAN_MAX, SCAN_MAX + 1, 5000])
@pytest.mark.parametrize("itype", [torch.int64, torch.int32])
@pytest.mark.parametrize("width", [24, 1000])
def test_table_write_by_index_keeps_the_last_and_leaves_the_rest(n, itype, width):
    P = 700
    g = torch.Generator().manual_seed(n)
    first = make((P, width), F32, 1)
    for pad in (False, True):
        t = QuantizedRows(P, width, dtype=torch.int8).write(first)
        before = t.read()
        ix = torch.randint(0, P, (n,), generator=g)
        if pad:                                            # a padded batch: indices outside the table
            ix[torch.rand(n, generator=g) < 0.3] = -1
            ix[0] = P
            ix[-1] = -(2 ** 31)
        new = make((n, width), F32, 2)
        t.write(new, ix.to(itype).cuda())
        want = before.clone()
        fresh = QuantizedRows.from_rows(new, dtype=torch.int8).read()
        for k, r in enumerate(ix.tolist()):
            if 0 <= r < P:
                want[r] = fresh[k]
        assert torch.equal(t.read(), want)
        assert bool((t._owner == -1).all())
        got = t.read(ix.to(itype).cuda(), norm_eps=0.0 if not pad else None)
        valid = ((ix >= 0) & (ix < P)).cuda()
        rows = want[ix.clamp(0, P - 1).cuda()]
        if pad:
            assert torch.equal(got, torch.where(valid[:, None], rows, torch.zeros_like(rows)))
        assert torch.equal(gather_rows(t, ix.to(itype).cuda()), torch.where(valid[:, None], rows, torch.zeros_like(rows)))


def test_table_ranges_strides_and_state():
    t = QuantizedRows(100, 48, dtype=E4M3)
    x = make((30, 200), BF16, 1)
    t.write(x[:, 3:51], 60)
    full = t.read()
    assert bool((full[:60] == 0).all()) and bool((full[90:] == 0).all())
    assert torch.equal(full[60:90], QuantizedRows.from_rows(x[:, 3:51].contiguous()).read())
    assert torch.equal(t.read(slice(58, 75)), full[58:75]) and t.read(slice(90, 10)).shape == (0, 48)
    t.write(x[:0, 3:51], 100)
    t.write(x[:0, 3:51], torch.empty(0, dtype=torch.int64, device="cuda"))
    assert t.read(torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 48)
    u = QuantizedRows(100, 48, dtype=E4M3)
    u.load_state_dict(t.state_dict())
    assert torch.equal(u.read(), full) and u.nbytes == 100 * 48 + 400
    assert QuantizedRows(0, 8).read().shape == (0, 8)
    empty = QuantizedRows(0, 8)
    ix = torch.tensor([0, -1], device="cuda")
    empty.write(torch.ones(2, 8, device="cuda"), ix)
    assert bool((empty.read(ix) == 0).all())
    # an invalid row is zero also where a zero row has no direction
    assert bool((t.read(torch.tensor([-1], device="cuda"), norm_eps=0.0) == 0).all())


def test_one_row_without_a_row_dimension_and_other_index_forms():
    import numpy as np
    x = make((300,), BF16, 1)
    assert torch.equal(rms_norm(x), rms_norm(x[None])[0])
    leaf = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(rms_norm(leaf), leaf, x)
    deep = x[None, None].clone().requires_grad_(True)
    d3, = torch.autograd.grad(rms_norm(deep), deep, x[None, None])
    assert dx.shape == (300,) and torch.equal(dx, d3[0, 0])
    t = QuantizedRows(9, 300, dtype=torch.int8)
    t.write(x[None], np.int64(4))
    assert torch.equal(t.read(slice(4, 5)), QuantizedRows.from_rows(x[None], dtype=torch.int8).read()) and bool((t.read(slice(5, 9)) == 0).all())
    every_second = torch.arange(18, device="cuda")[::2]                     # an index with a stride
    assert torch.equal(t.read(every_second.flip(0)), torch.cat((torch.zeros(4, 300, device="cuda"), t.read(every_second.flip(0)[4:]))))
    assert torch.equal(t.read(every_second)[2], t.read(slice(4, 5))[0])
    with pytest.raises(TypeError):
        t.write(x[None], 4.0)


def test_offsets_beyond_32_bits():
    """More than 2^32 code bytes, more than 2^31 elements of a norm."""
    P, F = 68_000_000, 64
    t = QuantizedRows(P, F, dtype=torch.int8)
    ix = torch.tensor([P - 1, 0, P - 2, 2 ** 26 + 1], device="cuda")
    x = make((4, F), F32, 1)
    t.write(x, ix)
    assert torch.equal(t.read(ix), QuantizedRows.from_rows(x, dtype=torch.int8).read())
    assert torch.equal(t.read(slice(P - 2, P)), t.read(ix[[2, 0]]))
    t.write(x[:2], P - 2)
    assert torch.equal(t.read(slice(P - 2, P)), QuantizedRows.from_rows(x[:2], dtype=torch.int8).read())
    del t
    n, F = 1_100_000, 2048
    a = torch.zeros(n, F, dtype=BF16, device="cuda")
    a[-3:] = make((3, F), BF16, 2)
    y = rms_norm(a)
    assert torch.equal(y[-3:], rms_norm(a[-3:].clone()))
    del y
    torch.cuda.empty_cache()


# ---- streams, graphs, devices ------------------------------------------------------------------------------------------------------
def test_captured_and_replayed():
    """Forward, backward, quantised norm, indexed write (both forms) and read in one graph; replays on new inputs equal the eager run."""
    N, F, P = 600, 96, 5000
    x, r, gy, gs = (make((N, F), BF16, k) for k in range(4))
    w = 1.0 + 0.1 * make((F,), F32, 9)
    ix = torch.randint(0, P, (N,), device="cuda")
    few = torch.tensor([3, 3, 4999, -1], device="cuda")

    def work(table):
        xa, ra, wa = (t.detach().requires_grad_(True) for t in (x, r, w))
        y, s = rms_norm(xa, wa, 1e-6, residual=ra)
        grads = torch.autograd.grad((y, s), (xa, ra, wa), (gy, gs))
        q, _ = rms_norm_quantized(x, w, 1e-6, residual=r, dtype=torch.int8, group=32)
        table.write(y.detach(), ix)
        table.write(s.detach()[:4], few)
        return [y.detach(), s.detach(), *grads, q.codes, q.scales, table.read(ix, norm_eps=1e-6), table.read(few)]

    cached, eager = QuantizedRows(P, F), QuantizedRows(P, F)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(cached)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(cached)
    for k in range(4):
        for t, seed in ((x, 20), (r, 21), (gy, 22), (gs, 23)):
            t.copy_(make((N, F), BF16, seed + 10 * k))
        ix.copy_(torch.randint(0, P, (N,), device="cuda"))
        few.copy_(torch.tensor([k, 7, k, 8], device="cuda"))
        graph.replay()
        got = [t.clone() for t in out]
        if k % 2:
            torch.cuda.synchronize()
        for a, b in zip(got, work(eager)):
            assert torch.equal(a, b)
    assert torch.equal(cached._owner, eager._owner) and bool((cached._owner == -1).all())


def test_two_streams_write_disjoint_rows():
    P, F, n = 40000, 32, 9000
    order = torch.randperm(P, device="cuda")
    a, b = order[:n], order[n:2 * n]
    xa, xb = make((n, F), F32, 1), make((n, F), F32, 2)
    t = QuantizedRows(P, F, dtype=torch.int8)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(s1):
            t.write(xa, a)
        with torch.cuda.stream(s2):
            t.write(xb, b)
    torch.cuda.synchronize()
    assert torch.equal(t.read(a), QuantizedRows.from_rows(xa, dtype=torch.int8).read())
    assert torch.equal(t.read(b), QuantizedRows.from_rows(xb, dtype=torch.int8).read())


def test_same_inputs_same_bits():
    x, w = make((20000, 48), BF16, 1).requires_grad_(True), torch.ones(48, device="cuda", requires_grad=True)
    gy = make((20000, 48), BF16, 2)
    first = torch.autograd.grad(rms_norm(x, w), (x, w), gy)
    for _ in range(3):
        again = torch.autograd.grad(rms_norm(x, w), (x, w), gy)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_refusals_on_the_device():
    x = torch.ones(4, 64, device="cuda")
    for call, error in [
            (lambda: rms_norm(x, torch.ones(63, device="cuda")), ValueError),
            (lambda: rms_norm(x, torch.ones(64)), ValueError),
            (lambda: rms_norm(x, torch.ones(64, device="cuda", dtype=F16)), TypeError),
            (lambda: rms_norm(x, residual=x[:2]), ValueError),
            (lambda: rms_norm(x, residual=x.half()), ValueError),
            (lambda: rms_norm(x, eps=0.0), ValueError),
            (lambda: rms_norm(x, eps=float("nan")), ValueError),
            (lambda: rms_norm(x.double()), TypeError),
            (lambda: rms_norm(torch.empty(3, 0, device="cuda")), ValueError),
            (lambda: rms_norm_quantized(x, group=48), ValueError),
            (lambda: rms_norm_quantized(x[:, :63], group=32), ValueError),
            (lambda: rms_norm_quantized(x, dtype=torch.uint8), TypeError),
            (lambda: rms_norm_quantized(x[0]), ValueError),
            (lambda: rms_norm_quantized(x.clone().requires_grad_(True)), RuntimeError),
            (lambda: QuantizedRows(4, 64).write(x, 1), ValueError),
            (lambda: QuantizedRows(4, 64).write(x, -1), ValueError),
            (lambda: QuantizedRows(5, 64).write(x), ValueError),
            (lambda: QuantizedRows(4, 32).write(x), ValueError),
            (lambda: QuantizedRows(4, 64).write(x, torch.arange(3, device="cuda")), ValueError),
            (lambda: QuantizedRows(4, 64).write(x, torch.arange(4)), ValueError),
            (lambda: QuantizedRows(4, 64).write(x, torch.ones(4, device="cuda")), ValueError),
            (lambda: QuantizedRows(4, 64).read(torch.ones(4, 1, device="cuda", dtype=torch.int64)), ValueError),
            (lambda: QuantizedRows(4, 64).read(slice(0, 4, 2)), ValueError),
            (lambda: QuantizedRows(4, 64).read(out_dtype=torch.float64), TypeError),
            (lambda: QuantizedRows(4, 64).read(norm_eps=-1.0), ValueError)]:
        with pytest.raises(error):
            call()
    with torch.no_grad():
        rms_norm_quantized(x.clone().requires_grad_(True))


# ---- together, as they are used -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("code,group", [(E4M3, None), (torch.int8, None), (E4M3, 32)])
def test_a_trained_table_in_8_bits_renders(code, group):
    """SegGaussianModel.compact_features: the render of the 8-bit table is the render of the values it stands for."""
    from instascene_amd import rasterizer as rz
    from instascene_amd import scenes
    from instascene_amd.harness import PipelineParams, SegGaussianModel
    from instascene_amd.render import render
    rz.set_mode("exact")
    sc = scenes.synthetic_scene(3000, 32, 5, math.log(0.04))
    cam = scenes.ring_cameras(6, 128, 96)[0].to("cuda")
    bg = torch.zeros(3, device="cuda")
    with torch.no_grad():
        m, plain = SegGaussianModel(sc, "cuda"), SegGaussianModel(sc, "cuda")
        full = render(cam, plain, PipelineParams(), bg)["seg_feature"]
        rows = row_normalize(plain._seg_feature, 1e-6)
        table = m.compact_features(code, group)
        assert m.get_seg_feature is table and table.nbytes * 3 < plain._seg_feature.nbytes
        got = render(cam, m, PipelineParams(), bg)["seg_feature"]
        plain._seg_feature = torch.nn.Parameter(table.read())
        plain._seg_cache = None
        want = render(cam, plain, PipelineParams(), bg)["seg_feature"]
        # the plain model normalises once more (getter, eps 1e-6; render, eps 1e-9): 1e-6 of the value
        assert bool(((got - want).abs() <= 4e-6).all())
        # the codes are half a step off: 2^-4 relative (e4m3), a 254th of the row's largest (int8), on rows of length 1
        step = 2.0 ** -4 if code == E4M3 else 1.0 / 254
        assert float((got - full).norm() / full.norm()) <= 2 * step
        assert torch.equal(gather_rows(m.get_seg_feature, torch.arange(9, device="cuda")), table.read(slice(0, 9)))
        check(table.read(), rows.double(), (step if code == E4M3 else step * rows.double().abs().amax(1, keepdim=True)) * (rows.double().abs() if code == E4M3 else 1.0)
              + 2.0 ** -10 * rows.double().abs().amax(1, keepdim=True) / 448 + 4 * U, "codes")
        with pytest.raises(RuntimeError):
            m.compact_features()


def test_a_trainer_hands_out_its_compacted_features_in_input_order():
    from instascene_amd import scenes
    from instascene_amd.harness import SegTrainer
    sc = scenes.synthetic_scene(2000, 16, 5, math.log(0.04))
    t = SegTrainer(sc, scenes.ring_cameras(6, 96, 64), device="cuda", sample_batchsize=512, n_labels=8, use_class_feat=True, seed=3)
    t.step(0)
    want = row_normalize(t.features_in_input_order(), 1e-6)
    t.model.compact_features(torch.int8)
    check(t.features_in_input_order(), want.double(), want.double().abs().amax(1, keepdim=True) * (0.5 / 127 + 4 * U), "input order")


def test_a_residual_table_is_trained_clipped_and_put_away():
    """All of it together, as a program uses it: a frozen base table and a trained one, rms_norm of their sum with a learned gain, the
    contrastive loss on gathered rows, the gradients clipped together, the steps; then the trained rows in 8 bits and read back by index.
    Every piece against the same step in 64 bits."""
    from instascene_amd.contrastive import contrastive_loss
    from instascene_amd.optim import clip_grad_norm_
    P, F, n = 3000, 32, 1024
    base = make((P, F), F32, 1)
    delta = torch.nn.Parameter(0.1 * make((P, F), F32, 2))
    gain = torch.nn.Parameter(1.0 + 0.1 * make((F,), F32, 3))
    labels = torch.randint(1, 9, (P,), device="cuda")
    opt = torch.optim.SGD([delta, gain], lr=1.0)
    for step in range(3):
        pick = torch.randint(0, P, (n,), device="cuda")
        opt.zero_grad()
        y, s = rms_norm(delta, gain, 1e-6, residual=base)
        (contrastive_loss(y[pick], labels[pick], num_labels=9) + 1e-3 * s.square().sum()).backward()
        with torch.enable_grad():
            d64, g64 = delta.detach().double().requires_grad_(True), gain.detach().double().requires_grad_(True)
            s64 = d64 + base.double()
            y64 = s64 / torch.sqrt(s64.square().mean(1, keepdim=True) + 1e-6) * g64
            leaf = y.detach()[pick].requires_grad_(True)                   # the loss' own gradient at y
            gl, = torch.autograd.grad(contrastive_loss(leaf, labels[pick], num_labels=9), leaf)
            gy = torch.zeros(P, F, dtype=torch.float64, device="cuda").index_add_(0, pick, gl.double())
            want = torch.autograd.grad((y64 * gy).sum() + 1e-3 * s64.square().sum(), (d64, g64))
        norm = math.sqrt(sum(float(w.square().sum()) for w in want))
        before = delta.detach().clone()
        got = clip_grad_norm_([delta, gain], 0.5 * norm)
        assert abs(float(got) - norm) <= 1e-5 * norm
        coef = 0.5 * norm / (norm + 1e-6)
        for p, w in ((delta, want[0]), (gain, want[1])):
            assert float((p.grad.double() - coef * w).norm()) <= 1e-5 * float((coef * w).norm())
        opt.step()
        assert torch.equal(delta, before - delta.grad)
    with torch.no_grad():
        q, s = rms_norm_quantized(delta, gain, 1e-6, residual=base, dtype=torch.int8)
        y = rms_norm(delta, gain, 1e-6, residual=base)[0]
        top = y.abs().amax(1, keepdim=True)
        check(q.read(), y.double(), top.double() * (0.5 / 127 + 60 * U), "8 bits")        # half a step of the row's largest / 127
        table = QuantizedRows(P, F, dtype=torch.int8)
        order = torch.randperm(P, device="cuda")
        table.write(y[order], order)
        check(table.read(), y.double(), top.double() * (0.5 / 127 + 60 * U), "written by index")
        assert torch.equal(gather_rows(table, order[:n]), table.read()[order[:n]])
        check(gather_rows(table, order[:n]).norm(dim=1), y[order[:n]].double().norm(dim=1), top[order[:n], 0].double() * math.sqrt(F) * 0.6 / 127, "lengths")
