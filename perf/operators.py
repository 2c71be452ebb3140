"""Measured cases of the row and gradient operators: root-mean-square norm of rows (with the residual's addition, its backward
pass and an 8-bit output), the 8-bit row table (written and read back), and the global gradient norm with clipping.

``own`` selects the framework's kernels; otherwise every operator runs in its plain form, elementary torch operations in 32 bits
rounded once at the end."""
import math
import random

import torch

own = False

EPS = 1e-6          # of the root-mean-square norm
NORM_EPS = 1e-6     # of the feature getter's row normalisation
QMAX = {"e4m3": 448.0, "int8": 127.0}
TINY = 2.0 ** -116  # a group whose largest magnitude lies below is stored as zeros
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def listed():
    return [
        # one new token's activation on its way into the next layer: latency alone counts
        dict(name="norm_token", op="norm", rows=1, width=4096, dtype="bf16", residual=True, backward=False),
        # an odd width and an odd number of rows: no row starts on a vector boundary
        dict(name="norm_ragged", op="norm", rows=2047, width=1021, dtype="fp16", residual=True, backward=True),
        # the feature table of the 1.5 M Gaussian scene, a frozen base plus the trained table, one training step
        dict(name="norm_table", op="norm", rows=1_500_000, width=32, dtype="fp32", residual=True, backward=True),
        # wide activations of a training step
        dict(name="norm_wide", op="norm", rows=8192, width=8192, dtype="bf16", residual=True, backward=True),
        # a few sequences that decode together, the 8-bit operand of the product that follows
        dict(name="quant_token", op="quant", rows=8, width=5120, dtype="bf16", residual=True, group=0),
        # a long prompt, scales in groups of 128
        dict(name="quant_prompt", op="quant", rows=16384, width=4096, dtype="bf16", residual=True, group=128),
        # one token's entry (8 heads of 128) appended to a cache and one read
        dict(name="cache_token", op="cache", table=65536, width=1024, dtype="bf16", code="e4m3", group=128, write=1, read=1, norm=False),
        # a training batch's rows of the 1.5 M Gaussian table, with repeated rows, read back normalised
        dict(name="cache_batch", op="cache", table=1_500_000, width=32, dtype="fp32", code="int8", group=0, write=8192, read=8192, norm=True),
        # the 5 M Gaussian table put away whole in 8 bits and read back whole for a render
        dict(name="cache_table", op="cache", table=5_000_000, width=64, dtype="fp32", code="e4m3", group=32, write=0, read=0, norm=True),
        # the norm of a small model's gradients, for a log line
        dict(name="gradnorm_small", op="gradnorm", layout="gaussians", rows=1000, tensors=6, largest=0, mixed=False, clip=False),
        # the six parameter groups of 300 k Gaussians, clipped in place
        dict(name="clip_gaussians", op="gradnorm", layout="gaussians", rows=300_000, tensors=6, largest=0, mixed=False, clip=True),
        # many tensors of three types and of every size, views of one bucket per type
        dict(name="clip_many", op="gradnorm", layout="ragged", rows=0, tensors=260, largest=4_000_000, mixed=True, clip=True),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(("norm", "quant", "cache", "gradnorm"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    if op == "norm":
        width = _log(rng, 4, 20000)
        return dict(op=op, rows=_log(rng, 1, min(3_000_000, (1 << 25) // width)), width=width, dtype=dtype,
                    residual=rng.random() < 0.7, backward=rng.random() < 0.6)
    if op == "quant":
        group = rng.choice((0, 32, 64, 128))
        width = _log(rng, 4, 20000) if group == 0 else group * _log(rng, 1, 16384 // group)
        return dict(op=op, rows=_log(rng, 1, min(3_000_000, (1 << 25) // width)), width=width, dtype=dtype,
                    residual=rng.random() < 0.7, group=group)
    if op == "cache":
        group = rng.choice((0, 32, 64, 128))
        width = _log(rng, 4, 4096) if group == 0 else group * _log(rng, 1, 4096 // group)
        table = _log(rng, 64, min(3_000_000, (1 << 27) // width))
        whole = rng.random() < 0.3
        most = min(table, (1 << 25) // width)
        return dict(op=op, table=table, width=width, dtype=dtype, code=rng.choice(("e4m3", "int8")), group=group,
                    write=0 if whole else _log(rng, 1, most), read=0 if whole else _log(rng, 1, most), norm=rng.random() < 0.5)
    if rng.random() < 0.4:
        return dict(op=op, layout="gaussians", rows=_log(rng, 100, 1_000_000), tensors=6, largest=0, mixed=False, clip=rng.random() < 0.6)
    return dict(op=op, layout="ragged", rows=0, tensors=_log(rng, 1, 300), largest=_log(rng, 1000, 3_000_000), mixed=rng.random() < 0.6,
                clip=rng.random() < 0.6)


def _sizes(case):
    """Numbers of elements and types of a gradient case's tensors."""
    if case["layout"] == "gaussians":       # xyz, f_dc, f_rest (degree 3), opacity, scaling, rotation
        return [(case["rows"] * k, "fp32") for k in (3, 3, 45, 1, 2, 4)]
    r = random.Random(case["tensors"] * 7919 + case["largest"])
    sizes = [(_log(r, 1, case["largest"]), r.choice(("fp32", "bf16", "fp16")) if case["mixed"] else "fp32") for _ in range(case["tensors"])]
    sizes[0] = (case["largest"], sizes[0][1])
    return sizes


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(shape, dtype, scale=1.0):
        return (torch.randn(shape, generator=gen, device=dev) * scale).to(dtype)

    if case["op"] in ("norm", "quant"):
        dt, shape = TYPES[case["dtype"]], (case["rows"], case["width"])
        st = dict(case=case, x=normal(shape, dt), weight=1.0 + 0.2 * torch.randn(case["width"], generator=gen, device=dev),
                  residual=normal(shape, dt, 2.0) if case["residual"] else None)
        if case.get("backward"):
            st["x"].requires_grad_(True)
            st["weight"].requires_grad_(True)
            st["gy"] = normal(shape, dt)
            if case["residual"]:
                st["residual"].requires_grad_(True)
                st["gs"] = normal(shape, dt)
        return st
    if case["op"] == "cache":
        dt, P, F = TYPES[case["dtype"]], case["table"], case["width"]
        n_w, n_r = case["write"] or P, case["read"] or P
        st = dict(case=case, rows=normal((n_w, F), dt),
                  to=None if case["write"] == 0 else torch.randint(0, P, (n_w,), generator=gen, device=dev),
                  at=None if case["read"] == 0 else torch.randint(0, P, (n_r,), generator=gen, device=dev))
        if case["read"] != 0:       # a few of the rows that are read were written by the same pass
            k = min(n_w, (n_r + 1) // 2)
            st["at"][:k] = st["to"][:k]
        if own:
            from instascene_amd.rows import QuantizedRows
            st["cache"] = QuantizedRows(P, F, dtype=CODES[case["code"]], group=case["group"] or None, device=dev)
        else:
            st["codes"] = torch.zeros((P, F), device=dev, dtype=CODES[case["code"]])
            st["scales"] = torch.zeros((P, F // (case["group"] or F)), device=dev)
        return st
    sizes = _sizes(case)
    st = dict(case=case, flat={}, fresh={}, grads=[])
    for t in sorted({t for _, t in sizes}):
        st["fresh"][t] = normal((sum(n for n, u in sizes if u == t),), TYPES[t], 0.01)
        st["flat"][t] = st["fresh"][t].clone()
    at = dict.fromkeys(st["flat"], 0)
    for n, t in sizes:
        st["grads"].append(st["flat"][t][at[t]:at[t] + n])
        at[t] += n
    total = sum(float(f.double().square().sum()) for f in st["fresh"].values())
    st["max_norm"] = 0.37 * math.sqrt(total)        # the step is clipped
    return st


# ---- plain forms ------------------------------------------------------------------------------------------------------------------
def _norm_plain(st):
    x, w = st["x"].detach(), st["weight"].detach()
    s32 = x.float()
    if st["residual"] is not None:
        s32 = s32 + st["residual"].detach().float()
    rstd = 1.0 / torch.sqrt((s32 * s32).mean(dim=1, keepdim=True) + EPS)
    h = s32 * rstd
    out = {"y": (h * w).to(x.dtype)}
    if st["residual"] is not None:
        out["s"] = s32.to(x.dtype)
    if st["case"]["backward"]:
        g = st["gy"].float()
        gw = g * w
        d = rstd * (gw - h * (gw * h).mean(dim=1, keepdim=True))
        if st["residual"] is not None:
            d = d + st["gs"].float()
        out["dx"] = d.to(x.dtype)
        if st["residual"] is not None:
            out["dr"] = out["dx"]
        out["dw"] = (g * h).sum(dim=0)
    return out


def _encode(t, code, group):
    """Codes and the largest magnitude of each group of ``group`` columns.  The quotients are formed in 64 bits: rounded to 32 first,
    those next to a border between two codes would fall on the wrong side."""
    v = t.reshape(t.shape[0], -1, group)
    top = v.abs().amax(dim=2, keepdim=True)
    top = torch.where(top < TINY, torch.zeros_like(top), top)
    scaled = v.double() * QMAX[code] / torch.where(top > 0, top, torch.full_like(top, math.inf)).double()
    if code == "int8":
        return scaled.round().to(torch.int8).reshape(t.shape), top.squeeze(2)
    mantissa = torch.frexp(scaled).mantissa           # e4m3: four significant bits from 2^-6 on, a spacing of 2^-9 below
    normal = scaled / mantissa * ((mantissa * 16).round() / 16)
    codes = torch.where(scaled.abs() < 2.0 ** -6, (scaled * 512).round() / 512, normal).to(torch.float8_e4m3fn)
    return codes.reshape(t.shape), top.squeeze(2)


def _quant_plain(st):
    case, w = st["case"], st["weight"]
    s32 = st["x"].float()
    if st["residual"] is not None:
        s32 = s32 + st["residual"].float()
    rstd = 1.0 / torch.sqrt((s32 * s32).mean(dim=1, keepdim=True) + EPS)
    codes, top = _encode(s32 * w, "e4m3", case["group"] or case["width"])
    out = {"codes": codes, "scales": top / QMAX["e4m3"] * rstd}
    if st["residual"] is not None:
        out["s"] = s32.to(st["x"].dtype)
    return out


def _cache_plain(st):
    case, codes, scales = st["case"], st["codes"], st["scales"]
    P, F = codes.shape
    group = case["group"] or F
    new, top = _encode(st["rows"].float(), case["code"], group)
    top = top / QMAX[case["code"]]
    if st["to"] is None:
        codes.copy_(new)
        scales.copy_(top)
    else:                       # a row that is written twice in one call keeps the later one
        place = torch.arange(st["to"].numel(), device=codes.device)
        last = torch.zeros(P, dtype=torch.int64, device=codes.device).scatter_reduce_(0, st["to"], place, "amax")[st["to"]]
        codes.view(torch.uint8)[st["to"]] = new.view(torch.uint8)[last]
        scales[st["to"]] = top[last]
    c, s = (codes, scales) if st["at"] is None else (codes.view(torch.uint8)[st["at"]].view(codes.dtype), scales[st["at"]])
    v = (c.float().reshape(-1, F // group, group) * s[:, :, None]).reshape(-1, F)
    if case["norm"]:
        v = v / (torch.sqrt((v * v).sum(dim=1, keepdim=True)) + NORM_EPS)
    return v.to(TYPES[case["dtype"]])


def _gradnorm_plain(st):
    total = torch.sqrt(torch.stack([g.float().square().sum() for g in st["grads"]]).sum())
    if not st["case"]["clip"]:
        return {"norm": total}
    torch._foreach_mul_(st["grads"], torch.clamp(st["max_norm"] / (total + 1e-6), max=1.0))
    return {"norm": total, "grads": st["flat"]}


# ---- one pass ---------------------------------------------------------------------------------------------------------------------
def run(st):
    case = st["case"]
    if case["op"] == "gradnorm" and case["clip"]:       # the new step's gradients arrive in the buckets
        torch._foreach_copy_(list(st["flat"].values()), list(st["fresh"].values()))
    if not own:
        return {"norm": _norm_plain, "quant": _quant_plain, "cache": _cache_plain, "gradnorm": _gradnorm_plain}[case["op"]](st)
    if case["op"] == "norm":
        from instascene_amd.rows import rms_norm
        if not case["backward"]:
            got = rms_norm(st["x"], st["weight"], EPS, residual=st["residual"])
            return {"y": got} if st["residual"] is None else {"y": got[0], "s": got[1]}
        if st["residual"] is None:
            y = rms_norm(st["x"], st["weight"], EPS)
            dx, dw = torch.autograd.grad(y, (st["x"], st["weight"]), st["gy"])
            return {"y": y, "dx": dx, "dw": dw}
        y, s = rms_norm(st["x"], st["weight"], EPS, residual=st["residual"])
        dx, dr, dw = torch.autograd.grad((y, s), (st["x"], st["residual"], st["weight"]), (st["gy"], st["gs"]))
        return {"y": y, "s": s, "dx": dx, "dr": dr, "dw": dw}
    if case["op"] == "quant":
        from instascene_amd.rows import rms_norm_quantized
        got = rms_norm_quantized(st["x"], st["weight"], EPS, residual=st["residual"], dtype=torch.float8_e4m3fn, group=case["group"] or None)
        q, s = got if st["residual"] is not None else (got, None)
        return {"codes": q.codes, "scales": q.scales} if s is None else {"codes": q.codes, "scales": q.scales, "s": s}
    if case["op"] == "cache":
        st["cache"].write(st["rows"], st["to"])
        return st["cache"].read(st["at"], out_dtype=TYPES[case["dtype"]], norm_eps=NORM_EPS if case["norm"] else None)
    from instascene_amd.optim import clip_grads_, grad_norm
    if not case["clip"]:
        return {"norm": grad_norm(st["grads"])}
    return {"norm": clip_grads_(st["grads"], st["max_norm"]), "grads": st["flat"]}


def work(case):
    if case["op"] in ("norm", "quant"):
        n, b = case["rows"] * case["width"], SIZE[case["dtype"]]
        if case["op"] == "quant":
            groups = case["rows"] * (case["width"] // (case["group"] or case["width"]))
            return {"bytes": n * (b * (3 if case["residual"] else 1) + 1) + 4 * groups + 4 * case["width"], "flops": 8 * n}
        forward = 4 if case["residual"] else 2                          # x, residual -> y, s
        # as one training step: the incoming gradients and the gradients of both inputs (one tensor); s, read again, is no input
        back = (0 if not case["backward"] else 3 if case["residual"] else 2)
        return {"bytes": n * b * (forward + back) + 8 * case["width"], "flops": n * (6 + (12 if back else 0))}
    if case["op"] == "cache":
        F, b = case["width"], SIZE[case["dtype"]]
        n_w, n_r = case["write"] or case["table"], case["read"] or case["table"]
        entry = F + 4 * (F // (case["group"] or F))
        ids = (8 * n_w if case["write"] else 0) + (8 * n_r if case["read"] else 0)
        return {"bytes": (n_w + n_r) * (F * b + entry) + ids, "flops": F * (4 * n_w + (4 if case["norm"] else 1) * n_r)}
    bytes_, n = sum(k * SIZE[t] for k, t in _sizes(case)), sum(k for k, _ in _sizes(case))
    # clipping: the gradients arrive (read, written), are read for the norm, and are scaled (read, written)
    return {"bytes": bytes_ * (5 if case["clip"] else 1), "flops": n * (3 if case["clip"] else 2)}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    with torch.no_grad():
        return {"norm": _exact_norm, "quant": _exact_norm, "cache": _exact_cache, "gradnorm": _exact_gradnorm}[case["op"]](case, st)


def _rounded(v, code):
    """The nearest value of the 8-bit type, ties to even, of |v| <= its largest."""
    if code == "int8":
        return torch.round(v)
    power = (v.contiguous().view(torch.int64) & 0x7FF0000000000000).view(torch.float64)     # the power of two at or below |v|
    step = power.clamp(min=2.0 ** -6) / 8
    return torch.round(v / step) * step


def _exact_norm(case, st):
    s = st["x"].detach().double()
    if case["residual"]:
        s += st["residual"].detach().double()
    w = st["weight"].detach().double()
    n = case["width"]
    inv = (torch.linalg.vector_norm(s, dim=1) ** 2 / n + EPS) ** -0.5
    if case["op"] == "quant":
        group = case["group"] or n
        y = (s * inv[:, None] * w).unflatten(1, (-1, group))
        scale = y.abs().max(dim=2).values / QMAX["e4m3"]
        out = {"codes": _rounded(y / scale[:, :, None], "e4m3").flatten(1).to(torch.float8_e4m3fn), "scales": scale}
    else:
        out = {"y": s * inv[:, None] * w}
        if case["backward"]:
            a = st["gy"].double() * w
            dot = torch.linalg.vecdot(a, s, dim=1)
            d = a * inv[:, None] - s * (inv ** 3 * dot / n)[:, None]
            if case["residual"]:
                d += st["gs"].double()
            out["dx"] = d
            if case["residual"]:
                out["dr"] = d
            out["dw"] = torch.mv((st["gy"].double() * s).T.contiguous(), inv)
    if case["residual"]:
        out["s"] = s
    return out


def _exact_cache(case, st):
    P, F = case["table"], case["width"]
    group = case["group"] or F
    v = st["rows"].double().unflatten(1, (-1, group))
    top = v.abs().max(dim=2, keepdim=True).values
    v = (_rounded(QMAX[case["code"]] * v / top.clamp(min=1e-300), case["code"]) * (top / QMAX[case["code"]])).flatten(1)
    if st["to"] is not None:
        to = st["to"].cpu()
        owner = torch.full((P,), -1, dtype=torch.int64)
        owner.numpy()[to.numpy()] = range(to.numel())       # in order: the later one stays
        owner = owner.to(v.device)[st["at"]]
        v = v[owner.clamp(min=0)] * (owner >= 0)[:, None]
    if case["norm"]:
        v = v / (torch.linalg.vector_norm(v, dim=1, keepdim=True) + NORM_EPS)
    return v


def _exact_gradnorm(case, st):
    total = math.sqrt(sum(float(f.double().square().sum()) for f in st["fresh"].values()))
    norm = torch.tensor(total, dtype=torch.float64)
    if not case["clip"]:
        return {"norm": norm}
    return {"norm": norm, "grads": {t: f.double() * min(1.0, st["max_norm"] / (total + 1e-6)) for t, f in st["fresh"].items()}}
