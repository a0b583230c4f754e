"""Plain 64-bit implementations of the attention layer's operators, each with the bound on what rounding may cost.

Bounds are worst-case sums over the roundings of the arithmetic that the operators document: products in fp32 (`u` is the
relative error of one product with its operands' roundings), sums in fp32, one rounding on store.
"""
import torch

import primitiv_b200 as pb

F16, F32 = 2.0 ** -11, 2.0 ** -24            # half a step, relative
TINY16 = 2.0 ** -25                          # half a step among halves too small for full precision
# one product: halves are exact in the first product, and p or ds is rounded for the second; 3xTF32 drops lo.lo (2^-22) and
# rounds lo (2^-22 more on either side); TF32 rounds both operands; 3xFP16 runs as 3xTF32
MODES = {
    "fp16": (pb.MODE_FP16, torch.float16, 0.0, F16),
    "3xtf32": (pb.MODE_FP32_3XTF32, torch.float32, 2.0 ** -20, 2.0 ** -20),
    "tf32": (pb.MODE_TF32, torch.float32, 2.0 ** -10, 2.0 ** -10),
    "3xfp16": (pb.MODE_FP32_3XFP16, torch.float32, 2.0 ** -20, 2.0 ** -20),
}


def store_rounding(dtype):
    # fp32: a weight below 2^-126 counts as zero, and so may each product with it; the 2^10 rows of a sum here, each with factors
    # below 2^16, make of that at most 2^-126 2^26
    return (F16, TINY16) if dtype == torch.float16 else (F32, 2.0 ** -100)


def rotary(x, angles, amplitude, rot, layout, back=False):
    """x: [tokens, heads, head] in 64 bits; angles: [tokens, rot / 2]."""
    cos, sin = (amplitude * torch.cos(angles))[:, None], (amplitude * torch.sin(angles))[:, None]
    if back:
        sin = -sin
    y = x.clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if layout == pb.ROTARY_PAIRS else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def attention(q, k, v, scale, causal, gy=None, mode="fp16"):
    """One head of one sequence, [rows, head] in 64 bits.  -> dict of values and dict of bounds: y, lse and, with gy, gq, gk, gv."""
    _, dtype, u1, u2 = MODES[mode]
    store, tiny = store_rounding(dtype)
    (lq, d), lk = q.shape, k.shape[0]
    seen = torch.ones(lq, lk, dtype=torch.bool, device=q.device)
    if causal:
        seen = seen.tril(lk - lq)
    empty = ~seen.any(1)
    s = (q @ k.t()) * scale
    # fp32 sums of d products, added by a unit that truncates (a whole step): every k-step adds at most three terms
    e_s = (abs(q) @ abs(k).t()) * abs(scale) * (u1 + (3 * d / 8 + 4) * 2 * F32)
    s = s.masked_fill(~seen, -float("inf"))
    top = s.max(1, keepdim=True).values if lk else torch.full((lq, 1), -float("inf"), dtype=q.dtype, device=q.device)
    top = torch.where(empty[:, None], torch.zeros_like(top), top)
    w = torch.exp(s - top)
    total = w.sum(1, keepdim=True)
    p = torch.where(empty[:, None], torch.zeros_like(w), w / total)
    lse = torch.where(empty, torch.full_like(top[:, 0], -float("inf")), (top + torch.log(total))[:, 0])
    # relative error of p: that of its score and of the row's sum, the exponent's argument, exp2 (2 units of 2^-22), lse as stored
    arg = (abs(torch.where(seen, s, torch.zeros_like(s))) + abs(torch.where(empty, torch.zeros_like(lse), lse))[:, None] + 1) * 4 * F32
    e_s = torch.where(seen, e_s, torch.zeros_like(e_s))
    e_row = (p * (e_s + arg)).sum(1, keepdim=True)
    e_p = e_s + arg + e_row + 2.0 ** -20
    y = p @ v
    run = (lk / 32 + 64) * 2 * F32            # tiles added in fp32, and the steps within one that truncates
    val = {"y": y, "lse": lse}
    # halves: a weight that is too small for a half beside the row's largest loses at most 2^-25 of that
    e_y = (p * (e_p + u2 + run)) @ abs(v) + (TINY16 * abs(v).sum(0)[None] if dtype == torch.float16 else 0.0)
    tol = {"y": e_y + store * abs(y) + tiny, "lse": (e_row[:, 0] + 2.0 ** -20 + run + (abs(torch.where(empty, torch.zeros_like(lse), lse)) + 1) * 4 * F32)}
    if gy is None:
        return val, tol
    dp = gy @ v.t()
    delta = (gy * y).sum(1, keepdim=True)
    ds = p * (dp - delta)
    val.update(gv=p.t() @ gy, gq=scale * ds @ k, gk=scale * ds.t() @ q)
    # delta is taken from y as it was stored
    e_dp = (abs(gy) @ abs(v).t()) * (u1 + (3 * d / 8 + 4) * 2 * F32)
    e_delta = (abs(gy) * (e_y + store * abs(y) + tiny)).sum(1, keepdim=True) + (abs(gy) * abs(y)).sum(1, keepdim=True) * d * F32
    # ds lies below 2^13 after its scale, so what is too small for a half loses 2^-25 / 2^12 of the largest possible
    bound = abs(gy).square().sum(1).sqrt().max() * abs(v).square().sum(1).sqrt().max() + abs(delta).max() if lq and lk else 0.0
    e_ds = p * (e_p * abs(dp - delta) + e_dp + e_delta) + abs(ds) * (u2 + run)
    if dtype == torch.float16:
        e_ds = e_ds + seen * (TINY16 / 2.0 ** 11) * bound
    run_q = (lq / 32 + 64) * 2 * F32
    tol["gv"] = (p * (e_p + u2 + run_q)).t() @ abs(gy) + store * abs(val["gv"]) + tiny
    if dtype == torch.float16:
        tol["gv"] = tol["gv"] + TINY16 / 8192 * abs(gy).sum(0)[None]
    tol["gq"] = abs(scale) * e_ds @ abs(k) + store * abs(val["gq"]) + tiny
    tol["gk"] = abs(scale) * (e_ds + abs(ds) * run_q).t() @ abs(q) + store * abs(val["gk"]) + tiny
    return val, tol
