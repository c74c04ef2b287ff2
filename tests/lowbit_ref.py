"""Plain 64-bit forms of the decoder operators, and the error that each type allows.

Bounds.  u is the relative size of one rounding to the output's type (2^-24, 2^-11, 2^-8 for fp32, fp16,
bf16).  Sums are held in fp32: a sum whose longest chain has L additions is off by at most about
L * 2^-23 times the sum of the magnitudes (2^-23, not 2^-24, for adders that truncate).
"""
import math

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def within(got, want, bound):
    """|got - want| <= bound everywhere (NaN fails), with the worst ratio in the message."""
    got, want = got.double().cpu(), want.double().cpu()
    bound = bound.double().cpu()
    off = (got - want).abs()
    same = got == want  # infinities
    bad = ~((off <= bound) | same)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} outside; worst off/bound "
                           f"{float((off / bound.clamp(min=1e-300))[bad].nan_to_num(math.inf).max()):.3g}")


def unpair(codes):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()


def w4_values(w):
    at = torch.arange(w.k, device=w.codes.device) // w.group
    z = 8.0 if w.zeros is None else w.zeros.double()[at].t()
    return (unpair(w.codes)[:, :w.k] - z) * w.scales.double()[at].t()


def rotate(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    h = x[..., :rot]
    a, b = (h[..., 0::2], h[..., 1::2]) if interleaved else (h[..., :rot // 2], h[..., rot // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    h = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([h, x[..., rot:]], -1)


def norm_rope(x, w, table, pos, eps, interleaved):
    """One side in 64 bits (differentiable)."""
    y = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    if w is not None:
        y = y * w
    if table is None:
        return y
    cos, sin = table.double()[pos.long()][:, None].chunk(2, -1)
    return rotate(y, cos, sin, interleaved)


def quantize4(x, group):
    """The cache format's own fp32 steps: codes (uint8 per channel), bf16 scales as fp32, zero points."""
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
    s = ((hi - lo) * torch.tensor(1 / 15, dtype=torch.float32)).bfloat16().float()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    inv = torch.where(s > 0, torch.ones_like(s) / s, torch.zeros_like(s))
    z = (-lo * inv).round().clamp(0, 15)
    c = ((g * inv[..., None]).round() + z[..., None]).clamp(0, 15)
    return c.to(torch.uint8).flatten(-2), s, z


def cache_words(s, z):
    return ((s.contiguous().view(torch.int32) >> 16) & 0xFFFF) | (z.to(torch.int32) << 16)


def cache_values(codes, params, group):
    s = (params << 16).view(torch.float32).double()
    z = ((params >> 16) & 255).double()
    return ((unpair(codes).unflatten(-1, (-1, group)) - z[..., None]) * s[..., None]).flatten(-2), s


def attention(q, cache, table, lens, scale, dtype):
    """(out, lse, bound on out, bound on lse) in 64 bits, one sequence and head at a time.

    Scores: the products are exact and summed in fp32 over codes of at most 15 and zero points of at most 15,
    so a score is off by about 2^-20 B, B = scale * sum |q| 16 s; weights are rounded to 8 bits or more before
    they meet the values in 16-bit calls, and hardly at all in fp32 ones."""
    b, tq, hq, d = q.shape
    hk, r = cache.heads, hq // cache.heads
    out = torch.zeros(b, tq, hq, d, dtype=torch.float64)
    lse = torch.full((b, tq, hq), -math.inf, dtype=torch.float64)
    ob, lb = torch.zeros_like(out), torch.zeros_like(lse)
    kc, kp, vc, vp = (x.cpu() for x in (cache.k_codes, cache.k_params, cache.v_codes, cache.v_params))
    table, lens, q = table.cpu(), lens.cpu(), q.double().cpu()
    for i in range(b):
        n = int(lens[i])
        if n == 0:
            continue
        at = table[i, :-(-n // cache.page_size)].long()
        for h in range(hk):
            def flat(x):
                return x[at, h].flatten(0, 1)[:n]

            k, ks = cache_values(flat(kc), flat(kp), cache.group)
            v, vs = cache_values(flat(vc), flat(vp), cache.group)
            ks, vs = (s.repeat_interleave(cache.group, 1) for s in (ks, vs))
            for j in range(tq):
                m = n - tq + j + 1
                if m <= 0:
                    continue
                rows = q[i, j, h * r:(h + 1) * r]
                a = scale * (rows @ k[:m].t())
                big = (abs(scale) * (rows.abs() @ (16 * ks[:m]).t())).amax(-1)
                p = torch.softmax(a, -1)
                o = p @ v[:m]
                e = 2.0 ** -20 * (8 + big) + (2.0 ** -8 if dtype != torch.float32 else 0.0)
                out[i, j, h * r:(h + 1) * r] = o
                lse[i, j, h * r:(h + 1) * r] = torch.logsumexp(a, -1)
                ob[i, j, h * r:(h + 1) * r] = UNIT[dtype] * o.abs() + e[:, None] * (p @ (16 * vs[:m]))
                lb[i, j, h * r:(h + 1) * r] = 2.0 ** -20 * (8 + big)
    return out, lse, ob, lb
