"""Plain 64-bit forms of the 8-bit prompt operators, and the error that each type allows (UNIT and `within` are lowbit_ref's)."""
import math

import torch

from tests.lowbit_ref import UNIT

SMALLEST = 2.0 ** -119


def rows(x, weight=None, residual=None, eps=None):
    """(codes fp64, scales fp64, h) of x [t, n]: the format's own roundings are those of h, of its product with the weight and
    the two of 127 (1 / largest); with eps the norm's factor is in the scales."""
    h = x if residual is None else (x.double() + residual.double()).float().to(x.dtype)
    u = h.double() if weight is None else (h.double() * weight.double()).float().double()
    top = u.abs().amax(-1)
    bad, small = ~top.isfinite(), top < SMALLEST
    inv = (127.0 * (1.0 / torch.where(bad | small, torch.ones_like(top), top)).float().double()).float().double()
    codes = (u * inv[:, None]).round()
    codes[bad | small] = 0
    scales = top / 127
    if eps is not None:
        scales = scales * (h.double().square().mean(-1) + eps).rsqrt()
    scales = torch.where(bad, math.nan, torch.where(small, 0.0, scales))
    return codes, scales, h


# A scale is off by its three roundings, the root's 2^-22 and half of the sum of squares' error: chains of at most 32 elements a lane,
# 5 steps of a warp and 32 warps (40 elements and the same in rows past 16384).
SCALE = 2.0 ** -22 + 80 * 2.0 ** -24


def linear(x_codes, x_scales, w_codes, w_scales, bias, dtype):
    """(y, bound): whole sums are exact; their conversion, two products and the addition round in fp32, the result to dtype.

    fp16 values below its smallest normal 2^-14 lie 2^-24 apart (10 bits behind the point of 2^-14), so that rounding to the nearest
    is off by up to 2^-25 whatever the value: 2^-11 of it holds from 2^-14 up only."""
    s = x_codes.double() @ w_codes.double().t()
    p = s * x_scales.double()[..., None] * w_scales.double()
    y = p if bias is None else p + bias.double()
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return y, UNIT[dtype] * y.abs() + 2.0 ** -22 * (p.abs() + y.abs()) + tiny


def attention(q, k, v, starts, k_starts, scale, dtype):
    """(out, lse, bound on out, bound on lse), one sequence and head at a time; rows outside every sequence stay NaN.

    A score is a sum of d products in fp32, off by at most d 2^-23 sum |scale q k|, its product with the base's factor by two roundings;
    a weight besides by 2^-21 (the exponential) and, in 16-bit calls, its rounding to 16 bits; their sums (of n keys: n / 4 additions a lane and
    16 more, or n / 16 in the tensor core; parts add up to 32 more where n is past 512) by (n / 4 + 16) 2^-23.  fp16 weights, 2^6 to 2^14
    where the largest has its place, are normal down to 2^-20 of it and off by 2^-25 of it at most below."""
    tq, hq, d = q.shape
    r = hq // k.shape[1]
    out = torch.full((tq, hq, d), math.nan, dtype=torch.float64)
    lse = torch.full((tq, hq), math.nan, dtype=torch.float64)
    ob, lb = torch.zeros_like(out), torch.zeros_like(lse)
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    starts, k_starts = starts.tolist(), k_starts.tolist()
    for i in range(len(starts) - 1):
        q0, q1, k0, k1 = starts[i], starts[i + 1], k_starts[i], k_starts[i + 1]
        seen = torch.arange(k1 - k0)[None] <= torch.arange(q1 - q0)[:, None] + (k1 - k0) - (q1 - q0)
        n = seen.sum(-1)
        for h in range(hq):
            kk, vv = k[k0:k1, h // r], v[k0:k1, h // r]
            a = torch.where(seen, scale * (q[q0:q1, h] @ kk.t()), -math.inf)
            big = torch.where(seen, abs(scale) * (q[q0:q1, h].abs() @ kk.abs().t()), 0.0)
            big = big.amax(-1) if k1 > k0 else torch.zeros(q1 - q0, dtype=torch.float64)
            p = torch.where(n[:, None] > 0, torch.softmax(a, -1), 0.0) if k1 > k0 else a
            o = p @ vv
            wide = p @ vv.abs()
            e = 2 * (d + 2) * 2.0 ** -23 * big + 2.0 ** -20 + (n / 4 + 16) * 2.0 ** -22 + (0 if dtype == torch.float32 else UNIT[dtype])
            out[q0:q1, h] = o
            lse[q0:q1, h] = torch.where(n > 0, torch.logsumexp(a, -1), -math.inf) if k1 > k0 else -math.inf
            ob[q0:q1, h] = UNIT[dtype] * o.abs() + e[:, None] * wide
            if dtype == torch.float16 and k1 > k0:  # no weight is smaller than the largest by more than its own rounding says, or 2^-25
                ob[q0:q1, h] += 2.0 ** -25 * (seen.double() @ vv.abs()) * p.amax(-1, keepdim=True)
            lb[q0:q1, h] = (d + 2) * 2.0 ** -23 * big + (n / 4 + 16) * 2.0 ** -23 + 2.0 ** -20 + 2.0 ** -23 * lse[q0:q1, h].abs().nan_to_num(posinf=0)
    return out, lse, ob, lb
