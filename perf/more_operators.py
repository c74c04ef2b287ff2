"""Cases of the 8-bit prompt operators: RMS norm with the residual's addition into 8-bit rows (rms_norm_s8) and the same
rounding without a norm (quantize_s8), linear layers of 8-bit rows (linear_s8), causal attention over packed prompts
(prompt_attention).

With ``own`` false, ``run`` computes an operator from elementary torch operations in 32 bits; with ``own`` true it
calls the package.  ``exact`` is each operator's definition in 64 bits.

8-bit rows.  A matrix [m, k] is codes int8 [m, 16 * ceil(k / 16)] and one fp32 scale a row; value = code * scale.
A row u is rounded as code = rint(u * fp32(127 / max|u|)), the product exact.  A norm's factor goes into the scale alone.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
PAIRS = 1 << 31  # (query row, key) pairs of all heads that the plain form holds at once


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a decode step of four sequences: latency
        dict(name="norm t4 4096 bf16", op="norm", dtype="bf16", t=4, n=4096, norm=True, residual=True),
        # a prompt of 8192 tokens between two layers
        dict(name="norm t8192 4096 f16", op="norm", dtype="f16", t=8192, n=4096, norm=True, residual=True),
        # odd sizes, the first layer of a prompt: nothing to add yet
        dict(name="norm t1021 5003 f32", op="norm", dtype="f32", t=1021, n=5003, norm=True, residual=False),
        # one token through a square projection: latency and the weight stream
        dict(name="linear m1 4096x4096 f16", op="linear", dtype="f16", m=1, n=4096, k=4096, bias=False),
        # a decode batch through an expansion: the weight stream
        dict(name="linear m16 16384x8192 bf16", op="linear", dtype="bf16", m=16, n=16384, k=8192, bias=True),
        # a short prompt, odd sizes, rows that are no multiple of 16 bytes
        dict(name="linear m77 5003x4091 f32", op="linear", dtype="f32", m=77, n=5003, k=4091, bias=True),
        # a long prompt: arithmetic
        dict(name="linear m8192 8192x8192 bf16", op="linear", dtype="bf16", m=8192, n=8192, k=8192, bias=False),
        # one question: latency
        dict(name="attention l77 f16", op="attention", dtype="f16", b=1, t=77, hq=12, hk=12, d=64, prefix=0, ragged=False, fused=True),
        # one long prompt, grouped heads read in place from a fused projection
        dict(name="attention l8192 bf16", op="attention", dtype="bf16", b=1, t=8192, hq=32, hk=8, d=128, prefix=0, ragged=False, fused=True),
        # prompts of many lengths packed into one call, some of them empty
        dict(name="attention b24 t8192 f16", op="attention", dtype="f16", b=24, t=8192, hq=32, hk=8, d=128, prefix=0, ragged=True, fused=True),
        # the next parts of six conversations whose first parts' keys and values are there
        dict(name="attention b6 t2048 prefix bf16", op="attention", dtype="bf16", b=6, t=2048, hq=32, hk=8, d=128, prefix=4096, ragged=True, fused=False),
        # full precision
        dict(name="attention b5 t1531 f32", op="attention", dtype="f32", b=5, t=1531, hq=16, hk=16, d=64, prefix=0, ragged=True, fused=False),
    ]


def draw(rng):
    def log(lo, hi):
        hi = max(lo, int(hi))
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    op = rng.choice(["norm", "norm", "linear", "linear", "linear", "attention", "attention", "attention"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "norm":
        n = log(256, 16384)
        if rng.random() < 0.6:
            n = -(-n // 64) * 64
        norm = rng.random() < 0.7
        return dict(op=op, dtype=dtype, t=log(1, (8192 * 4096) // n // (2 if dtype == "f32" else 1)), n=n, norm=norm,
                    residual=norm and rng.random() < 0.6)
    if op == "linear":
        m, n, k = log(1, 8192), log(256, 16384), log(256, 16384)
        if rng.random() < 0.6:
            n, k = -(-n // 64) * 64, -(-k // 64) * 64
        while n * k > 1 << 27:
            n = max(256, n // 2)
        return dict(op=op, dtype=dtype, m=min(m, (1 << 39) // (n * k)), n=n, k=k, bias=rng.random() < 0.5)
    dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
    hk = rng.choice([1, 2, 4, 8, 8, 12])
    hq = hk * rng.choice([1, 1, 2, 3, 4, 4, 5, 8])
    d = rng.choice([64, 64, 80, 128, 128, 128])
    b = log(1, 48)
    prefix = log(16, 4096) if rng.random() < 0.25 else 0
    most = PAIRS // (2 if dtype == "f32" else 1) // hq
    t = log(1, min(8192, (math.sqrt((b * prefix) ** 2 + 4 * most) - b * prefix) / 2))
    return dict(op=op, dtype=dtype, b=b, t=t, hq=hq, hk=hk, d=d, prefix=prefix, ragged=rng.random() < 0.7,
                fused=prefix == 0 and rng.random() < 0.5)


def lengths(c):
    """Tokens of each sequence, and its keys: the same tokens and those of its earlier part."""
    b = c["b"]
    share = [0 if i % 16 == 5 else 1 + (i * 7919 + 3) % 64 if c["ragged"] else 1 for i in range(b)]
    q = [c["t"] * s // sum(share) for s in share]
    q[0] += c["t"] - sum(q)
    return q, [n + (c["prefix"] * (1 + (i * 31 + 7) % 16) // 16 if n else 0) for i, n in enumerate(q)]


def work(c):
    e = BYTES[c["dtype"]]
    if c["op"] == "norm":  # stored in 8 bits, then read back
        x = c["t"] * c["n"]
        return {"bytes": x * (e * (4 if c["residual"] else 2) + 2) + 8 * c["t"] + (c["n"] * e if c["norm"] else 0),
                "flops": (7 if c["norm"] else 4) * x}
    if c["op"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + m * n * e + (n * e if c["bias"] else 0), "flops": 2 * m * n * k}
    q, k = lengths(c)
    seen = sum(n * m - n * (n - 1) // 2 for n, m in zip(q, k))
    return {"bytes": (2 * c["t"] * c["hq"] + 2 * sum(k) * c["hk"]) * c["d"] * e + 4 * c["t"] * c["hq"],
            "flops": 4 * c["d"] * c["hq"] * seen}


# ----------------------------------------------------------------------------------------------- inputs
def channels(n, g, dev):
    """Sizes of channels: mostly alike, a few much larger, as projections give them."""
    a = torch.rand(n, generator=g, device=dev) * 0.8 + 0.6
    return torch.where(torch.rand(n, generator=g, device=dev) < 0.02, a * 6, a)


def rounded(u):
    """Codes (as fp32) and the largest size of each row of u, fp32."""
    a = u.abs().amax(-1, keepdim=True)
    inv = torch.where(a > 0, 127 / a, torch.zeros_like(a))
    return (u.double() * inv.double()).round().float(), a


def rows_of(x):
    """x [m, k] as 8-bit rows."""
    c, a = rounded(x.float())
    codes = torch.zeros(x.shape[0], -(-x.shape[1] // 16) * 16, dtype=torch.int8, device=x.device)
    codes[:, :x.shape[1]] = c.to(torch.int8)
    return codes, (a / 127).squeeze(-1).contiguous()


def prepare(case, seed):
    c = dict(case)
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = {"case": c}
    if c["op"] == "norm":
        t, n = c["t"], c["n"]
        s["x"] = normal(t, n).mul_(channels(n, g, dev)).to(dt)
        s["w"] = (1 + 0.2 * normal(n)).to(dt) if c["norm"] else None
        s["residual"] = normal(t, n).mul_(channels(n, g, dev) * 3).to(dt) if c["residual"] else None
        return s
    if c["op"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        s["x_codes"], s["x_scales"] = rows_of(normal(m, k).mul_(channels(k, g, dev)))
        s["w_codes"], s["w_scales"] = rows_of(normal(n, k).mul_(k ** -0.5))
        s["bias"] = (normal(n) * 0.1).to(dt) if c["bias"] else None
        return s
    hq, hk, d = c["hq"], c["hk"], c["d"]
    q, k = lengths(c)
    if c["fused"]:  # queries, keys and values side by side in a projection's output
        x = normal(c["t"], hq + 2 * hk, d).mul_(channels(d, g, dev)).to(dt)
        s["q"], s["k"], s["v"] = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    else:
        s["q"] = normal(c["t"], hq, d).mul_(channels(d, g, dev)).to(dt)
        s["k"], s["v"] = (normal(sum(k), hk, d).mul_(channels(d, g, dev)).to(dt) for _ in range(2))
    s["starts"], s["k_starts"] = (torch.tensor([0] + n, device=dev).cumsum(0).to(torch.int32) for n in (q, k))
    s["scale"] = d ** -0.5
    return s


# --------------------------------------------------------------------------------------------- operators
def plain_norm(s):
    c = s["case"]
    x = s["x"]
    dt = x.dtype
    if s["residual"] is not None:  # the sum is rounded to the type that it is kept in; the state's own is left for the next pass
        x = (x.float() + s["residual"].float()).to(dt)
    h = x.float()
    codes, a = rounded(h * s["w"].float() if c["norm"] else h)
    scale = a / 127
    if c["norm"]:
        scale = scale * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    return [(codes * scale).to(dt), scale.squeeze(-1)] + ([x] if c["residual"] else [])


def plain_linear(s):
    c = s["case"]
    y = s["x_codes"][:, :c["k"]].float() @ s["w_codes"][:, :c["k"]].float().t()
    y = y * s["x_scales"][:, None] * s["w_scales"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[c["dtype"]])


def plain_attention(s):
    c = s["case"]
    hq, hk, d = c["hq"], c["hk"], c["d"]
    t, tk = s["q"].shape[0], s["k"].shape[0]
    i, j = (torch.arange(n, device="cuda") for n in (t, tk))
    of_q, of_k = (torch.searchsorted(st[1:], x.to(torch.int32), right=True) for st, x in ((s["starts"], i), (s["k_starts"], j)))
    # a sequence's last token and last key are in line
    last = (s["k_starts"][1:] - s["starts"][1:])[of_q] + i
    hidden = (of_q[:, None] != of_k) | (j > last[:, None])
    q = s["q"].float().view(t, hk, hq // hk, d).permute(1, 2, 0, 3).flatten(1, 2)
    a = (q @ s["k"].float().permute(1, 2, 0)).mul_(s["scale"]).view(hk, hq // hk, t, tk)
    a.masked_fill_(hidden, -math.inf)
    top = a.amax(-1, keepdim=True).clamp(min=-1e30)
    a = a.sub_(top).exp_()
    total = a.sum(-1, keepdim=True)
    o = (a.flatten(1, 2) @ s["v"].float().transpose(0, 1)).view(hk, hq // hk, t, d) / total.clamp(min=1e-30)
    lse = (top + total.log()).squeeze(-1).flatten(0, 1).t().contiguous()
    return [o.permute(2, 0, 1, 3).reshape(t, hq, d).to(s["q"].dtype), lse]


def own_norm(s):
    import my_own_cnn_b200 as b2q

    x, residual = s["x"], s["residual"]
    if s["w"] is None:
        rows = b2q.quantize_s8(x)
    elif residual is None:
        rows = b2q.rms_norm_s8(x, s["w"], eps=EPS)
    else:  # the sum into a buffer of its own: the state's residual is left for the next pass
        rows, total = b2q.rms_norm_s8(x, s["w"], residual=residual, residual_out=torch.empty_like(x), eps=EPS)
        return [rows.dequantize(x.dtype), rows.scales, total]
    return [rows.dequantize(x.dtype), rows.scales]


def own_linear(s):
    import my_own_cnn_b200 as b2q

    k = s["case"]["k"]
    x, w = b2q.S8Rows(s["x_codes"], s["x_scales"], k), b2q.S8Rows(s["w_codes"], s["w_scales"], k)
    return b2q.linear_s8(x, w, s["bias"], dtype=DTYPES[s["case"]["dtype"]])


def own_attention(s):
    import my_own_cnn_b200 as b2q

    return b2q.prompt_attention(s["q"], s["k"], s["v"], s["starts"], k_starts=s["k_starts"] if s["case"]["prefix"] else None,
                                scale=s["scale"], return_lse=True)


PLAIN = {"norm": plain_norm, "linear": plain_linear, "attention": plain_attention}
OWN = {"norm": own_norm, "linear": own_linear, "attention": own_attention}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ----------------------------------------------------------------------------------- definitions, 64 bits
def exact(case, seed):
    s, c = prepare(case, seed), dict(case)
    if c["op"] == "norm":
        return exact_norm(s, c)
    if c["op"] == "linear":
        k = c["k"]
        y = torch.empty(c["m"], c["n"], dtype=torch.float64, device="cuda")
        w = s["w_codes"][:, :k].double() * s["w_scales"].double()[:, None]
        for i in range(0, c["m"], 1024):
            torch.matmul(s["x_codes"][i:i + 1024, :k].double() * s["x_scales"][i:i + 1024].double()[:, None], w.t(),
                         out=y[i:i + 1024])
        return y if s["bias"] is None else y + s["bias"].double()
    hq, hk, d = c["hq"], c["hk"], c["d"]
    out = torch.zeros(c["t"], hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((c["t"], hq), -math.inf, dtype=torch.float64, device="cuda")
    at = at_k = 0
    for n, m in zip(*lengths(c)):
        if n:
            row = torch.arange(n, device="cuda")[:, None] + (m - n)
            seen = torch.arange(m, device="cuda") <= row
            for h in range(hq):
                k, v = (s[x][at_k:at_k + m, h // (hq // hk)].double() for x in ("k", "v"))
                a = s["scale"] * (s["q"][at:at + n, h].double() @ k.t())
                a = torch.where(seen, a, -math.inf)
                lse[at:at + n, h] = torch.logsumexp(a, -1)
                out[at:at + n, h] = torch.softmax(a, -1) @ v
        at, at_k = at + n, at_k + m
    return [out, lse]


def exact_norm(s, c):
    # the format's own roundings: the sum to the type that it is kept in, its product with the weight and 127 / largest to fp32
    h, residual = s["x"], s["residual"]
    if residual is not None:
        h = torch.add(h.double(), residual.double()).to(torch.float32).to(h.dtype)
    u = h.double()
    if c["norm"]:
        u = (u * s["w"].double()).to(torch.float32).double()
    largest = torch.maximum(u.max(-1).values, -u.min(-1).values)
    codes = torch.round(u * (127.0 / largest).to(torch.float32).double()[:, None])
    scale = largest / 127.0
    if c["norm"]:
        scale = scale / torch.sqrt((h.double() ** 2).sum(-1) / c["n"] + EPS)
    return [codes * scale[:, None], scale] + ([h.double()] if residual is not None else [])
