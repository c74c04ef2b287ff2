"""Cases of the 4-bit decoder operators: weight-only linear layers (linear_w4), per-head norms with the
position rotation and their gradient (qk_norm_rope, qk_norm_rope_bprop), the 4-bit paged cache
(kv4_append, kv4_read) and the attention over it (kv4_attention).

With ``own`` false, ``run`` computes an operator from elementary torch operations in 32 bits; with
``own`` true it calls the package.  ``exact`` is each operator's definition in 64 bits.

Formats.  A 4-bit code pair is one byte, low nibble first.  A weight matrix [N, K] is codes
[N, 16 * ceil(K / 32)] (rows padded to 16 bytes), bf16 scales and optional uint8 zero points
[ceil(K / group), N]; w = (code - zero) * scale, zero = 8 where there are no zero points.  A cache page is
codes [heads, page_size, D / 2] and one int32 per `group` channels: the bf16 scale's bits, and the zero
point in bits 16-23.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
MIN_NORMAL = 2.0 ** -126


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token through a small projection: latency
        dict(name="linear m1 768x768 f16", op="linear", dtype="f16", m=1, n=768, k=768, group=64, zeros=False, bias=False),
        # one token through a large projection: the weight stream
        dict(name="linear m1 8192x8192 bf16", op="linear", dtype="bf16", m=1, n=8192, k=8192, group=128, zeros=True, bias=False),
        # a decode batch through an expansion
        dict(name="linear m16 16384x8192 bf16", op="linear", dtype="bf16", m=16, n=16384, k=8192, group=64, zeros=True, bias=True),
        # odd sizes: a short last group, rows that are no multiple of a vector
        dict(name="linear m5 5003x4091 f32", op="linear", dtype="f32", m=5, n=5003, k=4091, group=32, zeros=True, bias=True),
        # a decode step of four sequences
        dict(name="norm t4 bf16", op="norm", dtype="bf16", t=4, hq=32, hk=8, d=128, rot=128, interleaved=False, fused=True),
        # a prompt, heads read in place from a fused projection
        dict(name="norm t8192 f16", op="norm", dtype="f16", t=8192, hq=32, hk=8, d=128, rot=128, interleaved=False, fused=True),
        # training: the gradient of a batch of sequences, half of each head rotated
        dict(name="norm bprop t4097 f32", op="norm_bprop", dtype="f32", t=4097, hq=16, hk=16, d=64, rot=32, interleaved=True, fused=False),
        # a decode batch, one new token a sequence
        dict(name="append t64 bf16", op="append", dtype="bf16", t=64, h=8, d=128, group=64, page=64, fused=True),
        # a long prompt, with padding tokens that are not stored
        dict(name="append t8191 f32", op="append", dtype="f32", t=8191, h=4, d=256, group=32, page=16, fused=False),
        # the start of one conversation: latency
        dict(name="attention b1 l77 f32", op="attention", dtype="f32", b=1, tq=1, hq=12, hk=12, d=64, group=32, page=16, longest=77, ragged=False),
        # a ragged serving batch, some sequences empty
        dict(name="attention b48 l8192 bf16", op="attention", dtype="bf16", b=48, tq=1, hq=32, hk=8, d=128, group=64, page=64, longest=8192, ragged=True),
        # two very long contexts, two tokens checked at once
        dict(name="attention b2 l131072 f16", op="attention", dtype="f16", b=2, tq=2, hq=32, hk=8, d=128, group=64, page=128, longest=131072, ragged=False),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    op = rng.choice(["linear", "linear", "norm", "norm_bprop", "append", "attention", "attention"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "linear":
        m, n, k = log(1, 16), log(256, 16384), log(256, 16384)
        if rng.random() < 0.5:
            n, k = -(-n // 64) * 64, -(-k // 64) * 64
        while n * k > 1 << 27:
            n = max(256, n // 2)
        return dict(op=op, dtype=dtype, m=m, n=n, k=k, group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.7,
                    bias=rng.random() < 0.5)
    if op in ("norm", "norm_bprop"):
        hq, hk = rng.choice([(32, 8), (16, 16), (24, 4), (40, 8), (7, 1), (64, 8)])
        d = rng.choice([64, 64, 80, 128, 128, 256])
        rot = rng.choice([d, d, d // 2])
        return dict(op=op, dtype=dtype, t=log(1, 8192 * 40 * 128 // ((hq + hk) * d * (2 if dtype == "f32" else 1))), hq=hq,
                    hk=hk, d=d, rot=rot, interleaved=rng.random() < 0.3, fused=rng.random() < 0.5)
    d = rng.choice([64, 128, 128, 256])
    group = rng.choice([32, 64, 64])
    page = rng.choice([16, 32, 48, 64, 128])
    if op == "append":
        h = rng.choice([1, 2, 4, 8, 8, 12])
        return dict(op=op, dtype=dtype, t=log(1, 8192 * 1024 // (max(4, h) * d)), h=h, d=d, group=group, page=page,
                    fused=rng.random() < 0.5)
    hk = rng.choice([1, 2, 4, 8, 8, 12])
    ratio = rng.choice([1, 2, 3, 4, 4, 5, 8])
    b, tq = log(1, 64), rng.choice([1, 1, 1, 2, 4])
    longest = log(1, min(131072, (1 << 27) // (b * hk * d) * 3 // 2, (1 << 31) // (b * tq * hk * ratio * d)))
    return dict(op=op, dtype=dtype, b=b, tq=tq, hq=hk * ratio, hk=hk, d=d, group=group, page=page, longest=longest,
                ragged=rng.random() < 0.6)


def lengths(c):
    """Tokens in the cache of each sequence, the new ones among them: the longest, and others down to none."""
    if not c["ragged"]:
        return [c["longest"]] * c["b"]
    return [0 if i % 16 == 5 else max(1, c["longest"] * (1 + (i * 7919 + 3) % 64) // 64) if i else c["longest"]
            for i in range(c["b"])]


def work(c):
    e = BYTES[c["dtype"]]
    if c["op"] == "linear":
        groups = -(-c["k"] // c["group"])
        b = c["n"] * c["k"] / 2 + groups * c["n"] * (3 if c["zeros"] else 2) + c["m"] * (c["k"] + c["n"]) * e
        return {"bytes": b + (c["n"] * e if c["bias"] else 0), "flops": 2 * c["m"] * c["n"] * c["k"]}
    if c["op"] in ("norm", "norm_bprop"):
        x = c["t"] * (c["hq"] + c["hk"]) * c["d"]
        rest = c["t"] * (4 + c["rot"] * 4) + 2 * c["d"] * e
        return ({"bytes": 2 * x * e + rest, "flops": 8 * x} if c["op"] == "norm" else
                {"bytes": 3 * x * e + rest + 2 * c["d"] * e, "flops": 16 * x})
    row = c["d"] // 2 + 4 * (c["d"] // c["group"])
    if c["op"] == "append":  # stored, then read back
        x = 2 * c["t"] * c["h"]
        return {"bytes": x * (2 * c["d"] * e + 2 * row) + 16 * c["t"], "flops": 8 * x * c["d"]}
    tokens = sum(lengths(c))
    rows = c["tq"] * c["hq"]
    return {"bytes": tokens * c["hk"] * 2 * row + 2 * c["b"] * rows * c["d"] * e + 4 * c["b"] * rows,
            "flops": 4 * tokens * rows * c["d"]}


# ----------------------------------------------------------------------------------------------- inputs
def quantize(x, group):
    """x [..., D] in 32 bits -> codes [..., D] uint8, scales and zero points [..., D / group] (float32)."""
    g = x.unflatten(-1, (-1, group))
    lo, hi = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
    s = ((hi - lo) * torch.tensor(1 / 15, dtype=torch.float32)).bfloat16().float()
    s = torch.where(s < MIN_NORMAL, torch.zeros_like(s), s)
    inv = torch.where(s > 0, 1 / s, torch.zeros_like(s))
    z = (-lo * inv).round().clamp(0, 15)
    c = ((g * inv[..., None]).round() + z[..., None]).clamp(0, 15)
    return c.to(torch.uint8).flatten(-2), s, z


def pair(c):
    return c[..., 0::2] | (c[..., 1::2] << 4)


def params_of(s, z):
    return ((s.view(torch.int32) >> 16) & 0xFFFF) | (z.to(torch.int32) << 16)


def channels(n, g, dev):
    """Sizes of channels: mostly alike, a few much larger, as projections give them."""
    a = torch.rand(n, generator=g, device=dev) * 0.8 + 0.6
    return torch.where(torch.rand(n, generator=g, device=dev) < 0.02, a * 6, a)


def rotation_table(positions, rot, dev):
    f = 10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
    a = torch.arange(positions, device=dev, dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], -1).float()


def prepare(case, seed):
    c = dict(case)
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = {"case": c}
    if c["op"] == "linear":
        m, n, k, group = c["m"], c["n"], c["k"], c["group"]
        groups, pitch = -(-k // group), -(-k // 32) * 16
        w = torch.zeros(n, groups * group, device=dev)
        w[:, :k] = normal(n, k) * (k ** -0.5)
        if c["zeros"]:
            codes, sc, z = quantize(w, group)
            s["zeros"] = z.t().to(torch.uint8).contiguous()
        else:  # symmetric: codes 1 to 15 around 8
            sc = (w.unflatten(1, (-1, group)).abs().amax(-1) / 7).bfloat16().float()
            codes = ((w.unflatten(1, (-1, group)) / sc[..., None]).round() + 8).clamp(0, 15).to(torch.uint8).flatten(1)
            s["zeros"] = None
        full = torch.zeros(n, 2 * pitch, dtype=torch.uint8, device=dev)
        full[:, :min(2 * pitch, groups * group)] = codes[:, :2 * pitch]
        s["codes"], s["scales"] = pair(full).contiguous(), sc.t().bfloat16().contiguous()
        s["x"] = (normal(m, k) * channels(k, g, dev)).to(dt)
        s["bias"] = (normal(n) * 0.1).to(dt) if c["bias"] else None
        return s
    if c["op"] in ("norm", "norm_bprop"):
        t, hq, hk, d = c["t"], c["hq"], c["hk"], c["d"]
        if c["fused"]:  # queries, keys and values side by side in a projection's output
            x = normal(t, hq + 2 * hk, d).mul_(channels(d, g, dev)).to(dt)
            s["q"], s["k"] = x[:, :hq], x[:, hq:hq + hk]
        else:
            s["q"] = normal(t, hq, d).mul_(channels(d, g, dev)).to(dt)
            s["k"] = normal(t, hk, d).mul_(channels(d, g, dev)).to(dt)
        s["qw"], s["kw"] = ((1 + 0.2 * normal(d)).to(dt) for _ in range(2))
        s["table"] = rotation_table(max(16384, t), c["rot"], dev)
        s["pos"] = torch.randint(0, 16384 - min(t, 8192), (1,), generator=g, device=dev, dtype=torch.int32) + torch.arange(
            t, device=dev, dtype=torch.int32) % 8192
        if c["op"] == "norm_bprop":
            s["dq"], s["dk"] = normal(t, hq, d).to(dt), normal(t, hk, d).to(dt)
        return s
    h, d, page, group = c["h" if c["op"] == "append" else "hk"], c["d"], c["page"], c["group"]
    if c["op"] == "append":
        t = c["t"]
        pages = -(-t // page) + 3
        if c["fused"]:
            x = normal(t, 2 * h, d).mul_(channels(d, g, dev)).to(dt)
            s["k"], s["v"] = x[:, :h], x[:, h:]
        else:
            s["k"], s["v"] = (normal(t, h, d).mul_(channels(d, g, dev)).to(dt) for _ in range(2))
        s["slots"] = page_slots(t, pages, page, g, dev)
        if not c["fused"]:  # padding tokens
            s["slots"] = torch.where(torch.rand(t, generator=g, device=dev) < 0.05, -1, s["slots"])
        for name in ("k", "v"):
            s[name + "_codes"] = torch.zeros(pages, h, page, d // 2, dtype=torch.uint8, device=dev)
            s[name + "_params"] = torch.zeros(pages, h, page, d // group, dtype=torch.int32, device=dev)
        return s
    b, lens = c["b"], lengths(c)
    per = -(-max(lens) // page) or 1
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + 2
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    held = torch.arange(per, device=dev)[None] < torch.tensor(counts, device=dev)[:, None]
    s["pages"] = torch.full((b, per), -1, dtype=torch.int32, device=dev)
    s["pages"][held] = order[:sum(counts)]
    # places of a last page that no token has reached hold what was there before: any bits
    filled = torch.zeros(pages, page, dtype=torch.bool, device=dev)
    at = torch.arange(per * page, device=dev).view(1, per, page) < s["lens"].view(b, 1, 1)
    filled[s["pages"][held].long()] = at[held]
    for name in ("k", "v"):
        codes = torch.empty(pages, h, page, d // 2, dtype=torch.uint8, device=dev)
        params = torch.empty(pages, h, page, d // group, dtype=torch.int32, device=dev)
        size = channels(h * d, g, dev).view(h, 1, d)
        step = max(1, (1 << 25) // (h * page * d))
        for i in range(0, pages, step):
            n = min(step, pages - i)
            cd, sc, z = quantize(normal(n, h, page, d).mul_(size), group)
            codes[i:i + n], params[i:i + n] = pair(cd), params_of(sc, z)
        params.masked_fill_(~filled[:, None, :, None], 0x7FC0)
        s[name + "_codes"], s[name + "_params"] = codes, params
    s["q"] = normal(b, c["tq"], c["hq"], d).to(dt)
    s["scale"] = d ** -0.5
    return s


def page_slots(t, pages, page, g, dev):
    """Slots of t consecutive tokens of one sequence whose pages lie anywhere."""
    order = torch.randperm(pages, generator=g, device=dev)
    i = torch.arange(t, device=dev)
    return order[i // page] * page + i % page


# --------------------------------------------------------------------------------------------- operators
def unpair(codes):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()


def values(codes, params, group):
    s = (params << 16).view(torch.float32)
    z = ((params >> 16) & 255).float()
    return ((unpair(codes).unflatten(-1, (-1, group)) - z[..., None]) * s[..., None]).flatten(-2)


def plain_linear(s):
    c = s["case"]
    n, k, group = c["n"], c["k"], c["group"]
    w = unpair(s["codes"])[:, :k]
    at = torch.arange(k, device=w.device) // group
    z = 8.0 if s["zeros"] is None else s["zeros"].float()[at].t()
    w = (w - z) * s["scales"].float()[at].t()
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def rotate(x, cos, sin, interleaved, back=False):
    rot = 2 * cos.shape[-1]
    head, rest = x[..., :rot], x[..., rot:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :rot // 2], head[..., rot // 2:])
    if back:
        sin = -sin
    a, b = a * cos - b * sin, b * cos + a * sin
    head = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([head, rest], -1)


def plain_norm(s):
    c = s["case"]
    cos, sin = s["table"][s["pos"].long()][:, None].chunk(2, -1)
    out = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        x = x.float()
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
        out.append(rotate(y, cos, sin, c["interleaved"]).to(w.dtype))
    return out


def plain_norm_bprop(s):
    c = s["case"]
    cos, sin = s["table"][s["pos"].long()][:, None].chunk(2, -1)
    dx, dw = [], []
    for x, w, dy in ((s["q"], s["qw"], s["dq"]), (s["k"], s["kw"], s["dk"])):
        x = x.float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        dn = rotate(dy.float(), cos, sin, c["interleaved"], back=True)
        dw.append((dn * x * r).sum((0, 1)).to(w.dtype))
        g = dn * w.float()
        dx.append((r * (g - x * r * r * (g * x).mean(-1, keepdim=True))).to(w.dtype))
    return dx + dw


def plain_append(s):
    c = s["case"]
    page, slots = c["page"], s["slots"]
    kept = (slots >= 0)[:, None, None]
    out = []
    for name in ("k", "v"):
        codes, sc, z = quantize(s[name].float(), c["group"])
        pg, at = slots.clamp(min=0) // page, slots.clamp(min=0) % page
        n = s[name + "_codes"].shape[0]
        # a padding token's row goes to a page of its own that is dropped
        pg = torch.where(slots >= 0, pg, n)
        for field, new in (("_codes", pair(codes)), ("_params", params_of(sc, z))):
            old = s[name + field]
            whole = torch.cat([old, old[:1]])
            whole[pg, :, at] = new
            old.copy_(whole[:n])
        pg = pg.clamp(max=n - 1)
        v = values(s[name + "_codes"][pg, :, at], s[name + "_params"][pg, :, at], c["group"])
        out.append(torch.where(kept, v, 0.0).to(s[name].dtype))
    return out


def plain_attention(s):
    c = s["case"]
    b, tq, hq, hk, d = c["b"], c["tq"], c["hq"], c["hk"], c["d"]
    at = s["pages"].clamp(min=0).long()
    total = at.shape[1] * c["page"]
    token = torch.arange(total, device=at.device)
    held = (token < s["lens"][:, None]).view(b, 1, total, 1)

    def gathered(name):  # [b, hk, tokens, d], zero where nothing is held
        codes, params = (s[name + f][at].permute(0, 2, 1, 3, 4).flatten(2, 3) for f in ("_codes", "_params"))
        return torch.where(held, values(codes, params, c["group"]), 0.0)

    q = s["q"].float().view(b, tq, hk, hq // hk, d).permute(0, 2, 1, 3, 4).flatten(2, 3)
    a = (q @ gathered("k").transpose(-1, -2)).mul_(s["scale"])
    until = s["lens"][:, None] - tq + 1 + torch.arange(tq, device=at.device)
    seen = (token < until[..., None]).view(b, 1, tq, 1, total)
    a = a.view(b, hk, tq, -1, total).masked_fill_(~seen, -math.inf)
    top = a.amax(-1, keepdim=True).clamp(min=-1e30)
    a = (a - top).exp_()
    total_weight = a.sum(-1, keepdim=True)
    o = a.flatten(2, 3) @ gathered("v")
    o = (o.view(b, hk, tq, -1, d) / total_weight.clamp(min=1e-30)).permute(0, 2, 1, 3, 4).reshape(b, tq, hq, d)
    lse = (top + total_weight.log()).squeeze(-1).permute(0, 2, 1, 3).reshape(b, tq, hq)
    return [o.to(s["q"].dtype), lse]


def own_linear(s):
    import my_own_cnn_b200 as b2q

    c = s["case"]
    w = b2q.W4Weight(s["codes"], s["scales"], s["zeros"], c["n"], c["k"], c["group"])
    return b2q.linear_w4(s["x"], w, s["bias"])


def own_norm(s):
    import my_own_cnn_b200 as b2q

    return b2q.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["table"], s["pos"], eps=1e-6,
                            interleaved=s["case"]["interleaved"])


def own_norm_bprop(s):
    import my_own_cnn_b200 as b2q

    return b2q.qk_norm_rope_bprop(s["dq"], s["dk"], s["q"], s["k"], s["qw"], s["kw"], s["table"], s["pos"], eps=1e-6,
                                  interleaved=s["case"]["interleaved"])


def own_append(s):
    import my_own_cnn_b200 as b2q

    cache = b2q.KV4Cache(s["k_codes"], s["k_params"], s["v_codes"], s["v_params"])
    b2q.kv4_append(cache, s["k"], s["v"], s["slots"])
    return b2q.kv4_read(cache, s["slots"], s["k"].dtype)


def own_attention(s):
    import my_own_cnn_b200 as b2q

    cache = b2q.KV4Cache(s["k_codes"], s["k_params"], s["v_codes"], s["v_params"])
    return b2q.kv4_attention(s["q"], cache, s["pages"], s["lens"], scale=s["scale"], return_lse=True)


PLAIN = {"linear": plain_linear, "norm": plain_norm, "norm_bprop": plain_norm_bprop, "append": plain_append,
         "attention": plain_attention}
OWN = {"linear": own_linear, "norm": own_norm, "norm_bprop": own_norm_bprop, "append": own_append,
       "attention": own_attention}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ----------------------------------------------------------------------------------- definitions, 64 bits
def exact(case, seed):
    s, c = prepare(case, seed), dict(case)
    if c["op"] == "linear":
        k = c["k"]
        y = torch.zeros(c["m"], c["n"], dtype=torch.float64, device="cuda")
        x = s["x"].double()
        for g0 in range(0, k, c["group"]):
            g1 = min(k, g0 + c["group"])
            by = s["codes"][:, g0 // 2:(g1 + 1) // 2].double()
            high = torch.floor(by / 16)
            low = by - 16 * high
            z = 8.0 if s["zeros"] is None else s["zeros"][g0 // c["group"]].double()
            even, odd = x[:, g0:g1:2], x[:, g0 + 1:g1:2]
            dot = even @ low.t() + odd @ high[:, :odd.shape[1]].t()
            y += (dot - z * x[:, g0:g1].sum(1, keepdim=True)) * s["scales"][g0 // c["group"]].double()
        return y if s["bias"] is None else y + s["bias"].double()
    if c["op"] in ("norm", "norm_bprop"):
        return exact_norm(s, c)
    if c["op"] == "append":
        out = []
        for name in ("k", "v"):
            x = s[name].double().reshape(c["t"], c["h"], c["d"] // c["group"], c["group"])
            low, high = x.min(-1).values.clamp_max(0), x.max(-1).values.clamp_min(0)
            # the scale is stored as bf16(fl32((high - low) * fl32(1 / 15))): the format's own roundings
            sc = ((high - low).float() * torch.tensor(1 / 15, dtype=torch.float32)).to(torch.bfloat16).double()
            z = torch.round(-low / sc)
            v = (torch.clamp(torch.round(x / sc[..., None]) + z[..., None], 0, 15) - z[..., None]) * sc[..., None]
            v[s["slots"] < 0] = 0
            out.append(v.reshape(c["t"], c["h"], c["d"]))
        return out
    b, tq, hq, hk, d = c["b"], c["tq"], c["hq"], c["hk"], c["d"]
    out = torch.zeros(b, tq, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, tq, hq), -math.inf, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lengths(c)):
        if n == 0:
            continue
        at = s["pages"][i, :-(-n // c["page"])].long()
        for h in range(hk):
            kv = []
            for name in ("k", "v"):
                by = s[name + "_codes"][at, h].reshape(-1, d // 2)[:n].to(torch.int16)
                bits = s[name + "_params"][at, h].reshape(-1, d // c["group"])[:n]
                x = torch.empty(n, d, dtype=torch.float64, device="cuda")
                x[:, 0::2], x[:, 1::2] = (by % 16).double(), (by // 16).double()
                sc = (bits % 65536).to(torch.int32).bitwise_left_shift(16).view(torch.float32).double()
                zero = (bits // 65536).double()
                kv.append((x - zero.repeat_interleave(c["group"], 1)) * sc.repeat_interleave(c["group"], 1))
            r = hq // hk
            for j in range(tq):
                m = n - tq + j + 1
                if m <= 0:
                    continue
                a = s["scale"] * (s["q"][i, j, h * r:(h + 1) * r].double() @ kv[0][:m].t())
                lse[i, j, h * r:(h + 1) * r] = torch.logsumexp(a, -1)
                out[i, j, h * r:(h + 1) * r] = torch.softmax(a, -1) @ kv[1][:m]
    return [out, lse]


def exact_norm(s, c):
    rot, d = c["rot"], c["d"]
    table = s["table"][s["pos"].long()].double()
    # the rotation of each pair of channels as multiplication by a complex number
    turn = torch.complex(table[:, :rot // 2], table[:, rot // 2:])[:, None]
    i = torch.arange(rot // 2, device="cuda")
    first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + rot // 2)

    def turned(x, by):
        y = x.clone()
        p = torch.complex(x[..., first], x[..., second]) * by
        y[..., first], y[..., second] = p.real, p.imag
        return y

    outs, grads = [], []
    for x, w, dy in ((s["q"], s["qw"], s.get("dq")), (s["k"], s["kw"], s.get("dk"))):
        x, w = x.double(), w.double()
        r = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) / d + 1e-6)
        if dy is None:
            outs.append(turned(x * r * w, turn))
            continue
        dn = turned(dy.double(), turn.conj())
        grads.append((dn * x * r).sum((0, 1)))
        gx = (dn * w * x).sum(-1, keepdim=True) / d
        outs.append(r * dn * w - r ** 3 * x * gx)
    return outs + grads
