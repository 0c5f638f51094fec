"""Rotary positions and cached attention: their plain forms, and the library's calls for them.

Four operators of a decoder with rotary positions and a key / value cache:

    rope        y = x turned by its position: pairs (a, b) of a head's first n_dims values become
                (a cos t - b sin t, a sin t + b cos t), t = position * frequency of the pair
    rope_back   the gradient of rope (the turn by -t)
    attn        softmax(scale * Q K^T + mask) V over a cache, with shared key / value heads,
                causal and ragged lengths, additive masks with per-head slopes, capped scores
    prefix      attn for sequences that share one long prefix: keys and values of the prefix are
                held once, each sequence has a cache of its own behind it

`run` computes the plain form in 32 bits (angles in 64) while `own` is false, and calls the
library while it is true. Tensors are laid out as a program keeps them: activations
[batch, token, head, dim], caches [batch, position, head, dim].
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    rope = dict(op="rope", batch=1, dim=128, n_dims=128, pairing="halves", src="f32", dst="f32", yarn=False, factors=False, last=8192)
    attn = dict(op="attn", batch=1, heads=32, kv_heads=8, dim=128, n_q=1, kv="f16", io="f16", causal=True, ragged=False, mask=False, bias=0.0, cap=0.0)
    prefix = dict(op="prefix", heads=32, kv_heads=8, dim=128, n_q=1, kv="f16", io="f16")
    return [
        # one new token of one sequence: the launch is all there is
        dict(rope, name="rope_token", tokens=1, heads=32),
        # the queries of a prompt, as the projection leaves them
        dict(rope, name="rope_prompt", tokens=4096, heads=32),
        # the keys of a long prompt, turned and rounded on their way into a 16-bit cache, positions
        # stretched past the trained context
        dict(rope, name="rope_into_cache", tokens=8192, heads=8, dst="f16", yarn=True, last=131072),
        # the gradient for a batch of prompts: neighbouring pairs, 32 of a head's 80 values turned
        dict(rope, name="rope_back_part", op="rope_back", batch=4, tokens=1000, heads=20, dim=80, n_dims=32, pairing="neighbours",
             src="bf16", dst="bf16", factors=True),
        # one token of a 12-head decoder with 64-value heads and a context of about a thousand
        dict(attn, name="attn_token", heads=12, kv_heads=12, dim=64, io="f32", n_kv=1000),
        # a serving batch: one token each, ragged contexts up to 8192
        dict(attn, name="attn_decode", batch=64, n_kv=8192, ragged=True),
        # one token of one sequence behind a very long context
        dict(attn, name="attn_long", n_kv=131072, kv="bf16", io="bf16"),
        # a long prompt
        dict(attn, name="attn_prompt", n_q=8192, n_kv=8192, kv="bf16", io="bf16"),
        # odd prompt lengths with a mask tensor and per-head slopes, 32-bit activations, 80-value heads
        dict(attn, name="attn_masked", batch=2, heads=16, kv_heads=16, dim=80, io="f32", n_q=777, n_kv=1900, causal=False, mask=True, bias=8.0),
        # a serving batch behind one system prompt
        dict(prefix, name="prefix_batch", seqs=64, prefix=8192, n_kv=512),
        # a few sequences behind a short prefix, 32-bit activations
        dict(prefix, name="prefix_few", seqs=3, heads=12, kv_heads=12, dim=64, io="f32", prefix=500, n_kv=60),
        # four draft tokens for each of 16 sequences behind a long document
        dict(prefix, name="prefix_draft", seqs=16, heads=32, kv_heads=4, n_q=4, prefix=32768, n_kv=1024, kv="bf16", io="bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    most = {"bytes": max(work(c)["bytes"] for c in listed()), "flops": max(work(c)["flops"] for c in listed())}
    while True:
        op = rng.choice(["rope", "rope", "rope_back", "attn", "attn", "attn", "prefix", "prefix"])
        if op in ("rope", "rope_back"):
            dim = 2 * rng.randint(8, 128)
            src = rng.choice(["f32", "f32", "f16", "bf16"])
            c = dict(op=op, batch=log(1, 8), tokens=log(1, 8192), heads=log(1, 64), dim=dim,
                     n_dims=dim if rng.random() < 0.6 else 2 * rng.randint(4, dim // 2), pairing=rng.choice(["halves", "neighbours"]),
                     src=src, dst="f16" if src == "f32" and rng.random() < 0.3 else src, yarn=rng.random() < 0.4,
                     factors=rng.random() < 0.3, last=log(8192, 1 << 20))
        else:
            kv_heads = log(1, 16)
            heads = kv_heads * rng.choice([1, 1, 2, 4, 4, 7, 8])
            dim = rng.choice([64, 64, 128, 128, 128, 256, 8 * rng.randint(4, 32)])
            kv, io = rng.choice([("f16", "f16"), ("bf16", "bf16"), ("f16", "f32")])
            c = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, kv=kv, io=io)
            if op == "attn":
                n_q = log(1, 8) if rng.random() < 0.5 else log(9, 4096)
                mask = rng.random() < 0.3
                c.update(batch=log(1, 64) if n_q <= 8 else log(1, 4), n_q=n_q, n_kv=n_q + log(1, 32768 if n_q <= 8 else 2048),
                         causal=not mask and rng.random() < 0.8, ragged=rng.random() < 0.5, mask=mask,
                         bias=8.0 if mask and rng.random() < 0.5 else 0.0, cap=30.0 if rng.random() < 0.2 else 0.0)
            else:
                n_q = log(1, 4)
                c.update(seqs=log(1, 96), n_q=n_q, prefix=log(16, 32768), n_kv=n_q + log(1, 1024))
        w = work(c)
        if all(w[k] <= most[k] for k in most) and _scores(c) <= 32 * 8192 * 8192:
            return c


def _scores(c):
    if c["op"] == "attn":
        return c["batch"] * c["heads"] * c["n_q"] * c["n_kv"]
    if c["op"] == "prefix":
        return c["seqs"] * c["heads"] * c["n_q"] * (c["prefix"] + c["n_kv"])
    return 0


def _least(c):
    """the shortest of a ragged batch's lengths"""
    return max(c["n_q"], c["n_kv"] // 2)


def work(c):
    if c["op"] in ("rope", "rope_back"):
        n = c["batch"] * c["tokens"] * c["heads"] * c["dim"]
        turned = c["batch"] * c["tokens"] * c["heads"] * c["n_dims"]
        return {"bytes": n * (SIZE[c["src"]] + SIZE[c["dst"]]) + 4 * c["tokens"], "flops": 3 * turned}
    kv, io, d = SIZE[c["kv"]], SIZE[c["io"]], c["dim"]
    if c["op"] == "attn":
        length = (c["n_kv"] + _least(c)) / 2 if c["ragged"] else c["n_kv"]
        seen = length - (c["n_q"] - 1) / 2 if c["causal"] else length   # keys of a mean row
        if c["mask"]:
            seen = seen - (c["n_q"] - 1) / 2                             # (the mask is causal too)
        rows = c["batch"] * c["heads"] * c["n_q"]
        b = 2 * rows * d * io + 2 * c["batch"] * c["kv_heads"] * length * d * kv + (2 * c["batch"] * c["n_q"] * c["n_kv"] if c["mask"] else 0)
        return {"bytes": b, "flops": 4 * rows * d * seen}
    length = (c["n_kv"] + _least(c)) / 2
    rows = c["seqs"] * c["heads"] * c["n_q"]
    b = 2 * rows * d * io + 2 * c["kv_heads"] * (c["prefix"] + c["seqs"] * length) * d * kv
    return {"bytes": b, "flops": 4 * rows * d * (c["prefix"] + length - (c["n_q"] - 1) / 2)}


# ---- inputs ------------------------------------------------------------------------------------


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype="f32", std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std).to(TYPES[dtype])

    def lengths(n):
        if c["op"] == "attn" and not c["ragged"]:
            return torch.full((n,), c["n_kv"], dtype=torch.int32, device="cuda")
        return torch.randint(_least(c), c["n_kv"] + 1, (n,), generator=g, device="cuda", dtype=torch.int32)

    s = {"case": c}
    if c["op"] in ("rope", "rope_back"):
        b, t, h, d = c["batch"], c["tokens"], c["heads"], c["dim"]
        s["x"] = normal(b, t, h, d, dtype=c["src"])
        first = int(torch.randint(0, c["last"] - t + 1, (1,), generator=g, device="cuda")) if c["last"] > t else 0
        s["pos"] = torch.arange(first, first + t, dtype=torch.int32, device="cuda")
        s["factors"] = 1.0 + 7.0 * torch.rand(c["n_dims"] // 2, generator=g, device="cuda") if c["factors"] else None
        # (a cache is longer than what one call writes: the rows of this call begin at row 7)
        if c["src"] != c["dst"]:
            s["cache"] = torch.zeros(b, t + 16, h, d, dtype=TYPES[c["dst"]], device="cuda")
            s["y"] = s["cache"][:, 7 : 7 + t]
        else:
            s["y"] = torch.empty(b, t, h, d, dtype=TYPES[c["dst"]], device="cuda")
        s["spec"] = dict(n_dims=c["n_dims"], freq_base=500000.0 if c["last"] > 8192 else 10000.0, n_ctx_orig=8192 if c["yarn"] else 0,
                         freq_scale=0.0625 if c["yarn"] else 1.0, ext_factor=1.0 if c["yarn"] else 0.0, attn_factor=1.0, beta_fast=32.0,
                         beta_slow=1.0)
        return s
    b = c["batch"] if c["op"] == "attn" else c["seqs"]
    s["scale"] = 1.0 / math.sqrt(c["dim"])
    # queries longer than the keys' norm asks for, so that some keys stand out
    s["q"] = normal(b, c["n_q"], c["heads"], c["dim"], dtype=c["io"], std=1.5)
    s["k"] = normal(b, c["n_kv"], c["kv_heads"], c["dim"], dtype=c["kv"])
    s["v"] = normal(b, c["n_kv"], c["kv_heads"], c["dim"], dtype=c["kv"])
    s["len"] = lengths(b)
    s["out"] = torch.empty(b, c["n_q"], c["heads"], c["dim"], dtype=TYPES[c["io"]], device="cuda")
    if c["op"] == "prefix":
        s["kp"] = normal(c["prefix"], c["kv_heads"], c["dim"], dtype=c["kv"])
        s["vp"] = normal(c["prefix"], c["kv_heads"], c["dim"], dtype=c["kv"])
        return s
    s["mask"] = None
    if c["mask"]:  # what a program with slopes passes: minus the distance, nothing behind the query
        i = torch.arange(c["n_kv"] - c["n_q"], c["n_kv"], device="cuda")[:, None]
        j = torch.arange(c["n_kv"], device="cuda")[None, :]
        far = -(i - j).float() if c["bias"] else torch.zeros(c["n_q"], c["n_kv"], device="cuda")
        far = far.masked_fill(j > i, -math.inf).expand(b, -1, -1).clone()
        hidden = torch.rand(b, 1, c["n_kv"], generator=g, device="cuda") < 0.1   # padding here and there
        s["mask"] = far.masked_fill(hidden, -math.inf).to(torch.float16)
    return s


# ---- the plain forms ---------------------------------------------------------------------------


def _frequencies(spec, device):
    """angle per position of each pair, in 64 bits, and the factor of the turned values"""
    n, base = spec["n_dims"], spec["freq_base"]
    i = torch.arange(n // 2, dtype=torch.float64, device=device)
    f = base ** (-2.0 * i / n)
    size = spec["attn_factor"]
    if spec["ext_factor"]:
        def turning(beta):
            return n * math.log(spec["n_ctx_orig"] / (beta * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(0, math.floor(turning(spec["beta_fast"]))), min(n - 1, math.ceil(turning(spec["beta_slow"])))
        kept = (1 - ((i - low) / max(0.001, high - low)).clamp(0, 1)) * spec["ext_factor"]
        f = f * (spec["freq_scale"] * (1 - kept) + kept)
        size *= 1 + 0.1 * math.log(1 / spec["freq_scale"])
    else:
        f = f * spec["freq_scale"]
    return f, size


def _plain_rope(s):
    c, x = s["case"], s["x"].float()
    n = c["n_dims"]
    f, size = _frequencies(s["spec"], x.device)
    if s["factors"] is not None:
        f = f / s["factors"].double()
    angle = s["pos"].double()[:, None] * f
    cos, sin = (angle.cos() * size).float()[:, None, :], (angle.sin() * size).float()[:, None, :]
    if c["op"] == "rope_back":
        sin = -sin
    y = x.clone()
    if c["pairing"] == "halves":
        a, b = x[..., : n // 2], x[..., n // 2 : n]
        y[..., : n // 2] = a * cos - b * sin
        y[..., n // 2 : n] = a * sin + b * cos
    else:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        y[..., 0:n:2] = a * cos - b * sin
        y[..., 1:n:2] = a * sin + b * cos
    s["y"].copy_(y)
    return s["y"]


def _grouped(q, kv_heads):
    """[b, i, h, d] -> [b, kv head, heads of the group * i, d], 32 bits"""
    b, n, h, d = q.shape
    return q.float().permute(0, 2, 1, 3).reshape(b, kv_heads, h // kv_heads * n, d)


def _plain_attn(s):
    c = s["case"]
    b, n, h, d = s["q"].shape
    hk, m = c["kv_heads"], c["n_kv"]
    k, v = s["k"].float().permute(0, 2, 1, 3), s["v"].float().permute(0, 2, 1, 3)
    x = torch.matmul(_grouped(s["q"], hk), k.transpose(2, 3)).mul_(s["scale"])
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    x = x.view(b, h, n, m)
    if s["mask"] is not None:
        add = s["mask"].float()[:, None]
        if c["bias"]:
            add = add * _slopes(h, c["bias"])[:, None, None]
        x += add
    j = torch.arange(m, device=x.device)
    seen = s["len"].long()[:, None, None]
    if c["causal"]:
        seen = seen - n + 1 + torch.arange(n, device=x.device)[:, None]
    x.masked_fill_((j >= seen)[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, hk, h // hk * n, m), v).view(b, h, n, d) / torch.where(total == 0, 1.0, total)
    s["out"].copy_(o.permute(0, 2, 1, 3))
    return s["out"]


def _slopes(heads, bias):
    """ALiBi's: a geometric sequence over the largest power of two of heads, its halves for the rest"""
    n = 1 << int(math.floor(math.log2(heads)))
    m0, m1 = 2.0 ** (-bias / n), 2.0 ** (-bias / 2 / n)
    return torch.tensor([m0 ** (i + 1) if i < n else m1 ** (2 * (i - n) + 1) for i in range(heads)], device="cuda")


def _plain_prefix(s):
    c = s["case"]
    b, n, h, d = s["q"].shape
    hk = c["kv_heads"]
    r = h // hk * n
    q = _grouped(s["q"], hk)
    kp, vp = s["kp"].float().permute(1, 0, 2), s["vp"].float().permute(1, 0, 2)
    k, v = s["k"].float().permute(0, 2, 1, 3), s["v"].float().permute(0, 2, 1, 3)
    shared = torch.matmul(q.permute(1, 0, 2, 3).reshape(hk, b * r, d), kp.transpose(1, 2)).view(hk, b, r, -1).transpose(0, 1)
    mine = torch.matmul(q, k.transpose(2, 3))
    j = torch.arange(c["n_kv"], device=q.device)
    seen = s["len"].long()[:, None, None] - n + 1 + torch.arange(n, device=q.device)[:, None]
    mine = mine.view(b, h, n, -1).masked_fill_((j >= seen)[:, None], -math.inf).view(b, hk, r, -1)
    p = torch.cat([shared, mine], -1).mul_(s["scale"])
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    front, back = p[..., : c["prefix"]], p[..., c["prefix"] :]
    o = torch.matmul(front.transpose(0, 1).reshape(hk, b * r, -1), vp).view(hk, b, r, d).transpose(0, 1) + torch.matmul(back, v)
    s["out"].copy_((o / total).reshape(b, h, n, d).permute(0, 2, 1, 3))
    return s["out"]


# ---- the library's calls -----------------------------------------------------------------------


def _described(s):
    """the library's descriptors of this state's buffers: a program makes them once for its buffers"""
    import os
    import sys

    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ggml-gfx906_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import mi355x_qmm as M

    c = s["case"]
    if c["op"] in ("rope", "rope_back"):
        spec = M.rope_spec(mode=M.ROPE_HALVES if c["pairing"] == "halves" else M.ROPE_NEIGHBOURS, **s["spec"])
        call = M.rope if c["op"] == "rope" else M.rope_back
        x, pos, y = M.from_torch(s["x"]), M.from_torch(s["pos"]), M.from_torch(s["y"])
        factors = None if s["factors"] is None else M.from_torch(s["factors"])
        return lambda: call(x, pos, y, spec, factors=factors)

    def heads_first(t):
        return M.from_torch(t.permute(0, 2, 1, 3))

    q, k, v, out, n = heads_first(s["q"]), heads_first(s["k"]), heads_first(s["v"]), M.from_torch(s["out"]), M.from_torch(s["len"])
    if c["op"] == "attn":
        spec = M.attn_spec(scale=s["scale"], max_bias=c["bias"], logit_softcap=c["cap"], causal=c["causal"])
        mask = None if s["mask"] is None else M.from_torch(s["mask"][:, None])
        return lambda: M.flash_attn(q, k, v, out, spec, mask=mask, kv_len=n)
    spec = M.attn_spec(scale=s["scale"], causal=True)
    kp, vp = M.from_torch(s["kp"].permute(1, 0, 2)), M.from_torch(s["vp"].permute(1, 0, 2))
    return lambda: M.flash_attn_prefix(q, kp, vp, k, v, out, spec, kv_len=n)


def run(s):
    if own:
        if "call" not in s:
            s["call"] = _described(s)
        s["call"]()
        return s["y"] if "y" in s else s["out"]
    return {"rope": _plain_rope, "rope_back": _plain_rope, "attn": _plain_attn, "prefix": _plain_prefix}[s["case"]["op"]](s)


# ---- the definitions in 64 bits ----------------------------------------------------------------


def _exact_rope(s):
    c, spec = s["case"], s["spec"]
    n = c["n_dims"]
    scale, size, low, high = spec["freq_scale"], spec["attn_factor"], 0.0, 0.0
    if spec["ext_factor"]:
        low, high = (n * math.log(spec["n_ctx_orig"] / (2 * math.pi * beta)) / math.log(spec["freq_base"]) / 2 for beta in (spec["beta_fast"], spec["beta_slow"]))
        low, high = max(0.0, float(math.floor(low))), min(n - 1.0, float(math.ceil(high)))
        size = size * (1.0 + 0.1 * math.log(1.0 / scale))
    turns = []
    for i in range(n // 2):
        f = spec["freq_base"] ** (-2.0 * i / n)
        ramp = min(1.0, max(0.0, (i - low) / max(0.001, high - low)))
        keep = (1.0 - ramp) * spec["ext_factor"]
        turns.append(f * scale * (1.0 - keep) + f * keep)
    turns = torch.tensor(turns, dtype=torch.float64, device="cuda")
    if s["factors"] is not None:
        turns /= s["factors"].double()
    angle = s["pos"].double().view(-1, 1, 1) * turns
    way = torch.polar(torch.full_like(angle, size), angle if c["op"] == "rope" else -angle)
    x = s["x"].double()
    head, tail = x[..., :n], x[..., n:]
    if c["pairing"] == "halves":
        z = torch.complex(head[..., : n // 2].contiguous(), head[..., n // 2 :].contiguous()) * way
        head = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], n // 2, 2).contiguous()) * way
        head = torch.view_as_real(z).flatten(-2)
    return torch.cat([head, tail], -1)


def _exact_attn(s):
    c = s["case"]
    b, n, h, d = s["q"].shape
    group = h // c["kv_heads"]
    out = torch.zeros(b, n, h, d, dtype=torch.float64, device="cuda")
    for i in range(b):
        own_len = int(s["len"][i])
        for head in range(h):
            k, v = s["k"][i, :own_len, head // group].double(), s["v"][i, :own_len, head // group].double()
            w = s["mask"][i, :, :own_len].double() if s.get("mask") is not None else torch.zeros(n, own_len, dtype=torch.float64, device="cuda")
            if c.get("bias"):
                p2 = 2 ** int(math.log2(h))
                w = w * (2.0 ** (-c["bias"] * (head + 1) / p2) if head < p2 else 2.0 ** (-c["bias"] / 2 * (2 * (head - p2) + 1) / p2))
            if c["op"] == "prefix" or c["causal"]:
                w = w + torch.full_like(w, -math.inf).triu(own_len - n + 1)
            if c["op"] == "prefix":
                k, v = torch.cat([s["kp"][:, head // group].double(), k]), torch.cat([s["vp"][:, head // group].double(), v])
                w = torch.cat([w.new_zeros(n, c["prefix"]), w], 1)
            x = s["q"][i, :, head].double() @ k.T.contiguous() * s["scale"]
            if c.get("cap"):
                x = (x / c["cap"]).tanh() * c["cap"]
            x = x + w
            p = (x - x.logsumexp(1, keepdim=True)).exp().nan_to_num(nan=0.0)   # (a row that sees nothing: zeros)
            out[i, :, head] = p @ v
    return out


def exact(c, seed):
    s = prepare(c, seed)
    return _exact_rope(s) if c["op"] in ("rope", "rope_back") else _exact_attn(s)
