"""Attention over a cache (ggml_mi355x_flash_attn) and behind a shared prefix
(ggml_mi355x_flash_attn_prefix) against the formula in 64 bits: types, head layouts, lengths from
none to long ones, odd sizes, strides, masks that leave rows empty, NaN in places that no row sees,
workspaces and captured graphs. Refusals run without a GPU (nothing is launched).

Tolerances. With u = 2^-24, S the largest scale * sum |q||k| of a row, X its largest |score| with the
mask, n keys, A = sum w |v| (w: the weights): a score is off by D u S (its sum) + 6 u X (scale, cap, factor
log2 e, mask, difference, exp2's argument), so a weight by that share of itself, doubled by the normalising
sum; exp2 and the running factors add 8 u; the sum over the keys n u A. A 16-bit result adds eps/2 A
(weights rounded before the product with v) and eps/2 |o|. Summed that is `bound`; the mean square of the
errors is held to the same with square roots in place of D and n (roundings that do not conspire)."""
import ctypes as C
import math

import numpy as np
import pytest

import mi355x_qmm as M

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PAIRS = [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32")]   # cache, activations
IDS = ["f16", "bf16", "f16-f32"]
U = 2.0**-24
NAN, INF = float("nan"), float("inf")


def rnd(shape, dtype, seed, std=1.0):
    x = np.random.default_rng(seed).standard_normal(shape).astype(np.float32) * std
    return torch.from_numpy(x).cuda().to(TYPES[dtype])


def slopes(H, bias):
    n = 1 << int(math.log2(H))
    return torch.tensor([2.0 ** (-bias / n * (h + 1)) if h < n else 2.0 ** (-bias / 2 / n * (2 * (h - n) + 1)) for h in range(H)],
                        dtype=torch.float64, device="cuda")


def formula(q, k, v, scale, lens, causal=False, mask=None, bias=0.0, cap=0.0, sinks=None, kp=None, vp=None):
    """o [B, n_q, H, D] and the allowances (elementwise, mean square per element), in 64 bits. q [B, n_q, H, D],
    k, v [B or fewer, n_kv, Hk, D], mask [B', H', n_q, n_kv]; unseen keys are left out, not weighted with 0"""
    B, n, H, D = q.shape
    io = q.dtype
    rep = B // k.shape[0]
    q = q.double()
    k, v = (t.double().repeat_interleave(rep, 0) for t in (k, v))
    m = k.shape[1]
    seen = torch.arange(m, device="cuda")[None, None, :] < lens.long()[:, None, None]
    if causal:
        seen = seen & (torch.arange(m, device="cuda") <= lens.long()[:, None, None] - n + torch.arange(n, device="cuda")[:, None])
    seen = seen[:, None].expand(B, H, n, m).clone()
    add = torch.zeros(B, H, n, m, dtype=torch.float64, device="cuda")
    if mask is not None:
        w = mask.double().repeat(B // mask.shape[0], H // mask.shape[1], 1, 1)
        seen &= w != -INF
        add = torch.where(w == -INF, 0.0, w) * (slopes(H, bias)[:, None, None] if bias else 1.0)
    if kp is not None:
        P = kp.shape[0]
        k, v = (torch.cat([p.double()[None].expand(B, -1, -1, -1), t], 1) for p, t in ((kp, k), (vp, v)))
        seen = torch.cat([torch.ones(B, H, n, P, dtype=torch.bool, device="cuda"), seen], -1)
        add = torch.cat([torch.zeros(B, H, n, P, dtype=torch.float64, device="cuda"), add], -1)
    g = H // k.shape[2]
    k, v = (t.repeat_interleave(g, 2).permute(0, 2, 1, 3) for t in (k, v))
    # (a key that no row sees may hold anything)
    used = seen.any(2)[..., None]
    k, v = torch.where(used, k, 0.0), torch.where(used, v, 0.0)
    qh = q.permute(0, 2, 1, 3)
    x = (qh @ k.transpose(2, 3).contiguous()) * scale
    size = ((qh.abs() @ k.abs().transpose(2, 3).contiguous()) * abs(scale)).masked_fill(~seen, 0).amax(-1) if x.shape[-1] else torch.zeros(B, H, n, dtype=torch.float64, device="cuda")
    if cap:
        x = cap * torch.tanh(x / cap)
    x = x + add
    big = x.abs().masked_fill(~seen, 0).amax(-1) if x.shape[-1] else torch.zeros_like(size)
    x = x.masked_fill(~seen, -INF)
    top = x.amax(-1, keepdim=True) if x.shape[-1] else torch.full((B, H, n, 1), -INF, dtype=torch.float64, device="cuda")
    if sinks is not None:
        top = torch.maximum(top, sinks.double()[:, None, None])
    top = torch.where(top == -INF, 0.0, top)
    p = (x - top).exp()
    total = p.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + (sinks.double()[:, None, None] - top).exp()
    w = p / torch.where(total == 0, 1.0, total)
    o, A = w @ v, w @ v.abs()
    keys = x.shape[-1]

    def allowed(d, ks):
        off = (2 * (d * size + 6 * big) + 8 + ks)[..., None] * U * A
        if io != torch.float32:
            e = torch.finfo(io).eps / 2
            off = off + e * A + e * o.abs() + torch.finfo(io).tiny * torch.finfo(io).eps
        return off.permute(0, 2, 1, 3)

    return o.permute(0, 2, 1, 3), allowed(D, keys), allowed(math.sqrt(D), math.sqrt(max(1, keys)))


def near(got, want):
    o, most, mean = want
    off = (got.double() - o).abs()
    assert torch.isfinite(got).all()
    assert (off <= most).all(), (float((off - most).max()), (off > most).nonzero()[:4].tolist())
    assert float(off.square().mean()) <= float(mean.square().mean()), (float(off.square().mean()) ** 0.5, float(mean.square().mean()) ** 0.5)


def call(q, k, v, scale, lens=None, causal=False, mask=None, bias=0.0, cap=0.0, sinks=None, kp=None, vp=None, work=None, out=None, stream=None):
    out = torch.full_like(q, NAN) if out is None else out
    hf = lambda t: M.from_torch(t.permute(0, 2, 1, 3))  # noqa: E731
    spec = M.attn_spec(scale, bias, cap, causal)
    opt = dict(sinks=None if sinks is None else M.from_torch(sinks), kv_len=None if lens is None else M.from_torch(lens), work=work, stream=stream)
    if kp is not None:
        M.flash_attn_prefix(hf(q), M.from_torch(kp.permute(1, 0, 2)), M.from_torch(vp.permute(1, 0, 2)), hf(k), hf(v), M.from_torch(out), spec, **opt)
    else:
        M.flash_attn(hf(q), hf(k), hf(v), M.from_torch(out), spec, mask=None if mask is None else M.from_torch(mask), **opt)
    torch.cuda.synchronize()
    return out


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def full(B, n):
    return torch.full((B,), n, dtype=torch.int32, device="cuda")


def operands(B, n, m, H, Hk, D, kv, io, seed=0, Bk=None):
    return rnd((B, n, H, D), io, seed, 1.5), rnd((Bk or B, m, Hk, D), kv, seed + 1), rnd((Bk or B, m, Hk, D), kv, seed + 2)


SIZES = [
    # B, n_q, n_kv, H, Hk, D
    (1, 1, 1, 1, 1, 8), (1, 1, 2, 4, 4, 64), (2, 1, 31, 8, 2, 128), (1, 1, 32, 8, 1, 64), (1, 1, 33, 12, 12, 64), (3, 1, 64, 7, 1, 128),
    (1, 1, 65, 32, 8, 128), (1, 1, 1000, 32, 8, 128), (2, 1, 129, 16, 1, 256), (1, 1, 257, 64, 2, 80), (1, 1, 5000, 4, 1, 128), (5, 1, 700, 32, 4, 64),
    (1, 2, 100, 8, 2, 128), (2, 3, 77, 21, 3, 96), (1, 4, 300, 32, 4, 128), (1, 8, 40, 8, 8, 72), (2, 5, 511, 16, 1, 64), (1, 17, 17, 8, 2, 64),
    (1, 31, 200, 2, 2, 40), (1, 33, 65, 4, 2, 128), (2, 64, 64, 3, 1, 128), (1, 127, 333, 8, 8, 64), (1, 130, 1025, 4, 1, 256), (1, 200, 200, 2, 2, 192),
    (1, 257, 300, 6, 2, 128), (2, 300, 300, 5, 5, 16), (1, 1, 128, 71, 1, 64), (1, 40, 90, 71, 71, 64), (1, 513, 900, 4, 2, 80),
]


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_matches_formula(size, kv, io):
    B, n, m, H, Hk, D = size
    q, k, v = operands(B, n, m, H, Hk, D, kv, io, seed=sum(size))
    s = 1 / math.sqrt(D)
    near(call(q, k, v, s), formula(q, k, v, s, full(B, m)))
    near(call(q, k, v, s, causal=True), formula(q, k, v, s, full(B, m), causal=True))


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("n", [1, 3, 40, 150])
@pytest.mark.parametrize("causal", [False, True])
def test_ragged_lengths_and_rows_without_keys(kv, io, n, causal):
    """lengths 0, 1, below n_q (causal: the first rows see nothing), around tile ends, full, and outside
    0 .. n_kv (clamped); what lies behind a length is NaN"""
    m = 400
    want_len = [0, 1, 2, 31, 32, 33, 39, 63, 64, 65, 128, 149, 151, 300, 399, 400]
    B = len(want_len) + 2
    q, k, v = operands(B, n, m, 8, 2, 64, kv, io, seed=n)
    clamped = ints(*want_len, 0, m)
    for b, c in enumerate(clamped.tolist()):
        k[b, c:], v[b, c:] = NAN, NAN
    lens = ints(*want_len, -7, 100000)
    got = call(q, k, v, 0.125, lens, causal=causal)
    near(got, formula(q, k, v, 0.125, clamped, causal=causal))
    assert (got[0] == 0).all() and (got[-2] == 0).all()
    if causal and n > 1:
        assert (got[1, : n - 1] == 0).all()


def mask_of(B, H, n, m, seed, width=None):
    """finite values, hidden keys, rows that hide everything, a row of the type's lowest value"""
    r = np.random.default_rng(seed)
    w = r.standard_normal((B, H, n, width or m)).astype(np.float16)
    w[r.random(w.shape) < 0.3] = -np.inf
    w[:, :, n // 2] = -np.inf
    w[:, :, n - 1] = np.float16(-65504)
    if n > 3:
        w[:, :, 0, : m - 1] = -np.inf          # one key left
        w[:, :, 1, min(m, 64):] = -np.inf      # the first keys only
    return torch.from_numpy(w).cuda()


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("n,m", [(1, 1), (1, 77), (4, 33), (7, 200), (65, 130), (150, 333), (129, 640)])
@pytest.mark.parametrize("bias", [0.0, 8.0])
@pytest.mark.parametrize("planes", [(1, 1), (2, 6), (1, 2), (2, 1)])
def test_masks(kv, io, n, m, bias, planes):
    """planes: the mask's batches and heads; wider than n_kv, so its rows have any alignment"""
    q, k, v = operands(2, n, m, 6, 2, 64, kv, io, seed=n + m)
    w = mask_of(planes[0], planes[1], n + 2, m, 5, width=m + 3)[:, :, 1 : n + 1]
    near(call(q, k, v, 0.125, mask=w, bias=bias), formula(q, k, v, 0.125, full(2, m), mask=w[..., :m], bias=bias))
    lens = ints(m // 2, m)
    near(call(q, k, v, 0.125, lens, causal=True, mask=w, bias=bias), formula(q, k, v, 0.125, lens, causal=True, mask=w[..., :m], bias=bias))


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("n", [1, 6, 300])
def test_masks_that_hide_whole_tiles(kv, io, n):
    """several sequences in one cache: each row sees a stretch of it somewhere, and what lies between is hidden
    from every row (and NaN)"""
    m = 1100
    q, k, v = operands(1, n, m, 8, 2, 64, kv, io, seed=2)
    w = torch.full((1, 1, n, m), -INF, dtype=torch.float16, device="cuda")
    for i in range(n):
        first = 700 if i % 3 == 0 else 100 + i % 7
        w[0, 0, i, first : first + 60 + i % 50] = 0.25 * (i % 4)
    dead = (w == -INF).all(2)[0, 0]
    k[:, dead], v[:, dead] = NAN, NAN
    near(call(q, k, v, 0.125, mask=w), formula(q, k, v, 0.125, full(1, m), mask=w))


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("n", [1, 4, 40, 140])
def test_unseen_keys_may_hold_anything(kv, io, n):
    """NaN and infinities in keys that the mask hides from some rows or the causal rule hides from the first:
    those rows are what they are without them"""
    m = 260
    q, k, v = operands(1, n, m, 4, 2, 128, kv, io, seed=3)
    hidden = torch.zeros(m, dtype=torch.bool)
    hidden[[0, 5, 31, 32, 100, 255, 259]] = True
    w = torch.zeros(1, 1, n, m, dtype=torch.float16, device="cuda")
    w[..., hidden.cuda()] = -INF
    bad = [t.clone() for t in (k, v)]
    for t, what in ((bad[0], [NAN, INF, -INF, NAN, INF, NAN, NAN]), (bad[1], [INF, NAN, NAN, -INF, NAN, INF, NAN])):
        for j, x in zip(hidden.nonzero().flatten().tolist(), what):
            t[:, j] = x
    near(call(q, bad[0], bad[1], 0.1, mask=w), formula(q, k, v, 0.1, full(1, m), mask=w))
    if n > 1:   # the last key is NaN: the causal rule keeps it from every row but the last
        k2, v2 = k.clone(), v.clone()
        k2[:, -1], v2[:, -1] = NAN, NAN
        got = call(q, k2, v2, 0.1, causal=True)
        o, most, _ = formula(q, k, v, 0.1, full(1, m), causal=True)
        assert torch.isnan(got[:, -1]).all() and ((got.double() - o).abs() <= most)[:, :-1].all()


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
def test_nan_and_infinity_that_a_row_sees(kv, io):
    """they reach that row, value for value as in the formula, and no other row"""
    q, k, v = operands(1, 40, 100, 2, 1, 64, kv, io, seed=9)
    q[0, 7, 1] = NAN
    v[0, 70, 0, 3], v[0, 80, 0, 5] = INF, -INF
    got = call(q, k, v, 0.125)
    assert torch.isnan(got[0, 7, 1]).all()
    keep = torch.ones(40, 2, dtype=torch.bool)
    keep[7, 1] = False
    rows = got[0][keep.cuda()]
    assert (rows[:, 3] == INF).all() and (rows[:, 5] == -INF).all()
    others = [i for i in range(64) if i not in (3, 5)]
    q2 = q.clone()
    q2[0, 7, 1] = 0
    o, most, _ = formula(q2, k, torch.where(torch.isfinite(v), v, 0), 0.125, full(1, 100))
    assert ((rows.double() - o[0][keep.cuda()]).abs() <= most[0][keep.cuda()])[:, others].all()


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("n", [1, 9, 150])
def test_negative_scale_under_a_cap(kv, io, n):
    q, k, v = operands(2, n, 333, 6, 2, 64, kv, io, seed=41)
    w = rnd((1, 1, n, 333), "f16", 42)
    kp, vp = rnd((100, 2, 64), kv, 43), rnd((100, 2, 64), kv, 44)
    for scale in (-0.125, -1.0):
        near(call(q, k, v, scale, cap=7.0), formula(q, k, v, scale, full(2, 333), cap=7.0))
        near(call(q, k, v, scale, cap=7.0, mask=w, causal=True), formula(q, k, v, scale, full(2, 333), cap=7.0, mask=w, causal=True))
        near(call(q, k, v, scale, cap=7.0, kp=kp, vp=vp), formula(q, k, v, scale, full(2, 333), cap=7.0, kp=kp, vp=vp))


LAUNCHES = [
    # B, n_q, n_kv, H, Hk, D: few row tiles, one for each CU, several (workgroups of 4 and 8 waves, their tiles of keys
    # shared or taken in turns, the keys split or not)
    (1, 300, 3000, 8, 2, 64), (1, 515, 1031, 16, 4, 128), (1, 300, 1500, 32, 8, 96), (1, 1024, 1030, 32, 8, 128), (1, 2049, 2049, 16, 8, 88),
    (2, 2048, 2050, 32, 4, 64), (2, 2048, 2048, 32, 4, 128), (4, 700, 900, 32, 8, 96), (2, 777, 1900, 16, 16, 80), (1, 600, 1000, 16, 2, 256),
    (1, 1000, 1500, 32, 8, 160), (2, 1500, 1500, 16, 16, 192), (3, 5, 900, 16, 2, 136),
]


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("size", LAUNCHES, ids=lambda s: "x".join(map(str, s)))
def test_row_tiles_of_every_launch(size, kv, io):
    """plain, causal with ragged lengths (one of none) and sinks, and masked with a cap, hidden NaN and rows that see
    nothing"""
    B, n, m, H, Hk, D = size
    q, k, v = operands(B, n, m, H, Hk, D, kv, io, seed=sum(size))
    s = 1 / math.sqrt(D)
    near(call(q, k, v, s), formula(q, k, v, s, full(B, m)))
    lens = torch.tensor([0 if i == 3 else max(0, m - 333 * i) for i in range(B)], dtype=torch.int32, device="cuda")
    sinks = rnd((H,), "f32", 5)
    near(call(q, k, v, s, lens=lens, causal=True, sinks=sinks), formula(q, k, v, s, lens, causal=True, sinks=sinks))
    w = rnd((1, 1, n, m), "f16", 8)
    w[0, 0, :, 5::3] = -INF
    w[0, 0, n // 2, :] = -INF
    w[0, 0, : min(n, 200), 128 : 128 + m // 2] = -INF
    k[:, 5::3], v[:, 5::3] = NAN, NAN
    near(call(q, k, v, s, mask=w, cap=20.0), formula(q, k, v, s, full(B, m), mask=w, cap=20.0))
    near(call(q, k, v, s, mask=w, bias=4.0), formula(q, k, v, s, full(B, m), mask=w, bias=4.0))


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("scale", [0.0, 1e-25, -0.125, 3.0e6])
def test_masks_beside_extreme_scales(kv, io, scale):
    """products that next to nothing or far too much multiplies, next to a finite mask"""
    q, k, v = operands(1, 70, 90, 2, 1, 64, kv, io, seed=31)
    w = (rnd((1, 1, 70, 90), "f32", 32) * 50).to(torch.float16)
    w[..., ::4] = -1000
    w[..., 1::9] = -INF
    near(call(q, k, v, scale, mask=w), formula(q, k, v, scale, full(1, 90), mask=w))


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("n", [1, 7, 1500])
@pytest.mark.parametrize("what", ["q", "k", "v", "all"])
def test_nan_throughout(kv, io, n, what):
    """rows that see NaN only, or behind the second key, are NaN; rows that see none of it are what they are"""
    q, k, v = operands(2, n, 1600, 8, 2, 128, kv, io, seed=n)
    kp, vp = rnd((300, 2, 128), kv, 51), rnd((300, 2, 128), kv, 52)
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if what in (name, "all"):
            t[:] = NAN
    assert torch.isnan(call(q, k, v, 0.09)).all() and torch.isnan(call(q, k, v, 0.09, kp=kp, vp=vp)).all()
    if what in ("k", "v"):
        q, k, v = operands(2, n, 1600, 8, 2, 128, kv, io, seed=n)
        (k if what == "k" else v)[:, 2:] = NAN
        lens = ints(1600, min(2, n))
        got = call(q, k, v, 0.09, lens, causal=True)
        assert torch.isnan(got[0]).all()
        o, most, _ = formula(q, k[:, :2], v[:, :2], 0.09, ints(2, min(2, n)), causal=True)
        assert ((got[1].double() - o[1]).abs() <= most[1]).all()


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("n", [1, 50])
def test_cap_sinks_and_large_scores(kv, io, n):
    q, k, v = operands(2, n, 150, 8, 2, 64, kv, io, seed=21)
    lens = ints(0, 150)
    sinks = torch.linspace(-30, 30, 8, device="cuda")
    near(call(q, k, v, 0.5, cap=20.0), formula(q, k, v, 0.5, full(2, 150), cap=20.0))
    near(call(q, k, v, 0.125, lens, sinks=sinks), formula(q, k, v, 0.125, lens, sinks=sinks))
    near(call(q, k, v, -0.125), formula(q, k, v, -0.125, full(2, 150)))
    near(call(q, k, v, 0.0), formula(q, k, v, 0.0, full(2, 150)))
    # scores in the hundreds, of both signs: the weights of all but a few keys underflow
    near(call(q * 8, k * 4, v, 1.0), formula(q * 8, k * 4, v, 1.0, full(2, 150)))


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
def test_running_maximum(kv, io):
    """scores that rise to the end, fall from the start, and one that stands out anywhere"""
    m, D = 700, 64
    v = rnd((1, m, 1, D), kv, 1)
    q = torch.zeros(1, 3, 1, D, dtype=TYPES[io], device="cuda")
    q[..., 0] = 1
    for x in (torch.linspace(-60, 60, m), torch.linspace(60, -60, m), torch.zeros(m).index_fill(0, torch.tensor([333]), 50.0)):
        k = torch.zeros(1, m, 1, D, dtype=TYPES[kv], device="cuda")
        k[0, :, 0, 0] = x.cuda().to(TYPES[kv])
        near(call(q, k, v, 1.0), formula(q, k, v, 1.0, full(1, m)))


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("n", [1, 70])
def test_layouts(kv, io, n):
    """heads outside positions, padded rows, slices of wider tensors, one cache for several batches"""
    B, m, H, Hk, D = 4, 190, 8, 2, 80
    q = rnd((B, H, n + 1, D + 16), io, 1, 1.5)[:, :, 1:, 8 : 8 + D].permute(0, 2, 1, 3)
    k = rnd((2, Hk, m + 5, D + 8), kv, 2)[:, :, 5:, :D].permute(0, 2, 1, 3)
    v = rnd((2, m, 3 * Hk, D), kv, 3)[:, :, Hk : 2 * Hk]
    buf = torch.full((B, n + 2, H + 1, D + 8), 3.0, dtype=TYPES[io], device="cuda")
    out = buf[:, 1:-1, :H, :D]
    near(call(q, k, v, 0.11, causal=True, out=out), formula(q, k, v, 0.11, full(B, m), causal=True))
    out.fill_(3.0)
    assert (buf == 3.0).all()


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
def test_offsets_past_32_bits(kv, io):
    """a cache whose heads lie 5 GiB apart, and positions far enough apart that the last begin past 4 GiB"""
    D, m = 64, 33
    store = torch.empty(9 * 2**30 // 2, dtype=TYPES[kv], device="cuda")
    for strides in ((D, 5 * 2**29, 0), (2**31 // 16, 64, 0)):
        k = torch.as_strided(store, (1, m, 2, D), (0, strides[0], strides[1], 1))
        v = torch.as_strided(store, (1, m, 2, D), (0, strides[0], strides[1], 1), 4096)
        k.copy_(rnd((1, m, 2, D), kv, 1))
        v.copy_(rnd((1, m, 2, D), kv, 2))
        for n in (1, 40):
            q = rnd((1, n, 4, D), io, 3, 1.5)
            near(call(q, k, v, 0.125), formula(q, k.contiguous(), v.contiguous(), 0.125, full(1, m)))


PREFIXES = [
    # sequences, n_q, prefix, n_kv, H, Hk, D
    (1, 1, 1, 1, 1, 1, 64), (3, 1, 500, 60, 12, 12, 64), (2, 1, 0, 50, 8, 2, 128), (5, 1, 33, 1, 8, 1, 128), (64, 1, 300, 40, 8, 2, 128),
    (4, 4, 1000, 70, 32, 4, 128), (2, 3, 64, 3, 7, 1, 80), (17, 1, 129, 31, 16, 4, 256), (1, 8, 4100, 20, 8, 2, 64), (9, 2, 257, 300, 14, 2, 96),
    (40, 1, 2000, 100, 32, 8, 64), (3, 40, 200, 50, 4, 2, 128), (130, 1, 70, 5, 1, 1, 64),
    (1, 1, 40, 9000, 8, 2, 128), (2, 3, 700, 5000, 8, 1, 64), (1, 50, 300, 4000, 8, 2, 128), (57, 3, 700, 20, 21, 3, 144), (4, 20, 500, 90, 8, 2, 192),   # long caches behind the prefix
]


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("size", PREFIXES, ids=lambda s: "x".join(map(str, s)))
def test_shared_prefix(size, kv, io):
    B, n, P, m, H, Hk, D = size
    q, k, v = operands(B, n, m, H, Hk, D, kv, io, seed=sum(size))
    kp, vp = rnd((P, Hk, D), kv, 7), rnd((P, Hk, D), kv, 8)
    s = 1 / math.sqrt(D)
    lens = torch.from_numpy(np.random.default_rng(1).integers(0, m + 1, B).astype(np.int32)).cuda()
    lens[0] = m
    for b, c in enumerate(lens.tolist()):
        k[b, c:], v[b, c:] = NAN, NAN
    for causal in (True, False):
        near(call(q, k, v, s, lens, causal=causal, kp=kp, vp=vp), formula(q, k, v, s, lens, causal=causal, kp=kp, vp=vp))


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
def test_prefix_equals_a_joined_cache(kv, io):
    """with sinks and a cap: the same as attention over the prefix copied before every own cache, to the
    allowance of either"""
    B, n, P, m, H, Hk, D = 3, 2, 210, 45, 8, 2, 64
    q, k, v = operands(B, n, m, H, Hk, D, kv, io, seed=5)
    kp, vp = rnd((P, Hk, D), kv, 7), rnd((P, Hk, D), kv, 8)
    sinks = torch.linspace(-4, 4, H, device="cuda")
    lens = ints(2, 30, 45)
    k2, v2 = (torch.cat([p[None].expand(B, -1, -1, -1), t], 1) for p, t in ((kp, k), (vp, v)))
    a = call(q, k, v, 0.125, lens, causal=True, cap=15.0, sinks=sinks, kp=kp, vp=vp)
    b = call(q, k2, v2, 0.125, lens + P, causal=True, cap=15.0, sinks=sinks)
    want = formula(q, k, v, 0.125, lens, causal=True, cap=15.0, sinks=sinks, kp=kp, vp=vp)
    near(a, want)
    near(b, want)


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("case", ["token", "prompt", "prefix"])
def test_repeats_bit_for_bit(kv, io, case):
    n, m = (1, 3000) if case != "prompt" else (200, 500)
    q, k, v = operands(2, n, m, 8, 2, 128, kv, io, seed=31)
    more = dict(kp=rnd((900, 2, 128), kv, 7), vp=rnd((900, 2, 128), kv, 8)) if case == "prefix" else {}
    first = call(q, k, v, 0.09, causal=True, **more)
    for _ in range(3):
        assert torch.equal(first, call(q, k, v, 0.09, causal=True, **more))


@gpu
@pytest.mark.parametrize("prefix", [False, True])
def test_callers_workspace_capture_and_replay(prefix):
    """two graphs with workspaces of their own, replayed at the same time on two streams; lengths change
    between replays"""
    graphs = []
    for seed in (1, 2):
        q, k, v = operands(2, 1, 4000, 8, 2, 128, "f16", "f16", seed=seed)
        kp, vp = (rnd((3000, 2, 128), "f16", seed + 9), rnd((3000, 2, 128), "f16", seed + 8)) if prefix else (None, None)
        hf = lambda t: M.from_torch(t.permute(0, 2, 1, 3))  # noqa: E731
        n = M.flash_attn_prefix_work_size(hf(q), M.from_torch(kp.permute(1, 0, 2)), hf(k)) if prefix else M.flash_attn_work_size(hf(q), hf(k))
        work = torch.empty(max(16, n), dtype=torch.uint8, device="cuda")
        lens, out = ints(4000, 17), torch.zeros_like(q)
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        keep = (M.from_torch(out), M.from_torch(lens))
        spec = M.attn_spec(0.09, causal=True)
        with torch.cuda.graph(g, stream=s):
            if prefix:
                M.flash_attn_prefix(hf(q), M.from_torch(kp.permute(1, 0, 2)), M.from_torch(vp.permute(1, 0, 2)), hf(k), hf(v), keep[0], spec,
                                    kv_len=keep[1], work=work, stream=s)
            else:
                M.flash_attn(hf(q), hf(k), hf(v), keep[0], spec, kv_len=keep[1], work=work, stream=s)
        graphs.append((g, s, q, k, v, kp, vp, lens, out, work))
    for r in range(4):
        for g, s, q, k, v, kp, vp, lens, out, work in graphs:
            q.normal_()
            lens.copy_(ints(4000 - 900 * r, 17 + 500 * r))
            out.zero_()
        torch.cuda.synchronize()
        for g, s, *_ in graphs:
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        for g, s, q, k, v, kp, vp, lens, out, work in graphs:
            assert torch.equal(out, call(q, k, v, 0.09, lens, causal=True, kp=kp, vp=vp))


@gpu
@pytest.mark.parametrize("small_first", [True, False])
def test_graph_keeps_its_workspace(small_first):
    """a call captured with the library's workspace is replayed after a later call on its stream needed a larger one"""
    q, k, v = operands(2, 1, 4000, 8, 2, 128, "f16", "f16", seed=4)
    big = operands(256, 4, 20, 32, 4, 128, "f16", "f16", seed=5)
    kp, vp = rnd((8000, 4, 128), "f16", 6), rnd((8000, 4, 128), "f16", 7)
    hf = lambda t: M.from_torch(t.permute(0, 2, 1, 3))  # noqa: E731
    need = M.flash_attn_work_size(hf(q), hf(k))
    assert 0 < need < 16 << 20 < M.flash_attn_prefix_work_size(hf(big[0]), M.from_torch(kp.permute(1, 0, 2)), hf(big[1]))
    s, out = torch.cuda.Stream(), torch.zeros_like(q)
    torch.cuda.synchronize()
    want = call(q, k, v, 0.09, stream=s)
    g = torch.cuda.CUDAGraph()
    d, spec = M.from_torch(out), M.attn_spec(0.09)
    with torch.cuda.graph(g, stream=s):
        M.flash_attn(hf(q), hf(k), hf(v), d, spec, stream=s)
    if not small_first:
        g.replay()
        torch.cuda.synchronize()
    large = call(*big, 0.09, kp=kp, vp=vp, stream=s)
    assert torch.equal(large, call(*big, 0.09, kp=kp, vp=vp))
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(large, call(*big, 0.09, kp=kp, vp=vp, stream=s))


@gpu
def test_streams_and_threads():
    """calls on two streams, and from two host threads on one, each with the library's workspace"""
    import threading

    sets = [operands(2, 1, 5000 + 1000 * i, 8, 2, 128, "f16", "f16", seed=i) for i in range(2)]
    want = [call(*s, 0.09) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    outs = [torch.zeros_like(s[0]) for s in sets]
    torch.cuda.synchronize()
    hf = lambda t: M.from_torch(t.permute(0, 2, 1, 3))  # noqa: E731
    for _ in range(8):
        for s, st, out in zip(sets, streams, outs):
            M.flash_attn(hf(s[0]), hf(s[1]), hf(s[2]), M.from_torch(out), M.attn_spec(0.09), stream=st)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    bad = []

    def worker(i):
        try:
            for _ in range(8):
                if not torch.equal(call(*sets[i], 0.09), want[i]):
                    bad.append(i)
        except Exception as e:  # noqa: BLE001
            bad.append(repr(e))

    ts = [threading.Thread(target=worker, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join(timeout=60)
    assert not bad, bad


@gpu
@pytest.mark.parametrize("kv,io", [("f16", "f32"), ("bf16", "bf16")], ids=["f16-f32", "bf16"])
def test_prompt_then_tokens_with_rotary_positions(kv, io):
    """used together: a prompt's keys turn into the cache, the prompt attends, then tokens one by one; every
    step against the formula over what the cache holds, and each token's row against the same row of one
    long prompt"""
    B, H, Hk, D, prompt, steps = 2, 8, 2, 64, 50, 6
    total = prompt + steps
    rope = M.rope_spec(D, M.ROPE_HALVES)
    xq, xk, xv = rnd((B, total, H, D), io, 1, 1.5), rnd((B, total, Hk, D), io, 2), rnd((B, total, Hk, D), kv, 3)
    cache_k = torch.full((B, 64, Hk, D), NAN, dtype=TYPES[kv], device="cuda")
    cache_v = cache_k.clone()
    rows = []
    for first, n in [(0, prompt)] + [(prompt + i, 1) for i in range(steps)]:
        pos = torch.arange(first, first + n, dtype=torch.int32, device="cuda")
        q = torch.empty(B, n, H, D, dtype=TYPES[io], device="cuda")
        M.rope(M.from_torch(xq[:, first : first + n]), M.from_torch(pos), M.from_torch(q), rope)
        M.rope(M.from_torch(xk[:, first : first + n]), M.from_torch(pos), M.from_torch(cache_k[:, first : first + n]), rope)
        cache_v[:, first : first + n] = xv[:, first : first + n]
        lens = full(B, first + n)
        o = call(q, cache_k, cache_v, 0.125, lens, causal=True)
        near(o, formula(q, cache_k, cache_v, 0.125, lens, causal=True))
        rows.append(o)
    q = torch.empty(B, total, H, D, dtype=TYPES[io], device="cuda")
    M.rope(M.from_torch(xq), M.from_torch(torch.arange(total, dtype=torch.int32, device="cuda")), M.from_torch(q), rope)
    o, most, _ = formula(q, cache_k[:, :total], cache_v[:, :total], 0.125, full(B, total), causal=True)
    assert ((torch.cat(rows, 1).double() - o).abs() <= most).all()


@gpu
def test_empty():
    for B, n, H in ((0, 1, 4), (1, 0, 4), (1, 1, 0)):
        q = torch.empty(B, n, H, 64, dtype=torch.float16, device="cuda")
        k = torch.empty(max(B, 1), 5, 1, 64, dtype=torch.float16, device="cuda")
        call(q, k, k, 1.0)
    q = rnd((2, 3, 4, 64), "f16", 1)
    k = torch.empty(2, 0, 2, 64, dtype=torch.float16, device="cuda")
    assert (call(q, k, k, 1.0) == 0).all()


# ---- refusals (no GPU: nothing is launched) ----------------------------------------------------


def desc(kind, ne, nb=None, ptr=0x10000):
    ne = list(ne) + [1] * (4 - len(ne))
    return M.tensor(kind, ptr, ne, nb or M.contiguous_nb(kind, ne))


def base():
    return dict(q=desc(M.F16, [64, 3, 8, 2]), k=desc(M.F16, [64, 50, 2, 2]), v=desc(M.F16, [64, 50, 2, 2]), mask=None, sinks=None, kv_len=None,
                dst=desc(M.F16, [64, 8, 3, 2]), params=M.attn_spec(0.125), work=None, work_bytes=0)


def rc(prefix=False, **change):
    a = dict(base(), **change)
    r = lambda x: None if x is None else C.byref(x)  # noqa: E731
    if prefix:
        a = dict(dict(kp=desc(M.F16, [64, 70, 2]), vp=desc(M.F16, [64, 70, 2])), **a)
        return M.lib().ggml_mi355x_flash_attn_prefix(r(a["q"]), r(a["kp"]), r(a["vp"]), r(a["k"]), r(a["v"]), r(a["sinks"]), r(a["kv_len"]), r(a["dst"]),
                                                     r(a["params"]), a["work"], a["work_bytes"], None)
    return M.lib().ggml_mi355x_flash_attn(r(a["q"]), r(a["k"]), r(a["v"]), r(a["mask"]), r(a["sinks"]), r(a["kv_len"]), r(a["dst"]), r(a["params"]),
                                          a["work"], a["work_bytes"], None)


@pytest.mark.parametrize("prefix", [False, True])
def test_refusals(prefix):
    wide = dict(q=desc(M.F16, [264, 3, 8, 2]), k=desc(M.F16, [264, 50, 2, 2]), v=desc(M.F16, [264, 50, 2, 2]), dst=desc(M.F16, [264, 8, 3, 2]))
    odd = dict(q=desc(M.F16, [20, 3, 8, 2]), k=desc(M.F16, [20, 50, 2, 2]), v=desc(M.F16, [20, 50, 2, 2]), dst=desc(M.F16, [20, 8, 3, 2]))
    changes = [
        wide, odd, dict(q=desc(M.BF16, [64, 3, 8, 2]), dst=desc(M.BF16, [64, 8, 3, 2])), dict(dst=desc(M.F32, [64, 8, 3, 2])),
        dict(k=desc(M.BF16, [64, 50, 2, 2]), v=desc(M.BF16, [64, 50, 2, 2]), q=desc(M.F32, [64, 3, 8, 2]), dst=desc(M.F32, [64, 8, 3, 2])),
        dict(k=desc(M.Q8_0, [64, 50, 2, 2])), dict(v=desc(M.F16, [64, 49, 2, 2])), dict(v=desc(M.F16, [32, 50, 2, 2])),
        dict(k=desc(M.F16, [64, 50, 3, 2]), v=desc(M.F16, [64, 50, 3, 2])), dict(k=desc(M.F16, [64, 50, 2, 4]), v=desc(M.F16, [64, 50, 2, 4])),
        dict(dst=desc(M.F16, [64, 3, 8, 2])), dict(dst=desc(M.F16, [64, 8, 3, 2], [2, 128, 1024, 0])),
        dict(q=desc(M.F16, [64, 3, 8, 2], ptr=0x10008)), dict(k=desc(M.F16, [64, 50, 2, 2], [2, 130, 6500, 13000])),
        dict(k=desc(M.F16, [64, 50, 2, 2], [4, 256, 12800, 25600])),
        dict(sinks=desc(M.F32, [7])), dict(sinks=desc(M.F16, [8])), dict(kv_len=desc(M.I32, [1])), dict(kv_len=desc(M.F32, [2])),
        dict(q=desc(M.F16, [64, 3, 8, 2], ptr=0)), dict(v=desc(M.F16, [64, 50, 2, 2], ptr=0)), dict(kv_len=desc(M.I32, [2], ptr=0)), dict(sinks=desc(M.F32, [8], ptr=0)),
        dict(params=M.attn_spec(NAN)), dict(params=M.attn_spec(INF)), dict(params=M.attn_spec(1.0, -1.0)), dict(params=M.attn_spec(1.0, 8.0)),
        dict(params=M.attn_spec(1.0, 0.0, -5.0)), dict(params=M.attn_spec(1.0, 0.0, NAN)), dict(params=M.attn_spec(1.0, 0.0, INF)), dict(params=M.attn_spec(1.0, 0.0, 1e20)), dict(params=M.AttnSpec(1.0, 0.0, 0.0, 2)),
        dict(q=None), dict(k=None), dict(v=None), dict(dst=None), dict(params=None),
    ]
    if prefix:
        changes += [dict(kp=desc(M.BF16, [64, 70, 2])), dict(vp=desc(M.F16, [64, 71, 2])), dict(kp=desc(M.F16, [64, 70, 1])), dict(kp=desc(M.F16, [64, 70, 2, 2])),
                    dict(kp=None), dict(vp=None), dict(kp=desc(M.F16, [64, 70, 2], ptr=0)), dict(k=desc(M.F16, [64, 50, 2, 1]), v=desc(M.F16, [64, 50, 2, 1]))]
    else:
        changes += [dict(mask=desc(M.F32, [50, 3])), dict(mask=desc(M.F16, [49, 3])), dict(mask=desc(M.F16, [50, 2])), dict(mask=desc(M.F16, [50, 3, 3])),
                    dict(mask=desc(M.F16, [50, 3, 1, 4])), dict(mask=desc(M.F16, [50, 3], ptr=0)), dict(mask=desc(M.F16, [50, 3], [4, 200, 600, 600]))]
    for c in changes:
        assert rc(prefix, **c) == -1, c


def test_refusals_of_what_no_grid_holds():
    def of(B, n, H, Hk, D=8):
        return dict(q=desc(M.F16, [D, n, H, B]), k=desc(M.F16, [D, 4, Hk, B]), v=desc(M.F16, [D, 4, Hk, B]), dst=desc(M.F16, [D, H, n, B]))

    for sizes in ((65536, 1, 1, 1), (1, 1, 65536, 1), (1, 1 << 24, 1, 1), (65535, 1, 128, 128), (64, 1 << 18, 64, 1)):
        assert rc(**of(*sizes)) == -1, sizes
    pre = dict(kp=desc(M.F16, [8, 70, 2]), vp=desc(M.F16, [8, 70, 2]))
    assert rc(True, **of(64, 1 << 14, 64, 2), **pre) == -1


def test_workspace_sizes_and_refusals():
    q, k, kp = desc(M.F16, [128, 1, 32, 1]), desc(M.F16, [128, 100000, 8, 1]), desc(M.F16, [128, 9000, 8])
    n, p = M.flash_attn_work_size(q, k), M.flash_attn_prefix_work_size(q, kp, k)
    for need, call_rc in ((n, lambda **w: rc(q=q, k=k, v=k, dst=desc(M.F16, [128, 32, 1, 1]), **w)),
                          (p, lambda **w: rc(True, q=q, kp=kp, vp=kp, k=k, v=k, dst=desc(M.F16, [128, 32, 1, 1]), **w))):
        if need:
            assert call_rc(work=0x10000, work_bytes=need - 1) == -1
        assert call_rc(work=0x10008, work_bytes=need) == -1
    L, b = M.lib(), C.c_size_t(0)
    assert L.ggml_mi355x_flash_attn_work_size(None, C.byref(k), C.byref(b)) == -1
    assert L.ggml_mi355x_flash_attn_work_size(C.byref(q), C.byref(k), None) == -1
    assert L.ggml_mi355x_flash_attn_work_size(C.byref(q), C.byref(desc(M.F16, [64, 10, 8])), C.byref(b)) == -1
    assert L.ggml_mi355x_flash_attn_prefix_work_size(C.byref(q), None, C.byref(k), C.byref(b)) == -1


def test_tensors_on_another_gpu_are_refused(monkeypatch):
    monkeypatch.setattr(M, "_several_gpus", True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    a = base()
    for name in ("q", "k", "v", "dst"):
        x = dict(a, **{name: desc(M.F16, [64, 3, 8, 2])})
        x[name].device = 1
        with pytest.raises(M.Mi355xError, match="GPU 1"):
            M.flash_attn(x["q"], x["k"], x["v"], x["dst"], x["params"], stream=0)
        with pytest.raises(M.Mi355xError, match="GPU 1"):
            M.flash_attn_prefix(x["q"], a["k"], a["v"], x["k"], x["v"], x["dst"], x["params"], stream=0)
        with pytest.raises(M.Mi355xError, match="GPU 1"):
            M.rope(x["q"], x["k"], x["v"] if name != "dst" else x["dst"], M.rope_spec(64), stream=0)
