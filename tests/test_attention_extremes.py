"""Attention at the ends of its types' ranges: the largest values of a cache, f32 queries whose row holds one value
far above the others, factors of nothing beside large products, infinities under a cap, and values that are not
finite in places that some rows see and others do not. Allowances are those of tests/test_attention.py, whose
`formula` leaves out what a row does not see."""
import math

import numpy as np
import pytest
from test_attention import IDS, INF, NAN, PAIRS, TYPES, call, formula, full, near, operands, rnd, torch

import mi355x_qmm as M

gpu = pytest.mark.gpu


# ---- large values ------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("n", [1, 9, 70, 600])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_largest_values(kv, io, n, D):
    """a key that takes nearly all of every row's weight and holds the type's largest values (a bf16 one overflows 32
    bits as soon as its weight is kept larger than 1), in the first tile, in a later one, and in a prefix; and one
    that exceeds the row's maximum by less than a rescale of the running sums asks for"""
    m, most = 700, torch.finfo(TYPES[kv]).max
    q, k, v = operands(1, n, m, 8, 2, D, kv, io, seed=n + D)
    kp, vp = rnd((90, 2, D), kv, 7), rnd((90, 2, D), kv, 8)
    q[..., 0], k[..., 0], kp[..., 0] = 8.0, 0.0, 0.0
    s = 1 / math.sqrt(D)
    # (e^18 = 6e7 over at most 790 keys; f16 results may not round past the largest value)
    stand_out = 18.0 / (8.0 * s)
    large = 0.99 * most
    for at in (3, 333, 699):
        k2, v2 = k.clone(), v.clone()
        k2[:, at, :, 0] = stand_out
        v2[:, at, :, ::2], v2[:, at, :, 1::2] = large, -large
        near(call(q, k2, v2, s), formula(q, k2, v2, s, full(1, m)))
        near(call(q, k2, v2, s, kp=kp, vp=vp), formula(q, k2, v2, s, full(1, m), kp=kp, vp=vp))
    kp2, vp2 = kp.clone(), vp.clone()
    kp2[50, :, 0] = stand_out
    vp2[50] = -large
    near(call(q, k, v, s, kp=kp2, vp=vp2), formula(q, k, v, s, full(1, m), kp=kp2, vp=vp2))
    # key 0 sets the maximum, key 400 lies 4.5 (6.5 powers of two) above it, all others far below
    q2, k3, v3 = torch.zeros_like(q), torch.zeros_like(k), v.clone()
    q2[..., 0] = 4.0
    k3[..., 0], k3[:, 0, :, 0], k3[:, 400, :, 0] = -30.0 / 4, 0.0, 4.5 / 4
    v3[:, 400], v3[:, 0] = large, large / 2
    near(call(q2, k3, v3, 1.0), formula(q2, k3, v3, 1.0, full(1, m)))


# ---- f32 queries -------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("n", [1, 5, 70, 600])
@pytest.mark.parametrize("D", [64, 80, 128, 192, 256])
@pytest.mark.parametrize("size", [30.0, 1000.0, 16384.0, -3.0e6])
def test_queries_with_one_large_value(n, D, size):
    """f32 queries with one value far above the rest over keys that hold next to nothing there: the rest keep their
    precision"""
    m = 300
    q, k, v = operands(2, n, m, 8, 2, D, "f16", "f32", seed=n + D)
    kp, vp = rnd((100, 2, D), "f16", 7), rnd((100, 2, D), "f16", 8)
    w = rnd((1, 1, n, m), "f16", 9)
    w[..., 1::7] = -INF
    q[..., 3] = size
    s = 1 / math.sqrt(D)
    for small in (0.0, 0.5 / abs(size)):
        k[..., 3], kp[..., 3] = small, small
        near(call(q, k, v, s), formula(q, k, v, s, full(2, m)))
        near(call(q, k, v, -s, causal=True), formula(q, k, v, -s, full(2, m), causal=True))
        near(call(q, k, v, s, mask=w, bias=8.0), formula(q, k, v, s, full(2, m), mask=w, bias=8.0))
        near(call(q, k, v, s, cap=5.0, kp=kp, vp=vp), formula(q, k, v, s, full(2, m), cap=5.0, kp=kp, vp=vp))


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("n", [1, 70])
@pytest.mark.parametrize("beside", [1.0, 3.0e4, 1.0e6])
def test_infinite_queries_under_a_cap(kv, io, n, beside):
    """a query value of infinity makes scores of infinity, whatever is beside it, and the cap makes them finite"""
    if beside > torch.finfo(TYPES[io]).max:
        beside = torch.finfo(TYPES[io]).max
    m, D, i, cap = 200, 64, n // 2, 3.0
    q, k, v = operands(1, n, m, 4, 2, D, kv, io, seed=3)
    q[..., 5] = beside
    k[..., 2] = torch.where(k[..., 2].abs() < 0.1, 0.5, k[..., 2].float()).to(k.dtype)
    q2 = q.clone()
    q2[0, i, 1, 2] = INF
    got = call(q2, k, v, 0.125, cap=cap)
    # its row: weights of 1 and e^-6, by the key's sign there; every other row as without it
    p = torch.exp(cap * torch.sign(k[0, :, 0, 2].double()) - cap)
    row = (p[:, None] * v[0, :, 0].double()).sum(0) / p.sum()
    A = (p[:, None] * v[0, :, 0].double().abs()).sum(0) / p.sum()
    eps = 0.0 if io == "f32" else torch.finfo(TYPES[io]).eps / 2
    allowed = ((2 * 6 * cap + 8 + m) * 2.0**-24 + 2 * eps) * A
    assert ((got[0, i, 1].double() - row).abs() <= allowed).all()
    o, most, _ = formula(q, k, v, 0.125, full(1, m), cap=cap)
    fine = (got.double() - o).abs() <= most
    fine[0, i, 1] = True
    assert fine.all()


# ---- factors of nothing ------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("n", [1, 70])
@pytest.mark.parametrize("scale", [0.0, 1.0e-40, -1.0e-38])
def test_next_to_no_factor_beside_large_products(kv, io, n, scale):
    """bf16 products reach 1e38, where even the smallest factor counts and a factor of 0 still leaves nothing"""
    size = 1.0e18 if kv == "bf16" else 100.0
    q, k, v = operands(2, n, 150, 4, 2, 64, kv, io, seed=11)
    q, k = q * size, k * size
    w = rnd((1, 1, n, 150), "f16", 12)
    scale = float(torch.tensor(scale, dtype=torch.float32))
    kp, vp = rnd((100, 2, 64), kv, 7) * size, rnd((100, 2, 64), kv, 8)
    near(call(q, k, v, scale), formula(q, k, v, scale, full(2, 150)))
    near(call(q, k, v, scale, mask=w), formula(q, k, v, scale, full(2, 150), mask=w))
    near(call(q, k, v, scale, kp=kp, vp=vp), formula(q, k, v, scale, full(2, 150), kp=kp, vp=vp))


# ---- values that are not finite ----------------------------------------------------------------


@gpu
@pytest.mark.parametrize("kv,io", PAIRS, ids=IDS)
@pytest.mark.parametrize("n", [1, 6, 50, 200])
@pytest.mark.parametrize("D", [40, 64, 96, 128, 184, 256])
def test_nonfinite_values_that_some_rows_see(kv, io, n, D):
    """NaN and infinities in single channels of values, in keys that some rows see: those channels of those rows, and
    nothing else"""
    m, H = 330, 4
    q, k, v = operands(1, n, m, H, 2, D, kv, io, seed=n + D)
    w = rnd((1, H, n, m), "f16", 5)
    r = torch.from_numpy(np.random.default_rng(6).random((H, n, m)) < 0.4).cuda()
    w[0][r] = -INF
    w[..., 7], w[..., 200] = 0.0, -INF
    marks = [(0, 3, NAN), (7, 1, INF), (31, 5, INF), (32, 5, -INF), (100, D - 1, -INF), (200, 4, NAN), (255, 6, NAN), (256, 7, INF), (329, 3, NAN)]
    k2, v2 = k.clone(), v.clone()
    k2[:, 200] = NAN
    for j, ch, x in marks:
        v2[0, j, :, ch] = x
    got = call(q, k2, v2, 0.1, mask=w)[0].double()
    o, most, _ = formula(q, k, torch.where(torch.isfinite(v2), v2, 0.0), 0.1, full(1, m), mask=w)
    want = o[0].clone()
    seen = (w[0] != -INF).permute(1, 0, 2)                     # [n, H, m]
    for j, ch, x in marks:
        # (a sum of weights above 0 times these: infinity, or NaN with one of the other sign)
        want[:, :, ch] = torch.where(seen[:, :, j], want[:, :, ch] + x, want[:, :, ch])
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    fine = torch.isfinite(want)
    assert (((got - o[0]).abs() <= most[0]) | ~fine).all(), float(((got - o[0]).abs() - most[0])[fine].max())


@gpu
@pytest.mark.parametrize("n", [1, 1000])
@pytest.mark.parametrize("what", ["hidden value", "hidden key", "seen value"])
def test_one_nan_costs_no_second(n, what):
    """the rows whose sums a NaN spoils are formed again, 32 at a time: 1500 keys of up to 1.5 us are 2.3 ms, some 50 of
    the calls of 45 us; a row at a time takes 2 us for each of its keys, 2000 calls"""
    m = 1500 if n > 1 else 4000
    q, k, v = operands(1, n, m, 8, 2, 128, "f16", "f32", seed=1)
    w = torch.zeros(1, 1, n, m, dtype=torch.float16, device="cuda")
    if what != "seen value":
        w[..., 700] = -INF
    out, spec, hf = torch.empty_like(q), M.attn_spec(0.09), lambda t: M.from_torch(t.permute(0, 2, 1, 3))

    def us():
        best = INF
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            a.record()
            for _ in range(2):
                M.flash_attn(hf(q), hf(k), hf(v), M.from_torch(out), spec, mask=M.from_torch(w))
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b) * 500)
        return best

    before = us()
    (k if what == "hidden key" else v)[0, 700, 0, 3] = NAN
    assert us() <= 100 * before
    assert torch.isnan(out).any() == (what == "seen value")


# ---- weights of 16-bit activations -------------------------------------------------------------


@gpu
@pytest.mark.parametrize("io", ["f16", "bf16"])
@pytest.mark.parametrize("size", [(3, 1, 1000, 8, 2, 128, 0), (1, 4, 700, 32, 4, 64, 0), (2, 2, 300, 14, 2, 96, 0), (1, 1, 5000, 16, 1, 256, 0), (2, 3, 90, 6, 2, 184, 0),
                                  (1, 8, 400, 8, 2, 128, 500), (4, 1, 200, 8, 1, 64, 900)], ids=lambda s: "x".join(map(str, s)))
def test_few_rows_keep_their_weights(io, size):
    """up to 32 rows a key head: nothing is rounded to 16 bits but the result. Weights of two terms are off by 2^-16 of
    them (bf16) or 2^-22 and, below f16's normal numbers, 2^-33 of the largest"""
    B, n, m, H, Hk, D, P = size
    q, k, v = operands(B, n, m, H, Hk, D, io, io, seed=sum(size))
    more = dict(kp=rnd((P, Hk, D), io, 7), vp=rnd((P, Hk, D), io, 8)) if P else {}
    s = 1 / math.sqrt(D)
    got = call(q, k, v, s, causal=True, **more).double()
    o, most, _ = formula(q.float(), k, v, s, full(B, m), causal=True, **more)
    size_of = {name: t.abs() for name, t in more.items() if name == "vp"}
    A, _, _ = formula(q.float(), k, v.abs(), s, full(B, m), causal=True, **{**more, **size_of})
    eps = torch.finfo(TYPES[io]).eps / 2
    weights = 2.0**-16 * A if io == "bf16" else 2.0**-22 * A + 2.0**-33 * (m + P) * float(v.abs().max())
    assert ((got - o).abs() <= most + weights + eps * o.abs() + torch.finfo(TYPES[io]).tiny * eps).all()
