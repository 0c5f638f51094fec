"""Attention at the ends of its types' ranges. Allowances are those of tests/test_attention.py, whose `formula` leaves
out what a row does not see."""
import math

import pytest
from test_attention import IDS, INF, PAIRS, TYPES, call, formula, full, near, operands, rnd, torch

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
