"""Attention at the ends of its types' ranges. Allowances are those of tests/test_attention.py, whose `formula` leaves
out what a row does not see."""
import math

import pytest
from test_attention import IDS, PAIRS, TYPES, call, formula, full, near, operands, rnd, torch

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
