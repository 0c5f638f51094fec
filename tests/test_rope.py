"""Rotary positions and their gradient (ggml_mi355x_rope, ggml_mi355x_rope_back) against the formula
in 64 and 80 bits: pairings, partial heads, stretched contexts, frequency factors, types, strides,
positions, in place and into a cache; the gradient also against differences. Refusals run without
a GPU (nothing is launched).

Tolerances, relative to the pair's length times the factor of the turned values: the angle's
remainder is rounded to 32 bits (2^-26 turns: 1.6 * 2^-24 radians), sine and cosine are off by 2 units
in the last place (2 * 2^-24), the factor, the two products and their sum round once each (4 * 2^-24):
under 10 * 2^-24 with the sum of both terms of a turned value (sqrt 2); then one rounding to the
result's type, eps/2 of the value, or half the smallest subnormal."""
import ctypes as C
import math

import numpy as np
import pytest

import mi355x_qmm as M

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def frequencies(spec):
    """radians per position of each pair in 80 bits, and the factor"""
    n, L = spec.n_dims, np.longdouble
    i = np.arange(n // 2, dtype=L)
    base, scale = L(spec.freq_base), L(spec.freq_scale)
    f = np.exp(-2 * i / n * np.log(base))
    size = L(spec.attn_factor)
    if spec.ext_factor != 0:
        low, high = (n * np.log(spec.n_ctx_orig / (L(beta) * 2 * L(math.pi))) / (2 * np.log(base)) for beta in (spec.beta_fast, spec.beta_slow))
        low, high = max(L(0), np.floor(low)), min(L(n - 1), np.ceil(high))
        mix = (1 - np.clip((i - low) / max(L(0.001), high - low), 0, 1)) * L(spec.ext_factor)
        f = f * (scale * (1 - mix) + mix)
        size = size * (1 + L(0.1) * np.log(1 / scale))
    else:
        f = f * scale
    return f, size


def turned(x, pos, spec, factors=None, back=False):
    """(y, the pairs' lengths times the factor) of x [batch, token, head, dim], pos [batch, token], in 64 bits"""
    f, size = frequencies(spec)
    if factors is not None:
        f = f / factors.astype(np.longdouble)[: len(f)]
    pi2 = np.longdouble("6.28318530717958647692528676655900576839")
    t = pos.astype(np.longdouble)[..., None] * f / pi2
    t = ((t - np.rint(t)) * pi2).astype(np.float64)[:, :, None, :]
    c, s = np.cos(t) * float(size), np.sin(t) * float(size) * (-1 if back else 1)
    n = spec.n_dims
    y, length = x.astype(np.float64).copy(), np.zeros(x.shape)
    ia, ib = (np.arange(n // 2), np.arange(n // 2) + n // 2) if spec.mode == M.ROPE_HALVES else (np.arange(0, n, 2), np.arange(1, n, 2))
    a, b = x[..., ia].astype(np.float64), x[..., ib].astype(np.float64)
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    length[..., ia] = length[..., ib] = np.hypot(a, b) * abs(float(size))
    return y, length


def near(got, want, length, dtype, extra=0.0):
    t = TYPES[dtype]
    allowed = length * (10 * 2.0**-24 + extra)
    if dtype != "f32":
        allowed = allowed + np.abs(want) * torch.finfo(t).eps / 2 * 1.001 + torch.finfo(t).tiny * torch.finfo(t).eps / 2
    off = np.abs(got.double().cpu().numpy() - want)
    assert (off <= allowed).all(), (off.max(), np.argwhere(off > allowed)[:4])


def run(x, pos, spec, out=None, factors=None, back=False):
    d = torch.empty_like(x) if out is None else out
    f = None if factors is None else torch.from_numpy(factors).cuda()
    p = torch.from_numpy(np.ascontiguousarray(pos)).cuda()
    (M.rope_back if back else M.rope)(M.from_torch(x), M.from_torch(p), M.from_torch(d), spec, factors=None if f is None else M.from_torch(f))
    torch.cuda.synchronize()
    return d


def values(shape, dtype, seed=0):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape).astype(np.float32)).cuda().to(TYPES[dtype])


SHAPES = [
    # batch, tokens, heads, dim, n_dims
    (1, 1, 1, 2, 2), (1, 1, 32, 128, 128), (1, 7, 3, 64, 64), (2, 33, 5, 80, 32), (1, 5, 2, 81, 18), (3, 129, 1, 96, 96),
    (1, 1000, 8, 128, 128), (2, 3, 4, 576, 512), (1, 17, 71, 20, 20), (1, 2, 1, 1000, 64), (1, 64, 1, 36, 34),
    (1, 2100, 13, 96, 96), (3, 4000, 3, 80, 40), (1, 1500, 20, 136, 64),   # several heads a thread, and their ends
    (2, 3001, 9, 44, 36), (1, 4100, 6, 30, 14), (3, 1500, 7, 81, 40), (1, 2500, 5, 204, 52),   # groups of 4, of 2, of no values
]


@gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("mode", [M.ROPE_NEIGHBOURS, M.ROPE_HALVES])
@pytest.mark.parametrize("src,dst", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("back", [False, True])
def test_matches_formula(shape, mode, src, dst, back):
    b, t, h, d, n = shape
    x = values((b, t, h, d), src, seed=d + t)
    pos = np.random.default_rng(t).integers(0, 8192, (1, t)).astype(np.int32)
    spec = M.rope_spec(n, mode)
    y = run(x, pos[0], spec, torch.full((b, t, h, d), 7.0, dtype=TYPES[dst], device="cuda"), back=back)
    near(y, *turned(x.double().cpu().numpy(), np.repeat(pos, b, 0), spec, back=back), dst)


@gpu
@pytest.mark.parametrize("mode", [M.ROPE_NEIGHBOURS, M.ROPE_HALVES])
@pytest.mark.parametrize("scaled", ["linear", "yarn", "factors", "all"])
def test_stretched(mode, scaled):
    kw = dict(freq_base=500000.0)
    if scaled in ("yarn", "all"):
        kw.update(freq_scale=1 / 16, ext_factor=1.0 if scaled == "yarn" else 0.75, n_ctx_orig=8192, attn_factor=1.25)
    elif scaled == "linear":
        kw.update(freq_scale=0.125)
    spec = M.rope_spec(128, mode, **kw)
    factors = (1 + 7 * np.random.default_rng(1).random(64)).astype(np.float32) if scaled in ("factors", "all") else None
    x = values((2, 40, 4, 128), "f32", 3)
    pos = np.random.default_rng(2).integers(0, 131072, (2, 40)).astype(np.int32)   # a row of positions per batch
    y = run(x, pos, spec, factors=factors)
    near(y, *turned(x.double().cpu().numpy(), pos, spec, factors), "f32")


@gpu
def test_far_and_negative_positions():
    """64-bit angles: two roundings of the turns made, 2^-52 of 2^31/2pi turns, beside the 32-bit ones"""
    pos = np.array([[0, 1, -1, 2**20 + 1, 2**24 + 1, 2**30 + 7, 2**31 - 1, -(2**31), -12345678]], dtype=np.int32)
    x = values((1, 9, 2, 128), "f32", 5)
    for mode in (M.ROPE_NEIGHBOURS, M.ROPE_HALVES):
        spec = M.rope_spec(128, mode)
        near(run(x, pos[0], spec), *turned(x.double().cpu().numpy(), pos, spec), "f32", extra=2 * 2.0**-52 * 2.0**31)


@gpu
@pytest.mark.parametrize("factors", [False, True])
def test_far_positions_to_their_roundings(factors):
    """the frequency and its product with the position are off by 2^-53 each of the radians made, a division by factors by
    as much again"""
    pos = np.array([[2**31 - 1 - 97 * i for i in range(20)] + [-(2**31) + 89 * i for i in range(20)]], dtype=np.int32)
    x = values((1, 40, 2, 128), "f32", 5)
    ff = (1 + 7 * np.random.default_rng(1).random(64)).astype(np.float32) if factors else None
    for mode in (M.ROPE_NEIGHBOURS, M.ROPE_HALVES):
        spec = M.rope_spec(128, mode)
        near(run(x, pos[0], spec, factors=ff), *turned(x.double().cpu().numpy(), pos, spec, ff), "f32", extra=(3 if factors else 2) * 2.0**-53 * 2.0**31)


@gpu
@pytest.mark.parametrize("mode", [M.ROPE_NEIGHBOURS, M.ROPE_HALVES])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_in_place_strides_and_what_lies_between(mode, dtype):
    """a strided view in place (the rows of q inside a fused qkv buffer, odd offsets): the bytes
    between its rows stay"""
    spec = M.rope_spec(20, mode)
    for first, dim in ((0, 24), (3, 25), (8, 24)):
        buf = values((2, 13, 3, 40), dtype, 6)
        before = buf.clone()
        view = buf[:, :, :, first : first + dim]
        pos = np.arange(100, 113, dtype=np.int32)[None]
        want = turned(view.double().cpu().numpy(), np.repeat(pos, 2, 0), spec)
        run(view, pos[0], spec, out=view)
        near(view, *want, dtype)
        assert torch.equal(buf[..., :first], before[..., :first]) and torch.equal(buf[..., first + dim :], before[..., first + dim :])


@gpu
def test_into_a_cache_slice():
    spec = M.rope_spec(128, M.ROPE_HALVES)
    cache = torch.full((2, 64, 4, 128), 5.0, dtype=torch.float16, device="cuda")
    x = values((2, 9, 4, 128), "f32", 8)
    pos = np.arange(30, 39, dtype=np.int32)[None]
    run(x, pos[0], spec, out=cache[:, 30:39])
    near(cache[:, 30:39], *turned(x.double().cpu().numpy(), np.repeat(pos, 2, 0), spec), "f16")
    assert (cache[:, :30] == 5).all() and (cache[:, 39:] == 5).all()


@gpu
def test_permuted_and_broadcast_source():
    """heads outside tokens, and one batch read for several (stride 0)"""
    spec = M.rope_spec(64, M.ROPE_HALVES)
    x = values((1, 5, 11, 64), "f32", 9).permute(0, 2, 1, 3).expand(3, 11, 5, 64)
    pos = np.arange(11, dtype=np.int32)[None]
    y = run(x, pos[0], spec, out=torch.empty(3, 11, 5, 64, device="cuda"))
    near(y, *turned(x.double().cpu().numpy(), np.repeat(pos, 3, 0), spec), "f32")


@gpu
@pytest.mark.parametrize("mode", [M.ROPE_NEIGHBOURS, M.ROPE_HALVES])
def test_gradient_is_the_transpose_and_matches_differences(mode):
    """<rope(x), g> = <x, rope_back(g)>, and the difference quotient of <rope(x), g> along v is
    <v, rope_back(g)> (rope is linear: the quotient has no error but rounding)"""
    spec = M.rope_spec(48, mode, freq_scale=0.25, ext_factor=1.0, n_ctx_orig=4096, attn_factor=0.8)
    shape = (2, 19, 3, 64)
    x, v, g = (values(shape, "f32", s) for s in (11, 12, 13))
    pos = np.arange(5000, 5019, dtype=np.int32)
    dx = run(g, pos, spec, back=True).double()
    size = max(1.0, abs(float(frequencies(spec)[1])))
    # every value of both sides is off by at most 10 * 2^-24 of its pair's length (the head comment)
    slack = 10 * 2.0**-24 * size
    def inner(a, b):
        return float((a.double() * b.double()).sum())
    lengths = float(x.double().norm() * g.double().norm()) * math.sqrt(2)
    assert abs(inner(run(x, pos, spec), g) - inner(x, dx)) <= 2 * slack * lengths
    h = 0.5
    quotient = (inner(run(x + h * v, pos, spec), g) - inner(run(x - h * v, pos, spec), g)) / (2 * h)
    most = float((x.double().norm() + h * v.double().norm()) * g.double().norm()) * math.sqrt(2)
    # (x + h v rounds once more, 2^-24 of its values)
    assert abs(quotient - inner(v, dx)) <= 2 * (slack + 2.0**-24 * size) * most / (2 * h) + slack * lengths * 2


@gpu
def test_nonfinite_values_stay_in_their_pair():
    spec = M.rope_spec(8, M.ROPE_HALVES)
    x = values((1, 2, 2, 12), "f32", 1)
    x[0, 0, 0, 1], x[0, 1, 1, 10] = float("nan"), float("inf")
    y = run(x, np.array([3, 4], dtype=np.int32), spec)
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[0, 0, 0, 1] = want[0, 0, 0, 5] = want[0, 1, 1, 10] = True
    assert torch.equal(bad, want)


@gpu
def test_empty():
    spec = M.rope_spec(8)
    for shape in ((1, 0, 4, 16), (1, 4, 0, 16), (0, 4, 4, 16)):
        x = torch.empty(shape, device="cuda")
        p = torch.zeros(shape[1], dtype=torch.int32, device="cuda")
        M.rope(M.from_torch(x), M.from_torch(p), M.from_torch(x), spec)


@gpu
def test_captured_and_replayed():
    spec = M.rope_spec(128, M.ROPE_HALVES)
    x, y = values((1, 4, 8, 128), "f32", 2), torch.empty(1, 4, 8, 128, device="cuda")
    p = torch.arange(4, dtype=torch.int32, device="cuda")
    X, P, Y = M.from_torch(x), M.from_torch(p), M.from_torch(y)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        M.rope(X, P, Y, spec)
    for k in range(4):
        p += 1000 * k
        x.normal_()
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        eager = torch.empty_like(y)
        M.rope(X, P, M.from_torch(eager), spec)
        assert torch.equal(y, eager)


# ---- refusals (no GPU: nothing is launched) ----------------------------------------------------


def desc(kind, ne, nb=None, ptr=0x10000):
    ne = list(ne) + [1] * (4 - len(ne))
    return M.tensor(kind, ptr, ne, nb or M.contiguous_nb(kind, ne))


def refused(src=None, pos=None, dst=None, spec=None, ff=None, back=False):
    M.lib()
    src = src or desc(M.F32, [64, 4, 8, 2])
    dst = dst or desc(M.F32, [64, 4, 8, 2], ptr=0x90000)
    pos = pos or desc(M.I32, [8])
    spec = spec or M.rope_spec(64)
    f = M.lib().ggml_mi355x_rope_back if back else M.lib().ggml_mi355x_rope
    return f(C.byref(src), C.byref(pos), None if ff is None else C.byref(ff), C.byref(dst), C.byref(spec), None)


@pytest.mark.parametrize("back", [False, True])
def test_refusals(back):
    e = -1
    for what in (
        dict(src=desc(M.I32, [64, 4, 8, 2])), dict(dst=desc(M.Q8_0, [64, 4, 8, 2])), dict(pos=desc(M.F32, [8])),
        dict(dst=desc(M.F32, [64, 4, 8, 1])), dict(dst=desc(M.F32, [32, 4, 8, 2])),
        dict(pos=desc(M.I32, [7])), dict(pos=desc(M.I32, [8, 3])), dict(pos=desc(M.I32, [8, 2, 2])), dict(pos=desc(M.I32, [8], [8, 64, 64, 64])),
        dict(src=desc(M.F32, [64, 4, 8, 2], [8, 512, 2048, 16384])),      # rows not contiguous
        dict(src=desc(M.F32, [64, 4, 8, 2], [4, 258, 1032, 8256])),       # rows at half a value
        dict(src=desc(M.F32, [64, 4, 8, 2], ptr=0x10002)),
        dict(dst=desc(M.F32, [64, 4, 8, 2], [4, 256, 1024, 0])),          # two results in one place
        dict(ff=desc(M.F32, [31])), dict(ff=desc(M.F16, [32])),
        dict(src=desc(M.F32, [64, 4, 8, 2], ptr=0)), dict(pos=desc(M.I32, [8], ptr=0)), dict(ff=desc(M.F32, [32], ptr=0)),
    ):
        assert refused(back=back, **what) == e, what
    for kw in (dict(n_dims=0), dict(n_dims=63), dict(n_dims=66), dict(n_dims=-2), dict(n_dims=64, mode=8), dict(n_dims=64, mode=24),
               dict(n_dims=64, freq_base=0.0), dict(n_dims=64, freq_base=-1.0), dict(n_dims=64, freq_base=math.inf),
               dict(n_dims=64, freq_scale=math.nan), dict(n_dims=64, ext_factor=1.0), dict(n_dims=64, ext_factor=1.0, n_ctx_orig=4096, freq_base=1.0),
               dict(n_dims=64, ext_factor=1.0, n_ctx_orig=4096, freq_scale=0.0), dict(n_dims=64, ext_factor=1.0, n_ctx_orig=4096, beta_slow=0.0),
               dict(n_dims=64, ext_factor=math.nan), dict(n_dims=64, attn_factor=math.inf)):
        assert refused(spec=M.rope_spec(**kw), back=back) == e, kw
    wide = [514, 1, 8, 1]
    assert refused(src=desc(M.F32, wide), dst=desc(M.F32, wide, ptr=0x900000), spec=M.rope_spec(514), back=back) == e


def test_null_arguments():
    L = M.lib()
    a, p, s = desc(M.F32, [64, 4, 8, 2]), desc(M.I32, [8]), M.rope_spec(64)
    R = C.byref
    for args in ((None, R(p), None, R(a), R(s), None), (R(a), None, None, R(a), R(s), None), (R(a), R(p), None, None, R(s), None),
                 (R(a), R(p), None, R(a), None, None)):
        assert L.ggml_mi355x_rope(*args) == -1 and L.ggml_mi355x_rope_back(*args) == -1
    with pytest.raises(M.Mi355xError):
        M.from_torch(torch.zeros(4))
