"""ROPE, ROPE_BACK and FLASH_ATTN_EXT nodes through the plugin's graph_compute and supports_op, driven by a
minimal ggml-like host (oracle/graph_host.cpp) in a process of its own: the results are those of the direct
API bit for bit (tests/test_rope.py and tests/test_attention.py hold that against the formulas), on the
first call, on the calls that capture and replay the graph, and after an operand changed."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HOST = os.path.join(ROOT, "oracle", "libgraph_host.so")

BODY = r'''
import ctypes as C, math, os, struct, sys
sys.path[:0] = [os.path.join(ROOT, "ggml-gfx906_amd")]
import torch
import mi355x_qmm as M
H = C.CDLL(os.path.join(ROOT, "oracle", "libgraph_host.so"), mode=C.RTLD_GLOBAL)
assert H.gh_open(M.LIB_PATH.encode()) == 1
M.lib()
ROPE, ROPE_BACK, ATTN = 47, 48, 67
def ints(*v):
    return [struct.unpack("i", struct.pack("f", x))[0] if isinstance(x, float) else x for x in v]
def node(op, d, src=(), params=()):
    p = ints(*params)
    return H.gh_tensor(op, d.type, d.ne, d.nb, C.c_void_p(d.data), (C.c_int * 10)(*src), len(src), (C.c_int32 * 16)(*p), len(p))
def leaf(d):
    return node(0, d)
def graph(*n):
    H.gh_graph((C.c_int * len(n))(*n), len(n))
def compute():
    torch.cuda.synchronize()
    assert H.gh_compute() == 0
g = torch.Generator(device="cuda").manual_seed(1)
def rnd(*s, dtype=torch.float32):
    return torch.randn(*s, generator=g, device="cuda").to(dtype)
def rope_params(n, mode, base=10000.0, scale=1.0, ext=0.0, attn=1.0, orig=4096):
    return (0, n, mode, 0, orig, base, scale, ext, attn, 32.0, 1.0)
F = M.from_torch
'''

GRAPH = BODY + r'''
B, n, Hq, Hk, D, m = 1, 20, 8, 2, 64, 96
def llama_like(n, first):
    """q and k turned, k and v copied into an f16 cache behind what it holds, masked attention"""
    xq, xk, xv = rnd(B, n, Hq, D), rnd(B, n, Hk, D), rnd(B, n, Hk, D)
    pos = torch.arange(first, first + n, dtype=torch.int32, device="cuda")
    kc, vc = rnd(B, m, Hk, D, dtype=torch.float16), rnd(B, m, Hk, D, dtype=torch.float16)
    ff = 1 + torch.rand(D // 2, generator=g, device="cuda")
    q, k, out = torch.zeros_like(xq), torch.zeros_like(xk), torch.zeros_like(xq)
    seen = torch.arange(m, device="cuda")[None] <= pos[:, None]
    mask = torch.zeros(64, m, device="cuda").masked_fill(torch.cat([~seen, torch.ones(64 - n, m, dtype=torch.bool, device="cuda")]), -math.inf).half()
    sinks = rnd(Hq)
    lp, lf = leaf(F(pos)), leaf(F(ff))
    rq = node(ROPE, F(q), (leaf(F(xq)), lp, lf), rope_params(D, 2, ext=1.0, scale=0.25))
    rk = node(ROPE, F(k), (leaf(F(xk)), lp, lf), rope_params(D, 2, ext=1.0, scale=0.25))
    ks, vs = kc[:, first : first + n], vc[:, first : first + n]
    ck = node(33, F(ks), (rk, leaf(F(ks))))
    cv = node(33, F(vs), (leaf(F(xv)), leaf(F(vs))))
    hf = lambda t: F(t.permute(0, 2, 1, 3))
    at = node(ATTN, F(out), (leaf(hf(q)), leaf(hf(kc)), leaf(hf(vc)), leaf(F(mask)), leaf(F(sinks))), (0.125, 0.0, 30.0, 10))
    for t in (rq, rk, ck, cv, at):
        assert H.gh_supports(t) == 1, t
    return (rq, rk, ck, cv, at), (xq, xk, xv, pos, kc, vc, ff, mask, sinks, out, q, k), first
def direct(state):
    (xq, xk, xv, pos, kc, vc, ff, mask, sinks, *_), first = state[1], state[2]
    n = xq.shape[1]
    spec = M.rope_spec(D, M.ROPE_HALVES, freq_scale=0.25, ext_factor=1.0, n_ctx_orig=4096)
    q, k, out, kc, vc = torch.empty_like(xq), torch.empty_like(xk), torch.empty_like(xq), kc.clone(), vc.clone()
    M.rope(F(xq), F(pos), F(q), spec, factors=F(ff))
    M.rope(F(xk), F(pos), F(k), spec, factors=F(ff))
    kc[:, first : first + n] = k
    vc[:, first : first + n] = xv
    hf = lambda t: F(t.permute(0, 2, 1, 3))
    M.flash_attn(hf(q), hf(kc), hf(vc), F(out), M.attn_spec(0.125, 0.0, 30.0), mask=F(mask), sinks=F(sinks))
    torch.cuda.synchronize()
    return out
for n, first in ((20, 0), (1, 50), (64, 32)):
    s = llama_like(n, first)
    graph(*s[0])
    for call in range(5):
        want = direct(s)
        s[1][9].zero_()
        compute()
        assert torch.equal(s[1][9], want), (n, call, (s[1][9] - want).abs().max())
        s[1][0].normal_(generator=g)
        s[1][3].add_(0 if call < 3 else 1)
    print("graph", n, "ok", flush=True)
for mode in (0, 2):
    x, y, pos = rnd(2, 5, 3, 80), rnd(2, 5, 3, 80), torch.arange(5, dtype=torch.int32, device="cuda")
    b = node(ROPE_BACK, F(y), (leaf(F(x)), leaf(F(pos))), rope_params(48, mode))
    assert H.gh_supports(b) == 1
    graph(b)
    want = torch.empty_like(x)
    M.rope_back(F(x), F(pos), F(want), M.rope_spec(48, mode))
    for _ in range(3):
        y.zero_()
        compute()
        assert torch.equal(y, want)
print("GRAPH_OK", flush=True)
'''

REFUSED = BODY + r'''
x, pos = rnd(1, 5, 3, 64), torch.arange(20, dtype=torch.int32, device="cuda")
p5 = leaf(F(pos[:5]))
for params in (rope_params(64, 8), rope_params(64, 24), rope_params(63, 0), rope_params(66, 0), rope_params(64, 2, ext=1.0, orig=0)):
    assert H.gh_supports(node(ROPE, F(torch.empty_like(x)), (leaf(F(x)), p5), params)) == 0, params
assert H.gh_supports(node(ROPE, F(torch.empty_like(x)), (leaf(F(x)), leaf(F(pos))), rope_params(64, 0))) == 0
assert H.gh_supports(node(ROPE, F(torch.empty_like(x)), (leaf(F(x.permute(0, 1, 3, 2))), p5), rope_params(64, 0))) == 0
hf = lambda t: leaf(F(t.permute(0, 2, 1, 3)))
def attn(q, k, v, *more, d=None, params=(0.125, 0.0, 0.0, 10)):
    return H.gh_supports(node(ATTN, F(d if d is not None else torch.empty_like(q)), (hf(q), hf(k), hf(v)) + more, params))
q, k = rnd(1, 4, 8, 64), rnd(1, 70, 2, 64, dtype=torch.float16)
mask = torch.zeros(4, 70, dtype=torch.float16, device="cuda")
assert attn(q, k, k) == 1 and attn(q, k, k, leaf(F(mask))) == 1 and attn(q, k, k, leaf(F(mask)), params=(0.125, 8.0, 0.0, 10)) == 1
assert attn(q, k, k, params=(0.125, 8.0, 0.0, 10)) == 0
assert attn(q, k, k, leaf(F(mask.float()))) == 0 and attn(q, k, k, leaf(F(mask[:3]))) == 0
assert attn(q, k.bfloat16(), k.bfloat16()) == 0 and attn(q, k.float(), k.float()) == 0 and attn(q, k, k[..., :32]) == 0
assert attn(rnd(1, 4, 8, 576), rnd(1, 70, 1, 576, dtype=torch.float16), rnd(1, 70, 1, 576, dtype=torch.float16)) == 0
assert attn(rnd(1, 4, 3, 64), k, k) == 0
print("REFUSED_OK", flush=True)
'''

VIEWS = BODY + r'''
q, k = rnd(1, 4, 8, 64), rnd(1, 70, 2, 64, dtype=torch.float16)
hf = lambda t: leaf(F(t.permute(0, 2, 1, 3)))
whole = leaf(F(rnd(100000)))
for of in range(3):
    for offset, want in ((0, 1), (16, 1), (4096 + 32, 1), (8, 0), (4096 + 2, 0)):
        src = [hf(q), hf(k), hf(k)]
        H.gh_view(src[of], whole, C.c_size_t(offset))
        assert H.gh_supports(node(ATTN, F(torch.empty_like(q)), src, (0.125, 0.0, 0.0, 10))) == want, (of, offset)
print("VIEWS_OK", flush=True)
'''


def run(body, word):
    if not os.path.exists(HOST):
        subprocess.check_call(["make", "-s", "-C", os.path.join(ROOT, "oracle")])
    r = subprocess.run([sys.executable, "-u", "-c", f"ROOT = {ROOT!r}\n" + body], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and word in r.stdout, (r.stdout[-1500:], r.stderr[-3000:])


@pytest.mark.gpu
def test_graph_equals_the_direct_calls():
    run(GRAPH, "GRAPH_OK")


@pytest.mark.gpu
def test_supports_op_declines():
    run(REFUSED, "REFUSED_OK")


@pytest.mark.gpu
def test_supports_op_sees_where_a_view_will_lie():
    """a graph is handed out before its tensors have data: a view at an odd offset is declined then, not when it runs"""
    run(VIEWS, "VIEWS_OK")
