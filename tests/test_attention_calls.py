"""Calls of the attention entry points that their documentation allows, and ones that must not reach the GPU."""
import types

import pytest
from test_attention import base, call, desc, formula, full, near, rc, rnd, torch

import mi355x_qmm as M

gpu = pytest.mark.gpu


@pytest.mark.parametrize("nb", [[2, 256, 256, 0], [2, 0, 256, 8192], [2, 256, 0, 256], [2, 0, 0, 0]])
def test_workspace_of_a_broadcast_query(nb):
    """one query for several batches, heads or positions: the size is that of queries of their own"""
    k, kp = desc(M.F16, [128, 9000, 8, 4]), desc(M.F16, [128, 9000, 8])
    q, own = desc(M.F16, [128, 2, 32, 4], nb), desc(M.F16, [128, 2, 32, 4])
    assert M.flash_attn_work_size(q, k) == M.flash_attn_work_size(own, k) > 0
    assert M.flash_attn_prefix_work_size(q, kp, k) == M.flash_attn_prefix_work_size(own, kp, k) > 0


@gpu
@pytest.mark.parametrize("n", [1, 40])
def test_broadcast_query_with_a_workspace(n):
    q = rnd((1, n, 1, 64), "f16", 1, 1.5).expand(3, n, 8, 64)
    k, v = rnd((3, 3000, 2, 64), "f16", 2), rnd((3, 3000, 2, 64), "f16", 3)
    hf = lambda t: M.from_torch(t.permute(0, 2, 1, 3))  # noqa: E731
    work = torch.empty(max(16, M.flash_attn_work_size(hf(q), hf(k))), dtype=torch.uint8, device="cuda")
    out = torch.empty(3, n, 8, 64, dtype=torch.float16, device="cuda")
    near(call(q, k, v, 0.125, work=work, out=out), formula(q, k, v, 0.125, full(3, 3000)))


def tensor_at(index, contiguous=True, kind="cuda"):
    """what the checks look at of a workspace tensor"""
    return types.SimpleNamespace(device=torch.device(kind, index), is_cuda=kind == "cuda", is_contiguous=lambda: contiguous, data_ptr=lambda: 0x10000,
                                 numel=lambda: 1 << 20, element_size=lambda: 1)


@pytest.mark.parametrize("work", [torch.empty(1 << 20, dtype=torch.uint8), torch.empty(16, dtype=torch.uint8).expand(1 << 16, 16), tensor_at(0, False)],
                         ids=["host", "host broadcast", "strided"])
def test_workspaces_that_a_kernel_may_not_write(work):
    """host memory would be written by the GPU, a broadcast one behind its end"""
    a = base()
    with pytest.raises(M.Mi355xError, match="workspace"):
        M.flash_attn(a["q"], a["k"], a["v"], a["dst"], a["params"], work=work, stream=0)
    with pytest.raises(M.Mi355xError, match="workspace"):
        M.flash_attn_prefix(a["q"], desc(M.F16, [64, 70, 2]), desc(M.F16, [64, 70, 2]), a["k"], a["v"], a["dst"], a["params"], work=work, stream=0)


def test_workspaces_on_another_gpu_are_refused(monkeypatch):
    monkeypatch.setattr(M, "_several_gpus", True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    a, work = base(), tensor_at(1)
    with pytest.raises(M.Mi355xError, match="GPU 1"):
        M.flash_attn(a["q"], a["k"], a["v"], a["dst"], a["params"], work=work, stream=0)
    with pytest.raises(M.Mi355xError, match="GPU 1"):
        M.flash_attn_prefix(a["q"], desc(M.F16, [64, 70, 2]), desc(M.F16, [64, 70, 2]), a["k"], a["v"], a["dst"], a["params"], work=work, stream=0)


@pytest.mark.parametrize("B,n,H,Hk,Bk", [(0, 3, 8, 2, 0), (0, 3, 8, 2, 1), (2, 3, 0, 0, 2), (2, 3, 0, 2, 2), (2, 0, 8, 2, 2), (0, 0, 0, 0, 0)])
@pytest.mark.parametrize("prefix", [False, True])
def test_calls_without_rows(prefix, B, n, H, Hk, Bk):
    """no sequences, no queries or no heads, beside a cache of none: nothing to do, and no workspace"""
    cache = desc(M.F16, [64, 50, Hk, Bk])
    q, kp = desc(M.F16, [64, n, H, B]), desc(M.F16, [64, 70, Hk])
    more = dict(kp=kp, vp=kp) if prefix else {}
    want = -1 if prefix and Bk != B else 0   # (behind a prefix every sequence has its own cache)
    assert rc(prefix, q=q, k=cache, v=cache, dst=desc(M.F16, [64, H, n, B]), **more) == want
    if not prefix:
        assert rc(q=q, k=cache, v=cache, dst=desc(M.F16, [64, H, n, B]), mask=desc(M.F16, [50, 3, H, B])) == 0
        assert rc(q=q, k=cache, v=cache, dst=desc(M.F16, [64, H, n, B]), mask=desc(M.F16, [50, 3])) == 0
    if want == 0:
        assert (M.flash_attn_prefix_work_size(q, kp, cache) if prefix else M.flash_attn_work_size(q, cache)) == 0


@pytest.mark.parametrize("prefix", [False, True])
def test_rows_without_a_cache_are_refused(prefix):
    assert prefix or rc(mask=desc(M.F16, [50, 3, 0, 1])) == rc(mask=desc(M.F16, [50, 3, 1, 0])) == -1
    for Hk, Bk in ((0, 2), (2, 0), (0, 0)):
        cache = desc(M.F16, [64, 50, Hk, Bk])
        more = dict(kp=desc(M.F16, [64, 70, Hk]), vp=desc(M.F16, [64, 70, Hk])) if prefix else {}
        assert rc(prefix, k=cache, v=cache, **more) == -1
