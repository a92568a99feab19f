"""Waits of the tcgen05 attention kernel that run out: its MMA issuer is told to stop after some tasks in
every CTA and the waits to expire after 20 ms (``SGLD_ATTEND_STALL``), so that the other roles wait for
what nobody signals, leave, and the kernel ends.  No row may then be left unwritten: it is right, or NaN
with a NaN log-sum-exp."""
import pytest
import torch

from sglang_decode.prompt import prompt_attention
from tests.attention_reference import check, prompt
from tests.test_gpu_prefix import Setup

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def pointers(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).int().cuda()


def case(lens, past, hq, hkv, d, dtype, pool):
    kv = [n + p for n, p in zip(lens, past)]
    q, k, v = (torch.randn(n, h, d, device="cuda").to(dtype) for n, h in ((sum(lens), hq), (sum(kv) + 5, hkv), (sum(kv) + 5, hkv)))
    index = torch.randperm(sum(kv) + 5, device="cuda")[:sum(kv)].int() if pool else None
    return q, k, v, kv, index


@pytest.mark.parametrize("stall", [0, 1, 3])
@pytest.mark.parametrize("lens,past,hq,hkv,d,dtype,pool,window", [
    ([4000], [0], 32, 8, 64, BF, False, -1),                    # boxes; 504 tasks, so that some CTA takes a fourth
    ([4000], [100], 32, 8, 64, FP, True, 500),                  # row copies
    ([300, 1, 0, 77], [0, 40, 3, -50], 8, 2, 128, BF, False, -1),
    ([3, 2], [2000, 3000], 8, 2, 128, FP, True, -1),            # split results, merged
])
def test_no_row_is_left_unwritten(cuda_device, monkeypatch, stall, lens, past, hq, hkv, d, dtype, pool, window):
    q, k, v, kv, index = case(lens, past, hq, hkv, d, dtype, pool)
    out, lse = torch.full_like(q, 5.0), torch.full(q.shape[:2], 5.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    call = lambda: prompt_attention(q, k, v, pointers(lens), kv_indptr=pointers(kv), kv_indices=index, window_left=window,
                                    out=out, lse=lse, status=status)
    monkeypatch.setenv("SGLD_ATTEND_STALL", f"{stall}:20000000")
    call()
    torch.cuda.synchronize()
    monkeypatch.delenv("SGLD_ATTEND_STALL")
    none = out.isnan().all(-1)
    assert torch.equal(none, out.isnan().any(-1)) and torch.equal(none, lse.isnan())
    if stall == 0 or sum(lens) == 4000:
        assert none.any() and status.item() == 1
    if stall == 0:
        seen = torch.cat([torch.arange(n, device="cuda") + m - n >= 0 for n, m in zip(lens, kv)])
        assert none[seen].all()                                 # (tiles that see no key need no issuer)
    want = prompt(q, k, v, lens, kv, index, window=window)
    check(out[~none], [x[~none] for x in want], dtype, max(kv), lse[~none])
    status.zero_()
    call()                                                      # nothing is left behind
    check(out, want, dtype, max(kv), lse)
    assert status.item() == 0


@pytest.mark.parametrize("page", [1, 64])
def test_shared_prefix(cuda_device, monkeypatch, page):
    s = Setup([5, 60, 0], 1000, 8, 2, 128, BF, page=page)
    monkeypatch.setenv("SGLD_ATTEND_STALL", "0:20000000")
    out = s.run().clone()
    assert out.isnan().all() and s.engine.layers[0].status.item() == 1
    monkeypatch.delenv("SGLD_ATTEND_STALL")
    s.engine.layers[0].status.zero_()
    s.check(s.run())


def test_waits_behind_rows_that_are_formed_again_go_on(cuda_device, monkeypatch):
    """The last 63 other tokens of each head see 16000 finite keys beside a masked NaN: a warp sums 32 of such
    rows for some 30 ms, and the waits expire after a millisecond without a step of it."""
    q, k, v, kv, index = case([16000], [0], 16, 4, 128, BF, False)
    clean = prompt_attention(q, k, v, pointers([16000]))
    v[15999] = float("nan")
    out, status = torch.full_like(q, 5.0), torch.zeros(1, dtype=torch.int32, device="cuda")
    monkeypatch.setenv("SGLD_ATTEND_STALL", "-1:1000000")
    prompt_attention(q, k, v, pointers([16000]), out=out, status=status)
    torch.cuda.synchronize()
    assert status.item() == 0
    check(out[-64:], prompt(q[-64:], k, v, [64], [16000]), BF, 16000)
    assert torch.equal(out[:-64], clean[:-64])
