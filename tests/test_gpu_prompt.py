"""Prompt attention on the GPU against the formula in 64 bits (tolerance: tests/attention_reference.py)."""
import ctypes
import random

import pytest
import torch

from sglang_decode import _native
from sglang_decode.prompt import prompt_attention
from tests.attention_reference import check, prompt

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def pointers(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).int().cuda()


def heads_major(x):
    """The same values with each head's rows in one run."""
    return x.transpose(0, 1).contiguous().transpose(0, 1)


def odd_rows(x):
    """The same values in rows that start off a 16-byte boundary."""
    y = torch.empty(*x.shape[:-1], x.shape[-1] + 1, dtype=x.dtype, device=x.device)
    y[..., 1:] = x
    return y[..., 1:]


def run(q_lens, past, hq, hkv, d, dtype, pool=False, layout="plain", cap=0.0, window=-1, scale=None, seed=0, edit=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv_lens = [n + p for n, p in zip(q_lens, past)]
    new = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)
    q = new(sum(q_lens), hq, d)
    rows = sum(kv_lens) + (7 if pool else 0)
    k, v = new(rows, hkv, d), new(rows, hkv, d)
    index = torch.randperm(rows, generator=g, device="cuda")[:sum(kv_lens)].int() if pool else None
    if edit is not None:
        q, k, v = edit(q, k, v)
    want = prompt(q, k, v, q_lens, kv_lens, index, scale, cap, window)
    if layout == "heads":
        k, v = heads_major(k), heads_major(v)
    if layout == "odd":
        q, k, v = odd_rows(q), odd_rows(k), odd_rows(v)
    if layout == "fused":
        x = torch.cat([t.flatten(1) for t in (q, k, v)], 1) if q.shape[0] == k.shape[0] else None
        q, k, v = (t.unflatten(1, (-1, d)) for t in x.split([hq * d, hkv * d, hkv * d], 1))
    lse = torch.full((q.shape[0], hq), 9.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = prompt_attention(q, k, v, pointers(q_lens), kv_indptr=pointers(kv_lens) if pool or any(past) else None,
                           kv_indices=index, scale=scale, logit_cap=cap, window_left=window, lse=lse, status=status)
    check(out, want, dtype, max(kv_lens, default=0), lse)
    assert status.item() == 0
    return out


@pytest.mark.parametrize("layout", ["plain", "odd"])      # the tcgen05 kernel, and the mma.sync kernel
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[1], [33], [128], [129], [16, 17], [300, 1, 0, 64, 2], [1000, 7, 513]])
def test_lengths(cuda_device, lens, d, layout):
    run(lens, [0] * len(lens), 8, 2, d, BF, layout=layout)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (6, 2), (5, 1), (7, 1), (28, 4), (16, 1), (12, 12), (32, 8)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_head_groups(cuda_device, hq, hkv, dtype):
    run([70, 1, 141], [0, 0, 0], hq, hkv, 128, dtype)
    run([70, 1, 141], [5, 300, 0], hq, hkv, 64, dtype, pool=True)


@pytest.mark.parametrize("lens,past", [([200, 40], [0, 33]), ([1], [700]), ([5, 300], [129, 0])])
def test_head_dim_256(cuda_device, lens, past):
    run(lens, past, 8, 1, 256, BF, pool=True)
    run(lens, past, 4, 4, 256, FP, cap=20.0)


@pytest.mark.parametrize("layout", ["plain", "heads", "fused", "odd"])
def test_layouts(cuda_device, layout):
    run([100, 260, 1], [0, 0, 0], 8, 2, 128, BF, layout=layout)
    if layout != "fused":
        run([100, 260, 1], [3, 500, 64], 8, 2, 128, FP, layout=layout, pool=True)


@pytest.mark.parametrize("layout", ["plain", "odd"])
@pytest.mark.parametrize("window", [0, 1, 63, 128, 500])
def test_windows(cuda_device, window, layout):
    run([400, 1, 700], [0, 900, 130], 8, 2, 64, FP, pool=True, window=window, layout=layout)


@pytest.mark.parametrize("layout", ["plain", "odd"])
@pytest.mark.parametrize("window", [0, 39, 40, 41, 170, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1])
def test_windows_through_the_c_abi(cuda_device, window, layout):
    """Any int32 window, 2^31 - 1 as "none" among them, with tiles whose first queries lie before key 0."""
    q_lens, kv_lens = [100, 7], [41, 129]
    q, k, v = (torch.randn(n, h, 128, device="cuda").to(BF) for n, h in ((107, 8), (170, 2), (170, 2)))
    want = prompt(q, k, v, q_lens, kv_lens, window=window)
    if layout == "odd":
        q, k, v = odd_rows(q), odd_rows(k), odd_rows(v)
    out, lse = torch.full((107, 8, 128), 5.0, device="cuda", dtype=BF), torch.zeros(107, 8, device="cuda")
    q_indptr, kv_indptr = pointers(q_lens), pointers(kv_lens)
    a = _native.PromptArgs()
    a.q, a.k, a.v, a.out, a.lse = (x.data_ptr() for x in (q, k, v, out, lse))
    a.q_indptr, a.kv_indptr = q_indptr.data_ptr(), kv_indptr.data_ptr()
    for name, x in (("q", q), ("k", k), ("v", v), ("out", out)):
        getattr(a, name + "_stride")[:] = x.stride()
    a.kv_extent, a.tokens, a.seqs, a.query_heads, a.kv_heads, a.head_dim, a.dtype = 170, 107, 2, 8, 2, 128, 1
    a.window_left, a.scale = window, 128 ** -0.5
    size = _native.load().sgld_prompt_workspace_bytes(ctypes.byref(a))
    workspace = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert _native.load().sgld_prompt_attention(ctypes.byref(a), workspace.data_ptr(), size, stream) == 0
    check(out, want, BF, 129, lse)


@pytest.mark.parametrize("layout", ["plain", "odd"])
def test_soft_cap_and_scale(cuda_device, layout):
    run([300, 20], [0, 70], 8, 2, 128, BF, cap=5.0, layout=layout)
    run([300, 20], [0, 70], 8, 2, 64, FP, cap=30.0, scale=1.5, layout=layout)
    run([300, 20], [0, 70], 8, 2, 64, FP, scale=0.01, layout=layout)


@pytest.mark.parametrize("layout", ["plain", "odd"])
def test_small_scores_under_a_large_cap_keep_their_precision(cuda_device, layout):
    """One key a row: the LSE is the capped score, which is small beside the cap.  Its error: the score's
    sum (40 roundings of 2^-23 of scale |q||k|), then fewer than 16 roundings of 2^-24 relative."""
    q, k, v = (torch.randn(300, h, 128, device="cuda").to(BF) * 0.1 for h in (4, 4, 4))
    want = prompt(q, k, v, [300], [300], cap=50.0, window=0)
    if layout == "odd":
        q, k, v = odd_rows(q), odd_rows(k), odd_rows(v)
    lse = torch.zeros(300, 4, device="cuda")
    prompt_attention(q, k, v, pointers([300]), logit_cap=50.0, window_left=0, lse=lse)
    ds = want[3] - 2.0 ** -21 * 50                      # the reference's allowance without its cap term
    assert ((lse.double() - want[1]).abs() <= ds + 16 * 2.0 ** -24 * want[1].abs() + 2.0 ** -22).all()


@pytest.mark.parametrize("layout", ["plain", "odd"])
@pytest.mark.parametrize("lens,past", [([1], [5000]), ([1, 1, 1], [4000, 0, 129]), ([9], [2999]), ([3, 0, 2], [0, 77, 3000])])
def test_few_rows_over_many_keys(cuda_device, lens, past, layout):
    """The keys are split and the split results merged."""
    run(lens, past, 8, 2, 128, BF, pool=True, layout=layout)
    run(lens, past, 16, 1, 64, FP, layout=layout)


def test_more_queries_than_keys(cuda_device):
    """Queries before key 0 see nothing: zeros, and -inf."""
    for layout in ("plain", "odd"):
        run([50, 200, 3], [-20, -150, -3], 8, 2, 128, BF, pool=True, layout=layout)


def test_many_sequences(cuda_device):
    rng = random.Random(3)
    lens = [rng.choice([0, 1, 2, 17, 40, 90, 131]) for _ in range(150)]
    run(lens, [rng.choice([0, 3, 200]) for _ in lens], 8, 2, 64, BF, pool=True)


def test_scores_that_rise_and_outgrow_the_running_maximum(cuda_device):
    def rise(q, k, v):
        k = k.abs() * torch.linspace(0.1, 6, k.shape[0], device="cuda")[:, None, None].to(k.dtype)
        return q.abs(), k, v
    for layout in ("plain", "odd"):
        run([900], [0], 4, 1, 128, BF, edit=rise, layout=layout)
        run([300], [600], 4, 1, 64, FP, edit=rise, pool=True, layout=layout)


def test_many_windowed_sequences_and_the_largest_group(cuda_device):
    rng = random.Random(4)
    lens = [rng.choice([1, 5, 64, 300]) for _ in range(140)]            # more than are sorted
    run(lens, [rng.choice([0, 50, 400]) for _ in lens], 16, 1, 64, FP, pool=True, window=100)
    lens = lens[:100]
    run(lens, [rng.choice([0, 50, 400]) for _ in lens], 4, 2, 128, BF, pool=True, window=100)
    run([40, 300], [500, 0], 16, 1, 256, BF, pool=True, window=70, cap=10.0)


def test_expanded_tensors(cuda_device):
    """Heads or rows that share memory (stride 0) are read as they are."""
    q, k, v = (torch.randn(150, h, 128, device="cuda").to(BF) for h in (8, 1, 1))
    for kk, vv in ((k.expand(150, 2, 128), v.expand(150, 2, 128)), (k[:1].expand(150, 1, 128), v)):
        out = prompt_attention(q, kk, vv, pointers([150]))
        check(out, prompt(q, kk, vv, [150], [150]), BF, 150)
    qq = q[:, :1].expand(150, 8, 128)
    check(prompt_attention(qq, k, v, pointers([150])), prompt(qq, k, v, [150], [150]), BF, 150)


@pytest.mark.parametrize("layout", ["plain", "odd"])
@pytest.mark.parametrize("d", [64, 256])
def test_small_weights_keep_their_bits(cuda_device, layout, d):
    """2000 keys of weight 2^-18.4 beside one whose value is zero: the result is theirs alone."""
    q = torch.zeros(1, 4, d, device="cuda", dtype=FP)
    k, v = (torch.zeros(2001, 1, d, device="cuda", dtype=FP) for _ in range(2))
    q[..., 0], k[700, :, 0] = 1.0, 12.734375
    v[:], v[700] = 1.0, 0.0
    want = prompt(q, k, v, [1], [2001], scale=1.0)
    if layout == "odd":
        q, k, v = odd_rows(q), odd_rows(k), odd_rows(v)
    lse = torch.zeros(1, 4, device="cuda")
    out = prompt_attention(q, k, v, pointers([1]), kv_indptr=pointers([2001]), scale=1.0, lse=lse)
    check(out, want, FP, 2001, lse)


def test_two_long_sequences(cuda_device):
    run([2050, 1200], [0, 0], 4, 2, 128, BF)


@pytest.mark.parametrize("d,layout", [(128, "plain"), (64, "plain"), (128, "odd"), (256, "plain")])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(cuda_device, d, layout):
    def edit(q, k, v):
        v[70, 0, 3] = float("nan")        # key 70 of the first sequence: its rows before see nothing of it
        v[150, 1] = float("inf")
        k[90, 0] = float("nan")
        v[200:] = float("nan")            # the second sequence's
        return q, k, v
    run([200, 40], [0, 0], 8, 2, d, BF, edit=edit, layout=layout)


@pytest.mark.parametrize("layout", ["plain", "odd"])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 128), (8, 2, 64), (16, 1, 128)])
def test_whole_tiles_beside_a_masked_value_that_is_not_finite(cuda_device, layout, hq, hkv, d):
    """Only the last key is NaN: all rows of its tiles but the last are formed again, in the place where
    their first results were stored, also as split results."""
    def edit(q, k, v):
        v[-1] = float("nan")
        return q, k, v
    run([300], [0], hq, hkv, d, BF, edit=edit, layout=layout)
    run([40], [3000], hq, hkv, d, FP, edit=edit, layout=layout)


BAD = {
    "one early key": lambda v: v[5, :, 3].fill_(float("nan")),
    "all from the middle on": lambda v: v[v.shape[0] // 2:].fill_(float("nan")),
    "an infinity in every 64 keys": lambda v: v[::64, :, 7].fill_(float("inf")),
    "both infinities and a NaN, dims apart": lambda v: (v[70, :, 0].fill_(float("inf")), v[90, :, 0].fill_(-float("inf")),
                                                        v[90, :, 1].fill_(-float("inf")), v[131, :, 1].fill_(float("nan")),
                                                        v[-1, :, 2].fill_(float("inf"))),
    "the last keys": lambda v: v[-3:].fill_(-float("inf")),
}


@pytest.mark.parametrize("d,layout", [(128, "plain"), (64, "plain"), (64, "odd"), (128, "odd"), (256, "plain")])
@pytest.mark.parametrize("bad", list(BAD))
def test_what_a_row_becomes_beside_values_that_are_not_finite(cuda_device, bad, d, layout):
    """Rows that see them, in the dims that have them, and no others; causal, on cache slots, in a window
    whose lower edge passes them, and as split results."""
    def edit(q, k, v):
        v = v.clone()
        BAD[bad](v)
        return q, k, v
    run([333], [0], 8, 2, d, BF, edit=edit, layout=layout)
    run([150, 40], [300, 0], 4, 4, d, FP, edit=edit, layout=layout, pool=True, cap=15.0)
    run([333], [100], 16, 1, d, BF, edit=edit, layout=layout, window=70)
    run([3], [1500], 8, 2, d, FP, edit=edit, layout=layout)


@pytest.mark.parametrize("layout", ["plain", "odd"])
def test_sums_that_pass_the_largest_number_on_the_way(cuda_device, layout):
    """Values of 2^124 under equal weights: their weighted sum before the division does not fit fp32."""
    q, k = (torch.zeros(300, h, 128, device="cuda", dtype=BF) for h in (4, 4))
    v = torch.full((300, 4, 128), 2.0 ** 124, device="cuda", dtype=BF)
    if layout == "odd":
        q, k, v = odd_rows(q), odd_rows(k), odd_rows(v)
    out = prompt_attention(q, k, v, pointers([300]))
    check(out, prompt(q, k, v, [300], [300]), BF, 300)


@pytest.mark.parametrize("bad", ["one early key", "all from the middle on", "an infinity in every 64 keys", "K"])
def test_bad_values_in_a_long_prompt_cost_no_second_pass_for_each_row(cuda_device, bad):
    """4096 tokens of 16 heads.  A walk of every row over its own keys would be 1.3e8 dependent steps of
    1.7 us (measured so at 1024 tokens) by 1184 warps, 190 ms; whole warps search 2048 tiles of at most
    4096 keys.  The best of three runs is bounded by a fifth of the walk."""
    q, k, v = (torch.randn(4096, h, 128, device="cuda").to(BF) for h in (16, 4, 4))
    if bad == "K":
        k[5] = float("nan")
    else:
        BAD[bad](v)
    status, ends = torch.zeros(1, dtype=torch.int32, device="cuda"), pointers([4096])
    out = prompt_attention(q, k, v, ends, status=status)
    times = []
    for _ in range(3):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        prompt_attention(q, k, v, ends, out=out, status=status)
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end))
    assert min(times) < 38 and status.item() == 0
    some = torch.tensor([0, 4, 5, 6, 63, 64, 65, 1000, 2047, 2048, 2049, 4095], device="cuda")
    finite = torch.isfinite(out[some])
    rows = some[:, None]
    seen = {"K": rows >= 5, "one early key": rows >= 5, "all from the middle on": rows >= 2048,
            "an infinity in every 64 keys": rows >= 0}[bad][:, None].expand(-1, 16, 128).clone()
    if bad not in ("K", "all from the middle on"):
        dim = 3 if bad == "one early key" else 7
        seen[..., :dim] = seen[..., dim + 1:] = False
    assert torch.equal(finite, ~seen)


@pytest.mark.parametrize("layout", ["plain", "odd"])
def test_rows_behind_the_last_sequence_stay(cuda_device, layout):
    q, k, v = (torch.randn(300, h, 128, device="cuda").to(BF) for h in (8, 2, 2))
    for t in (q, k, v):
        t[131:] = float("nan")
    if layout == "odd":
        q, k, v = odd_rows(q), odd_rows(k), odd_rows(v)
    out, lse = torch.full((300, 8, 128), 5.0, device="cuda", dtype=BF), torch.full((300, 8), 5.0, device="cuda")
    prompt_attention(q, k, v, pointers([100, 31]), out=out, lse=lse)
    assert (out[131:] == 5).all() and (lse[131:] == 5).all()
    check(out[:131], prompt(q[:131], k, v, [100, 31], [100, 31]), BF, 100, lse[:131])
    # the split form
    out.fill_(5.0)
    lse.fill_(5.0)
    index = torch.arange(131, device="cuda").repeat(20).int()
    prompt_attention(q[:4], k, v, pointers([1, 2]), kv_indptr=pointers([1000, 1620]), kv_indices=index, out=out[:4], lse=lse[:4])
    assert (out[3:] == 5).all() and (lse[3:] == 5).all()
    check(out[:3], prompt(q[:3], k, v, [1, 2], [1000, 1620], index), BF, 1620, lse[:3])


@pytest.mark.parametrize("layout", ["plain", "odd"])
def test_indices_outside_the_pool_read_as_zeros(cuda_device, layout):
    q, k, v = (torch.randn(200, h, 128, device="cuda").to(BF) for h in (8, 2, 2))
    index = torch.randperm(200, device="cuda").int()
    index[[3, 77]], index[[150, 199]] = -1, 200
    index[100] = 2 ** 31 - 1
    want = prompt(q, k, v, [200], [200], torch.where((index >= 0) & (index < 200), index, -1))
    if layout == "odd":
        q, k, v = odd_rows(q), odd_rows(k), odd_rows(v)
    out = prompt_attention(q, k, v, pointers([200]), kv_indptr=pointers([200]), kv_indices=index)
    check(out, want, BF, 200)


def test_nothing_to_do(cuda_device):
    z = lambda n, h: torch.zeros(n, h, 128, device="cuda", dtype=BF)
    assert prompt_attention(z(0, 4), z(0, 2), z(0, 2), pointers([0, 0])).shape == (0, 4, 128)
    out = torch.full((3, 4, 128), 5.0, device="cuda", dtype=BF)
    prompt_attention(z(3, 4), z(3, 2), z(3, 2), pointers([]), out=out)
    assert (out == 5).all()
    out = prompt_attention(z(3, 4), z(0, 2), z(0, 2), pointers([3]), kv_indptr=pointers([0]), out=out)
    assert (out == 0).all()
    out.fill_(5.0)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    prompt_attention(z(3, 4), z(9, 2), z(9, 2), pointers([3]), kv_indptr=pointers([0]), kv_indices=none, out=out)
    assert (out == 0).all()


def test_which_kernel_runs(cuda_device):
    lib, q, k = _native.load(), torch.zeros(64, 8, 128, device="cuda", dtype=BF), torch.zeros(64, 2, 128, device="cuda", dtype=BF)
    a = _native.PromptArgs()
    a.q = a.out = q.data_ptr()
    a.k = a.v = k.data_ptr()
    a.q_indptr = q.data_ptr()
    a.q_stride[:] = a.out_stride[:] = q.stride()
    a.k_stride[:] = a.v_stride[:] = k.stride()
    a.kv_extent = a.tokens = 64
    a.seqs, a.query_heads, a.kv_heads, a.head_dim, a.dtype, a.window_left, a.scale = 1, 8, 2, 128, 1, -1, 0.1
    import ctypes
    assert lib.sgld_prompt_kernel_kind(ctypes.byref(a)) == 2          # tcgen05 + TMA
    a.q = q.data_ptr() + 2
    assert lib.sgld_prompt_kernel_kind(ctypes.byref(a)) == 0          # mma.sync


def test_side_streams_and_graph_replay(cuda_device):
    cases = []
    for seed, lens in ((1, [150, 33]), (2, [500])):
        g = torch.Generator(device="cuda").manual_seed(seed)
        q, k, v = (torch.randn(sum(lens), h, 128, generator=g, device="cuda").to(BF) for h in (8, 2, 2))
        cases.append((q, k, v, pointers(lens), prompt_attention(q, k, v, pointers(lens))))
    few = (cases[1][0][:1], *cases[1][1:3])
    few_args = dict(kv_indptr=pointers([500]))
    few_want = prompt_attention(*few, pointers([1]), **few_args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [torch.zeros_like(c[0]) for c in cases]
    for _ in range(3):
        for s, c, o in zip(streams, cases, outs):
            with torch.cuda.stream(s):
                prompt_attention(*c[:4], out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(o, c[4]) for o, c in zip(outs, cases))
    graph, out, few_out = torch.cuda.CUDAGraph(), torch.zeros_like(outs[0]), torch.zeros_like(few_want)
    q, k, v, indptr, want = cases[0]
    one = pointers([1])
    with torch.cuda.graph(graph):
        prompt_attention(q, k, v, indptr, out=out)
        prompt_attention(*few, one, **few_args, out=few_out)
    for _ in range(2):
        out.zero_()
        few_out.zero_()
        graph.replay()
        assert torch.equal(out, want) and torch.equal(few_out, few_want)
    indptr.copy_(pointers([183, 0]))                                   # other lengths in the same buffers
    graph.replay()
    check(out, prompt(q, k, v, [183, 0], [183, 0]), BF, 183)


def test_refusals(cuda_device):
    q, k, v = (torch.zeros(10, h, 128, device="cuda", dtype=BF) for h in (8, 2, 2))
    p = pointers([10])
    bad = [
        dict(q=q.float()), dict(k=k.half()), dict(v=v[:5]), dict(q=q[:, :3]), dict(k=k[..., :64], v=v[..., :64]),
        dict(q=q[..., :96], k=k[..., :96], v=v[..., :96]), dict(q=q.repeat(1, 5, 1)), dict(indptr=p.long()), dict(indptr=p.cpu()),
        dict(indptr=p[:0]), dict(kv_indptr=pointers([5, 5])), dict(kv_indices=p), dict(kv_indptr=p, kv_indices=p.long()),
        dict(out=q[:4]), dict(out=q.half()), dict(lse=torch.zeros(10, 7, device="cuda")), dict(lse=torch.zeros(10, 8, device="cuda", dtype=BF)),
        dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(logit_cap=-1.0), dict(logit_cap=float("inf")),
        dict(out=q), dict(out=q[:, :1].expand(10, 8, 128)), dict(out=torch.zeros(11, 8, 128, device="cuda", dtype=BF)[:10], q=None),
        dict(window_left=-2), dict(status=torch.zeros(1, device="cuda")), dict(k=k.cpu()),
    ]
    for changes in bad:
        args = dict(dict(q=q, k=k, v=v, indptr=p), **changes)
        if args["q"] is None:                       # rows 1.. of out's own memory
            args["q"] = args["out"]._base[1:]
        with pytest.raises(ValueError):
            prompt_attention(args.pop("q"), args.pop("k"), args.pop("v"), args.pop("indptr"), **args)
