"""Shared-prefix decode on the GPU against attention over prefix + own tokens in 64 bits
(tolerance: tests/attention_reference.py)."""
import pytest
import torch

from sglang_decode.config import DecodeConfig, Mode
from sglang_decode.runtime.engine import DecodeEngine
from sglang_decode.runtime.prefix import SharedPrefixEngine
from sglang_decode.workloads import split_hints, update_plan
from tests.attention_reference import attend, check

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


class Setup:
    """One batch: a pool, the prefix's slots or pages, each request's own tokens, and an engine."""

    def __init__(self, lens, prefix, hq, hkv, d, dtype, page=1, capacity=None, max_splits=8, mode=-1, seed=0, prefix_capacity=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        cap = capacity or len(lens)
        self.lens, self.n, self.hq, self.hkv, self.d, self.dtype, self.page = lens, prefix, hq, hkv, d, dtype, page
        need = [-(-x // page) for x in [prefix] + lens]
        pages = sum(need) + 5
        order = torch.randperm(pages, generator=g, device="cuda").int()
        new = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)
        self.k, self.v, self.q = new(pages, page, hkv, d), new(pages, page, hkv, d), new(len(lens), hq, d)
        self.prefix = order[:need[0]].clone()
        self.config = DecodeConfig(batch_capacity=cap, max_splits=max_splits, max_context=max(max(lens), 1), query_heads=hq,
                                   kv_heads=hkv, head_dim=d, page_size=page)
        at = need[0]
        table = torch.full((cap, self.config.max_pages), -1, dtype=torch.int32, device="cuda")
        for r, x in enumerate(need[1:]):
            table[r, :x] = order[at:at + x]
            at += x
        self.table = table
        if page == 1:
            self.k, self.v = self.k[:, 0], self.v[:, 0]
            self.pages = order[need[0]:at].clone()
            self.indptr = torch.tensor([0] + lens + [0] * (cap - len(lens))).cumsum(0).int().cuda()
        else:
            self.pages, self.indptr = table, None
        self.engine = SharedPrefixEngine(self.config, prefix_capacity or len(self.prefix) * page, dtype=dtype, force_mode=int(mode))
        update_plan(self.engine, lens, split_hints(lens, max_splits))

    def rows(self, pages, n):
        return (pages.long()[:, None] * self.page + torch.arange(self.page, device="cuda")).flatten()[:n]

    def want(self, prefix=None, cap=0.0, scale=None):
        n = self.n if prefix is None else prefix
        k, v = (x.reshape(-1, self.hkv, self.d) for x in (self.k, self.v))
        shared = self.rows(self.prefix, n)
        bad = (shared < 0) | (shared >= k.shape[0])
        parts = [torch.zeros(len(self.lens), self.hq, *s, dtype=torch.float64, device="cuda") for s in ((self.d,), (), (self.d,), ())]
        g = self.hq // self.hkv
        for r, x in enumerate(self.lens):
            rows = torch.cat([shared.clamp(0, k.shape[0] - 1), self.rows(self.table[r, :-(-x // self.page)], x)])
            zero = torch.zeros(len(rows), dtype=torch.bool, device="cuda")
            zero[:n] = bad
            for h in range(self.hkv):
                kk, vv = (torch.where(zero[:, None], 0, t[rows, h]) for t in (k, v))
                for dst, src in zip(parts, attend(self.q[r, h * g:(h + 1) * g], kk, vv, self.d ** -0.5 if scale is None else scale, cap)):
                    dst[r, h * g:(h + 1) * g] = src
        return parts

    def run(self, **more):
        if "prefix_length" not in more:
            more["prefix_length"] = torch.tensor([self.n], dtype=torch.int32, device="cuda")
        self.engine.prepare()
        return self.engine.execute(self.q, self.k, self.v, self.pages, self.prefix, indptr=self.indptr, **more)

    def check(self, out, **more):
        b = len(self.lens)
        check(out[:b], self.want(**more), self.dtype, self.n + max(self.lens))
        assert (out[b:] == 0).all()
        assert self.engine.layers[0].status.item() == 0


CASES = [  # own lengths, prefix, hq, hkv, d, dtype, page
    ([1], 1, 1, 1, 128, BF, 1),
    ([5, 0, 33, 300], 700, 8, 2, 128, BF, 1),
    ([5, 0, 33, 300], 129, 28, 4, 128, FP, 1),
    ([64, 1, 17], 1000, 16, 1, 128, BF, 16),
    ([64, 1, 17], 130, 6, 2, 64, FP, 64),
    ([100] * 20, 513, 7, 1, 64, BF, 1),
    ([30, 200], 257, 4, 2, 256, BF, 16),
    ([3] * 33, 90, 10, 2, 256, FP, 1),
    ([(37 * i) % 200 for i in range(70)], 2000, 32, 8, 128, BF, 16),
    ([(37 * i) % 90 + 1 for i in range(130)], 4099, 5, 1, 128, FP, 1),
    ([0, 0, 0], 300, 8, 2, 128, BF, 1),
    ([40, 3], 0, 8, 2, 128, BF, 1),
]


@pytest.mark.parametrize("lens,prefix,hq,hkv,d,dtype,page", CASES)
def test_matches_attention_over_prefix_and_own_tokens(cuda_device, lens, prefix, hq, hkv, d, dtype, page):
    s = Setup(lens, prefix, hq, hkv, d, dtype, page)
    out = s.run()
    s.check(out)
    assert s.engine.layers[0].counter.tolist() == [0, 0]
    first = out.clone()
    assert torch.equal(s.run(), first)                    # the same bits again, no state left behind


@pytest.mark.parametrize("mode", list(Mode))
def test_every_mode_and_spare_capacity(cuda_device, mode):
    s = Setup([5, 260, 0, 33, 100], 300, 8, 2, 128, BF, capacity=9, mode=mode)
    s.check(s.run())


def test_soft_cap_scale_and_whole_prefix_by_default(cuda_device):
    s = Setup([5, 60], 320, 8, 2, 128, FP, page=16)
    s.check(s.run(logit_cap=8.0, scale=0.3, prefix_length=None), cap=8.0, scale=0.3)


def test_length_on_the_device_bounds_the_prefix(cuda_device):
    s = Setup([5, 60, 0], 900, 8, 2, 128, BF)
    length = torch.zeros(1, dtype=torch.int32, device="cuda")
    for n, seen in ((0, 0), (1, 1), (128, 128), (500, 500), (900, 900), (4000, 900), (-3, 0)):
        length.fill_(n)
        s.check(s.run(prefix_length=length), prefix=seen)


def test_new_rows_are_written_before_the_decode(cuda_device):
    s = Setup([5, 60, 7], 200, 8, 2, 128, BF)
    kn, vn = (torch.randn(3, 2, 128, device="cuda").to(BF) for _ in range(2))
    last = torch.stack([s.table[r, x - 1] for r, x in enumerate(s.lens)]).long()
    out = s.run(k_new=kn, v_new=vn, new_loc=last)
    assert torch.equal(s.k[last], kn) and torch.equal(s.v[last], vn)
    s.check(out)


def test_head_major_odd_and_strided_pools(cuda_device):
    s = Setup([5, 60, 7], 300, 8, 2, 128, BF)
    k, v = s.k, s.v
    s.k, s.v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
    s.check(s.run())
    wide = torch.zeros(*k.shape[:2], 129, dtype=BF, device="cuda")
    wide[..., 1:] = k
    s.k = wide[..., 1:]
    s.check(s.run())
    s.k, s.v, s.q = k, v, torch.cat([s.q, s.q], 2)[..., 64:192]
    s.check(s.run())


def test_prefix_slots_outside_the_pool_read_as_zeros(cuda_device):
    for page in (1, 16):
        s = Setup([5, 60], 512, 8, 2, 128, BF, page=page)
        s.prefix[3], s.prefix[7] = -1, s.k.shape[0]
        s.check(s.run())


def test_values_outside_the_prefix_do_not_matter(cuda_device):
    s = Setup([5, 60], 200, 8, 2, 128, BF, page=64)
    used = torch.cat([s.rows(s.prefix, 200)] + [s.rows(s.table[r, :1], x) for r, x in enumerate(s.lens)])
    for x in (s.k, s.v):
        flat = x.view(-1, 2, 128)
        keep = flat[used].clone()
        flat.fill_(float("nan"))
        flat[used] = keep
    s.check(s.run())


def test_an_inactive_row_and_a_broken_plan(cuda_device):
    s = Setup([5, 60, 7], 200, 8, 2, 128, BF)
    s.engine.plan.active.fill_(2)
    out = s.run()
    check(out[:2], [x[:2] for x in s.want()], BF, 300)
    assert (out[2] == 0).all()
    s.engine.plan.lengths[0] = -5
    assert s.run().isnan().all()


def test_no_index_of_own_tokens(cuda_device):
    """Empty ``pages``: the prefix alone, and a NaN row where the plan gives a request own tokens."""
    s = Setup([0, 0, 0], 300, 8, 2, 128, BF)
    assert s.pages.numel() == 0
    s.check(s.run())
    assert s.engine.kernel_kind() == "none"
    s.engine.plan.lengths[1] = 1            # (the capacity: more is a broken plan)
    out = s.run().clone()
    assert out[1].isnan().all() and s.engine.layers[0].status.item() == 512
    check(out[::2], [x[::2] for x in s.want()], BF, 300)
    assert s.engine.layers[0].counter.tolist() == [0, 0]
    s.engine.plan.lengths[1] = 0
    s.engine.layers[0].status.zero_()
    s.check(s.run())


def test_smaller_prefix_than_the_capacity_and_layers(cuda_device):
    s = Setup([9, 30], 640, 32, 8, 128, BF, prefix_capacity=20000)
    s.check(s.run())
    with pytest.raises(ValueError):
        SharedPrefixEngine(s.config, -1)
    small = SharedPrefixEngine(s.config, 639)
    with pytest.raises(ValueError):
        small.execute(s.q, s.k, s.v, s.pages, s.prefix, indptr=s.indptr)


def test_graph_replay_with_a_growing_prefix(cuda_device):
    s = Setup([9, 30, 0, 200], 1500, 8, 2, 128, BF)
    length = torch.tensor([1500], dtype=torch.int32, device="cuda")
    s.run(prefix_length=length)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.run(prefix_length=length)
    for n in (1500, 3, 1001):
        length.fill_(n)
        graph.replay()
        s.check(out, prefix=n)


def test_agrees_with_the_plain_engine_over_joined_sequences(cuda_device):
    s = Setup([9, 30, 200], 400, 8, 2, 128, BF)
    config = DecodeConfig(batch_capacity=3, max_splits=8, max_context=600, query_heads=8, kv_heads=2, head_dim=128, page_size=1)
    plain = DecodeEngine(config, dtype=BF)
    lens = [400 + x for x in s.lens]
    update_plan(plain, lens)
    plain.prepare()
    joined = torch.cat([torch.cat([s.prefix, s.table[r, :x]]) for r, x in enumerate(s.lens)])
    indptr = torch.tensor([0] + lens).cumsum(0).int().cuda()
    got = plain.execute(s.q, s.k, s.v, joined, indptr=indptr)
    check(got, s.want(), BF, 600)
    s.check(s.run())


def test_a_pool_of_one_page(cuda_device):
    """Its page stride is never used: any value is accepted."""
    s = Setup([9], 7, 8, 2, 128, BF, page=16)
    page = torch.randn(1, 16, 2, 128, device="cuda").to(BF)
    s.k, s.v = (x.as_strided(x.shape, (8 * 1000, 256, 128, 1)) for x in (page, page.flip(1).contiguous()))
    s.prefix.fill_(0)
    s.table[:, 0] = 0
    out = s.run()
    k, v = s.k[0], s.v[0]
    rows = torch.cat([torch.arange(7, device="cuda"), torch.arange(9, device="cuda")])
    for h in range(2):
        heads = slice(4 * h, 4 * h + 4)
        check(out[0, heads], attend(s.q[0, heads], k[rows, h], v[rows, h], 128 ** -0.5), BF, 16)


def test_two_engines_on_two_streams(cuda_device):
    setups = [Setup([9, 30, 200], 700, 8, 2, 128, BF, seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in setups]
    lengths = [torch.tensor([s.n], dtype=torch.int32, device="cuda") for s in setups]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        outs = []
        for s, stream, n in zip(setups, streams, lengths):
            with torch.cuda.stream(stream):
                outs.append(s.run(prefix_length=n))
    torch.cuda.synchronize()
    for s, out in zip(setups, outs):
        s.check(out)


def test_refusals(cuda_device):
    s = Setup([9, 30], 64, 8, 2, 128, BF)
    p = s.prefix
    for changes in (dict(prefix=p.long()), dict(prefix=p.cpu()), dict(prefix=p[None]), dict(prefix=p[::2]), dict(scale=0.0),
                    dict(scale=-1.0), dict(logit_cap=-1.0), dict(prefix_length=torch.zeros(1, device="cuda")),
                    dict(prefix_length=torch.zeros(2, dtype=torch.int32, device="cuda")), dict(q=s.q.half()),
                    dict(k=s.k.to(torch.float8_e4m3fn), v=s.v.to(torch.float8_e4m3fn)), dict(v=s.v[:-1]),
                    dict(new_loc=torch.zeros(2, dtype=torch.int64, device="cuda"))):
        a = dict(dict(q=s.q, k=s.k, v=s.v, pages=s.pages, prefix=p, indptr=s.indptr), **changes)
        with pytest.raises(ValueError):
            s.engine.execute(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("pages"), a.pop("prefix"), **a)
    t = Setup([9, 30], 64, 8, 2, 128, BF, page=16)
    apart = torch.zeros(t.k.shape[0], 20, 2, 128, dtype=BF, device="cuda")[:, :16]
    with pytest.raises(ValueError):
        t.engine.execute(t.q, apart, apart, t.pages, t.prefix)
