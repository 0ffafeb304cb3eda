"""Attention of requests that share their first rows, on the GPU, against the definition in 64 bits and against the
attention that reads every request's rows."""
import numpy as np
import pytest
import torch

import paged_util as U

pytestmark = pytest.mark.gpu


class Groups:
    """Requests in groups: (rows shared, [rows of their own], [query rows]) each, on shuffled pages.  Shared rows are
    whole pages plus, where `prefix` is none, rows that the members hold alike on pages of their own."""

    def __init__(self, pkg, groups, page, nq, nkv, dtype=torch.float16, seed=0, strength=1.0, base=0, growth=None):
        rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
        self.page, self.nq, self.nkv, self.sizes = page, nq, nkv, [len(own) for _, own, _ in groups]
        cdiv = lambda a: -(-a // page)
        self.lens = [p + o for p, own, _ in groups for o in own]
        self.rows = [r for _, _, rows in groups for r in rows]
        pages = sum(cdiv(p) + sum(cdiv(p + o) - p // page for o in own) for p, own, _ in groups)
        perm = iter((base + rng.permutation(pages + 5)).astype(np.int32).tolist())
        self.pool = pkg.q4_pool(base + pages + 5, nkv, page)
        self.table = np.full((len(self.lens), max(1, max(map(cdiv, self.lens)))), -1, np.int32)
        self.ks, self.vs, i = [], [], 0
        make = lambda n: [(torch.randn(n, nkv, 128, generator=g) * s).to(dtype) for s in (strength, 0.5)]
        for p, own, _ in groups:
            common = [next(perm) for _ in range(p // page)]
            k0, v0 = make(p)
            for o in own:
                k1, v1 = make(o)
                k, v = torch.cat([k0, k1]), torch.cat([v0, v1])
                if growth:
                    k = (k.double() * growth(torch.arange(p + o).double())[:, None, None]).to(dtype)
                mine = common + [next(perm) for _ in range(cdiv(p + o) - p // page)]
                self.table[i, :len(mine)] = mine
                if p + o:
                    pos = np.arange(p + o)
                    slots = torch.from_numpy((np.array(mine, np.int64)[pos // page] * page + pos % page).astype(np.int32)).cuda()
                    pkg.q4_append(k.cuda(), v.cuda(), slots, self.pool)
                self.ks.append(U.q4_values(k))
                self.vs.append(U.q4_values(v))
                i += 1
        self.q = torch.randn(sum(self.rows), nq, 128, generator=g).to(dtype).cuda()
        i32 = lambda v: torch.tensor(np.array(v), dtype=torch.int32).cuda()
        self.d_table, self.d_lens, self.starts = i32(self.table), i32(self.lens), i32(np.concatenate([[0], np.cumsum(self.rows)]))

    def attend(self, pkg, causal, scale=None, **kw):
        plan = pkg.paged_prefix_plan(self.d_table, self.d_lens, kw.pop("sizes", self.sizes), self.page, self.starts,
                                     max(max(self.rows), 1), causal, kw.pop("max_group", None), kw.pop("least", 0))
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = pkg.q4_prefix_attention(self.q, self.pool, self.d_table, plan, scale, status=status, **kw)
        return out, plan, int(status)

    def check(self, pkg, causal, scale=None, **kw):
        out, plan, status = self.attend(pkg, causal, scale, **kw)
        assert status == 0
        want, bound = U.attention(self.q, self.ks, self.vs, self.rows, U.scale_of(128) if scale is None else scale, causal)
        # (the join multiplies both sides by an exponential and adds them in fp32: 2^-18 of the weights)
        tol = U.attention_tolerance(want, bound, out.dtype) + bound[0] * 2.0 ** -18
        err = (out.double().cpu() - want).abs()
        assert bool((err <= tol).all()), float((err - tol).max())
        plain = pkg.q4_attention(self.q, self.pool, self.d_table, self.d_lens, self.starts, max(max(self.rows), 1), causal,
                                 scale=scale)
        assert bool(((out.double() - plain.double()).abs().cpu() <= 2 * tol).all())
        return plan


HEADS = [(4, 1), (8, 8), (12, 4), (5, 1), (40, 8)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("nq,nkv", HEADS)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_two_groups_of_single_tokens(pkg, causal, nq, nkv, page):
    d = Groups(pkg, [(512, [1, 40, 300], [1, 1, 1]), (256, [5, 64], [1, 1])], page, nq, nkv, torch.bfloat16, seed=page + nq)
    plan = d.check(pkg, causal)
    assert plan.prefix.tolist() == [512, 256]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("members,rows", [(2, 1), (3, 4), (9, 2), (33, 5), (70, 1), (2, 33)])
def test_sizes_of_groups_and_blocks(pkg, dtype, members, rows):
    rng = np.random.default_rng(members)
    own = [int(x) for x in rng.integers(rows, 90, members)]
    ragged = [int(x) for x in rng.integers(0, rows + 1, members)]
    ragged[0] = rows
    d = Groups(pkg, [(1003, own, ragged), (0, [rows], [rows]), (70, own[:2], [rows, 1])], 32, 8, 2, dtype, seed=rows)
    for causal in (True, False):
        plan = d.check(pkg, causal)
        assert plan.prefix.tolist()[1] == 0 and plan.prefix.tolist()[0] == 1003 // 32 * 32 or sum(r > 0 for r in ragged) < 2


def test_prefixes_end_where_a_query_row_ends(pkg):
    """Causal rows that see less than the shared rows, requests without rows of their own, and ones without any."""
    d = Groups(pkg, [(128, [0, 0, 3], [7, 1, 2]), (64, [0, 0], [64, 80]), (48, [0, 0, 0], [0, 0, 3]), (0, [0, 0], [2, 1])], 16, 8, 2)
    plan = d.check(pkg, True)
    assert plan.prefix.tolist() == [112, 0, 0, 0]        # 128 - 7 + 1 rows seen by the first row; rows behind length 0
    plan = d.check(pkg, False)
    assert plan.prefix.tolist() == [128, 64, 0, 0]
    assert plan.own_lens.tolist()[:5] == [0, 0, 3, 0, 0]


def test_members_that_sit_out_or_hold_other_pages(pkg):
    d = Groups(pkg, [(320, [10, 20, 30, 40], [1, 0, 2, 1])], 16, 8, 2, seed=3)
    d.table[1] = 0                                        # no query rows: its pages do not matter
    d.d_table = torch.from_numpy(d.table).cuda()
    assert d.check(pkg, True).prefix.tolist() == [320]
    d.table[3, 4] = d.table[2, 4] = -1                    # a page outside the pool, in both: hidden for one, shared by two
    d.d_table = torch.from_numpy(d.table).cuda()
    plan = d.attend(pkg, True)[1]
    assert plan.prefix.tolist() == [64]                   # the first member has it
    out, plain = d.attend(pkg, True)[0], pkg.q4_attention(d.q, d.pool, d.d_table, d.d_lens, d.starts, 2, True)
    assert float((out.double() - plain.double()).abs().max()) <= 2e-2 * float(plain.abs().max())
    d.table[0, 4] = -1
    d.d_table = torch.from_numpy(d.table).cuda()
    out, plan, _ = d.attend(pkg, True)
    assert plan.prefix.tolist() == [320]
    plain = pkg.q4_attention(d.q, d.pool, d.d_table, d.d_lens, d.starts, 2, True)
    assert float((out.double() - plain.double()).abs().max()) <= 2e-2 * float(plain.abs().max())


def test_what_spares_little_is_not_shared(pkg):
    d = Groups(pkg, [(160, [10, 20, 30], [1, 1, 2]), (96, [5, 5], [1, 1])], 16, 8, 2, seed=9)
    for least, want in ((0, [160, 96]), (2 * 160 + 96, [160, 96]), (2 * 160 + 97, [0, 0]), (1 << 40, [0, 0])):
        assert d.check(pkg, True, least=least).prefix.tolist() == want


def test_requests_of_no_group_and_groups_on_the_device(pkg):
    d = Groups(pkg, [(0, [50], [1]), (160, [10, 20, 30], [1, 1, 2]), (0, [33], [2])], 16, 8, 2, seed=4)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    assert d.check(pkg, True, sizes=i32([1, 4]), max_group=3).prefix.tolist() == [160]
    assert d.check(pkg, True, sizes=i32([-3, 1, 4, 2, 99]), max_group=3).prefix.tolist() == [0, 160, 0, 0]   # kept ascending
    assert d.check(pkg, True, sizes=[5]).prefix.tolist() == [0]
    _, _, status = d.attend(pkg, True, sizes=i32([0, 5]), max_group=2)
    assert status == 64                                   # more query rows in a group than promised
    assert not d.attend(pkg, True, sizes=i32([1, 4]), max_group=1)[1].shares


def test_groups_on_the_device_that_the_host_rule_misjudges(pkg):
    # one group of three beside empty ones, and groups of three that the caller states as groups of one
    d = Groups(pkg, [(128, [30, 1, 70], [2, 2, 2])], 64, 8, 2, seed=12)
    bounds = torch.tensor([0, 0, 0, 3, 3], dtype=torch.int32, device="cuda")
    assert d.check(pkg, True, sizes=bounds, max_group=3).prefix.tolist()[2] == 128
    assert d.check(pkg, True, sizes=bounds, max_group=3, least=256).prefix.tolist()[2] == 128
    assert d.check(pkg, True, sizes=bounds, max_group=3, least=257).prefix.tolist() == [0] * 4
    whole = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    assert d.check(pkg, True, sizes=whole, max_group=1).prefix.tolist() == [0]


@pytest.mark.parametrize("rows", [1, 5, 33])
def test_pages_beyond_4_gb(pkg, rows):
    d = Groups(pkg, [(512, [3, 100, 64], [rows] * 3)], 256, 16, 8, seed=15, base=16000)
    assert d.pool.nbytes > 1 << 32
    # whole pages that the first member's first row sees: of 515 - (rows - 1) rows
    assert d.check(pkg, True).prefix.tolist() == [(516 - rows) // 256 * 256]


def test_no_rows_and_nobody_with_rows(pkg):
    d = Groups(pkg, [(64, [3, 5], [0, 0]), (64, [2, 2], [0, 0])], 64, 4, 2, seed=16)
    plan = pkg.paged_prefix_plan(d.d_table, d.d_lens, d.sizes, 64, d.starts, 4, True, least=0)
    assert plan.prefix.tolist() == [0, 0] and plan.own_lens.tolist() == d.lens
    assert pkg.q4_prefix_attention(d.q, d.pool, d.d_table, plan).shape == (0, 4, 128)
    out = torch.full((3, 4, 128), 5.0, dtype=torch.float16, device="cuda")     # rows that no request owns
    pkg.q4_prefix_attention(torch.zeros_like(out), d.pool, d.d_table, plan, out=out)
    assert bool((out == 5).all())


@pytest.mark.parametrize("nq,nkv,rows", [(2, 1, 1), (12, 1, 1), (4, 1, 9)])
def test_as_many_requests_as_there_may_be(pkg, nq, nkv, rows):
    # 2,048 requests in 64 groups, and in 1,024 pairs
    d = Groups(pkg, [(16, [i % 3 for i in range(32)], [rows] * 32)] * 64, 16, nq, nkv, seed=13)
    assert d.check(pkg, False).prefix.tolist() == [16] * 64
    d = Groups(pkg, [(32, [1, 2], [rows, rows])] * 1024, 16, nq, nkv, seed=14)
    assert d.check(pkg, False).prefix.tolist() == [32] * 1024


@pytest.mark.parametrize("strength,scale", [(1.0, None), (300.0, None), (30.0, 1.0), (1.0, 1e-20), (3e4, 3e4)])
def test_large_and_small_scores(pkg, strength, scale):
    """Weights that live on one side, on both, on one key, or on none in particular.  (Where scores pass 2^24 a
    key's weight against another's is beyond fp32: compare with the attention that reads all rows.)"""
    d = Groups(pkg, [(256, [20, 300, 1], [3, 1, 2])], 16, 8, 2, torch.bfloat16, seed=5, strength=strength)
    if strength < 1e4:
        d.check(pkg, True, scale)
    else:
        out, _, _ = d.attend(pkg, True, scale)
        plain = pkg.q4_attention(d.q, d.pool, d.d_table, d.d_lens, d.starts, 3, True, scale=scale)
        assert torch.equal(out, plain) and bool(torch.isfinite(out).all())


GROWTH = {"up": lambda pos: 1 + pos / 40, "down": lambda pos: 40 / (1 + pos / 40), "steps": lambda pos: 1 + 30 * (pos // 128 % 3)}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("growth", GROWTH)
@pytest.mark.parametrize("members,nq,nkv", [(20, 4, 1), (33, 16, 2), (70, 4, 1), (3, 4, 1)])
def test_scores_that_grow_or_fall_along_the_cache(pkg, dtype, growth, members, nq, nkv):
    # (every tile of shared rows passes the references of the tiles before, or none does)
    d = Groups(pkg, [(1424, [1 + i % 7 for i in range(members)], [1 + i % 3 for i in range(members)])], 16, nq, nkv, dtype,
               seed=21, growth=GROWTH[growth])
    assert d.check(pkg, False).prefix.tolist() == [1424]


@pytest.mark.parametrize("rows", [1, 3, 5, 9])
def test_query_rows_of_all_magnitudes_in_bf16(pkg, rows):
    d = Groups(pkg, [(700, [5] * 30, [rows] * 30)], 64, 8, 2, torch.bfloat16, seed=22)
    size = torch.arange(d.q.shape[0], device="cuda") % 7 - 3
    d.q *= (2.0 ** (14 * size))[:, None, None].to(torch.bfloat16)
    d.q[0] = 0
    d.check(pkg, False)


def test_shared_pages_that_are_not_there(pkg):
    # entries outside the pool hide their rows, as in q4_attention
    d = Groups(pkg, [(1024, [9] * 40, [1] * 40)], 32, 16, 4, seed=23)
    hidden = [0, 5, 17, 31]
    d.d_table[:, hidden] = torch.tensor([-1, 10 ** 6, -7, 2 ** 30], dtype=torch.int32, device="cuda")
    out, plan, status = d.attend(pkg, False)
    assert plan.prefix.tolist() == [1024]
    keep = torch.tensor([p // 32 not in hidden for p in range(1024 + 9)])
    want, bound = U.attention(d.q, [k[keep] for k in d.ks], [v[keep] for v in d.vs], d.rows, U.scale_of(128), False)
    tol = U.attention_tolerance(want, bound, out.dtype) + bound[0] * 2.0 ** -18
    assert bool(((out.double().cpu() - want).abs() <= tol).all())


def test_without_starts_and_with_strided_queries(pkg):
    d = Groups(pkg, [(200, [9, 70, 3, 28], [3, 3, 3, 3])], 32, 12, 4, seed=6)
    want, _, _ = d.attend(pkg, True)
    wide = torch.zeros(12, 20, 128, dtype=torch.float16, device="cuda")
    wide[:, 3:15] = d.q
    plan = pkg.paged_prefix_plan(d.d_table, d.d_lens, [4], 32, max_rows=3, causal=True, least=0)
    assert torch.equal(pkg.q4_prefix_attention(wide[:, 3:15], d.pool, d.d_table, plan), want)
    out = torch.empty_like(want)
    ws = pkg.q4_prefix_workspace(50, 5, 9, 12, 4)        # a larger one serves
    for _ in range(3):
        assert pkg.q4_prefix_attention(d.q, d.pool, d.d_table, plan, out=out, workspace=ws) is out
        assert torch.equal(out, want)
    empty = pkg.paged_prefix_plan(d.d_table, d.d_lens, [4], 32, torch.zeros(5, dtype=torch.int32).cuda(), 3, True, least=0)
    assert pkg.q4_prefix_attention(d.q[:0], d.pool, d.d_table, empty).shape == (0, 12, 128)


def test_a_run_of_forked_requests_through_the_cache(pkg):
    """fork, reserve, rotary positions, append, plan, attend: as the ordinary attention over the same cache."""
    g = torch.Generator().manual_seed(7)
    cache = pkg.PagedKVCacheQ4(2, 120, 2, 6, 1024, 16, forkable=True)
    rope = pkg.Rope(128, 1e4)

    def rows(n, heads):
        return torch.randn(n, heads, 128, generator=g).half().cuda()

    step = cache.reserve([333, 0, 0, 100, 0, 0])
    for l in range(2):
        cache.append(l, pkg.apply_rope(rows(433, 2), rope, step), rows(433, 2), step)
    cache.fork([0, 0, 3, 3], [1, 2, 4, 5], [333, 320, 100, 100])
    for new in ([1] * 6, [4, 4, 0, 3, 2, 4]):
        step = cache.reserve(new)
        plan = cache.prefix_plan(step, [3, 3], max(new), least=0)
        assert plan.prefix.tolist() == [320, 96]
        for l in range(2):
            cache.append(l, pkg.apply_rope(rows(sum(new), 2), rope, step), rows(sum(new), 2), step)
            q = pkg.apply_rope(rows(sum(new), 8), rope, step)
            got, want = cache.attend(l, q, step, max(new), plan=plan), cache.attend(l, q, step, max(new))
            # (two roundings to f16, and the two orders of summation)
            assert float((got.double() - want.double()).abs().max()) <= 4 * 2.0 ** -11 * float(want.abs().max())
        cache.trim(1)
    cache.check()
    with pytest.raises(ValueError, match="plan"):
        cache.attend(0, q, step, max(new), causal=False, plan=plan)
    with pytest.raises(ValueError, match="plan"):
        cache.attend(0, q, step, max(new), window=5, plan=plan)


def test_streams_and_graphs(pkg):
    d = Groups(pkg, [(300, [9, 70, 3, 28], [3, 3, 3, 1])], 16, 8, 2, seed=8)
    want, _, _ = d.attend(pkg, True)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(d.attend(pkg, True)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    groups, ws = torch.tensor([0, 4], dtype=torch.int32).cuda(), pkg.q4_prefix_workspace(10, 3, 4, 8, 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = pkg.paged_prefix_plan(d.d_table, d.d_lens, groups, 16, d.starts, 3, True, max_group=4, least=0)
        out = pkg.q4_prefix_attention(d.q, d.pool, d.d_table, plan, workspace=ws)
        with pytest.raises(ValueError, match="graph"):
            pkg.paged_prefix_plan(d.d_table, d.d_lens, [4], 16, d.starts, 3, True)
    d.q.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, d.attend(pkg, True)[0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("count", [5, 40])
def test_groups_of_many_rows_and_all_lengths(pkg, dtype, count):
    # several items a CTA, of one tile to ten, with 65 to 300 query rows a kv head
    lens = [16, 128, 144, 384, 640, 1280, 256]
    d = Groups(pkg, [(lens[i % 7], [1 + (i + j) % 5 for j in range(17 + i % 4 * 19)], [1] * (17 + i % 4 * 19)) for i in range(count)],
               16, 8, 2, dtype, seed=31)
    plan = d.check(pkg, True)
    assert plan.prefix.tolist() == [lens[i % 7] for i in range(count)]


def test_large_groups_on_two_streams_and_in_graphs(pkg):
    d = Groups(pkg, [(2048, [1 + i % 9 for i in range(40)], [1] * 40), (1000, [3] * 70, [1] * 70)], 16, 16, 4, torch.bfloat16, seed=32)
    want = d.attend(pkg, True)[0]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(d.attend(pkg, True)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    groups = torch.tensor([0, 40, 110], dtype=torch.int32, device="cuda")
    graphs = []
    for _ in range(2):       # (two graphs that share a workspace, one after the other)
        ws = graphs[0][2] if graphs else pkg.q4_prefix_workspace(110, 1, 70, 16, 4)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan = pkg.paged_prefix_plan(d.d_table, d.d_lens, groups, 16, d.starts, 1, True, max_group=70, least=0)
            graphs.append((graph, pkg.q4_prefix_attention(d.q, d.pool, d.d_table, plan, workspace=ws), ws))
    d.q.mul_(0.5)
    want = d.attend(pkg, True)[0]
    for _ in range(3):
        for graph, _, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out, _ in graphs)
