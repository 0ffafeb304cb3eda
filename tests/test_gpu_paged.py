"""The paged 4-bit K/V cache on the GPU against 64-bit restatements
(paged_util.py), through the package's public operators."""
import numpy as np
import pytest
import torch

import paged_util as U

pytestmark = pytest.mark.gpu
i32 = torch.int32


def _dev(x):
    return torch.tensor(np.array(x), dtype=i32).cuda()


# ---------------------------------------------------------------- reserve and release
def _check_reserve(pkg, lens, new, pages, table, free, head, page, num_slots):
    t_dev, status = _dev(table), torch.zeros(1, dtype=i32).cuda()
    step = pkg.paged_reserve(_dev(lens), _dev(new), _dev(pages), t_dev, _dev(free), _dev([head]), page, num_slots, status)
    table = table.copy()
    starts, slots, lens2, pages2, head2, bits = U.reserve(lens, new, pages, table, free, head, page, num_slots)
    assert step.starts.tolist() == starts
    assert step.slots.tolist() == slots
    assert step.lens.tolist() == lens2 and step.pages.tolist() == pages2
    assert step.head.tolist() == [head2] and status.tolist() == [bits]
    assert np.array_equal(t_dev.cpu().numpy(), table)
    return step, table


@pytest.mark.parametrize("n,page,ctx,rows", [(1, 64, 0, 1), (1, 16, 15, 2), (3, 32, 100, 40), (511, 16, 70, 5),
                                             (512, 64, 300, 16), (513, 128, 900, 33), (2048, 16, 40, 3)])
def test_reserve_matches_definition(pkg, n, page, ctx, rows):
    rng = np.random.default_rng(n + page)
    lens = rng.integers(0, ctx + 1, n).tolist()
    new = rng.integers(0, rows + 1, n).tolist()
    pg = U.Paging(lens, page, seed=n, spare=sum(-(-(a + b) // page) for a, b in zip(lens, new)),
                  max_pages=-(-(ctx + rows) // page) + 1)
    pages = list(pg.pages)
    _check_reserve(pkg, lens, new, pages, pg.table, pg.free, pg.head, page, sum(new) + 5)
    _check_reserve(pkg, lens, new, pages, pg.table, pg.free, pg.head, page, sum(new))


@pytest.mark.parametrize("case", ["dry", "dry_late", "long", "slots", "spare_pages", "no_rows", "negative"])
def test_reserve_turns_requests_away(pkg, case):
    lens, new, page = [10, 64, 0, 33, 7], [60, 1, 200, 2, 3], 32
    pg = U.Paging(lens, page, seed=3, spare=20, max_pages=9)
    pages, free, num_slots = list(pg.pages), pg.free, sum(new)
    if case == "dry":
        free = free[:pg.head + 3]         # request 2 finds too few, 3 needs none
    elif case == "dry_late":
        free = free[:pg.head]
    elif case == "long":
        new[1] = 32 * 9 + 1
        num_slots = sum(new)
    elif case == "slots":
        num_slots = 262
    elif case == "spare_pages":           # pages kept from an earlier trim are used first
        pg.table[0, pages[0]:pages[0] + 2] = pg.free[pg.head:pg.head + 2]
        pages[0] += 2
        free, head = np.concatenate([pg.free[:pg.head + 2], pg.free[pg.head + 2:]]), pg.head + 2
        _check_reserve(pkg, lens, new, pages, pg.table, free, head, page, num_slots)
        return
    elif case == "no_rows":
        new, num_slots = [0] * 5, 0
    elif case == "negative":
        lens[3], new[0], num_slots = -4, -1, sum(new) - 60
    _check_reserve(pkg, lens, new, pages, pg.table, free, pg.head, page, num_slots)


def test_reserve_keeps_inputs_and_strided_table(pkg):
    lens, new, page = [5, 40], [30, 30], 16
    pg = U.Paging(lens, page, spare=10, max_pages=5)
    wide = torch.full((2, 9), -7, dtype=i32).cuda()
    wide[:, :5] = _dev(pg.table)
    ins = [_dev(lens), _dev(new), _dev(pg.pages), _dev(pg.free), _dev([pg.head])]
    keep = [t.clone() for t in ins]
    a = pkg.paged_reserve(ins[0], ins[1], ins[2], wide[:, :5], ins[3], ins[4], page, 60)
    b = pkg.paged_reserve(ins[0], ins[1], ins[2], wide[:, :5], ins[3], ins[4], page, 60)   # the same again
    table = pg.table.copy()
    U.reserve(lens, new, pg.pages, table, pg.free, pg.head, page, 60)
    assert np.array_equal(wide[:, :5].cpu().numpy(), table) and bool((wide[:, 5:] == -7).all())
    assert all(torch.equal(x, y) for x, y in zip(ins, keep))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("n,page,ctx", [(1, 16, 0), (1, 64, 1000), (7, 16, 3000), (600, 32, 200), (2048, 16, 50)])
def test_release_matches_definition(pkg, n, page, ctx):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, ctx + 1, n).tolist()
    keep = [int(rng.integers(0, a + 1)) if rng.random() < 0.8 else a + 100 for a in lens]
    pg = U.Paging(lens, page, seed=n)
    free_dev = pg.dev("free")
    pages, head = pkg.paged_release(_dev(keep), pg.dev("pages"), pg.dev("table"), free_dev, _dev([pg.head]), page)
    free = pg.free.copy()
    left, head2 = U.release(keep, pg.pages, pg.table, free, pg.head, page)
    assert pages.tolist() == left and head.tolist() == [head2]
    assert np.array_equal(free_dev.cpu().numpy(), free)


def test_release_refuses_more_pages_than_were_lent(pkg):
    pg = U.Paging([100, 50], 16)
    free_dev, status = pg.dev("free"), torch.zeros(1, dtype=i32).cuda()
    pages, head = pkg.paged_release(_dev([0, 0]), pg.dev("pages"), pg.dev("table"), free_dev, _dev([2]), 16, status)
    assert pages.tolist() == pg.pages and head.tolist() == [2] and status.tolist() == [8]
    assert np.array_equal(free_dev.cpu().numpy(), pg.free)


# ---------------------------------------------------------------- append and read
def _kv(rows, nkv, dtype, seed, kind="normal"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, rows, nkv, 128, generator=g)
    if kind == "ties":        # halves of the step, and maxima that are a scale times 7.5
        x = torch.randint(-15, 16, x.shape, generator=g) * 0.5 * 2.0 ** torch.randint(-6, 7, (2, rows, nkv, 1), generator=g)
    elif kind == "wide":      # every magnitude that f16 has, subnormal ones among them
        x = x * 2.0 ** torch.randint(-26, 14, x.shape, generator=g)
    elif kind == "tiny":
        x = x * 2.0 ** -20
    return x.to(dtype).unbind(0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["normal", "ties", "wide", "tiny"])
@pytest.mark.parametrize("rows,nkv,page", [(1, 1, 16), (37, 3, 32), (300, 8, 64), (129, 2, 256)])
def test_append_and_read_are_the_definition(pkg, dtype, kind, rows, nkv, page):
    """The rounding is defined to the last bit: equality, in both types, at shuffled slots."""
    k, v = _kv(rows, nkv, dtype, rows + nkv, kind)
    num_pages = -(-rows // page) + 2
    slots = torch.randperm(num_pages * page, generator=torch.Generator().manual_seed(1))[:rows].to(i32).cuda()
    pool = pkg.q4_pool(num_pages, nkv, page)
    status = torch.zeros(1, dtype=i32).cuda()
    pkg.q4_append(k.cuda(), v.cuda(), slots, pool, status)
    for out in (torch.float16, torch.bfloat16):
        kk, vv = pkg.q4_read(pool, slots, out)
        assert kk.dtype is out
        assert torch.equal(kk.double().cpu(), U.q4_values(k)) and torch.equal(vv.double().cpu(), U.q4_values(v))
    assert status.tolist() == [0]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_saturates_and_reports_what_is_not_finite(pkg, dtype):
    k = torch.ones(6, 1, 128).to(dtype)
    k[0, 0, 3] = float("nan")
    k[1, 0, 20] = float("inf")
    k[2, 0, 40] = float("-inf")
    k[3] = float("nan")
    k[4, 0, :2] = torch.tensor([60000.0, -60000.0]).to(dtype)
    if dtype is torch.bfloat16:
        k[5, 0, 0] = 3e38
    pool, slots = pkg.q4_pool(1, 1, 16), torch.arange(6, dtype=i32).cuda()
    status = torch.zeros(1, dtype=i32).cuda()
    pkg.q4_append(k.cuda(), k.cuda(), slots, pool, status)
    kk, vv = pkg.q4_read(pool, slots)
    assert bool(torch.isfinite(kk).all()) and torch.equal(kk, vv)
    assert torch.equal(kk.double().cpu(), U.q4_values(k))
    assert kk[1, 0, 20] == 64512 and kk[2, 0, 40] == -64512 and not kk[3].any() and kk[0, 0, 3] == 0
    assert status.tolist() == [16]


def test_append_takes_slices_of_a_fused_projection_and_skips_rows(pkg):
    nq, nkv, rows = 4, 2, 50
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(rows, (nq + 2 * nkv) * 128, generator=g).to(torch.bfloat16).cuda()
    k = wide[:, nq * 128:(nq + nkv) * 128].view(rows, nkv, 128)
    v = wide[:, (nq + nkv) * 128:].view(rows, nkv, 128)
    slots = torch.arange(rows, dtype=i32).cuda() + 10
    slots[7], slots[8], slots[9] = -1, 64, 2 ** 31 - 1
    pool = pkg.q4_pool(2, nkv, 32)
    pkg.q4_append(k, v, slots, pool)
    kk, vv = pkg.q4_read(pool, slots)
    there = torch.tensor([0 <= s < 64 for s in slots.tolist()])
    want = U.q4_values(k.cpu()) * there[:, None, None]
    assert torch.equal(kk.double().cpu(), want)
    assert torch.equal(vv.double().cpu(), U.q4_values(v.cpu()) * there[:, None, None])
    assert not pool[0].view(nkv, 2, 2304)[:, 0, :10 * 64].any()      # rows 0..9 of K were not touched
    odd = torch.randn(rows, nkv, 132, generator=g).to(torch.float16).cuda()[:, :, 1:129]    # unaligned: copied first
    pkg.q4_append(odd, odd, slots, pool)
    assert torch.equal(pkg.q4_read(pool, slots)[0].double().cpu(), U.q4_values(odd.cpu()) * there[:, None, None])


def test_rows_one_at_a_time_equal_rows_together(pkg):
    k, v = _kv(70, 2, torch.float16, 9)
    a, b = pkg.q4_pool(3, 2, 32), pkg.q4_pool(3, 2, 32)
    slots = torch.arange(70, dtype=i32).cuda()
    pkg.q4_append(k.cuda(), v.cuda(), slots, a)
    for r in range(70):
        pkg.q4_append(k[r:r + 1].cuda(), v[r:r + 1].cuda(), slots[r:r + 1], b)
    assert torch.equal(a, b)


# ---------------------------------------------------------------- attention
class Case:
    def __init__(self, pkg, lens, rows, nq, nkv, page, dtype, seed=0, garbage=False, first_page=0, qscale=1.0):
        self.pg = U.Paging(lens, page, seed=seed, first_page=first_page)
        self.rows, self.nq, self.nkv = rows, nq, nkv
        self.pool = pkg.q4_pool(self.pg.num_pages, nkv, page)
        if garbage:
            self.pool.fill_(0xFF)        # never written: every scale reads back as a NaN
        g = torch.Generator().manual_seed(seed + 100)
        self.k, self.v = [], []
        for a, slots in zip(lens, self.pg.slots):
            k = torch.randn(a, nkv, 128, generator=g).to(dtype)
            v = (torch.randn(a, nkv, 128, generator=g) * 0.5).to(dtype)
            if a:
                pkg.q4_append(k.cuda(), v.cuda(), slots.cuda(), self.pool)
            self.k.append(U.q4_values(k))
            self.v.append(U.q4_values(v))
        self.q = (torch.randn(sum(rows), nq, 128, generator=g) * qscale).to(dtype).cuda()
        self.starts = _dev(np.concatenate([[0], np.cumsum(rows)]))

    def check(self, pkg, out=None, scale=None, **kw):
        mine = out is None
        if mine:
            status = torch.zeros(1, dtype=i32).cuda()
            out = pkg.q4_attention(self.q, self.pool, self.pg.dev("table"), self.pg.dev("lens"), starts=self.starts,
                                   max_rows=max(self.rows + [1]), scale=scale, status=status, **kw)
            assert status.tolist() == [0]
        ref, bound = U.attention(self.q, self.k, self.v, self.rows, scale or 128 ** -0.5, **kw)
        err = (out.double().cpu() - ref).abs()
        tol = U.attention_tolerance(ref, bound, self.q.dtype)
        bad = ~(err <= tol)
        assert not bool(bad.any()), (int(bad.sum()), bad.numel(), float((err / tol).nan_to_num(1e9).max()),
                                     bad.nonzero()[:4].tolist())
        return out


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 130, 257, 1000]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq,nkv,page", [(8, 2, 64), (5, 1, 16), (2, 2, 32), (7, 1, 128), (16, 1, 256)])
@pytest.mark.parametrize("rows", [1, 3])
def test_attention_over_lengths_and_heads(pkg, dtype, nq, nkv, page, rows):
    c = Case(pkg, LENS, [rows] * len(LENS), nq, nkv, page, dtype, seed=nq)
    c.check(pkg)
    c.check(pkg, causal=True)


@pytest.mark.parametrize("rows", [[16, 0, 5, 1, 33], [64, 32, 2, 0, 7]])
@pytest.mark.parametrize("nq,nkv", [(8, 2), (10, 2), (1, 1)])
def test_attention_of_ragged_blocks(pkg, rows, nq, nkv):
    c = Case(pkg, [100, 40, 3, 500, 64], rows, nq, nkv, 32, torch.float16, seed=nq)
    c.check(pkg, causal=True)
    c.check(pkg)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sink,window", [(0, 1), (0, 64), (3, 70), (64, 128), (100, 30), (500, 500), (64, 1000)])
def test_attention_sink_and_window(pkg, causal, sink, window):
    lens = [1, 63, 64, 200, 333, 512, 700]
    for rows in (1, 9):
        c = Case(pkg, lens, [rows] * len(lens), 4, 1, 64, torch.bfloat16, seed=sink)
        c.check(pkg, causal=causal, sink=sink, window=window)


def test_attention_rows_that_see_nothing_are_zeros(pkg):
    c = Case(pkg, [0, 3, 20], [4, 8, 2], 4, 2, 16, torch.float16)
    out = c.check(pkg, causal=True)
    assert not out[:4].any()          # no cached row
    assert not out[4:9].any()         # rows 0..4 of 8 over 3 cached rows end before the first key
    assert bool(out[9:].any())


def test_attention_never_reads_unwritten_rows(pkg):
    """Pool bits that no append wrote (scales that read as NaN) stay out of every result."""
    for rows in (1, 5, 40):
        c = Case(pkg, [1, 17, 70, 200], [rows] * 4, 8, 2, 64, torch.float16, garbage=True)
        c.check(pkg, causal=True)
        c.check(pkg)


def test_attention_hides_pages_outside_the_pool(pkg):
    c = Case(pkg, [200, 90], [2, 2], 4, 2, 32, torch.float16)
    table = c.pg.dev("table")
    table[0, 1], table[0, 3] = -1, c.pg.num_pages      # rows 32..63 and 96..127
    out = pkg.q4_attention(c.q, c.pool, table, c.pg.dev("lens"), starts=c.starts, max_rows=2)
    keep = torch.ones(200, dtype=torch.bool)
    keep[32:64] = keep[96:128] = False
    c.k[0], c.v[0] = c.k[0][keep], c.v[0][keep]
    c.check(pkg, out=out)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_attention_hidden_rows_cannot_spoil_visible_ones(pkg, value):
    """Rows of NaN or infinity behind the causal mask, and queries beside a query of NaN."""
    c = Case(pkg, [40], [10], 4, 2, 16, torch.bfloat16)
    bad = torch.full((4, 2, 128), value).to(torch.bfloat16)
    pkg.q4_append(bad.cuda(), bad.cuda(), c.pg.slots[0][36:].cuda(), c.pool)      # the last four keys
    out = pkg.q4_attention(c.q, c.pool, c.pg.dev("table"), c.pg.dev("lens"), starts=c.starts, max_rows=10, causal=True)
    ref, bound = U.attention(c.q, c.k, c.v, c.rows, 128 ** -0.5, causal=True)
    err = (out.double().cpu() - ref).abs()[:6]
    assert bool((err <= U.attention_tolerance(ref, bound, torch.bfloat16)[:6]).all())
    c.q[3, 1] = float("nan")
    out2 = pkg.q4_attention(c.q, c.pool, c.pg.dev("table"), c.pg.dev("lens"), starts=c.starts, max_rows=10, causal=True)
    assert bool(torch.isnan(out2[3, 1]).all())
    out2[3, 1] = out[3, 1]
    assert torch.equal(out, out2)


@pytest.mark.parametrize("dtype,qscale", [(torch.float16, 30.0), (torch.bfloat16, 30.0), (torch.bfloat16, 1e-6),
                                          (torch.bfloat16, 1e6)])
def test_attention_of_sharp_and_flat_softmax(pkg, dtype, qscale):
    """Scores far apart (the running maximum moves), and query rows outside float16's range."""
    c = Case(pkg, [300, 65], [2, 2], 4, 1, 64, dtype, qscale=qscale)
    c.check(pkg, scale=128 ** -0.5 * (1e-5 if qscale == 1e6 else 1.0))


def test_attention_raises_the_maximum_late(pkg):
    """Keys that grow along the cache: every tile raises the running maximum."""
    c = Case(pkg, [640], [1], 4, 1, 64, torch.float16)
    k = torch.zeros(640, 1, 128)
    k[:, 0, 0] = torch.linspace(0, 120, 640)
    k = k.to(torch.float16)
    pkg.q4_append(k.cuda(), (k * 0.01).cuda(), c.pg.slots[0].cuda(), c.pool)
    c.k[0], c.v[0] = U.q4_values(k), U.q4_values(k * 0.01)
    c.q[:] = 0
    c.q[:, :, 0] = torch.tensor([10.0, 5.0, -10.0, 1.0]).cuda()
    c.check(pkg)


def test_attention_split_over_many_ctas_and_repeated(pkg):
    """One long request is cut over the whole GPU; a workspace serves calls of other shapes in between, and
    the same call gives the same bits."""
    c = Case(pkg, [20000], [1], 4, 1, 64, torch.float16)
    d = Case(pkg, [3, 900, 64, 0, 5000], [2, 1, 0, 2, 2], 8, 2, 16, torch.bfloat16)
    ws = pkg.q4_attention_workspace(5, 2, 8, 1)
    outs = []
    for _ in range(2):
        for x in (c, d):
            outs.append(pkg.q4_attention(x.q, x.pool, x.pg.dev("table"), x.pg.dev("lens"), starts=x.starts,
                                         max_rows=max(x.rows), workspace=ws))
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
    c.check(pkg, out=outs[0])
    d.check(pkg, out=outs[1])


def test_attention_many_requests(pkg):
    """More requests than threads of a CTA, most of them idle or tiny."""
    rng = np.random.default_rng(0)
    lens = rng.integers(0, 40, 1100).tolist()
    rows = [int(x) for x in rng.integers(0, 2, 1100)]
    c = Case(pkg, lens, rows, 2, 1, 16, torch.float16)
    c.check(pkg)


def test_attention_strided_queries_default_starts_and_streams(pkg):
    lens = [70, 5, 129]
    c = Case(pkg, lens, [2, 2, 2], 4, 2, 32, torch.float16)
    wide = torch.zeros(6, (4 + 2 * 2) * 128, dtype=torch.float16).cuda()
    wide[:, :512] = c.q.view(6, 512)
    side = torch.cuda.Stream()
    args = (c.pool, c.pg.dev("table"), c.pg.dev("lens"))
    ref = pkg.q4_attention(c.q, *args, starts=c.starts, max_rows=2)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = pkg.q4_attention(wide[:, :512].view(6, 4, 128), *args, max_rows=2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, ref)
    c.check(pkg, out=out)


def test_offsets_beyond_32_bits(pkg):
    """Pages that lie more than 4 GiB into the pool."""
    nkv, page = 8, 64
    first = (2 ** 32) // (nkv * 4 * 2304) + 10
    c = Case(pkg, [130, 40], [1, 3], 16, nkv, page, torch.float16, first_page=first)
    assert c.pool.numel() > 2 ** 32 and int(c.pg.table.max()) >= first
    c.check(pkg, causal=True)
    k, _ = pkg.q4_read(c.pool, c.pg.slots[0].cuda())
    assert torch.equal(k.double().cpu(), c.k[0])


# ---------------------------------------------------------------- the cache object
def test_cache_follows_requests_through_steps(pkg):
    """Reserve, append, attend, trim and release of requests that come and go, against plain lists."""
    nkv, nq, page, n = 2, 8, 16, 4
    cache = pkg.PagedKVCacheQ4(2, 40, nkv, n, 200, page_size=page)
    rows_of = [[[] for _ in range(n)] for _ in range(2)]
    g = torch.Generator().manual_seed(0)
    for step_no, (new, drop, done) in enumerate([([20, 0, 5, 1], [0, 0, 2, 0], []), ([3, 40, 1, 1], [1, 8, 0, 0], [2]),
                                                 ([4, 4, 0, 4], [3, 0, 0, 3], [0, 3]), ([50, 1, 9, 0], [0, 0, 0, 0], [])]):
        step = cache.reserve(new)
        T = sum(new)
        for layer in range(2):
            k, v = (torch.randn(T, nkv, 128, generator=g).to(torch.float16) for _ in range(2))
            q = torch.randn(T, nq, 128, generator=g).to(torch.float16).cuda()
            cache.append(layer, k.cuda(), v.cuda(), step)
            out = cache.attend(layer, q, step, max(new))
            at = 0
            for i, m in enumerate(new):
                rows_of[layer][i] += list(zip(k[at:at + m], v[at:at + m]))
                at += m
            ks = [U.q4_values(torch.stack([a for a, _ in r])) if r else torch.zeros(0, nkv, 128).double()
                  for r in rows_of[layer]]
            vs = [U.q4_values(torch.stack([b for _, b in r])) if r else torch.zeros(0, nkv, 128).double()
                  for r in rows_of[layer]]
            ref, bound = U.attention(q, ks, vs, new, 128 ** -0.5, causal=True)
            assert bool(((out.double().cpu() - ref).abs() <= U.attention_tolerance(ref, bound, torch.float16)).all())
            for i in range(n):
                got, _ = cache.read(layer, i, len(rows_of[layer][i]))
                assert torch.equal(got.double().cpu(), ks[i])
        cache.trim(torch.tensor(drop, dtype=i32).cuda() if step_no % 2 else drop)
        cache.release(done)
        for layer in range(2):
            for i in range(n):
                del rows_of[layer][i][len(rows_of[layer][i]) - drop[i]:]
                if i in done:
                    rows_of[layer][i].clear()
        lens = [len(r) for r in rows_of[0]]
        assert cache.lens.tolist() == lens
        assert cache.free_page_count() == 40 - sum(-(-a // page) for a in lens)
        cache.check()
    held = [int(p) for i in range(n) for p in cache.table[i, :int(cache.pages[i])]]
    free = cache.free_pages[int(cache.head):].tolist()
    assert sorted(held + free) == list(range(40))            # every page is somewhere, once
    cache.reserve([150, 150, 150, 150])
    with pytest.raises(RuntimeError, match="free pages"):
        cache.check()
    cache.check()


def test_operators_refuse_bad_arguments(pkg):
    pool = pkg.q4_pool(4, 2, 32)
    q = torch.zeros(2, 4, 128, dtype=torch.float16).cuda()
    kv = torch.zeros(2, 2, 128, dtype=torch.float16).cuda()
    table, lens, slots = torch.zeros(2, 2, dtype=i32).cuda(), _dev([1, 1]), _dev([0, 1])
    A = pkg.q4_attention
    for bad in [lambda: A(q[:, :3], pool, table, lens), lambda: A(q.float(), pool, table, lens),
                lambda: A(q, pool.view(4, 2, 2, -1)[:, :, :, :2000], table, lens), lambda: A(q, pool, table.long(), lens),
                lambda: A(q, pool, table, lens.long()), lambda: A(q, pool, table, lens, max_rows=0),
                lambda: A(q, pool, table, lens, max_rows=2), lambda: A(q, pool, table, lens, sink=4),
                lambda: A(q, pool, table, lens, window=-1), lambda: A(q, pool, table, lens, scale=float("nan")),
                lambda: A(q, pool, table, lens, starts=_dev([0, 1])), lambda: A(q, pool, table, lens, out=q[:1]),
                lambda: A(q, pool, table, lens, workspace=torch.zeros(64, dtype=torch.uint8).cuda()),
                lambda: A(q.cpu(), pool, table, lens), lambda: A(q[:, :, :64], pool, table, lens),
                lambda: pkg.q4_append(kv, kv[:1], slots, pool), lambda: pkg.q4_append(kv, kv.bfloat16(), slots, pool),
                lambda: pkg.q4_append(kv, kv, slots[:1], pool), lambda: pkg.q4_append(kv[:, :1], kv[:, :1], slots, pool),
                lambda: pkg.q4_read(pool, slots, torch.float32), lambda: pkg.q4_read(pool, slots.long()),
                lambda: pkg.q4_pool(4, 2, 48), lambda: pkg.q4_pool(0, 2),
                lambda: pkg.paged_reserve(lens, lens, lens, table, slots, _dev([0]), 48, 4),
                lambda: pkg.paged_reserve(lens, lens, lens, table, slots, _dev([0]), 32, -1),
                lambda: pkg.paged_reserve(lens, lens[:1], lens, table, slots, _dev([0]), 32, 4),
                lambda: pkg.paged_release(lens, lens, table.t(), slots, _dev([0]), 32),
                lambda: pkg.PagedKVCacheQ4(0, 4, 2, 1, 10), lambda: pkg.q4_attention_workspace(1, 1, 3, 2)]:
        with pytest.raises(ValueError):
            bad()
    # nothing to do is not an error
    assert A(q[:0], pool, table, lens, starts=_dev([0, 0, 0])).shape == (0, 4, 128)
    pkg.q4_append(kv[:0], kv[:0], slots[:0], pool)
    assert pkg.q4_read(pool, slots[:0])[0].shape == (0, 2, 128)


# ---------------------------------------------------------------- blocks of query rows (more than 16 a kv head)
@pytest.mark.parametrize("lens,rows,nq,nkv", [
    ([20000], [16], 4, 1),                                      # one item over the whole GPU
    ([9000, 0, 3000, 130], [16, 8, 20, 3], 8, 2),               # few items, whole CTAs to each
    ([40000] + [100] * 70, [5] * 71, 8, 2),                     # too uneven for that: equal runs
    ([2000, 2100, 1900, 1, 2050], [40, 32, 33, 40, 0], 10, 2),  # groups of 80 columns, one not full
])
def test_block_attention_shares_out_the_work(pkg, lens, rows, nq, nkv):
    c = Case(pkg, lens, rows, nq, nkv, 64, torch.float16, seed=len(lens))
    c.check(pkg, causal=True)
    a = c.check(pkg, sink=64, window=1000)
    assert torch.equal(a, c.check(pkg, sink=64, window=1000))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("step", [0.02, 0.3])
def test_block_attention_raises_the_maximum_late(pkg, causal, step):
    """Keys that grow along the cache, by less and by more than a tile's reference allows; one query the other way."""
    L = 1500
    c = Case(pkg, [L], [12], 4, 1, 64, torch.float16)
    k = torch.zeros(L, 1, 128)
    k[:, 0, 0] = torch.linspace(0, step * L, L)
    k = k.to(torch.float16)
    v = (torch.randn(L, 1, 128, generator=torch.Generator().manual_seed(1)) * 0.5).to(torch.float16)
    pkg.q4_append(k.cuda(), v.cuda(), c.pg.slots[0].cuda(), c.pool)
    c.k[0], c.v[0] = U.q4_values(k), U.q4_values(v)
    c.q[:] = 0
    c.q[:, :, 0] = torch.tensor([10.0, 5.0, -10.0, 1.0]).cuda()
    c.check(pkg, causal=causal)


@pytest.mark.parametrize("dtype,qscale", [(torch.float16, 30.0), (torch.bfloat16, 30.0), (torch.bfloat16, 1e-6),
                                          (torch.bfloat16, 1e6)])
@pytest.mark.parametrize("nq,nkv", [(4, 1), (5, 1), (4, 4)])
def test_block_attention_of_sharp_and_flat_softmax(pkg, dtype, qscale, nq, nkv):
    c = Case(pkg, [300, 65, 900, 129], [8, 6, 17, 1], nq, nkv, 32, dtype, qscale=qscale)
    if qscale == 1e6:
        c.q[3] *= 1e-9                    # rows of very different sizes in one block
    c.check(pkg, scale=128 ** -0.5 * (1e-5 if qscale == 1e6 else 1.0), causal=True)


def test_operators_in_a_cuda_graph(pkg):
    """A captured step gives the same bits at every replay, on changed rows."""
    c = Case(pkg, [700, 33], [5, 5], 8, 2, 64, torch.float16)
    ws = pkg.q4_attention_workspace(2, 5, 8, 2)
    slots = torch.cat([s[-5:] for s in c.pg.slots]).to(i32).cuda()
    k = torch.randn(10, 2, 128).half().cuda()
    table, lens = c.pg.dev("table"), c.pg.dev("lens")

    def step():
        pkg.q4_append(k, k, slots, c.pool)
        return pkg.q4_attention(c.q, c.pool, table, lens, starts=c.starts, max_rows=5, causal=True, workspace=ws)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2):
        k.copy_(torch.randn(10, 2, 128, generator=torch.Generator().manual_seed(seed)).half())
        graph.replay()
        got = out.clone()
        assert torch.equal(got, step())


def test_cache_object_used_on_two_streams(pkg):
    """The same steps on one stream, and on two that take turns."""
    g = torch.Generator().manual_seed(3)
    rows = [torch.randn(40, 2, 128, generator=g).half().cuda() for _ in range(6)]
    outs = []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for two in (False, True):
        cache, got = pkg.PagedKVCacheQ4(1, 64, 2, 2, 400, 16), []
        for i, k in enumerate(rows):
            st = streams[i % 2 if two else 0]
            st.wait_stream(torch.cuda.current_stream())
            st.wait_stream(streams[1 - i % 2 if two else 0])
            with torch.cuda.stream(st):
                step = cache.reserve([25, 15])
                cache.append(0, k, k, step)
                got.append(cache.attend(0, k.repeat(1, 2, 1), step, 25))
                cache.trim([3, 2])
                cache.release()
        torch.cuda.synchronize()
        cache.check()
        outs.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_cache_object_refuses(pkg):
    cache = pkg.PagedKVCacheQ4(1, 8, 2, 2, 100, 16)
    for bad in (lambda: cache.trim(-1), lambda: cache.trim([1, -1]), lambda: cache.trim(torch.ones(3, dtype=i32).cuda()),
                lambda: cache.trim(torch.ones(2).cuda()), lambda: cache.release([2]), lambda: cache.read(0, 2, 1),
                lambda: cache.read(0, 0, 1000), lambda: cache.reserve(torch.ones(2, dtype=i32).cuda())):
        with pytest.raises(ValueError):
            bad()
    cache.reserve([20, 5])
    cache.trim(torch.tensor([-4, 3], dtype=i32).cuda())       # a negative count on the device trims nothing
    assert cache.lens.tolist() == [20, 2]
    cache.trim(torch.tensor([30, 0]).cuda())
    assert cache.lens.tolist() == [0, 2]


def test_cache_object_keeps_one_workspace(pkg):
    """Steps of every size share the stream's workspace, grown where one needs more."""
    cache = pkg.PagedKVCacheQ4(1, 64, 1, 1, 600, 16)
    q = torch.randn(40, 4, 128, generator=torch.Generator().manual_seed(5)).half().cuda()
    for m in (1, 40, 3, 17, 25, 2, 30):
        step = cache.reserve([m])
        cache.append(0, q[:m, :1], q[:m, :1], step)
        out = cache.attend(0, q[:m], step, m)
        assert torch.equal(out, pkg.q4_attention(q[:m], cache.pools[0], cache.table, cache.lens, step.starts, m, True))
    cache.check()
    assert len(cache._workspace) == 1
