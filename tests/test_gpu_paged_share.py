"""Pages that several requests hold, on the GPU: every operator against its sequential restatement, and the cache
object over whole lives of requests against the rows that it was given."""
import random

import pytest
import torch

import paged_util as U
from share_util import Shared

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda").reshape(-1)


class Device:
    """The same state on the device."""

    def __init__(self, pkg, model):
        self.pkg, self.page = pkg, model.page
        n = model.n
        self.lens, self.pages, self.head, self.status = i32([0] * n), i32([0] * n), i32([0]), i32([0])
        self.table = torch.full((n, model.max_pages), -1, dtype=torch.int32, device="cuda")
        self.free = i32(model.free)
        self.holders = pkg.page_holders(len(model.free))
        self.refused = i32([0] * n)

    def fork(self, src, dst, rows=None):
        self.lens, self.pages = self.pkg.paged_fork(i32(src), i32(dst), self.lens, self.pages, self.table, self.holders, self.page,
                                                    None if rows is None else i32(rows), self.status, self.refused)

    def reserve(self, new, num_slots):
        step, copies = self.pkg.paged_reserve_forked(self.lens, i32(new), self.pages, self.table, self.free, self.head,
                                                     self.holders, self.page, num_slots, self.status, self.refused)
        self.lens, self.pages, self.head = step.lens, step.pages, step.head
        return step, copies

    def release(self, keep):
        self.pages, self.head = self.pkg.paged_release_forked(i32(keep), self.pages, self.table, self.free, self.head, self.holders,
                                                              self.page, self.status)

    def check(self, model):
        assert self.lens.tolist() == model.lens and int(self.status) == model.status
        assert self.pages.tolist() == [len(r) for r in model.held] and int(self.head) == model.head
        table = self.table.tolist()
        for i, row in enumerate(model.held):
            assert table[i][:len(row)] == row, i
        assert self.free.tolist()[model.head:] == model.free[model.head:]
        owners, holders = model.owners(), self.holders.tolist()
        assert holders[0] == [max(owners.get(p, 0) - 1, 0) for p in range(len(holders[0]))]
        assert not any(holders[1])


@pytest.mark.parametrize("n,num_pages,page,max_pages,seed", [(1, 4, 16, 4, 0), (6, 40, 16, 12, 1), (40, 90, 32, 9, 2),
                                                             (700, 3000, 16, 20, 3), (2048, 9000, 16, 16, 4), (9, 12, 64, 6, 5)])
def test_operators_match_their_restatement(pkg, n, num_pages, page, max_pages, seed):
    rng = random.Random(seed)
    model = Shared(n, num_pages, page, max_pages)
    dev = Device(pkg, model)
    for step in range(14):
        # forks of random requests into empty ones, and some that cannot be
        m = rng.randint(0, n)
        src = [rng.randint(-1 if step % 5 == 4 else 0, n - (step % 5 != 4)) for _ in range(m)]
        empty = [i for i in range(n) if not model.lens[i] and not model.held[i]]
        dst = [rng.choice(empty) if empty and rng.random() < 0.9 else rng.randint(0, n - 1) for _ in range(m)]
        rows = [rng.randint(-2, page * max_pages) for _ in range(m)] if step % 2 else None
        model.fork(src, dst, rows)
        dev.fork(src, dst, rows)
        dev.check(model)
        new = [rng.choice([0, 1, 1, 2, rng.randint(0, 3 * page)]) if rng.random() < 0.8 else 0 for _ in range(n)]
        num_slots = max(0, sum(new) - (rng.randint(0, 40) if step % 4 == 3 else 0))
        starts, slots, copies, served = model.reserve(new, num_slots)
        got, got_copies = dev.reserve(new, num_slots)
        assert got.starts.tolist() == starts and got.slots.tolist() == slots
        assert [tuple(c) for c in got_copies.tolist()] == copies
        assert all(r == (not s) for r, s, b in zip(dev.refused.tolist(), served, new) if b > 0)
        dev.check(model)
        # trims, finished requests, and every third time no release (pages behind the rows stay)
        model.lens = [0 if rng.random() < 0.1 else max(0, a - rng.choice([0, 0, 1, page, 2 * page])) for a in model.lens]
        dev.lens = i32(model.lens)
        if step % 3 != 2:
            model.release(model.lens)
            dev.release(model.lens)
            dev.check(model)
    model.release([0] * n)
    dev.release([0] * n)
    dev.check(model)
    assert model.head == 0 and sorted(model.free) == list(range(num_pages))


def test_a_request_that_writes_behind_a_trim_into_others_pages_is_turned_away(pkg):
    model = Shared(3, 20, 16, 8)
    dev = Device(pkg, model)
    for s in (model, dev):
        s.reserve([40, 0, 0], 40)
        s.fork([0], [1])
    model.lens[0] = 10
    dev.lens = i32(model.lens)
    for s in (model, dev):
        s.reserve([3, 0, 0], 3)           # stays on the page of its rows, which is copied
    dev.check(model)
    model.reserve([30, 0, 0], 30)
    dev.reserve([30, 0, 0], 30)
    assert model.status == 256
    dev.check(model)
    model.release(model.lens)
    dev.release(model.lens)
    model.reserve([30, 0, 0], 30)
    dev.reserve([30, 0, 0], 30)
    dev.check(model)
    assert model.lens[0] == 43


def test_page_counts_that_do_not_fit_change_nothing(pkg):
    """More pages come back than the free list lent: everything stays, and the status says so."""
    dev = Device(pkg, Shared(2, 8, 16, 4))
    dev.reserve([33, 0], 33)
    dev.head = i32([1])
    free, table = dev.free.clone(), dev.table.clone()
    dev.release([0, 0])
    assert int(dev.status) == 8 and dev.pages.tolist() == [3, 0] and int(dev.head) == 1
    assert torch.equal(dev.free, free) and torch.equal(dev.table, table) and not bool(dev.holders.any())
    # a page named twice, and one outside the pool
    dev = Device(pkg, Shared(2, 8, 16, 4))
    dev.reserve([33, 0], 33)
    dev.table[0, 1] = dev.table[0, 0]
    dev.table[0, 2] = 999
    dev.release([0, 0])
    assert int(dev.status) == 8 and int(dev.head) == 2 and not bool(dev.holders.any())


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("nkv,layers", [(1, 1), (3, 2), (8, 70)])
def test_page_copies(pkg, page, nkv, layers):
    g = torch.Generator(device="cuda").manual_seed(page)
    num = 9
    pools = [torch.randint(0, 256, (num, nkv, page // 16, 2304), generator=g, device="cuda", dtype=torch.uint8)
             for _ in range(layers)]
    want = [p.clone() for p in pools]
    copies = [(0, 1, 1), (-1, -1, 0), (2, 3, page), (4, 4, 5), (5, 99, 3), (-7, 6, 3), (6, 7, page // 2 + 1), (0, 8, 0), (8, 5, 10 ** 6)]
    for w in want:
        for a, b, r in copies:
            if 0 <= a < num and 0 <= b < num and a != b and r > 0:
                k = min(-(-r // 16), page // 16)
                w[b, :, :k] = w[a, :, :k]
    pkg.q4_copy_pages(pools, torch.tensor(copies, dtype=torch.int32).cuda())
    for p, w in zip(pools, want):
        assert torch.equal(p, w)
    many = torch.full((5000, 3), -1, dtype=torch.int32, device="cuda")
    many[4999] = torch.tensor([1, 2, 16])
    for w in want:
        w[2, :, :1] = w[1, :, :1]
    pkg.q4_copy_pages(pools, many)
    pkg.q4_copy_pages(pools, many[:0])
    pkg.q4_copy_pages([], many)
    for p, w in zip(pools, want):
        assert torch.equal(p, w)


def test_copies_of_pages_beyond_4_gb(pkg):
    pool = torch.zeros(16000, 8, 16, 2304, dtype=torch.uint8, device="cuda")
    pool[3] = torch.randint(0, 256, (8, 16, 2304), device="cuda", dtype=torch.uint8)
    pkg.q4_copy_pages([pool], torch.tensor([[3, 15999, 256], [-1, -1, 0]], dtype=torch.int32).cuda())
    pkg.q4_copy_pages([pool], torch.tensor([[15999, 7, 100]], dtype=torch.int32).cuda())
    assert pool.nbytes > 1 << 32 and torch.equal(pool[15999], pool[3])
    assert torch.equal(pool[7, :, :7], pool[3, :, :7]) and not bool(pool[7, :, 7:].any()) and not bool(pool[15998].any())


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("page,seed", [(16, 0), (64, 1)])
def test_lives_of_forked_requests_keep_their_rows(pkg, capturable, page, seed):
    """Random forks, appends, trims and releases: every request reads back the rows that it was given."""
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    n, layers, nkv, max_len = 10, 2, 2, 20 * 16
    cache = pkg.PagedKVCacheQ4(layers, 400, nkv, n, max_len, page, capturable=capturable, forkable=True)
    rows = [[[] for _ in range(n)] for _ in range(layers)]       # the stored (k, v) of each request's rows
    for step in range(60):
        what = rng.random()
        empty = [i for i in range(n) if not rows[0][i]]
        if what < 0.3 and len(empty) < n and empty:
            dst = rng.sample(empty, rng.randint(1, len(empty)))
            full = [i for i in range(n) if i not in empty]
            src = [rng.choice(full) for _ in dst]
            keep = [rng.randint(1, len(rows[0][s])) for s in src] if rng.random() < 0.5 else None
            cache.fork(src, dst, keep)
            for l in range(layers):
                for j, (s, d) in enumerate(zip(src, dst)):
                    rows[l][d] = list(rows[l][s][:keep[j] if keep else None])
        elif what < 0.75:
            new = [min(rng.choice([0, 1, 3, 20]), max_len - len(rows[0][i])) for i in range(n)]
            st = cache.reserve(new)
            for l in range(layers):
                k, v = (torch.randn(sum(new), nkv, 128, generator=g).half() for _ in range(2))
                cache.append(l, k.cuda(), v.cuda(), st)
                kq, vq, at = U.q4_values(k), U.q4_values(v), 0
                for i, m in enumerate(new):
                    rows[l][i] += [(kq[r], vq[r]) for r in range(at, at + m)]
                    at += m
        elif what < 0.9:
            drop = [rng.choice([0, 1, 5, 40]) for _ in range(n)]
            cache.trim(drop)
            for l in range(layers):
                rows[l] = [r[:max(0, len(r) - d)] for r, d in zip(rows[l], drop)]
            if rng.random() < 0.5:
                cache.release()
        else:
            done = rng.sample(range(n), 2)
            cache.release(done)
            for l in range(layers):
                for d in done:
                    rows[l][d] = []
        if step % 3 == 0:
            cache.check()
            assert cache.lens.tolist() == [len(r) for r in rows[0]]
            for l in range(layers):
                for i in range(n):
                    if rows[l][i]:
                        k, v = cache.read(l, i, len(rows[l][i]))
                        assert torch.equal(k.double().cpu(), torch.stack([r[0] for r in rows[l][i]])), (step, l, i)
                        assert torch.equal(v.double().cpu(), torch.stack([r[1] for r in rows[l][i]])), (step, l, i)
    cache.release(range(n))
    cache.check()
    assert cache.free_page_count() == 400 and not bool(cache.holders.any())


def test_a_captured_step_of_forked_requests(pkg):
    """reserve, append, attend, trim and release in one graph, replayed: the same rows as eager steps."""
    def build():
        cache = pkg.PagedKVCacheQ4(1, 64, 1, 4, 512, 16, capturable=True, forkable=True)
        st = cache.reserve([37, 0, 0, 0])
        g = torch.Generator().manual_seed(5)
        cache.append(0, *(torch.randn(37, 1, 128, generator=g).half().cuda() for _ in range(2)), st)
        cache.fork(0, [1, 2, 3])
        return cache, [torch.randn(12, n, 128, generator=g).half().cuda() for n in (1, 1, 2)]

    def step(cache, k, v, q, new, drop):
        st = cache.reserve(new, num_slots=12)
        cache.append(0, k, v, st)
        out = cache.attend(0, q, st, 3)
        cache.trim(drop)
        cache.release()
        return out

    new, drop = i32([3, 3, 3, 3]), i32([1, 0, 2, 3])
    eager, (k, v, q) = build()
    outs = []
    for i in range(5):
        outs.append(step(eager, k * (i + 1), v, q, new, drop))
    cache, (k, v, q) = build()
    first = step(cache, k, v, q, new, drop)         # (warm-up, and the first step)
    kk = k.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache, kk, v, q, new, drop)
    assert torch.equal(first, outs[0])
    for i in range(1, 5):
        kk.copy_(k * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, outs[i]), i
    assert cache.lens.tolist() == eager.lens.tolist() and cache.pages.tolist() == eager.pages.tolist()
    cache.check()


def test_cache_refusals(pkg):
    plain = pkg.PagedKVCacheQ4(1, 8, 1, 4, 64, 16)
    with pytest.raises(RuntimeError, match="forkable"):
        plain.fork(0, [1])
    cache = pkg.PagedKVCacheQ4(1, 8, 1, 4, 64, 16, forkable=True)
    cache.reserve([20, 0, 0, 0])
    for src, dst, rows in ((0, [1, 1], None), (0, [4], None), (4, [1], None), ([0, 0], [1], None), (0, [1], -1), (-1, [1], None)):
        with pytest.raises(ValueError):
            cache.fork(src, dst, rows)
    cache.fork(0, [1])
    cache.fork(0, [1])                          # holds rows already: skipped, and reported
    with pytest.raises(RuntimeError, match="fork"):
        cache.check()
    assert cache.lens.tolist() == [20, 20, 0, 0]
    cache.fork(torch.tensor([0], dtype=torch.int32).cuda(), torch.tensor([2], dtype=torch.int32).cuda(), 16)
    assert cache.lens.tolist() == [20, 20, 16, 0] and cache.pages.tolist() == [2, 2, 1, 0]
    cache.fork(0, [])
    # pages run out: the requests behind are turned away and keep their rows
    cache.reserve([50, 1, 1, 0])
    with pytest.raises(RuntimeError, match="outgrew"):
        cache.check()
    cache.release([0, 1, 2])
    assert cache.free_page_count() == 8
