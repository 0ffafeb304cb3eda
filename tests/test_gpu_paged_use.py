"""The paged 4-bit cache in use beside other work: overlapping calls, CUDA
graphs, refused requests, and the ends of the operators' ranges."""
import numpy as np
import pytest
import torch

import paged_util as U
from test_gpu_paged import Case, _dev

pytestmark = pytest.mark.gpu
i32 = torch.int32


# ---------------------------------------------------------------- overlapping calls

def test_block_calls_overlap_on_streams_of_different_priority(pkg):
    """Calls that share items over the whole GPU, on two streams that take SMs from each other: no CTA may depend on
    another one's residency, and each call gives the bits that it gives alone."""
    cases = [Case(pkg, [6000, 50], [16, 16], 8, 2, 64, torch.float16, seed=s) for s in (1, 2)]
    spaces = [pkg.q4_attention_workspace(2, 16, 8, 2) for _ in cases]
    tables = [(c.pg.dev("table"), c.pg.dev("lens")) for c in cases]
    alone = [c.check(pkg, causal=True) for c in cases]
    status = torch.zeros(2, dtype=i32).cuda()
    outs = [[torch.empty_like(c.q) for _ in range(40)] for c in cases]
    filler = torch.randn(1 << 22, device="cuda")
    streams = [torch.cuda.Stream(priority=0), torch.cuda.Stream(priority=-1)]
    torch.cuda.synchronize()
    for k in range(40):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                if i == 0:
                    filler.mul_(1.0)                    # leaves SMs to the two grids one by one
                pkg.q4_attention(cases[i].q, cases[i].pool, *tables[i], starts=cases[i].starts, max_rows=16, causal=True,
                                 out=outs[i][k], status=status[i:i + 1], workspace=spaces[i])
    torch.cuda.synchronize()
    assert status.tolist() == [0, 0]
    assert all(torch.equal(o, alone[i]) for i in range(2) for o in outs[i])


# ---------------------------------------------------------------- the ends of the ranges
@pytest.mark.parametrize("rows,nq", [(12, 1), (400, 1)])
@pytest.mark.parametrize("sink,window", [(0, 2 ** 31 - 1), (5, 2 ** 31 - 1), (0, 2 ** 31 - 400), (0, 304), (7, 305)])
def test_windows_wider_than_the_cache_hide_nothing(pkg, rows, nq, sink, window):
    """Also where there are more query rows than cached rows, so that lengths less rows are negative."""
    for L in (8, 300):
        c = Case(pkg, [L], [rows], nq, 1, 16, torch.float16, seed=L)
        c.check(pkg, causal=True, sink=sink, window=window)


@pytest.mark.parametrize("rows,most", [([2, 5, 1], 4), ([20, 33, 7], 32)])
def test_more_query_rows_than_max_rows_are_reported(pkg, rows, most):
    """Both kernels: the other requests' rows are right, and the status word names what happened."""
    c = Case(pkg, [90, 200, 31], rows, 4, 2, 32, torch.float16)
    args = (c.q, c.pool, c.pg.dev("table"), c.pg.dev("lens"))
    ref = c.check(pkg, causal=True)
    status = torch.zeros(1, dtype=i32).cuda()
    out = pkg.q4_attention(*args, starts=c.starts, max_rows=most, causal=True, status=status)
    assert status.tolist() == [64]
    for a, b in ((0, rows[0]), (rows[0] + rows[1], sum(rows))):
        err, tol = (out[a:b] - ref[a:b]).double().abs(), 2.0 ** -9 * ref[a:b].double().abs() + 2.0 ** -9
        assert bool((err <= tol).all())
    for starts in ([0, 3, 2, 3], [-1, 0, 1, 2], [0, 1, 2, sum(rows) + 1]):      # not ascending, or outside q
        status.zero_()
        pkg.q4_attention(*args, starts=_dev(starts), max_rows=sum(rows), causal=True, status=status)
        assert status.tolist() == [64], starts


def test_the_cache_object_reports_more_query_rows_than_max_rows(pkg):
    cache = pkg.PagedKVCacheQ4(1, 8, 2, 2, 100, 16)
    x = torch.zeros(8, 2, 128).half().cuda()
    step = cache.reserve([3, 5])
    cache.append(0, x, x, step)
    cache.attend(0, x, step, 5)
    cache.check()
    cache.attend(0, x, step, 4)
    with pytest.raises(RuntimeError, match="max_rows"):
        cache.check()


@pytest.mark.parametrize("rows,prefix", [(4096, 0), (1031, 700)])
def test_prompt_in_a_cache_of_many_long_slots(pkg, rows, prefix):
    """256 slots of up to 32,768 rows, 32 / 8 heads: one request's prompt, from empty or behind cached rows."""
    nq, nkv, at = 32, 8, 37
    cache = pkg.PagedKVCacheQ4(1, 90, nkv, 256, 32768, 64)
    g = torch.Generator().manual_seed(rows)
    k, v = ((torch.randn(prefix + rows, nkv, 128, generator=g) * s).half() for s in (1.0, 0.5))
    q = torch.randn(rows, nq, 128, generator=g).half()
    for a, b in ((0, prefix), (prefix, prefix + rows)):
        if a < b:
            step = cache.reserve([b - a if i == at else 0 for i in range(256)])
            cache.append(0, k[a:b].cuda(), v[a:b].cuda(), step)
    out = cache.attend(0, q.cuda(), step, rows).cpu()
    cache.check()
    ks, vs = U.q4_values(k), U.q4_values(v)
    for j in [0, 1, 19, 20, 63, 64, 500, rows - 2, rows - 1]:      # groups of 20 rows
        end = prefix + j + 1
        ref, bound = U.attention(q[j:j + 1], [ks[:end]], [vs[:end]], [1], 128 ** -0.5)
        assert bool(((out[j:j + 1].double() - ref).abs() <= U.attention_tolerance(ref, bound, torch.float16)).all()), j


@pytest.mark.parametrize("rows,nkv,length", [(16, 256, 2 ** 21), (512, 64, 2 ** 21)])
def test_starts_out_of_order_never_outgrow_the_tile_sums(pkg, rows, nkv, length):
    """Every other request claims all of q: more than 2^32 tiles together.  Nothing runs, and the status says why."""
    n = 2048
    pool = pkg.q4_pool(1, nkv, 256)
    q = torch.zeros(rows, nkv, 128, dtype=torch.float16).cuda()
    table = torch.full((n, length // 256), -1, dtype=i32).cuda()
    starts = torch.zeros(n + 1, dtype=i32).cuda()
    starts[1::2] = rows
    status = torch.zeros(1, dtype=i32).cuda()
    group = 16 if rows == 16 else 80
    tiles = length // (64 if rows == 16 else 128) * nkv * -(-rows // group)
    assert tiles * (n // 2) > 2 ** 32
    pkg.q4_attention(q, pool, table, torch.full((n,), length, dtype=i32).cuda(), starts=starts, max_rows=rows, status=status)
    assert status.tolist() == [64]


# ---------------------------------------------------------------- CUDA graphs of the cache object
def _rows(seed, rows, heads=2):
    return torch.randn(rows, heads, 128, generator=torch.Generator().manual_seed(seed)).half().cuda()


def _same_state(a, b):
    return all(torch.equal(getattr(a, n), getattr(b, n)) for n in ("lens", "pages", "head", "table", "free_pages", "status"))


@pytest.mark.parametrize("rows", [(2, 1, 0), (30, 7, 21)])
def test_captured_steps_go_on_where_the_last_one_ended(pkg, rows):
    """Replays of a captured step, with eager steps between them, against the same steps without a graph."""
    total, most = sum(rows), max(rows)
    k, q = _rows(1, total), _rows(2, total, 4)
    new, drop = _dev(rows), _dev([1, 0, 0])
    a, b = (pkg.PagedKVCacheQ4(1, 64, 2, 3, 400, 16, capturable=c) for c in (True, False))

    def step(cache):
        st = cache.reserve(new, num_slots=total)
        cache.append(0, k, k, st)
        out = cache.attend(0, q, st, most)
        cache.trim(drop)
        cache.release()
        return st, out

    for _ in range(2):
        step(a), step(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st, out = step(a)
    assert _same_state(a, b)                          # a capture runs nothing
    for i in range(4):
        k.copy_(_rows(10 + i, total))
        graph.replay()
        want_st, want = step(b)
        assert torch.equal(out, want) and all(torch.equal(x, y) for x, y in zip(st, want_st))
        assert _same_state(a, b), i
        if i == 1:
            st_a, _ = step(a)
            st_b, _ = step(b)
            assert torch.equal(st_a.slots, st_b.slots) and _same_state(a, b)
            a.release([1])
            b.release([1])
    a.check()


def test_the_cache_object_refuses_captures_that_it_cannot_follow(pkg):
    cache = pkg.PagedKVCacheQ4(1, 8, 2, 2, 100, 16)
    new, q = _dev([1, 1]), _rows(3, 2)
    step = cache.reserve(new, num_slots=2)
    lens = cache.lens.clone()
    fixed = pkg.PagedKVCacheQ4(1, 8, 2, 2, 100, 16, capturable=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q.add_(0)
        for call in (lambda: cache.reserve(new, num_slots=2), lambda: cache.attend(0, q, step, 1), lambda: cache.trim(1),
                     lambda: cache.release()):
            with pytest.raises(RuntimeError, match="capturable"):
                call()
        for call in (lambda: fixed.reserve([1, 1]), lambda: fixed.trim([1, 1]), lambda: fixed.release([0])):
            with pytest.raises(ValueError, match="CUDA graph"):
                call()
    graph.replay()
    assert torch.equal(cache.lens, lens) and fixed.lens.tolist() == [0, 0]
    cache.check()


def _two_caches(pkg, length, **kw):
    caches = [pkg.PagedKVCacheQ4(1, 96, 1, 1, 6000, 64, **kw) for _ in range(2)]
    k = _rows(5, length, 1)
    for c in caches:
        step = c.reserve([length])
        c.append(0, k, k, step)
    return caches, step


@pytest.mark.parametrize("rows,heads", [(1, 8), (16, 4)])      # either kernel, the cached rows cut over many CTAs
def test_a_graph_never_shares_the_objects_workspace(pkg, rows, heads):
    """A captured attention writes into none of the object's workspaces, whichever is made, grown or dropped meanwhile."""
    (cache, plain), _ = _two_caches(pkg, 5000, capturable=True)
    q, big = _rows(6, rows, heads), _rows(7, 40, 8)
    starts = pkg.PagedStep(_dev([0, rows]), None, None, None, None)
    large = pkg.PagedStep(_dev([0, 40]), None, None, None, None)
    want, want_big = plain.attend(0, q, starts, rows), plain.attend(0, big, large, 40)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        assert torch.equal(cache.attend(0, q, starts, rows), want)      # an eager call on the capturing stream first
    side.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = cache.attend(0, q, starts, rows)
        graphs.append((g, out))
    with torch.cuda.stream(side):
        eager = cache._workspace[side.cuda_stream]
        eager.fill_(0x55)                                # (not used again: the larger call below takes its place)
        for g, out in reversed(graphs):
            g.replay()
        assert bool((eager == 0x55).all())
        for g, out in graphs:
            assert torch.equal(out, want)
        del eager, cache._workspace[side.cuda_stream]
        assert torch.equal(cache.attend(0, big, large, 40), want_big)
        held = cache._workspace[side.cuda_stream].clone()
        spare = torch.full((1 << 24,), 0x66, dtype=torch.uint8, device="cuda")     # where a freed workspace might lie
        for g, out in graphs:
            out.zero_()
            g.replay()
            assert torch.equal(out, want)
        assert torch.equal(held, cache._workspace[side.cuda_stream]) and bool((spare == 0x66).all())
    side.synchronize()
    cache.check()


def test_attend_takes_a_workspace(pkg):
    (cache, plain), _ = _two_caches(pkg, 3000)
    q, step = _rows(6, 1, 8), pkg.PagedStep(_dev([0, 1]), None, None, None, None)
    ws = pkg.q4_attention_workspace(1, 1, 8, 1)
    assert torch.equal(cache.attend(0, q, step, 1, workspace=ws), plain.attend(0, q, step, 1))
    assert not cache._workspace and len(plain._workspace) == 1
    with pytest.raises(ValueError, match="workspace"):
        cache.attend(0, q, step, 1, workspace=ws[:64])


def test_threads_on_streams_of_their_own_use_workspaces_of_their_own(pkg):
    """Two host threads attend at once; neither takes the other's stream."""
    import threading
    (cache, plain), _ = _two_caches(pkg, 5000)
    q, step = _rows(6, 16, 4), pkg.PagedStep(_dev([0, 16]), None, None, None, None)
    want = plain.attend(0, q, step, 16)
    torch.cuda.synchronize()
    outs = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(200):
                outs[i].append(cache.attend(0, q, step, 16))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert len(cache._workspace) == 2 and all(torch.equal(o, want) for part in outs for o in part)
    cache.check()


# ---------------------------------------------------------------- requests that reserve turns away
@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("why", ["dry", "long", "slots"])
def test_trim_keeps_the_rows_of_a_request_that_was_turned_away(pkg, why, capturable):
    """The documented loop (reserve, append, trim, release, then check) on a request that could not be served."""
    cache = pkg.PagedKVCacheQ4(1, 7 if why == "dry" else 40, 2, 3, 64 if why == "long" else 200, 16, capturable=capturable)
    rows = _rows(1, 50)
    first = cache.reserve([12, 30, 8])
    cache.append(0, rows, rows, first)
    held = cache.read(0, 1, 30)[0]
    new = [4, 40, 4] if why == "slots" else [4, 36, 4] if why == "long" else [4, 60, 4]
    step = cache.reserve(_dev(new), num_slots=40 if why == "slots" else 100)
    served = {"dry": [16, 30, 12], "long": [16, 30, 12], "slots": [16, 30, 8]}[why]     # (what follows is over the slots too)
    assert step.lens.tolist() == served
    cache.append(0, _rows(2, step.slots.numel()), _rows(3, step.slots.numel()), step)
    drop = [2, 15, 2]
    cache.trim(_dev(drop) if why != "long" else drop)
    cache.release()
    after = [14, 30, 8 if why == "slots" else 10]
    assert cache.lens.tolist() == after and cache.pages.tolist() == [-(-a // 16) for a in after]
    assert torch.equal(cache.read(0, 1, 30)[0], held)
    cache.reserve([1, 0, 1])                              # it sits out: still what it held
    cache.trim(1)
    assert cache.lens.tolist() == after
    with pytest.raises(RuntimeError):
        cache.check()
    cache.trim([0, 3, 0])                                 # told: rows that it holds may be dropped
    assert cache.lens.tolist() == [after[0], 27, after[2]]
    cache.reserve([0, 5, 0])
    cache.trim(2)                                         # served again
    assert cache.lens.tolist() == [after[0] - 2, 30, after[2] - 2]
    cache.check()


def test_trim_in_a_graph_keeps_the_rows_of_a_request_that_was_turned_away(pkg):
    cache = pkg.PagedKVCacheQ4(1, 4, 2, 2, 400, 16, capturable=True)
    new = _dev([10, 3])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.reserve(new, num_slots=13)
        cache.trim(2)
        cache.release()
    for want in [[8, 1], [16, 2], [24, 3], [32, 4], [40, 5], [40, 6], [40, 7]]:      # 50 rows would need a fourth page
        graph.replay()
        assert cache.lens.tolist() == want
    with pytest.raises(RuntimeError, match="free pages"):
        cache.check()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_trim_counts_at_the_ends_of_their_type(pkg, dtype):
    cache = pkg.PagedKVCacheQ4(1, 8, 2, 3, 100, 16)
    cache.reserve([20, 5, 7])
    ends = torch.iinfo(dtype)
    cache.trim(torch.tensor([ends.min, ends.min + 3, 2], dtype=dtype).cuda())      # negative: nothing
    assert cache.lens.tolist() == [20, 5, 5]
    cache.trim(torch.tensor([ends.max, 0, -1], dtype=dtype).cuda())
    assert cache.lens.tolist() == [0, 5, 5]


# ---------------------------------------------------------------- what waits for the device
def test_only_check_and_free_page_count_wait_for_the_device(pkg):
    cache = pkg.PagedKVCacheQ4(1, 16, 2, 3, 100, 16)
    x, q, new = _rows(1, 6), _rows(2, 6, 4), _dev([1, 2, 3])
    drop = _dev([0, 1, 1])
    torch.cuda.synchronize()
    mode = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        for step in (cache.reserve([1, 2, 3]), cache.reserve(new, num_slots=6)):
            cache.append(0, x, x, step)
            cache.attend(0, q, step, 3)
        cache.trim(drop)
        cache.trim([1, 0, 0])
        cache.trim(1)
        cache.release()
        cache.release([0, 2])
        for wait in (cache.check, cache.free_page_count):
            with pytest.raises(RuntimeError, match="synchroniz"):
                wait()
    finally:
        torch.cuda.set_sync_debug_mode(mode)
    assert cache.lens.tolist() == [0, 2, 0]
    cache.check()


# ---------------------------------------------------------------- arguments
def test_rows_that_the_kernels_cannot_read_in_place_are_copied(pkg):
    """Contiguous but not on 16 bytes; one row, or one head, of any stride."""
    g = torch.Generator().manual_seed(4)
    flat = torch.randn(4096, generator=g).half().cuda()
    pool, slots = pkg.q4_pool(2, 2, 16), _dev([3, 17, 9])
    shifted = flat[1:1 + 3 * 2 * 128].view(3, 2, 128)
    assert shifted.is_contiguous() and shifted.data_ptr() % 16
    row = flat.as_strided((1, 2, 128), (77, 128, 1))
    for x in (shifted, row):
        pkg.q4_append(x, x, slots[:x.shape[0]], pool)
        assert torch.equal(pkg.q4_read(pool, slots[:x.shape[0]])[1].double().cpu(), U.q4_values(x.cpu()))
    one, head = pkg.q4_pool(2, 1, 16), flat.as_strided((3, 1, 128), (256, 33, 1))
    pkg.q4_append(head, head, slots, one)
    assert torch.equal(pkg.q4_read(one, slots)[0].double().cpu(), U.q4_values(head.cpu()))
    c = Case(pkg, [70], [3], 2, 1, 32, torch.float16)
    want = c.check(pkg)
    q = torch.cat([c.q.flatten()[:1], c.q.flatten()])[1:].view_as(c.q)
    assert q.data_ptr() % 16
    assert torch.equal(pkg.q4_attention(q, c.pool, c.pg.dev("table"), c.pg.dev("lens"), max_rows=3), want)


def test_attention_writes_between_query_rows_but_not_over_them(pkg):
    c = Case(pkg, [70], [2], 4, 2, 32, torch.float16)
    want = c.check(pkg)
    args = (c.pool, c.pg.dev("table"), c.pg.dev("lens"))
    wide = torch.zeros(2, 16 * 128, dtype=torch.float16).cuda()
    q = wide[:, :512].view(2, 4, 128)
    q.copy_(c.q)
    gap = wide.flatten()[512:512 + 1024].view(2, 4, 128)       # behind row 0, in front of row 1
    assert pkg.q4_attention(q, *args, max_rows=2, out=gap) is gap and torch.equal(gap, want) and torch.equal(q, c.q)
    with pytest.raises(ValueError, match="overlaps"):
        pkg.q4_attention(c.q, *args, max_rows=2, out=c.q)
    with pytest.raises(ValueError, match="overlaps"):
        pkg.q4_attention(q, *args, max_rows=2, out=wide.flatten()[256:1280].view(2, 4, 128))


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("dtype,size,key", [(torch.bfloat16, -1e37, 1.0), (torch.bfloat16, -1e31, 1.0), (torch.bfloat16, 1e31, 1.0),
                                            (torch.float16, 6e4, 6e4), (torch.float16, -6e4, 6e4), (torch.float16, 300.0, 3e3)])
def test_scores_far_beyond_the_mantissa(pkg, dtype, size, key, rows):
    """Every score of a row is huge: equal keys weigh the same, and of two keys the larger score wins."""
    c = Case(pkg, [200, 200], [rows, rows], 2, 1, 64, dtype)
    k = torch.full((200, 1, 128), key)
    v = [torch.randn(200, 1, 128, generator=torch.Generator().manual_seed(s)).to(dtype) for s in (1, 2)]
    pkg.q4_append(k.to(dtype).cuda(), v[0].cuda(), c.pg.slots[0].cuda(), c.pool)
    k[150] *= 0.5 if size < 0 else 1.0
    k[:150] *= 1.0 if size < 0 else 0.5
    k[151:] *= 1.0 if size < 0 else 0.5
    pkg.q4_append(k.to(dtype).cuda(), v[1].cuda(), c.pg.slots[1].cuda(), c.pool)
    c.q.fill_(size)
    status = torch.zeros(1, dtype=i32).cuda()
    out = pkg.q4_attention(c.q, c.pool, c.pg.dev("table"), c.pg.dev("lens"), max_rows=rows, status=status, scale=0.01).double().cpu()
    v = [U.q4_values(x)[:, 0] for x in v]
    for got, want in ((out[:rows], v[0].mean(0)), (out[rows:], v[1][150])):
        # the output's rounding, P exact (1 or 0), 200 fp32 additions of values below 5
        assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 5 * 200 * 2.0 ** -24).all())
    assert status.tolist() == [0]


def test_the_caches_memory_stays_until_every_stream_is_done_with_it(pkg):
    """A cache made on one stream, appended to on another and dropped while that one is busy."""
    cache = pkg.PagedKVCacheQ4(1, 200, 2, 3, 400, 16)
    x = _rows(1, 40)
    step = cache.reserve([40, 0, 0])
    pool = cache.pools[0]
    size, at = pool.numel(), pool.data_ptr()
    del pool
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)                  # about 0.1 s
        cache.append(0, x, x, step)
        busy = torch.cuda.Event()
        busy.record()
    del cache, step
    taken = torch.empty(size, dtype=torch.uint8, device="cuda")
    still = not busy.query()
    assert not still or taken.data_ptr() != at
    assert still, "the side stream was done too soon to tell"
    side.synchronize()
