"""Plans of shared prefixes on the GPU, against their definition on the host."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(np.array(v), dtype=torch.int32).cuda()


def definition(table, lens, rows, bounds, page, causal, least):
    """(prefix of each group, skip and own rows of each request)."""
    prefix, spared = [], 0
    for a, b in zip(bounds, bounds[1:]):
        mine = [i for i in range(a, b) if rows[i] > 0]
        pages = 0
        if len(mine) > 1:
            pages = min(max(lens[i] - (rows[i] - 1 if causal else 0), 0) // page for i in mine)
            same = (table[mine, :pages] == table[mine[0], :pages]).all(0)
            pages = pages if same.all() else int(np.argmin(same))
            spared += (len(mine) - 1) * pages * page
        prefix.append(pages * page)
    if spared < least:
        prefix = [0] * len(prefix)
    skip = [0] * len(lens)
    for k, (a, b) in enumerate(zip(bounds, bounds[1:])):
        for i in range(a, b):
            skip[i] = prefix[k] // page if rows[i] > 0 else 0
    return prefix, skip, [n - s * page for n, s in zip(lens, skip)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,g,columns,page", [(40, 1, 700, 16), (40, 5, 300, 32), (300, 17, 65, 64), (2048, 600, 33, 16),
                                              (2048, 1, 40, 16), (2, 1, 1, 256)])
def test_plans_match_the_definition(pkg, n, g, columns, page, causal):
    """Members that differ at random columns, in the order that makes each of them shorten the prefix of those before it,
    and in others: many warps compare while the limit falls."""
    rng = np.random.default_rng(n + g + columns)
    for trial in range(8):
        bounds = [0] + sorted(rng.integers(0, n + 1, g).tolist()) if g > 1 else [0, n]
        table = np.zeros((n, columns), np.int32)
        for a, b in zip(bounds, bounds[1:]):
            table[a:b] = rng.integers(0, 1 << 20, columns)
            at = rng.integers(0, 3 * columns, max(b - a, 1))
            at = np.sort(at)[::-1] if trial % 2 else at
            for i, c in zip(range(a + 1, b), at):
                table[i, c:] += 1 + i
        lens = (rng.integers(0, columns * page + 1, n) if trial % 3 == 0 else np.full(n, columns * page)).tolist()
        rows = rng.integers(0, 4, n).tolist()
        starts = i32(np.concatenate([[0], np.cumsum(rows)]))
        want = definition(table, lens, rows, bounds, page, causal, 0)[0]
        total = sum((sum(r > 0 for r in rows[a:b]) - 1) * p for a, b, p in zip(bounds, bounds[1:], want) if p)
        for least in (0, total, total + 1):
            plan = pkg.paged_prefix_plan(i32(table), i32(lens), i32(bounds), page, starts, 3, causal, n, least)
            got = plan.prefix.tolist(), plan.skip.tolist(), plan.own_lens.tolist()
            assert got == definition(table, lens, rows, bounds, page, causal, least), (trial, least)


@pytest.mark.parametrize("nkv,members,shares", [(64, 9, True), (64, 8, False), (8, 9, False), (128, 5, True), (128, 4, False)])
def test_a_plan_of_the_cache_asks_for_rows_by_its_kv_heads(pkg, nkv, members, shares):
    """2^20 rows times kv heads spared, of 2,048 rows that 4 to 9 requests share."""
    cache = pkg.PagedKVCacheQ4(1, 30, nkv, members, 2304, 256, forkable=True)
    cache.reserve([2048] + [0] * (members - 1))
    cache.fork(0, list(range(1, members)))
    step = cache.reserve([1] * members)
    assert cache.prefix_plan(step, [members], 1).prefix.tolist() == [2048 if shares else 0]
    assert cache.prefix_plan(step, [members], 1, least=1).prefix.tolist() == [2048]
    cache.check()
