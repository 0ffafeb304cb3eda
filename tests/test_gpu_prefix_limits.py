"""Prefix attention where groups or steps are larger than a plan was told, or than its bounds: on the GPU, against the
definition in 64 bits and against the attention that reads every request's rows."""
import pytest
import torch

import paged_util as U
from test_gpu_prefix_attention import Groups

pytestmark = pytest.mark.gpu


def close(pkg, d, out, causal):
    """out against the definition, with the tolerance of the other prefix tests."""
    want, bound = U.attention(d.q, d.ks, d.vs, d.rows, U.scale_of(128), causal)
    tol = U.attention_tolerance(want, bound, out.dtype) + bound[0] * 2.0 ** -18
    err = (out.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("members,rows,nq,nkv,told", [(5, 1, 8, 2, 2), (40, 2, 8, 2, 2), (70, 3, 8, 2, 8), (150, 1, 16, 2, 16),
                                                      (150, 2, 4, 4, 50), (33, 5, 5, 1, 3), (90, 1, 1, 1, 5)])
def test_groups_on_the_device_larger_than_told(pkg, members, rows, nq, nkv, told):
    """Their rows are all right; the status says that they were more than promised."""
    d = Groups(pkg, [(288, [1 + i % 40 for i in range(members)], [rows] * members)], 16, nq, nkv, seed=members)
    bounds = torch.tensor([0, members], dtype=torch.int32, device="cuda")
    out, plan, status = d.attend(pkg, False, sizes=bounds, max_group=told)
    assert plan.prefix.tolist() == [288] and status == 64
    close(pkg, d, out, False)
    # the same without a status word, over a workspace that holds other numbers
    ws = torch.full((pkg.q4_prefix_workspace(d.q.shape[0], rows, told, nq, nkv).nbytes,), 255, dtype=torch.uint8, device="cuda")
    ws[:4096] = 0
    assert torch.equal(pkg.q4_prefix_attention(d.q, d.pool, d.d_table, plan, workspace=ws), out)


def test_a_prompt_chunk_among_many_single_tokens(pkg):
    """300 requests behind one prompt, of which one brings 257 rows: 300 x 257 is more than 65,536, the rows are not."""
    members = 300
    rows = [257 if i == 7 else 1 for i in range(members)]
    d = Groups(pkg, [(512, [r + i % 3 for i, r in enumerate(rows)], rows)], 64, 4, 1, seed=1)
    out, plan, status = d.attend(pkg, True)
    assert status == 0 and plan.shares and plan.prefix.tolist() == [512]
    close(pkg, d, out, True)
    ws = pkg.q4_prefix_workspace(2000, 257, members, 4, 1)
    assert torch.equal(pkg.q4_prefix_attention(d.q, d.pool, d.d_table, plan, workspace=ws), out)


@pytest.mark.parametrize("rows,least", [([40000, 30000], 0), ([65536, 1], 0), ([33000, 33000], 1 << 40)])
def test_more_query_rows_than_a_group_takes(pkg, rows, least):
    """Then every request is read on its own, by the ordinary attention."""
    d = Groups(pkg, [(64, [5, 70], rows)], 16, 1, 1, seed=2)
    out, plan, status = d.attend(pkg, False, least=least)
    want = pkg.q4_attention(d.q, d.pool, d.d_table, d.d_lens, d.starts, max(rows), False)
    assert status == 0 and torch.equal(out, want)
    ws = pkg.q4_prefix_workspace(sum(rows), max(rows), 2, 1, 1)
    assert torch.equal(pkg.q4_prefix_attention(d.q, d.pool, d.d_table, plan, workspace=ws), want)


def test_a_forked_prompt_is_read_through_a_plan(pkg):
    """A prefill of 1,015 rows for 65 samples (65 x 1,015 > 65,536), as the paged example makes it: one member of the group
    has rows.  Then all of them."""
    samples, prompt = 65, 1015
    g = torch.Generator().manual_seed(3)
    cache = pkg.PagedKVCacheQ4(1, 400, 2, samples, 1200, 16, forkable=True)
    draw = lambda n, heads: torch.randn(n, heads, 128, generator=g).half().cuda()
    for new in ([prompt] + [0] * (samples - 1), [1] * samples, [1200 - prompt - 1] + [1] * (samples - 1)):
        step = cache.reserve(new)
        for least in (None, 0):
            plan = cache.prefix_plan(step, [samples], max(new), least=least)
            q = draw(sum(new), 4)
            cache.append(0, draw(sum(new), 2), draw(sum(new), 2), step)
            got, want = cache.attend(0, q, step, max(new), plan=plan), cache.attend(0, q, step, max(new))
            # (two roundings to f16, and the two orders of summation)
            assert float((got.double() - want.double()).abs().max()) <= 4 * 2.0 ** -11 * float(want.abs().max())
        if new[0] == prompt:
            cache.fork(0, list(range(1, samples)))
    cache.check()
