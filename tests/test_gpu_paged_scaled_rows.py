"""Block attention over the 4-bit cache with bf16 query rows of which some have to be scaled to become f16 and others not,
in all orders: on the GPU against the definition in 64 bits."""
import pytest
import torch

import paged_util as U

pytestmark = pytest.mark.gpu

# exponents of the 64 query rows of a kv head, by the place in the instruction's columns
ORDERS = {"first eight": lambda i: -20 if i < 8 else 0, "behind eight": lambda i: 0 if i < 8 else -20,
          "every other": lambda i: -20 * (i % 2), "every other eight": lambda i: 18 * (i // 8 % 2), "last": lambda i: 30 * (i == 63),
          "first": lambda i: -30 * (i == 0), "all": lambda i: -9, "none": lambda i: 0, "one in eight": lambda i: -60 * (i % 8 == 5)}


@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("rows,nq,nkv", [(16, 4, 1), (16, 8, 2), (32, 5, 1), (5, 16, 4)])
def test_rows_that_are_scaled_among_others(pkg, order, rows, nq, nkv):
    g = torch.Generator().manual_seed(rows)
    lens, page = [300, 77, 1000], 32
    P = U.Paging(lens, page)
    pool, ks, vs = pkg.q4_pool(P.num_pages, nkv, page), [], []
    for n, slots in zip(lens, P.slots):
        k, v = torch.randn(n, nkv, 128, generator=g).bfloat16(), torch.randn(n, nkv, 128, generator=g).bfloat16()
        pkg.q4_append(k.cuda(), v.cuda(), slots.cuda(), pool)
        ks.append(U.q4_values(k))
        vs.append(U.q4_values(v))
    group = nq // nkv
    size = torch.tensor([[ORDERS[order]((j * group + h % group) % 64) for h in range(nq)] for j in range(rows)])
    q = (torch.randn(3, rows, nq, 128, generator=g) * 2.0 ** size[..., None]).flatten(0, 1).bfloat16()
    q[rows] = 0                                             # a row of zeros is not scaled
    want, bound = U.attention(q, ks, vs, [rows] * 3, U.scale_of(128), True)
    out = pkg.q4_attention(q.cuda(), pool, P.dev("table"), P.dev("lens"), max_rows=rows, causal=True)
    err, tol = (out.double().cpu() - want).abs(), U.attention_tolerance(want, bound, torch.bfloat16)
    assert bool((err <= tol).all()), float((err - tol).max())
