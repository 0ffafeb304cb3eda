"""Prefix attention where groups are larger than a plan was told, on the GPU against the definition in 64 bits."""
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
