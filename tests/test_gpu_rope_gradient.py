"""Gradients through rotary positions: against the formula in 64 bits and against differences."""
import pytest
import torch

from test_gpu_rope import TYPES, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,dim,rot", [(1, 1, 128, 128), (37, 6, 128, 128), (19, 3, 96, 42), (5, 7, 2, 2)])
def test_gradient_is_the_formulas(pkg, dtype, interleaved, rows, heads, dim, rot):
    """y = f R x, so the gradient of x is f R^T that of y: the rotation backwards, rounded once."""
    g = torch.Generator().manual_seed(rows + dim)
    rope = pkg.Rope(dim, 1e4, rot, interleaved, {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64})
    pos = torch.randint(0, 5000, (rows,), generator=g, dtype=torch.int32)
    x = torch.randn(rows, heads, dim, generator=g).to(TYPES[dtype]).cuda().requires_grad_()
    up = torch.randn(rows, heads, dim, generator=g).to(TYPES[dtype]).cuda()
    for inverse in (False, True):
        y = pkg.apply_rope(x, rope, pos.cuda(), inverse=inverse)
        assert y.requires_grad
        check(y.detach(), x.detach(), rope, pos, inverse)
        y.backward(up)
        check(x.grad, up, rope, pos, not inverse)
        x.grad = None


def test_gradient_is_the_limit_of_differences(pkg):
    # the map is linear: a difference of any size is exact but for rounding, 2^-20 of |a| + |b| each way (test_gpu_rope.py)
    g = torch.Generator().manual_seed(1)
    rope, pos = pkg.Rope(64, 1e4, 48), torch.randint(0, 9999, (21,), generator=g).cuda()
    x, h, up = (torch.randn(21, 3, 64, generator=g).cuda() for _ in range(3))
    x.requires_grad_()
    pkg.apply_rope(x, rope, pos).backward(up)
    with torch.no_grad():
        change = ((pkg.apply_rope(x + h, rope, pos).double() - pkg.apply_rope(x - h, rope, pos).double()) / 2 * up.double()).sum()
        size = (up.abs().double() * (x.abs() + h.abs()).double()).sum() * 4
        assert abs(float(change - (x.grad.double() * h.double()).sum())) <= float(size) * 2.0 ** -20


def test_gradients_of_steps_slices_and_broadcasts(pkg):
    """Rows of no request take part in nothing: their gradient is zero.  Broadcast heads add theirs up."""
    g = torch.Generator().manual_seed(2)
    rope = pkg.Rope(128, 1e4)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    step = pkg.PagedStep(i32([0, 3, 3, 8]), i32([]), i32([10, 4, 500]), i32([1, 1, 8]), i32([10]))
    pos = torch.tensor([7, 8, 9] + list(range(495, 500)))
    qkv = torch.randn(12, 9, 128, generator=g).cuda().requires_grad_()
    up = torch.randn(12, 6, 128, generator=g).cuda()
    y = pkg.apply_rope(qkv[:, 1:7], rope, step)
    y.backward(up)
    check(qkv.grad[:8, 1:7], up[:8], rope, pos, inverse=True)
    assert not bool(qkv.grad[8:].any()) and not bool(qkv.grad[:, 0].any()) and not bool(qkv.grad[:, 7:].any())

    one = torch.randn(8, 1, 128, generator=g).cuda().requires_grad_()
    pkg.apply_rope(one.expand(8, 6, 128), rope, pos.cuda()).backward(up[:8])
    each = pkg.apply_rope(up[:8], rope, pos.cuda(), inverse=True)
    torch.testing.assert_close(one.grad, each.sum(1, keepdim=True), rtol=0, atol=6 * 2.0 ** -24 * float(each.abs().sum(1).max()))


def test_gradient_of_a_gradient_and_what_asks_for_none(pkg):
    g = torch.Generator().manual_seed(3)
    rope, pos = pkg.Rope(32, 1e4), torch.arange(5).cuda()
    x = torch.randn(5, 2, 32, generator=g).cuda().requires_grad_()
    up = torch.randn(5, 2, 32, generator=g).cuda().requires_grad_()
    (grad,) = torch.autograd.grad(pkg.apply_rope(x, rope, pos), x, up, create_graph=True)
    (back,) = torch.autograd.grad(grad, up, x.detach())
    assert torch.equal(back, pkg.apply_rope(x.detach(), rope, pos))
    with torch.no_grad():
        assert not pkg.apply_rope(x, rope, pos).requires_grad
        assert pkg.apply_rope(x, rope, pos, out=torch.empty_like(x)).shape == x.shape
    for out in (torch.empty(5, 2, 32, device="cuda"), x):
        with pytest.raises(ValueError, match="gradient"):
            pkg.apply_rope(x, rope, pos, out=out)
    with pytest.raises(ValueError, match="gradient"):
        pkg.apply_rope(x.detach(), rope, pos, out=torch.empty_like(x).requires_grad_())


def test_positions_changed_before_the_backward_pass_are_an_error(pkg):
    rope, i32 = pkg.Rope(32, 1e4), lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    x = torch.randn(5, 2, 32, device="cuda").requires_grad_()
    step = pkg.PagedStep(i32([0, 2, 5]), i32([]), i32([4, 9]), i32([1, 1]), i32([2]))
    for positions, changed in ((i32([1, 2, 3, 4, 5]), None), (step, step.starts), (step, step.lens)):
        y = pkg.apply_rope(x, rope, positions)
        (positions if changed is None else changed).add_(1)
        with pytest.raises(RuntimeError, match="inplace"):
            y.sum().backward()


def test_gradients_on_another_stream_and_in_a_graph(pkg):
    g = torch.Generator().manual_seed(4)
    rope, pos = pkg.Rope(128, 1e4), torch.arange(40).cuda()
    x = torch.randn(40, 4, 128, generator=g).cuda().requires_grad_()
    up = torch.randn(40, 4, 128, generator=g).cuda()
    run = lambda: torch.autograd.grad(pkg.apply_rope(x, rope, pos), x, up)[0]
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    up.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, 2 * want)
