"""Rotary positions on the GPU against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def reference(x, rope, pos, inverse=False):
    """y [rows, heads, dim] in 64 bits and the largest error that the kernel's arithmetic allows."""
    freq = rope.turns.cpu() * (2 * math.pi)
    x, r = x.detach().cpu().double(), rope.rotary_dim
    angle = pos.cpu().double()[:, None, None] * freq
    cos, sin = angle.cos() * rope.factor, angle.sin() * rope.factor * (-1 if inverse else 1)
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if rope.interleaved else (x[..., :r // 2], x[..., r // 2:r])
    u, v, size = a * cos - b * sin, b * cos + a * sin, (a.abs() + b.abs()) * rope.factor
    join = (lambda s, t: torch.stack([s, t], -1).flatten(-2)) if rope.interleaved else (lambda s, t: torch.cat([s, t], -1))
    rest = x[..., r:]
    # The angle's fraction of a turn in fp32 is off by 2^-25 turns (2^-22.3 rad), sine and cosine by 2^-23, the
    # factor and the three operations of a channel by 2^-24 each: below 2^-20 of |a| + |b|.
    return torch.cat([join(u, v), rest], -1), torch.cat([join(size, size) * 2.0 ** -20, torch.zeros_like(rest)], -1)


def check(got, x, rope, pos, inverse=False):
    want, bound = reference(x, rope, pos, inverse)
    half = torch.finfo(got.dtype).eps / 2        # the output's rounding
    tol = bound + want.abs() * half + (2.0 ** -25 if got.dtype is torch.float16 else 0.0)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), f"off by {float((err - tol).max())} more than allowed"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,dim,rot", [(1, 1, 128, 128), (1, 64, 128, 128), (257, 40, 128, 128), (33, 5, 80, 40),
                                                (19, 3, 96, 42), (70, 2, 192, 90), (5, 7, 2, 2), (12, 1, 1024, 1024),
                                                (9, 4, 64, 26), (1000, 3, 256, 64)])
def test_rope_matches_the_definition(pkg, dtype, interleaved, rows, heads, dim, rot):
    g = torch.Generator().manual_seed(rows + dim)
    x = torch.randn(rows, heads, dim, generator=g).to(TYPES[dtype]).cuda()
    pos = torch.randint(0, 1 << 20, (rows,), generator=g, dtype=torch.int32)
    rope = pkg.Rope(dim, 1e6, rot, interleaved)
    check(pkg.apply_rope(x, rope, pos.cuda()), x, rope, pos)


@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 8.0}, {"rope_type": "ntk", "factor": 4.0},
                                     {"type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096}])
def test_far_and_negative_positions_in_64_bits(pkg, scaling):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(64, 2, 128, generator=g).half().cuda()
    pos = torch.randint(-(1 << 30), 1 << 30, (64,), generator=g)
    pos[:4] = torch.tensor([0, 1, (1 << 31) + 5, -1])
    rope = pkg.Rope(128, 1e4, scaling=scaling)
    check(pkg.apply_rope(x, rope, pos.cuda()), x, rope, pos)


def test_strides_slices_and_odd_bases(pkg):
    g = torch.Generator().manual_seed(4)
    rope, pos = pkg.Rope(128, 1e4), torch.arange(50, dtype=torch.int32).cuda()
    wide = torch.randn(50, 48, 128, generator=g).bfloat16().cuda()
    for x in (wide[:, :40], wide[:, 3:4], wide.transpose(0, 1)[:48, :48].transpose(0, 1)[:48],
              torch.randn(50 * 3 * 128 + 1, generator=g).half().cuda()[1:].view(50, 3, 128),
              torch.randn(1, 1, 128, generator=g).cuda().expand(50, 2, 128),
              torch.randn(50, 128, 3, generator=g).cuda().transpose(1, 2)):
        p = pos[:x.shape[0]]
        check(pkg.apply_rope(x, rope, p), x, rope, p)


@pytest.mark.parametrize("rot", [128, 58])
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_touches_only_its_slice(pkg, rot, interleaved):
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(77, 48, 128, generator=g).half().cuda()
    before, rope = wide.clone(), pkg.Rope(128, 1e4, rot, interleaved)
    pos = torch.randint(0, 5000, (77,), generator=g, dtype=torch.int32).cuda()
    part = wide[:, 4:40]
    assert pkg.apply_rope(part, rope, pos, out=part) is part
    check(part, before[:, 4:40], rope, pos)
    assert torch.equal(wide[:, :4], before[:, :4]) and torch.equal(wide[:, 40:], before[:, 40:])


def test_positions_of_a_step_and_rows_of_no_request(pkg):
    cache = pkg.PagedKVCacheQ4(1, 64, 1, 5, 512, 16)
    cache.reserve([7, 0, 30, 1, 4])
    step = cache.reserve([3, 0, 1, 0, 9])
    x = torch.randn(16, 2, 128, generator=torch.Generator().manual_seed(6)).half().cuda()      # 13 rows are the step's
    rope, out = pkg.Rope(128, 1e4), torch.full((16, 2, 128), 7.0).half().cuda()
    pkg.apply_rope(x, rope, step, out=out)
    pos = torch.tensor([7, 8, 9, 30] + list(range(4, 13)))
    check(out[:13], x[:13], rope, pos)
    assert bool((out[13:] == 7).all())


def test_inverse_is_the_gradient_and_turns_back(pkg):
    g = torch.Generator().manual_seed(7)
    x, w = (torch.randn(6, 3, 64, generator=g).cuda() for _ in range(2))
    pos = torch.randint(0, 1000, (6,), generator=g, dtype=torch.int32).cuda()
    rope = pkg.Rope(64, 1e4, 48, True, {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 128})
    back = pkg.apply_rope(w, rope, pos, inverse=True)
    check(back, w, rope, pos, inverse=True)
    # sum(w * rope(x)) is linear in x: its difference along a direction is the gradient's product with it
    d = torch.randn(6, 3, 64, generator=g).cuda()
    moved = sum(float((w.double() * pkg.apply_rope(s * d, rope, pos).double()).sum()) * s for s in (1, -1)) / 2
    want = float((back.double() * d.double()).sum())
    # (6 * 3 * 64 products of two rotated values of size ~1, each off by 2^-20 of |a| + |b|)
    assert abs(moved - want) <= 1152 * 4 * 2.0 ** -20 * 4
    plain = pkg.Rope(64, 1e4)
    again = pkg.apply_rope(pkg.apply_rope(x, plain, pos), plain, pos, inverse=True)
    assert float((again - x).abs().max()) <= 2 * 2 * 2.0 ** -20 * 8


def test_streams_graphs_and_no_rows(pkg):
    rope = pkg.Rope(128, 1e4)
    x = torch.randn(300, 8, 128, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    pos = torch.arange(300, dtype=torch.int32).cuda()
    want = pkg.apply_rope(x, rope, pos)
    assert pkg.apply_rope(x[:0], rope, pos[:0]).shape == (0, 8, 128)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = pkg.apply_rope(x, rope, pos)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.apply_rope(x, rope, pos)
    x.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, pkg.apply_rope(x, rope, pos))


def test_long_rows_past_32_bits(pkg):
    """Elements behind 2^31 of a fused projection's rows."""
    rope, rows = pkg.Rope(128, 1e4), 17000
    wide = torch.empty(rows, 1024, 128, dtype=torch.float16, device="cuda")       # 4.5 GB
    part = wide[:, 1000:1003]
    part.copy_(torch.randn(rows, 3, 128, generator=torch.Generator().manual_seed(9)))
    pos = torch.arange(rows, dtype=torch.int32).cuda()
    got = pkg.apply_rope(part, rope, pos)
    check(got[-50:], part[-50:], rope, pos[-50:])
    check(got[:50], part[:50], rope, pos[:50])
