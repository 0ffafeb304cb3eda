"""Greedy requests of ``verify_drafts``: logits are compared as they are, as argmax compares them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [5, 1001, 40000])
def test_logits_beyond_1e30_keep_their_order(pkg, dtype, vocab):
    """Distinct values beyond +-1e30, masks of different depths below it, infinities: the first largest, also beside
    sampled requests in the call."""
    inf = float("inf")
    x = torch.full((8, 2, vocab), -1.0, dtype=dtype)
    x[0, :, 1], x[0, :, 4] = 2e30, 3e30
    x[1, :, 2], x[1, :, 3] = 1e31, inf
    x[2] = -inf
    x[2, :, 1], x[2, :, 3] = -3e38, -2e30          # every entry masked, one of them less
    x[3] = -3e38
    x[3, :, 4] = -1.5e30
    x[4, :, vocab - 1] = 1e30
    x[4, :, 0] = 1e29
    x[5, :, 1:3] = inf                             # a tie: the first one
    x[6, :, 0], x[6, :, vocab - 1] = -1e30, 5e37
    x[7] = -inf
    x[7, :, vocab - 1] = torch.finfo(dtype).min
    x = x.cuda()
    best = x.float().argmax(-1).int()
    assert best[:, 0].tolist() == [4, 3, 3, 4, vocab - 1, 1, vocab - 1, vocab - 1]
    u = torch.rand(8, 2, generator=torch.Generator().manual_seed(vocab)).cuda()
    for draft in (best[:, :1].contiguous(), torch.ones(8, 1, dtype=torch.int32, device="cuda")):
        want = pkg.accept(draft, best)
        for temperature in (0.0, torch.zeros(8, device="cuda"), torch.full((8,), -2.0, device="cuda")):
            got = pkg.verify_drafts(x, draft, u, temperature)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(pkg.sample_tokens(x[:, 1], u[:, 0].contiguous(), 0.0), best[:, 1])


def test_rows_without_a_token(pkg):
    """NaN counts as -inf, and a row with nothing above it refuses its draft and gives -1."""
    x = torch.zeros(3, 2, 100, device="cuda")
    x[0, 0] = float("nan")
    x[1] = -float("inf")
    x[2, 0, :50] = float("nan")
    x[2, 0, 77] = 1.0
    d = torch.tensor([[0], [5], [77]], dtype=torch.int32, device="cuda")
    for temperature in (0.0, 1e-5):
        got = pkg.verify_drafts(x, d, torch.zeros(3, 2, device="cuda"), temperature)
        assert got[0].tolist() == [0, 0, 1] and got[1].tolist() == [-1, -1, 0]
