"""Verification of drafts by sampling on the GPU against the definition in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# Largest relative error of an accepted draft's probability: the exponents' rounding (2^-24 of at most 40, times ln 2),
# 2^-22 of the exponential and 2^-23 of log2(e) / T times an exponent, as weights of a sum in 64 bits.
NEAR = 2.0 ** -17


def probabilities(x, temp):
    """softmax(x / temp) of one row in 64 bits; zeros where nothing is left."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    x = np.where(x == -np.inf, x, np.clip(x, -1e30, 1e30))
    if not temp >= 1e-5:
        p = np.zeros_like(x)
        if x.max() > -np.inf:
            p[int(np.argmax(x))] = 1.0
        return p
    if x.max() == -np.inf:
        return np.zeros_like(x)
    with np.errstate(over="ignore", under="ignore"):
        e = np.where(x == -np.inf, 0.0, np.exp((x - x.max()) / temp) if np.isfinite(temp) else 1.0)
    return e / e.sum()


def reference(logits, drafts, u, temps, probs=None, counts=None):
    """(accepted, token, whether a comparison was within rounding of its border) of every request."""
    logits, drafts, u = logits.double().cpu().numpy(), drafts.cpu().numpy(), u.double().cpu().numpy()
    n, block, vocab = logits.shape
    out = []
    for i in range(n):
        count = block - 1 if counts is None else min(max(int(counts[i]), 0), block - 1)
        near = False
        for j in range(count + 1):
            p = probabilities(logits[i, j], float(temps[i]))
            q = np.zeros(vocab)
            if j < count:
                d = int(drafts[i, j])
                if probs is not None:
                    q = np.nan_to_num(probs[i, j].double().cpu().numpy()).clip(min=0)
                elif 0 <= d < vocab:
                    q[d] = 1.0
                if 0 <= d < vocab:
                    near = near or 0 < abs(u[i, j] * q[d] - p[d]) < NEAR * p[d] and p[d] < 1.0
                    if u[i, j] * q[d] < p[d]:
                        continue
            r = np.maximum(p - q, 0.0)
            if not r.sum() > 0:
                r = p
            c = np.cumsum(r)
            token = -1
            if c[-1] > 0:
                over = np.nonzero((c > u[i, -1] * c[-1]) & (r > 0))[0]
                token = int(over[0]) if len(over) else int(np.nonzero(r > 0)[0][-1])
                near = near or 0 < u[i, -1] < 1 and bool(np.abs(c / c[-1] - u[i, -1]).min() < 1e-12)   # (at 0 and 1 nothing is near)
            out.append((j, token, near))
            break
    return out


def check(pkg, logits, drafts, u, temps, probs=None, counts=None, scalar=False):
    n = logits.shape[0]
    t = temps if scalar else torch.tensor(temps, dtype=torch.float32).cuda()
    acc, tok = pkg.verify_drafts(logits, drafts, u, t, draft_probs=probs, num_drafts=counts)
    each = [temps] * n if scalar else torch.tensor(temps, dtype=torch.float32).tolist()
    want = reference(logits, drafts, u, each, probs, None if counts is None else counts.tolist())
    got = list(zip(acc.tolist(), tok.tolist()))
    bad = [(i, g, w) for i, (g, w) in enumerate(zip(got, want)) if g != w[:2] and not w[2]]
    assert not bad, bad[:5]
    assert sum(w[2] for w in want) <= max(1, n // 20)
    return got


def inputs(n, block, vocab, dtype, seed, keep=0.7, noise=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, block, vocab, generator=g) * noise
    drafts = torch.randint(0, vocab, (n, block - 1), generator=g, dtype=torch.int32)
    lift = torch.where(torch.rand(n, block - 1, generator=g) < keep, x[:, :-1].logsumexp(-1) + 2.5, -1.0)
    x[:, :-1].scatter_(2, drafts.long()[..., None], lift[..., None])
    return x.to(TYPES[dtype]).cuda(), drafts.cuda(), torch.rand(n, block, generator=g).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,block,vocab", [(1, 16, 151936), (1, 1, 1000), (3, 5, 32003), (40, 8, 5003), (200, 4, 517), (7, 32, 64),
                                           (5, 3, 1), (600, 2, 2), (2, 20, 7)])
def test_verify_matches_the_definition(pkg, dtype, n, block, vocab):
    x, d, u = inputs(n, block, vocab, dtype, n + vocab)
    rng = np.random.default_rng(vocab)
    check(pkg, x, d, u, rng.choice([0.0, 0.5, 1.0, 1.7], n).tolist())
    check(pkg, x, d, u, 0.8, scalar=True)


@pytest.mark.parametrize("n,block,vocab", [(1, 6, 32003), (30, 5, 1001), (3, 4, 151936)])
def test_sampled_drafts(pkg, n, block, vocab):
    x, d, u = inputs(n, block, vocab, "f32", 11)
    g = torch.Generator().manual_seed(12)
    q = torch.softmax(x[:, :-1].cpu() + torch.randn(n, block - 1, vocab, generator=g), -1).cuda()
    check(pkg, x, d, u, [1.0, 0.7, 0.0][:n] * (n // min(n, 3)), probs=q)
    check(pkg, x, d, u, 1.0, probs=q.transpose(1, 2).contiguous().transpose(1, 2), scalar=True)


def test_ragged_drafts_and_drafts_outside_the_vocabulary(pkg):
    x, d, u = inputs(9, 6, 999, "bf16", 13, keep=1.0)
    counts = torch.tensor([0, 1, 2, 3, 4, 5, 99, -3, 5], dtype=torch.int32).cuda()
    got = check(pkg, x, d, u, [1.0] * 9, counts=counts)
    assert got[0][0] == 0 and got[7][0] == 0
    d[:, 2] = torch.tensor([-1, 999, 2 ** 31 - 1, -2 ** 31, 0, 5, 998, -7, 1000], dtype=torch.int32).cuda()
    check(pkg, x, d, u, [1.0, 0.0, 1.0, 0.0, 1.0, 1.0, 1.0, 1.0, 0.6])


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_rows(pkg, dtype):
    """-inf, the type's lowest value, NaN and infinities, in some entries and in all."""
    x, d, u = inputs(12, 4, 700, dtype, 14, keep=1.0)
    low, inf, nan = torch.finfo(TYPES[dtype]).min, float("inf"), float("nan")
    x[0, :, 100:] = -inf
    x[1, :, 100:] = low
    x[2, :, ::2] = nan
    x[3, 1] = -inf                  # nothing left at the second place
    x[4, 0] = nan
    x[5, 0] = low                   # all the same
    x[6, 0, 17] = inf
    x[6, 0, 500] = inf
    x[7, 0] = -inf
    x[7, 0, 699] = low              # one entry
    x[8, :, :] = 0.0
    x[9, 3] = -inf                  # the row behind the last draft
    x[10, 0] = low
    x[10, 0, 3] = -inf
    u[3, 0] = u[9, :3] = 0.0
    got = check(pkg, x, d, u, [1.0] * 12)
    assert got[4] == (0, -1) and got[9] == (3, -1) and got[7][1] == 699
    check(pkg, x, d, u, [0.0] * 12)
    check(pkg, x, d, u, [1e-5, 1e-4, 50.0, 1e6, float("inf"), 0.9e-5, -1.0, float("nan"), 3e38, float("inf"), 2e-5, 1e10])


def test_the_largest_vocabulary(pkg):
    # rows that have no usable reference are read entry by entry, while the other warps wait
    vocab = 2 ** 22
    g = torch.Generator().manual_seed(11)
    x = torch.randn(2, 3, vocab, generator=g).to(torch.float16)
    x[0, 0, vocab - 2] = x[0, 1, 77] = float("inf")
    x[0, 2, 5] = float("nan")
    d = torch.tensor([[vocab - 2, 77], [vocab - 1, 0]], dtype=torch.int32)
    u = torch.rand(2, 3, generator=g)
    check(pkg, x.cuda(), d.cuda(), u.cuda(), [1.0, 0.7])


def test_rows_past_32_bits(pkg):
    n, block, vocab = 3, 3, 1001
    x, d, u = inputs(n, block, vocab, "f16", 12)
    wide = torch.empty(n * block, 1 << 28, dtype=torch.float16, device="cuda").view(n, block, -1)     # 4.8 GB
    wide[:, :, 7:7 + vocab] = x
    view = wide[:, :, 7:7 + vocab]
    assert check(pkg, view, d, u, [1.0, 0.7, 0.0]) == check(pkg, x, d, u, [1.0, 0.7, 0.0])


def test_no_requests(pkg):
    none = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda")
    accepted, tokens = pkg.verify_drafts(none(0, 4, 100), none(0, 3, dtype=torch.int32), none(0, 4))
    assert accepted.shape == tokens.shape == (0,)
    assert pkg.sample_tokens(none(0, 100), none(0)).shape == (0,)


def test_random_numbers_at_their_ends(pkg):
    x, d, _ = inputs(4, 3, 300, "f32", 15, keep=1.0)
    for v in (0.0, 1.0 - 2.0 ** -24, 1.0):
        check(pkg, x, d, torch.full((4, 3), v).cuda(), [1.0, 0.0, 0.5, 2.0])
    x[:, :, 200:] = float("-inf")
    got = check(pkg, x, d, torch.full((4, 3), 1.0 - 2.0 ** -24).cuda(), [5.0] * 4)
    assert all(t < 200 for _, t in got)


def test_strided_and_unaligned_logits(pkg):
    x, d, u = inputs(6, 5, 1003, "bf16", 16)
    wide = torch.zeros(6, 9, 2011, dtype=torch.bfloat16).cuda()
    part = wide[:, 2:7, 5:1008]
    part.copy_(x)
    for view in (part, x.transpose(1, 2).contiguous().transpose(1, 2), x[:, :1].expand(6, 5, 1003),
                 x.transpose(0, 1).contiguous().transpose(0, 1)):
        check(pkg, view, d, u, [1.0, 0.5, 0.0, 2.0, 1.0, 1.0])


def test_greedy_requests_give_what_accept_gives(pkg):
    x, d, u = inputs(64, 16, 4001, "f16", 17, keep=0.9)
    x[:, :, 7] = x.amax(-1)           # ties: the first one
    acc, tok = pkg.verify_drafts(x, d, u, 0.0)
    want_acc, want_tok = pkg.accept(d, x.float().argmax(-1).int())
    first = torch.where(x == x.amax(-1, keepdim=True), torch.arange(4001, device="cuda"), 9999).amin(-1).int()
    want_acc, want_tok = pkg.accept(d, first)
    assert torch.equal(acc, want_acc) and torch.equal(tok, want_tok)


def test_sample_tokens(pkg):
    x, _, u = inputs(50, 1, 777, "f32", 18)
    tok = pkg.sample_tokens(x[:, 0], u[:, 0], 0.9)
    assert tok.tolist() == [w[1] for w in reference(x, torch.zeros(50, 0), u, [0.9] * 50)]


def test_tokens_are_distributed_as_the_targets_samples(pkg):
    """Drafts sampled from another distribution, accepted and replaced: the first token of each request is a
    sample of p.  400,000 of them: a frequency is within 5 standard deviations (of at most 0.5 / sqrt(n))."""
    g = torch.Generator(device="cuda").manual_seed(19)
    n, vocab = 400_000, 11
    logits = torch.randn(vocab, generator=g, device="cuda")
    q = torch.softmax(torch.randn(vocab, generator=g, device="cuda") * 1.5, -1)
    drafts = torch.multinomial(q.expand(4, -1), n // 4, replacement=True, generator=g).reshape(n, 1).int()
    u = torch.rand(n, 2, generator=g, device="cuda")
    acc, tok = pkg.verify_drafts(logits.expand(n, 2, vocab), drafts, u, 0.7, draft_probs=q.expand(n, 1, vocab))
    first = torch.where(acc > 0, drafts[:, 0], tok)
    seen = torch.bincount(first.long(), minlength=vocab).double().cpu() / n
    p = torch.softmax(logits.double().cpu() / 0.7, -1)
    assert float((seen - p).abs().max()) < 5 * 0.5 / n ** 0.5
    # a draft is accepted with probability sum min(p, q)
    assert abs(float((acc > 0).double().mean()) - float(torch.minimum(p, q.double().cpu()).sum())) < 5 * 0.5 / n ** 0.5


def test_streams_and_graphs(pkg):
    x, d, u = inputs(20, 8, 3001, "bf16", 20)
    want = pkg.verify_drafts(x, d, u, 1.0)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = pkg.verify_drafts(x, d, u, 1.0)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.verify_drafts(x, d, u, 1.0)
    u.copy_(torch.rand(20, 8, generator=torch.Generator().manual_seed(21)))
    graph.replay()
    torch.cuda.synchronize()
    want = pkg.verify_drafts(x, d, u, 1.0)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
