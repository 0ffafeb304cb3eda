"""The operators of sampled continuations together, as the decode loops use them: forked requests over the paged
cache, attention that reads their prompt once, rotary positions, and drafts verified by sampling."""
import importlib.util
import os

import pytest
import torch

from oracle import dflash_oracle as O
from helpers import gpu_model, tiny_cfg
from test_gpu_paged_generate import EX, _assert_greedy
from toy_target import ToyTarget

pytestmark = pytest.mark.gpu


def _models(pkg, prompts, samples, rows, least=0):
    ocfg = tiny_cfg(mask_token_id=999)
    target = EX.PagedTarget(ocfg.vocab_size, ocfg.hidden_size, 3, 4, 2, 512, 3, max_seqs=prompts * samples, max_len=160,
                            page_size=16, seed=3, samples=samples, least=least)
    ocfg.num_target_features = 3
    q8, _ = O.synth_weights(ocfg, seed=4)
    q8["lm_head"] = target.E.float().cpu()
    return target, gpu_model(pkg, ocfg, q8, max_batch=prompts * samples, max_ctx=max(rows, 64))


def test_greedy_samples_of_a_prompt_are_its_greedy_text(pkg):
    """Forked requests that attend to their shared prompt through a plan: every one decodes greedily."""
    lengths, samples = [40, 1, 67], 3
    target, draft = _models(pkg, len(lengths), samples, samples * sum(lengths))
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, 999, (m,), generator=g).tolist() for m in lengths]
    outs, _, cache = EX.generate(target, draft, prompts, 30)
    assert cache.free_page_count() == target.num_pages and not bool(cache.holders.any())
    for i, out in enumerate(outs):
        prompt = prompts[i // samples]
        assert out[:len(prompt)] == prompt and len(out) == len(prompt) + 30
        _assert_greedy(target, prompt, out)
    draft.close()


def test_sampled_continuations_differ_and_repeat(pkg):
    # The tied random embedding gives the token before a logit of sqrt(256) = 16 over others of spread 1, a probability of
    # 0.9999 at temperature 1; at 8 it is exp(2) in 999 + exp(2), below 1 %.
    lengths, samples, temperature = [33, 16], 4, 8.0
    target, draft = _models(pkg, len(lengths), samples, samples * sum(lengths))
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randint(0, 999, (m,), generator=g).tolist() for m in lengths]
    runs = []
    for _ in range(2):
        outs, accepted, cache = EX.generate(target, draft, prompts, 20, temperature, torch.Generator("cuda").manual_seed(8))
        assert cache.free_page_count() == target.num_pages
        assert all(0 <= a < draft.block_size for step in accepted for a in step)
        runs.append(outs)
    assert runs[0] == runs[1]                               # of the same random numbers
    for i in range(len(lengths)):
        mine = runs[0][i * samples:(i + 1) * samples]
        assert len({tuple(o) for o in mine}) == samples     # 20 tokens of a thousand likely ones each
        assert all(o[:lengths[i]] == prompts[i] and len(o) == lengths[i] + 20 for o in mine)
    draft.close()


@pytest.mark.parametrize("layered", [False, True])
def test_spec_generate_with_a_temperature(pkg, layered):
    ocfg = tiny_cfg(mask_token_id=999)
    target = ToyTarget(ocfg.vocab_size, ocfg.hidden_size, seed=11, layered=layered)
    q8, _ = O.synth_weights(ocfg, seed=12)
    q8["lm_head"] = target.E.float().cpu()
    model = gpu_model(pkg, ocfg, q8, max_batch=1, max_ctx=32)
    prompt = torch.randint(0, ocfg.vocab_size, (20,), generator=torch.Generator().manual_seed(13)).tolist()
    run = lambda t, seed: pkg.spec_generate(target, model, prompt, 40, temperature=t,
                                            generator=torch.Generator("cuda").manual_seed(seed))[0]
    # at a temperature that leaves the first largest logit alone the text is the greedy one
    assert run(1e-5, 1) == target.greedy(prompt, 40)
    a, b, c = run(1.0, 1), run(1.0, 1), run(1.0, 2)
    assert a == b and a != c and len(a) == 60 and a[:20] == prompt
    model.close()


def test_sample_with_a_temperature(pkg):
    x = torch.randn(3, 4, 50, generator=torch.Generator().manual_seed(1)).cuda()
    u = torch.rand(3, 4, generator=torch.Generator().manual_seed(2)).cuda()
    got = pkg.sample(x, 0.7, u)
    c = torch.softmax(x.double() / 0.7, -1).cumsum(-1)
    assert got.shape == (3, 4) and torch.equal(got, torch.searchsorted(c, u.double()[..., None], right=True)[..., 0])
    assert pkg.sample(x.double(), 0.7, u).tolist() == got.tolist()
    assert pkg.sample(x, 0.7).shape == (3, 4)
    assert torch.equal(pkg.sample(x), x.argmax(-1))
    with pytest.raises(NotImplementedError):
        pkg.sample(x.cpu(), 0.7)
