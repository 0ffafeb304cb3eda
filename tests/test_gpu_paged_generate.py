"""The paged operators together, as the example uses them: a target whose K/V
lives in the 4-bit cache, decoded speculatively alone and in a ragged batch."""
import importlib.util
import os

import pytest
import torch

from oracle import dflash_oracle as O
from helpers import gpu_model, tiny_cfg

pytestmark = pytest.mark.gpu

_path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_generate.py")
_spec = importlib.util.spec_from_file_location("paged_generate", _path)
EX = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(EX)


def _models(pkg, max_seqs, max_ctx_rows=64, num_pages=None, page_size=16):
    ocfg = tiny_cfg(mask_token_id=999)
    target = EX.PagedTarget(ocfg.vocab_size, ocfg.hidden_size, 3, 4, 2, 512, ocfg.num_target_features - 2,
                            max_seqs=max_seqs, max_len=160, num_pages=num_pages, page_size=page_size, seed=3)
    ocfg.num_target_features = 3
    q8, _ = O.synth_weights(ocfg, seed=4)
    q8["lm_head"] = target.E.float().cpu()
    draft = gpu_model(pkg, ocfg, q8, max_batch=max_seqs, max_ctx=max(max_ctx_rows, 64))
    return target, draft


def _assert_greedy(target, prompt, out):
    """Every generated token has the largest logit of its position, computed in
    one forward over the whole text, up to a tenth of the logits' spread.

    The two runs round differently (f16 products of other shapes, other splits
    of the softmax sums): about 10 roundings of 2^-11 a layer through 3 layers
    and the head are 1.5 % of a logit's spread, 4 standard deviations of the
    difference of two of 1000 logits are 8 %."""
    cache = target.make_cache()
    logits = target.forward(torch.tensor([out], device=target.device), cache, [len(out)] + [0] * (target.max_seqs - 1))[0]
    cache.check()
    for at in range(len(prompt), len(out)):
        row = logits[0, at - 1].double()
        assert row.max() - row[out[at]] <= 0.1 * row.std(), at


def test_spec_generate_over_the_paged_cache(pkg):
    target, draft = _models(pkg, 1)
    prompt = torch.randint(0, 999, (37,), generator=torch.Generator().manual_seed(5)).tolist()
    out, stats = pkg.spec_generate(target, draft, prompt, 48)
    assert out[:37] == prompt and stats.total_tokens == 48
    _assert_greedy(target, prompt, out)
    draft.close()


@pytest.mark.parametrize("page_size", [16, 64])
def test_ragged_batch_over_the_paged_cache(pkg, page_size):
    lengths = [1, 20, 53, 7, 16]
    target, draft = _models(pkg, len(lengths), sum(lengths), page_size=page_size)
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, 999, (m,), generator=g).tolist() for m in lengths]
    outs, accepted, cache = EX.generate(target, draft, prompts, 30)
    assert cache.free_page_count() == target.num_pages
    assert all(0 <= a < draft.block_size for step in accepted for a in step)
    for prompt, out in zip(prompts, outs):
        assert out[:len(prompt)] == prompt and len(out) == len(prompt) + 30
        _assert_greedy(target, prompt, out)
    draft.close()


def test_batch_that_outgrows_the_pages_is_reported(pkg):
    target, draft = _models(pkg, 2, num_pages=4)
    with pytest.raises(RuntimeError, match="too few free pages"):
        EX.generate(target, draft, [[1] * 30, [2] * 30], 40)
    draft.close()


def test_ragged_batch_with_accepted_drafts(pkg, monkeypatch):
    """Drafts that are right for a while: blocks are kept in part, requests finish at different steps."""
    lengths = [9, 1, 33, 18]
    target, draft = _models(pkg, len(lengths), sum(lengths))
    g = torch.Generator().manual_seed(8)
    prompts = [torch.randint(0, 999, (m,), generator=g).tolist() for m in lengths]
    texts = EX.generate(target, draft, prompts, 60)[0]

    class Knowing:
        """Proposes the known text, wrong from a position on that differs by request and step."""
        def __init__(self, model, n):
            self.at, self.steps = [0] * n, 0

        def step(self, seqs, noise, features, rows):
            assert features.shape[0] == sum(rows) and noise.shape[0] == len(seqs)
            drafts = []
            for i, m in zip(seqs, rows):
                self.at[i] += m                            # the anchor's place in the text
                known = (texts[i] + [0] * draft.block_size)[self.at[i] + 1:self.at[i] + draft.block_size]
                wrong = (self.steps * 3 + i * 2) % draft.block_size
                drafts.append([t if k < wrong else (t + 1) % 999 for k, t in enumerate(known)])
            self.steps += 1
            return torch.tensor(drafts, dtype=torch.int32, device=target.device), None, None

        def prefill(self, *a):
            return self.step(*a)[0]

        def release(self, seqs):
            pass

        def close(self):
            pass

    monkeypatch.setattr(EX.sd, "DraftServer", Knowing)
    outs, accepted, cache = EX.generate(target, draft, prompts, 40)
    assert cache.free_page_count() == target.num_pages
    assert len({len(step) for step in accepted}) > 1 and max(map(max, accepted)) >= 5
    for prompt, out in zip(prompts, outs):
        assert len(out) == len(prompt) + 40
        _assert_greedy(target, prompt, out)
    draft.close()
