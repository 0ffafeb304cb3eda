"""The sampled decode loops end with an error where verification gives no result or the logits leave no token."""
import importlib
from types import SimpleNamespace

import pytest
import torch

from toy_target import ToyTarget


class Draft:
    """What spec_generate asks of a drafter, on the host."""
    mask_token_id, block_size, device, config = 90, 4, torch.device("cpu"), SimpleNamespace(vocab_size=91)

    def make_cache(self, **_):
        return []

    def draft_tokens(self, noise, hidden, cache=None, **_):
        return torch.tensor([[1, 2, 3]], dtype=torch.int32)


def test_spec_generate_ends_on_results_that_are_none(pkg, monkeypatch):
    gen = importlib.import_module("mirror-sd_b200.generate")
    target, trims = ToyTarget(91, 16, device="cpu"), []
    cache = target.make_cache()
    cache.trim = trims.append
    target.make_cache = lambda: cache
    i32 = lambda v: torch.tensor([v], dtype=torch.int32)
    first, verified = 5, (0, 6)
    monkeypatch.setattr(gen, "sample", lambda *a: torch.tensor(first))
    monkeypatch.setattr(gen, "verify_drafts", lambda *a: tuple(map(i32, verified)))
    assert pkg.spec_generate(target, Draft(), [1, 2], 3, temperature=1.0)[0] == [1, 2, 5, 6, 6]
    count = len(trims)
    for verified, what in (((-1, -1), "wait"), ((2, -1), "no token"), ((3, -1), "no token")):
        with pytest.raises(RuntimeError, match=what):
            pkg.spec_generate(target, Draft(), [1, 2], 9, temperature=1.0)
        assert len(trims) == count          # before anything is dropped
    first = -1
    with pytest.raises(RuntimeError, match="no token"):
        pkg.spec_generate(target, Draft(), [1, 2], 9, temperature=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), -float("inf")])
def test_loops_end_on_logits_that_leave_no_token(pkg, bad):
    from oracle import dflash_oracle as O
    from helpers import gpu_model, tiny_cfg
    from test_gpu_paged_generate import EX
    ocfg = tiny_cfg(mask_token_id=999)
    q8, _ = O.synth_weights(ocfg, seed=12)
    toy = ToyTarget(ocfg.vocab_size, ocfg.hidden_size, seed=11)
    model = gpu_model(pkg, ocfg, q8, max_batch=1, max_ctx=32)
    real, calls = toy.forward, []

    def forward(ids, cache):
        calls.append(ids)
        logits, feats = real(ids, cache)
        return (logits, feats) if len(calls) < 2 else (torch.full_like(logits, bad), feats)

    toy.forward = forward
    with pytest.raises(RuntimeError, match="no token"):
        pkg.spec_generate(toy, model, [1, 2, 3], 20, temperature=1.0)
    assert len(calls) == 2
    with pytest.raises(RuntimeError, match="no token"):      # at the first token
        pkg.spec_generate(toy, model, [1, 2, 3], 20, temperature=1.0)
    model.close()

    ocfg = tiny_cfg(mask_token_id=999)
    target = EX.PagedTarget(ocfg.vocab_size, ocfg.hidden_size, 3, 4, 2, 512, 3, max_seqs=2, max_len=160, page_size=16, seed=3, samples=2)
    ocfg.num_target_features = 3
    q8, _ = O.synth_weights(ocfg, seed=4)
    draft = gpu_model(pkg, ocfg, q8, max_batch=2, max_ctx=64)
    head = target.lm_head
    for good_calls in (0, 1):
        done = [0]
        paged = EX.PagedTarget.forward

        def forward(ids, cache, new_rows=None):
            target.lm_head = head if done[0] < good_calls else torch.full_like(head, float("nan"))
            done[0] += 1
            return paged(target, ids, cache, new_rows)

        target.forward = forward
        with pytest.raises(RuntimeError, match="no token"):
            EX.generate(target, draft, [[5, 6, 7]], 20, 1.0)
    draft.close()
