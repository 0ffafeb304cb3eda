"""Batched speculative decoding of a target model whose K/V lives in the paged
4-bit cache.

A small decoder-only transformer with random weights (there is no checkpoint
here) is the target.  Its attention layers keep their keys and values in a
``PagedKVCacheQ4``; the block drafter proposes, the target verifies the blocks
of all requests in one packed forward, and what was rejected is trimmed on the
GPU.  Requests differ in length, finish at different times and give their pages
back.  With --samples a prompt is read once and forked: its continuations hold
its pages together, and attention reads them once for all; with --temperature
they are sampled and differ.

    python examples/paged_generate.py [--requests 8] [--new-tokens 64] [--samples 4 --temperature 0.8]

``PagedTarget`` also is a target for ``spec_generate``, one request at a time:
its cache is the paged cache itself.
"""
import argparse
import importlib
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sd = importlib.import_module("mirror-sd_b200")

HEAD_DIM = 128


class PagedTarget:
    """RMSNorm, RoPE, grouped-query attention over the cache, SwiGLU; tied
    embedding.  ``forward`` takes the packed new tokens of all requests."""

    def __init__(self, vocab, hidden, layers, heads, kv_heads, inter, features, max_seqs=1, max_len=4096,
                 num_pages=None, page_size=64, rope_theta=1e4, seed=0, device="cuda", samples=1, least=None):
        g = torch.Generator().manual_seed(seed)
        w = lambda o, i, gain=1.0: (torch.randn(o, i, generator=g) * gain * i ** -0.5).to(device, torch.float16)
        self.device, self.heads, self.kv_heads = torch.device(device), heads, kv_heads
        self.max_seqs, self.max_len, self.page_size = max_seqs, max_len, page_size
        self.num_pages = num_pages or max_seqs * -(-max_len // page_size)
        self.features = features             # number of layers whose output the drafter reads, the last ones
        self.samples, self.least = samples, least    # requests side by side that go on from one prompt
        self.E = torch.randn(vocab, hidden, generator=g).to(device, torch.bfloat16)
        self.layers = [dict(qkv=w((heads + 2 * kv_heads) * HEAD_DIM, hidden), o=w(hidden, heads * HEAD_DIM),
                            gate_up=w(2 * inter, hidden), down=w(hidden, inter)) for _ in range(layers)]
        self.lm_head = (self.E.float() * hidden ** -0.5).to(torch.float16)
        self.rope = sd.Rope(HEAD_DIM, rope_theta, device=device)

    def make_cache(self):
        return sd.PagedKVCacheQ4(len(self.layers), self.num_pages, self.kv_heads, self.max_seqs, self.max_len,
                                 self.page_size, self.device, forkable=self.samples > 1)

    def embed(self, ids):
        return self.E[ids]

    def forward(self, ids, cache, new_rows=None):
        """ids [1, T]: the new tokens of request 0, then of request 1, ...
        (new_rows[i] of request i).  Returns logits [1, T, V] and the features
        [1, T, F * hidden], and leaves the T tokens' rows in the cache."""
        new_rows = [ids.shape[1]] if new_rows is None else new_rows
        step, plan = cache.reserve(new_rows), None
        if self.samples > 1:
            plan = cache.prefix_plan(step, [self.samples] * (self.max_seqs // self.samples), max(new_rows), least=self.least)
        norm = lambda x: torch.nn.functional.rms_norm(x, x.shape[-1:]).half()
        x, feats, nq, nkv = self.E[ids[0]].float(), [], self.heads, self.kv_heads
        for i, L in enumerate(self.layers):
            qkv = (norm(x) @ L["qkv"].T).view(-1, nq + 2 * nkv, HEAD_DIM)
            qk, v = norm(qkv[:, :nq + nkv]), qkv[:, nq + nkv:]            # per-head norms of q and k
            qk = sd.apply_rope(qk, self.rope, step)                       # each row at its place in its request
            cache.append(i, qk[:, nq:], v, step)
            o = cache.attend(i, qk[:, :nq], step, max(new_rows), plan=plan)
            x = x + (o.flatten(1) @ L["o"].T).float()
            gate, up = (norm(x) @ L["gate_up"].T).chunk(2, dim=-1)
            x = x + ((torch.nn.functional.silu(gate) * up) @ L["down"].T).float()
            if i >= len(self.layers) - self.features:
                feats.append(x.to(torch.bfloat16))
        return (norm(x) @ self.lm_head.T)[None], torch.cat(feats, dim=-1)[None]


@torch.no_grad()
def generate(target, draft, prompts, max_new_tokens, temperature=0.0, generator=None):
    """Speculative decoding of all prompts together, ``target.samples`` times each
    (sequence k of prompt i is number i * samples + k), greedy or sampled.  Returns
    the sequences, the accepted drafts of every step, and the cache."""
    S, B, dev = target.samples, draft.block_size, target.device
    prompts = [p for p in prompts for _ in range(S)]
    n = len(prompts)
    cache, server = target.make_cache(), sd.DraftServer(draft, n)
    out = [list(p) for p in prompts]
    accepted = []
    numbers = lambda *shape: torch.rand(*shape, device=dev, generator=generator) if temperature else None
    firsts = [len(p) if i % S == 0 else 0 for i, p in enumerate(prompts)]      # each prompt is read once
    logits, feats = target.forward(torch.tensor([sum(prompts[::S], [])], device=dev), cache, firsts)
    if S > 1:
        others = [i for i in range(n) if i % S]
        cache.fork([i - i % S for i in others], others)
        feats = torch.cat([f for f in feats.split([len(p) for p in prompts[::S]], dim=1) for _ in range(S)], dim=1)
    ends = torch.tensor(firsts[::S]).cumsum(0).repeat_interleave(S) - 1
    for i, t in enumerate(sd.sample(logits[0, ends.to(dev)], temperature, numbers(n)).tolist()):
        out[i].append(t)
    cache.check()
    if min(o[-1] for o in out) < 0:
        raise RuntimeError("the target's logits leave a request no token")
    rows, fresh = [len(p) for p in prompts], True       # context rows that each request brings
    active = list(range(n))
    while active:
        anchors = torch.tensor([out[i][-1] for i in active], device=dev)
        block = torch.full((len(active), B), draft.mask_token_id, device=dev)
        block[:, 0] = anchors
        noise = target.embed(block)
        if fresh:
            drafts, fresh = server.prefill(active, noise, feats[0], rows), False
        else:
            drafts = server.step(active, noise, feats[0], rows)[0]
        verify = torch.cat([anchors[:, None], drafts.long()], dim=1)
        new_rows = [B if i in active else 0 for i in range(n)]
        logits, feats = target.forward(verify.reshape(1, -1), cache, new_rows)
        if temperature:
            acc, corr = sd.verify_drafts(logits.view(-1, B, logits.shape[-1]), drafts, numbers(len(active), B), temperature)
        else:
            acc, corr = sd.accept(drafts, logits.argmax(-1).view(-1, B).int())
        where = torch.tensor(active, device=dev)
        cache.trim(torch.zeros(n, dtype=torch.int32, device=dev).index_copy(0, where, B - 1 - acc.int()))
        a, c, d = acc.tolist(), corr.tolist(), drafts.tolist()      # the step's one host synchronisation
        cache.check()                                               # a request without pages ends the run
        if min(a + c) < 0:                                          # and so does one that verify_drafts could not serve
            raise RuntimeError("drafts could not be verified, or the target's logits leave a request no token")
        accepted.append(a)
        for k, i in enumerate(active):
            out[i] += d[k][:a[k]] + [c[k]]
        done = [i for i in active if len(out[i]) - len(prompts[i]) >= max_new_tokens]
        cache.release(done)                                         # their pages, and spare ones of the others
        server.release(done)
        left = [k for k, i in enumerate(active) if i not in done]
        if left:
            feats = torch.cat([feats[:, k * B:k * B + a[k] + 1] for k in left], dim=1)
        rows, active = [a[k] + 1 for k in left], [active[k] for k in left]
    server.close()
    return [o[:len(p) + max_new_tokens] for o, p in zip(out, prompts)], accepted, cache


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--new-tokens", type=int, default=64)
    ap.add_argument("--samples", type=int, default=1)
    ap.add_argument("--temperature", type=float, default=0.0)
    a = ap.parse_args()
    n = a.requests * a.samples
    cfg = sd.DFlashConfig(hidden_size=1024, num_hidden_layers=2, intermediate_size=2048, num_attention_heads=16,
                          num_key_value_heads=4, head_dim=HEAD_DIM, vocab_size=8192, block_size=16, mask_token_id=8191)
    cfg.target_layer_ids = [0, 1, 2]
    target = PagedTarget(cfg.vocab_size, cfg.hidden_size, 4, 16, 4, 2048, 3, max_seqs=n, max_len=2048, samples=a.samples)
    weights, _ = sd.synth_weights_q8(cfg, seed=1, num_target_features=3)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, cfg.vocab_size, (int(m),), generator=g).tolist()
               for m in torch.randint(1, 1024, (a.requests,), generator=g)]
    draft = sd.DFlashDraftModel(cfg, weights, target.E, max_batch=n, max_ctx=2048, max_block=cfg.block_size,
                                max_ctx_rows=a.samples * sum(map(len, prompts)))
    generate(target, draft, prompts, 2 * cfg.block_size, a.temperature)
    torch.cuda.synchronize()
    t = time.perf_counter()
    out, accepted, cache = generate(target, draft, prompts, a.new_tokens, a.temperature)
    torch.cuda.synchronize()
    t = time.perf_counter() - t
    mean = sum(map(sum, accepted)) / sum(map(len, accepted))
    print(f"{n} requests, {n * a.new_tokens} tokens in {t:.2f} s, {len(accepted)} verify steps, "
          f"{mean:.2f} drafts accepted a step (random weights), all {cache.free_page_count()} pages free again")
    draft.close()


if __name__ == "__main__":
    main()
