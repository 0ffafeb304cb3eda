"""Acceptance of drafts by sampling (csrc/verify.cu), where ``accept`` is greedy.

The drafter proposes greedily or samples; either way the tokens that come out
are distributed as the target's own samples at its temperature.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _native as N


def verify_drafts(logits, drafts, uniforms, temperature: Union[float, torch.Tensor] = 1.0, draft_probs=None, num_drafts=None):
    """How many of each request's drafts the target accepts, and the token that
    follows them: (accepted [n], tokens [n]), int32.

    logits [n, block, V] (f16, bf16 or f32): the target's at the block's
    positions, row j those of the token behind [anchor, drafts][j]; drafts
    [n, block - 1] int32; uniforms [n, block] f32, random numbers in [0, 1).
    temperature: a number or [n] f32 on the device; below 1e-5 a request is
    greedy and gives what ``accept`` gives for the first largest logits, compared
    as they are.  (Sampled requests take logits beyond +-1e30 for that.)

    Draft j is accepted while uniforms[j] * q(draft) < p_j(draft) with p_j =
    softmax(logits_j / temperature) and q its probability in ``draft_probs``
    [n, block - 1, V] f32, what it was sampled from (1 where the drafts were not
    sampled: no ``draft_probs``).  The token behind the accepted ones is sampled
    from max(p - q, 0) at the refused place, or from p behind the last draft,
    with the last random number: the first token in vocabulary order whose
    running sum passes it.  num_drafts [n] int32: how many of its drafts a
    request uses, where not all.  Rows behind a refused draft do not count, but
    may be read: they must hold what they will hold when the call is made.

    V is 2^22 at most.  NaN logits count as -inf; a row that leaves no token refuses its draft and
    gives token -1.  accepted -1 (and token -1) means that a bounded wait on the device expired and
    nothing is known of the request: check both before they become slices and indices."""
    return N.load_paged().verify(logits, drafts, uniforms, temperature, draft_probs, num_drafts)


def sample_tokens(logits, uniforms, temperature: Union[float, torch.Tensor] = 1.0):
    """One token a row of logits [n, V], each from its random number in
    uniforms [n]: ``verify_drafts`` without drafts.  -1 for a row that leaves none."""
    if logits.dim() != 2:
        raise ValueError(f"logits must be [n, V], got {tuple(logits.shape)}")
    none = torch.empty(logits.shape[0], 0, dtype=torch.int32, device=logits.device)
    return verify_drafts(logits[:, None], none, uniforms[:, None], temperature)[1]
