"""Rotary positions of query and key rows (csrc/rope.cu).

The drafter's own forward turns its rows inside its kernels; a target model's
rows are turned here before they are cached and attended, wherever they lie:

    rope = Rope(head_dim, theta)
    qk = apply_rope(qkv[:, :NQ + NKV], rope, step)     # or positions [rows]
    cache.append(layer, qk[:, NQ:], v, step)
"""
from __future__ import annotations

import math
from typing import Optional, Union

import torch

from . import _native as N
from .paged import PagedStep

SCALINGS = ("linear", "ntk", "yarn")


def rope_frequencies(rotary_dim: int, theta: float = 1e4, scaling: Optional[dict] = None):
    """(frequencies [rotary_dim / 2] in radians a position, float64; factor of
    cosine and sine).  theta ** (-2 i / rotary_dim), for longer contexts than a
    model was trained on changed by ``scaling``, a dict with "type" (or
    "rope_type") and "factor" s:

    linear  every frequency over s
    ntk     theta * s ** (r / (r - 2)): the lowest frequency over s, the highest kept
    yarn    pairs that turn "beta_fast" (32) times or more within
            "original_max_position_embeddings" positions are kept, those that turn
            "beta_slow" (1) times or less divided by s, between them a ramp;
            the factor is "attention_factor", by default 0.1 ln s + 1
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} must be even and positive")
    if not theta > 0 or not math.isfinite(theta):
        raise ValueError(f"theta {theta} must be positive and finite")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    kind = None if scaling is None else scaling.get("rope_type", scaling.get("type"))
    if kind in (None, "default") and (scaling is None or kind == "default"):
        return theta ** (-2 * i / rotary_dim), 1.0
    if kind not in SCALINGS:
        raise ValueError(f"rope scaling {kind!r} is none of {SCALINGS}")
    s = float(scaling["factor"])
    if not s >= 1 or not math.isfinite(s):
        raise ValueError(f"rope scaling factor {s} must be at least 1")
    if kind == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs two frequencies or more")
        return (theta * s ** (rotary_dim / (rotary_dim - 2))) ** (-2 * i / rotary_dim), 1.0
    freq = theta ** (-2 * i / rotary_dim)
    if kind == "linear":
        return freq / s, 1.0
    if not theta > 1:
        raise ValueError("yarn scaling needs theta above 1")
    length = float(scaling["original_max_position_embeddings"])
    if not length > 0:
        raise ValueError("original_max_position_embeddings must be positive")

    def pair_that_turns(times):      # the pair that turns so often within the original length
        return rotary_dim * math.log(length / (times * 2 * math.pi)) / (2 * math.log(theta))

    low = max(math.floor(pair_that_turns(float(scaling.get("beta_fast", 32.0)))), 0)
    high = min(math.ceil(pair_that_turns(float(scaling.get("beta_slow", 1.0)))), rotary_dim - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    factor = scaling.get("attention_factor")
    return freq * (1 - ramp) + freq / s * ramp, float(0.1 * math.log(s) + 1.0 if factor is None else factor)


class Rope:
    """The frequencies of one model on one device.  ``rotary_dim`` (default
    head_dim): the channels that are turned, the first ones of a head;
    ``interleaved``: pairs (2 i, 2 i + 1) and not (i, i + rotary_dim / 2)."""

    def __init__(self, head_dim: int, theta: float = 1e4, rotary_dim: Optional[int] = None, interleaved: bool = False,
                 scaling: Optional[dict] = None, device="cuda"):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim < 2 or head_dim > 1024 or head_dim % 2:
            raise ValueError(f"head_dim {head_dim} must be even and at most 1024")
        if rotary_dim > head_dim:
            raise ValueError(f"rotary_dim {rotary_dim} is more than head_dim {head_dim}")
        freq, self.factor = rope_frequencies(rotary_dim, theta, scaling)
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, rotary_dim, bool(interleaved)
        self.turns = (freq / (2 * math.pi)).to(device)


class _Turned(torch.autograd.Function):
    """Rows turned; their gradient is that of the result turned back (and again, so it has one itself)."""

    @staticmethod
    def forward(ctx, x, rope, positions, inverse):
        step = isinstance(positions, PagedStep)
        ctx.rope, ctx.inverse, ctx.step = rope, not inverse, positions if step else None
        ctx.save_for_backward(*(positions[:1] + positions[2:3] if step else (positions,)))   # (changed in place meanwhile: an error)
        # (rows of no request of a step are left unwritten: as a gradient they are zero)
        out = torch.zeros_like(x, memory_format=torch.contiguous_format) if step else None
        return _turn(x, rope, positions, out, inverse)

    @staticmethod
    def backward(ctx, grad):
        saved = ctx.saved_tensors
        positions = saved[0] if ctx.step is None else ctx.step._replace(starts=saved[0], lens=saved[1])
        return _Turned.apply(grad, ctx.rope, positions, ctx.inverse), None, None, None


def _turn(x, rope, positions, out, inverse):
    starts = lens = None
    if isinstance(positions, PagedStep):
        starts, lens, positions = positions.starts, positions.lens, None
    return N.load_paged().rope(x, rope.turns, rope.factor, rope.rotary_dim, rope.interleaved, inverse, positions, starts, lens,
                               out)


def apply_rope(x, rope: Rope, positions: Union[torch.Tensor, PagedStep], out=None, inverse: bool = False):
    """x [rows, heads, head_dim] (f16, bf16 or f32; strided rows and heads) with
    its rows turned to their positions, in a new tensor or in ``out`` (x itself,
    or memory apart from x).  positions: int32 or int64 [rows], or the
    ``PagedStep`` whose packed rows x holds (rows of no request are then left
    unwritten).  inverse: turned back, which is also the gradient of x from that
    of the result, and what autograd gets where x requires one (then without
    ``out``, and rows of no request are zeros).  Angles are formed in 64 bits; the
    result is rounded once."""
    if x.dim() == 3 and x.shape[2] != rope.head_dim:
        raise ValueError(f"x has heads of {x.shape[2]} channels, the positions are for {rope.head_dim}")
    if positions is None:
        raise ValueError("positions must be a tensor or a PagedStep")
    if torch.is_grad_enabled() and (x.requires_grad or (out is not None and out.requires_grad)):
        if out is not None:
            raise ValueError("apply_rope writes to out without a gradient: leave it to a new tensor, or use torch.no_grad()")
        return _Turned.apply(x, rope, positions, inverse)
    return _turn(x, rope, positions, out, inverse)
