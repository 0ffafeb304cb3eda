"""Refusals of the decode operators without a GPU: the C entry points check before any CUDA call."""
import ctypes
import math

import pytest
import torch

P = ctypes.c_void_p(4096)      # never dereferenced: the checks fail first


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg._native.load()


def _refused(pkg, status, text):
    assert status == pkg._native.DFLASH_ERR_INVALID
    assert text in pkg._native.last_error(), pkg._native.last_error()


def test_rope_refuses_bad_arguments(pkg, lib):
    def rope(x=P, x_row=256, x_head=128, type=0, rows=4, heads=2, dim=128, rot=128, turns=P, factor=1.0, positions=P, starts=None,
             lens=None, n=0, out=ctypes.c_void_p(1 << 20), out_row=256, out_head=128):
        return lib.dflash_rope(x, x_row, x_head, type, rows, heads, dim, rot, 0, 0, turns, factor, positions, 0, starts, lens, n,
                               out, out_row, out_head, None)

    _refused(pkg, rope(x=None), "NULL")
    _refused(pkg, rope(out=None), "NULL")
    _refused(pkg, rope(turns=None), "NULL")
    _refused(pkg, rope(type=3), "type")
    _refused(pkg, rope(rows=-1), "rows")
    _refused(pkg, rope(heads=0), "heads")
    _refused(pkg, rope(heads=65536), "heads")
    for dim in (0, 127, 1026):
        _refused(pkg, rope(dim=dim), "head dim")
    for rot in (0, 63, 130):
        _refused(pkg, rope(rot=rot), "rotary dim")
    _refused(pkg, rope(factor=math.inf), "factor")
    _refused(pkg, rope(positions=None), "either")
    _refused(pkg, rope(starts=P), "either")
    _refused(pkg, rope(positions=None, starts=P, lens=P), "n 0")
    _refused(pkg, rope(positions=None, starts=P, lens=P, n=2049), "n 2049")
    _refused(pkg, rope(x=ctypes.c_void_p(4097)), "aligned")
    _refused(pkg, rope(type=2, out=ctypes.c_void_p((1 << 20) + 2)), "aligned")
    _refused(pkg, rope(out_row=255), "overlap")
    _refused(pkg, rope(out_head=127), "overlap")
    _refused(pkg, rope(out_row=0), "overlap")
    _refused(pkg, rope(out=P, out_row=512), "out overlaps x")
    _refused(pkg, rope(out=ctypes.c_void_p(4096 + 2 * 128)), "out overlaps x")
    _refused(pkg, rope(x_row=-256, out=ctypes.c_void_p(4096 - 256 * 2)), "out overlaps x")
    assert rope(rows=0, x=None, out=None) == 0


def test_verify_refuses_bad_arguments(pkg, lib):
    def verify(logits=P, type=1, n=2, block=3, vocab=10, drafts=P, u=P, temps=None, temp=1.0, out=P):
        return lib.dflash_verify_drafts(logits, 30, 10, type, n, block, vocab, drafts, u, temps, temp, None, 0, 0, None, out, P, None)

    _refused(pkg, verify(logits=None), "NULL")
    _refused(pkg, verify(drafts=None), "NULL")
    _refused(pkg, verify(u=None), "NULL")
    _refused(pkg, verify(out=None), "NULL")
    _refused(pkg, verify(type=-1), "type")
    for kw in (dict(n=-1), dict(block=0), dict(vocab=0), dict(vocab=2 ** 31 - 1), dict(vocab=2 ** 22 + 1), dict(n=2 ** 28)):
        _refused(pkg, verify(**kw), "block")
    for t in (-0.1, math.nan, math.inf):
        _refused(pkg, verify(temp=t), "temperature")
    _refused(pkg, verify(logits=ctypes.c_void_p(4097)), "aligned")
    assert verify(n=0) == 0


def test_python_operators_refuse_bad_tensors(pkg):
    rope, x = pkg.Rope(64, device="cpu"), torch.zeros(4, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.apply_rope(x, rope, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="64"):
        pkg.apply_rope(torch.zeros(4, 2, 128), rope, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="positions"):
        pkg.apply_rope(x, rope, None)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.verify_drafts(torch.zeros(1, 2, 8), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 2))
    with pytest.raises(ValueError, match="tensor"):
        pkg.verify_drafts([1.0], None, None)
    with pytest.raises(ValueError):
        pkg.sample_tokens(torch.zeros(1, 2, 8), torch.zeros(1))


def test_frequencies(pkg):
    f, factor = pkg.rope_frequencies(8, 100.0)
    assert factor == 1.0 and torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64))
    assert torch.allclose(pkg.rope_frequencies(8, 100.0, {"type": "linear", "factor": 4.0})[0], f / 4)
    ntk = pkg.rope_frequencies(8, 100.0, {"rope_type": "ntk", "factor": 4.0})[0]
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]), float(f[-1]) / 4)
    yarn, factor = pkg.rope_frequencies(128, 1e4, {"type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096})
    f = pkg.rope_frequencies(128, 1e4)[0]
    assert torch.equal(yarn[:20], f[:20]) and torch.allclose(yarn[-16:], f[-16:] / 8) and math.isclose(factor, 0.1 * math.log(8) + 1)
    assert bool((yarn <= f).all() and (yarn >= f / 8 * (1 - 1e-12)).all() and (yarn[:-1] > yarn[1:]).all())
    for bad in (dict(type="other", factor=2.0), dict(type="linear", factor=0.5), dict(type="ntk", factor=math.inf), dict(factor=2.0),
                dict(type="yarn", factor=2.0, original_max_position_embeddings=0)):
        with pytest.raises(ValueError):
            pkg.rope_frequencies(8, 1e4, bad)
    for kw in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, theta=0.0), dict(rotary_dim=8, theta=math.inf)):
        with pytest.raises(ValueError):
            pkg.rope_frequencies(**kw)
    for kw in (dict(head_dim=7), dict(head_dim=2048), dict(head_dim=64, rotary_dim=66)):
        with pytest.raises(ValueError):
            pkg.Rope(device="cpu", **kw)
