"""Host side of the paged 4-bit cache without a GPU: what its kernels may rely
on, importing and building, and refusals at the ends of the ranges."""
import ctypes
import importlib.util
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mirror-sd_b200", "csrc")


def _source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def test_paged_kernels_do_not_wait_for_other_ctas():
    """They are launched as ordinary grids, so a CTA may not poll for what another one writes: it may never be resident."""
    for name in ("paged.cu", "q4_cache.cu", "q4_attention.cu", "q4_attention_tc.cu", "q4_attn.cuh"):
        text = _source(name)
        assert "ld_acquire" not in text and "nanosleep" not in text, name


# ---------------------------------------------------------------- refusals of the C entries
P = ctypes.c_void_p(4096)      # never dereferenced: the checks fail first, or there is no device


def _attend(lib, n=1, width=8, page=64, rows=1, max_rows=1, nq=2, nkv=2, window=0, starts=None, q=P,
            out=ctypes.c_void_p(1 << 44), q_row=256):
    return lib.dflash_q4_attention(q, q_row, 128, 0, P, 16, page, P, width, width, P, starts, n, rows, max_rows, nq, nkv, 1,
                                   0, window, 0.1, out, None, P, 1 << 30, None)


def _refused(pkg, status, text):
    assert status == pkg._native.DFLASH_ERR_INVALID
    assert text in pkg._native.last_error(), pkg._native.last_error()


def test_attention_refuses_tables_beyond_its_32_bit_sums(pkg):
    """Keys, tile ends and window ends of a request are counted in 32 bits."""
    lib = pkg._native.load()
    _refused(pkg, _attend(lib, width=2 ** 24 + 1), "2^30")
    _refused(pkg, _attend(lib, width=2 ** 25 - 1, window=5), "2^30")


def test_prompts_of_full_size_caches_are_taken(pkg):
    """One request's prompt in a cache of many slots and long tables: the tiles that exist are bounded by the rows of q."""
    lib = pkg._native.load()
    for kw in (dict(n=256, width=512, rows=4096, max_rows=4096, nq=32, nkv=8),
               dict(n=64, width=2048, rows=4096, max_rows=4096, nq=32, nkv=8),
               dict(n=16, width=2048, rows=8192, max_rows=8192, nq=64, nkv=8),
               dict(n=2048, width=512, rows=2048, max_rows=1, nq=32, nkv=8)):
        status = _attend(lib, starts=P, q_row=kw["nq"] * 128, **kw) if not torch.cuda.is_available() else 0
        assert status != pkg._native.DFLASH_ERR_INVALID, (kw, pkg._native.last_error())
    _refused(pkg, _attend(lib, n=2048, width=2 ** 22, rows=65536, max_rows=65536, nq=32, nkv=8, starts=P, q_row=4096),
             "too large")


def test_tile_sums_stay_in_range():
    """The device's sum of tile counts, restated: full is full, in any order of additions."""
    full = 2 ** 31 - 1
    add = lambda a, b: min((a + b) % 2 ** 32, full)
    rng = np.random.default_rng(0)
    for top in (10, 2 ** 20, 2 ** 30, full):
        v = [int(x) for x in rng.integers(0, top, 64)]
        tree = v
        while len(tree) > 1:
            tree = [add(a, b) for a, b in zip(tree[::2], tree[1::2])]
        line = 0
        for x in v:
            line = add(line, x)
        assert tree[0] == line == min(sum(v), full)


# ---------------------------------------------------------------- importing and building
ROOT = os.path.dirname(CSRC[:-len("/csrc")])


def test_package_imports_on_a_torch_without_cuda():
    code = ("import importlib, torch\n"
            "for n in [n for n in dir(torch._C) if n.startswith('_cuda_')]:\n"
            "    delattr(torch._C, n)\n"
            "pkg = importlib.import_module('mirror-sd_b200')\n"
            "assert pkg.PagedKVCacheQ4 and pkg.DFlashConfig\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


@pytest.fixture
def builder(tmp_path, monkeypatch):
    """build.py with an output folder of its own and a library that need not be compiled again."""
    spec = importlib.util.spec_from_file_location("dflash_build", os.path.join(ROOT, "mirror-sd_b200", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    for name, file in (("LIB_DIR", ""), ("LIB", "lib.so"), ("BINDING", "binding.so")):
        monkeypatch.setattr(b, name, str(tmp_path / file))
    b.compiled = []

    def library(verbose):
        b.compiled.append("library")
        with open(b.LIB, "w") as f:
            f.write("library")

    monkeypatch.setattr(b, "_build_library", library, raising=False)
    return b


def _as_binding(b, monkeypatch, *how):
    def command(out):
        if out:
            b.compiled.append("binding")
        return ["cp", *how, os.path.join(CSRC, b.BINDING_SOURCE), out]
    monkeypatch.setattr(b, "_binding_command", command)


def test_library_builds_without_torch(builder, monkeypatch, capsys):
    monkeypatch.setattr(builder.importlib.util, "find_spec", lambda name: None)
    assert builder.build() == builder.LIB and os.path.exists(builder.LIB) and not os.path.exists(builder.BINDING)
    assert "torch is not installed" in capsys.readouterr().out
    builder.build()
    assert builder.compiled == ["library"]


def test_library_is_there_when_the_binding_does_not_compile(builder, monkeypatch):
    _as_binding(builder, monkeypatch, "--no-such-flag")
    for _ in range(2):
        with pytest.raises(RuntimeError, match="binding"):
            builder.build()
    assert os.path.exists(builder.LIB) and not os.path.exists(builder.BINDING)
    assert builder.compiled == ["library", "binding", "binding"]


def test_binding_is_built_again_for_another_torch(builder, monkeypatch):
    _as_binding(builder, monkeypatch)
    builder.build()
    builder.build()
    assert builder.compiled == ["library", "binding"] and os.path.exists(builder.BINDING)
    assert torch.__version__.split("+")[0] in builder._torch_version()
    monkeypatch.setattr(builder, "_torch_version", lambda: "99.0")
    builder.build()
    builder.build()
    assert builder.compiled == ["library", "binding", "binding"]


def test_attention_refuses_an_output_over_its_queries(pkg):
    """Strided query rows: the output may lie beside them, in front or behind, or in the gap between two rows."""
    lib = pkg._native.load()
    at = lambda byte: ctypes.c_void_p((1 << 20) + byte)
    call = lambda byte, rows, row, **kw: _attend(lib, rows=rows, max_rows=rows, q=at(0), out=at(byte), q_row=row, **kw)
    size = lambda rows: rows * 2 * 256
    for rows, row, byte in ((4, 256, 0), (4, 256, 16), (4, 256, -16), (4, 256, size(4) - 16), (4, 256, 16 - size(4)),
                            (3, 1024, 2048), (3, 1024, 1024), (3, 1024, 4096 + 496), (3, 0, 0), (3, 0, 496), (2, 4096, 8192),
                            (2, 4096, 8192 - 16), (3, -256, 0), (3, -256, -1024)):
        _refused(pkg, call(byte, rows, row), "overlaps")
    if not torch.cuda.is_available():           # (past the check there is no device)
        for rows, row, byte in ((4, 256, size(4)), (4, 256, -size(4)), (3, 1024, 4096 + 512), (3, 0, 512), (2, 4096, 512),
                                (2, 4096, 8192 - 1024), (1, 4096, 8192), (3, -256, 512), (3, -256, -1024 - size(3))):
            assert call(byte, rows, row) != pkg._native.DFLASH_ERR_INVALID, (rows, row, byte, pkg._native.last_error())


def test_trim_and_tracked_reserve_refuse_bad_arguments(pkg):
    lib = pkg._native.load()
    _refused(pkg, lib.dflash_paged_trim(None, P, 0, P, 4, P, None), "NULL")
    _refused(pkg, lib.dflash_paged_trim(P, None, 3, None, 4, None, None), "NULL")
    _refused(pkg, lib.dflash_paged_trim(P, None, 3, None, 0, P, None), "n 0")
    _refused(pkg, lib.dflash_paged_trim(P, None, 3, None, 2049, P, None), "n 2049")
    _refused(pkg, lib.dflash_paged_reserve_tracked(P, P, P, 4, 48, P, 8, 8, P, 10, P, P, P, 4, ctypes.c_void_p(8192),
                                                   ctypes.c_void_p(8192), ctypes.c_void_p(8192), P, None, None), "page_size")


def test_a_workspace_serves_every_smaller_number_of_rows(pkg):
    size = pkg._native.load().dflash_q4_attention_workspace_size
    for nq, nkv in ((1, 1), (4, 1), (5, 1), (32, 8), (40, 8), (16, 1), (64, 2)):
        sizes = [size(rows, nq, nkv) for rows in range(1, 300)]
        assert all(sizes) and sizes == sorted(sizes), (nq, nkv)
