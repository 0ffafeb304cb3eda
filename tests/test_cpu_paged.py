"""Host side of the paged 4-bit cache without a GPU: argument checks of the C
entry points (they run before any CUDA call) and of the Python operators, and
the restatements that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest
import torch

import paged_util as U


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg._native.load()


def _refused(pkg, status, text):
    assert status == pkg._native.DFLASH_ERR_INVALID
    assert text in pkg._native.last_error(), pkg._native.last_error()


P = ctypes.c_void_p(4096)      # never dereferenced: the checks fail first


def test_paged_entry_points_refuse_bad_arguments(pkg, lib):
    def reserve(n=4, page=64, ld=8, width=8, num_pages=10, slots=P, num_slots=4, out=ctypes.c_void_p(8192), lens=P):
        return lib.dflash_paged_reserve(lens, P, P, n, page, P, ld, width, P, num_pages, P, P, slots, num_slots, out, out,
                                        out, None, None)

    _refused(pkg, reserve(lens=None), "NULL")
    _refused(pkg, reserve(n=0), "n 0")
    _refused(pkg, reserve(n=2049), "n 2049")
    _refused(pkg, reserve(page=8), "page_size")
    _refused(pkg, reserve(page=48), "page_size")
    _refused(pkg, reserve(page=512), "page_size")
    _refused(pkg, reserve(ld=7), "table_ld")
    _refused(pkg, reserve(width=0), "max_pages")
    _refused(pkg, reserve(n=2000, ld=2 ** 21, width=2 ** 21), "too large")
    _refused(pkg, reserve(num_pages=2 ** 26), "2^31")
    _refused(pkg, reserve(num_slots=-1), "num_slots")
    _refused(pkg, reserve(slots=None), "NULL")
    _refused(pkg, reserve(out=P), "must not be the inputs")
    _refused(pkg, lib.dflash_paged_release(P, P, 4, 64, P, 8, 8, P, 10, P, P, P, None, None), "must not be the inputs")
    _refused(pkg, lib.dflash_paged_release(None, P, 4, 64, P, 8, 8, P, 10, P, P, P, None, None), "NULL")


def test_q4_entry_points_refuse_bad_arguments(pkg, lib):
    def append(k=P, row=256, head=128, rows=4, nkv=2, pool=P, num_pages=4, page=64, slots=P):
        return lib.dflash_q4_append(k, row, head, P, 256, 128, 0, slots, rows, nkv, pool, num_pages, page, None, None)

    _refused(pkg, append(pool=None), "NULL")
    _refused(pkg, append(k=None), "NULL")
    _refused(pkg, append(slots=None), "NULL")
    _refused(pkg, append(k=ctypes.c_void_p(4104)), "aligned")
    _refused(pkg, append(pool=ctypes.c_void_p(4104)), "aligned")
    _refused(pkg, append(row=252), "strides")
    _refused(pkg, append(head=4), "strides")
    _refused(pkg, append(rows=-1), "rows")
    _refused(pkg, append(nkv=0), "nkv")
    _refused(pkg, append(page=24), "page_size")
    _refused(pkg, append(num_pages=0), "num_pages")
    _refused(pkg, append(num_pages=2 ** 25), "2^31")
    assert append(rows=0) == 0                       # nothing to do: no launch

    def read(rows=4, k=P, page=64):
        return lib.dflash_q4_read(P, 4, page, P, rows, 2, 0, k, P, None)

    _refused(pkg, read(k=None), "NULL")
    _refused(pkg, read(page=1), "page_size")
    assert read(rows=0) == 0

    def attend(q=P, row=1024, page=64, n=2, rows=2, max_rows=1, nq=8, nkv=2, sink=0, window=0, scale=0.1, starts=None,
               ws=P, nbytes=1 << 30, width=8):
        return lib.dflash_q4_attention(q, row, 128, 0, P, 16, page, P, 8, width, P, starts, n, rows, max_rows, nq, nkv, 0,
                                       sink, window, scale, P, None, ws, nbytes, None)

    _refused(pkg, attend(q=None), "NULL")
    _refused(pkg, attend(ws=None), "NULL")
    _refused(pkg, attend(q=ctypes.c_void_p(4100)), "aligned")
    _refused(pkg, attend(row=1028), "strides")
    _refused(pkg, attend(page=100), "page_size")
    _refused(pkg, attend(nq=7), "multiple")
    _refused(pkg, attend(nq=1), "multiple")
    _refused(pkg, attend(max_rows=0), "max_rows")
    _refused(pkg, attend(max_rows=70000, starts=P), "max_rows")
    _refused(pkg, attend(rows=3), "without starts")
    _refused(pkg, attend(sink=-1), "sink")
    _refused(pkg, attend(sink=4), "sink needs a window")
    _refused(pkg, attend(window=-4), "window")
    _refused(pkg, attend(scale=float("inf")), "finite")
    _refused(pkg, attend(scale=0.0), "positive")
    _refused(pkg, attend(scale=-0.1), "positive")
    _refused(pkg, attend(nbytes=100), "workspace too small")
    _refused(pkg, attend(width=9), "table_ld")
    assert attend(rows=0, starts=P) == 0


def test_sizes(pkg, lib):
    assert lib.dflash_q4_page_bytes(8, 64) == 8 * 4 * 2304           # 4.5 bits a channel, K and V
    assert lib.dflash_q4_page_bytes(8, 64) * 8 == 64 * 8 * 2 * 128 * 4.5
    assert lib.dflash_q4_page_bytes(0, 64) == 0 and lib.dflash_q4_page_bytes(8, 40) == 0
    size = lib.dflash_q4_attention_workspace_size
    assert size(1, 32, 8) > 4096 and size(16, 32, 8) >= size(1, 32, 8)
    assert size(0, 32, 8) == 0 and size(1, 32, 7) == 0


def test_python_operators_refuse_cpu_tensors(pkg):
    pool = torch.zeros(2, 1, 2, 2304, dtype=torch.uint8)
    with pytest.raises(ValueError):
        pkg.q4_read(pool, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        pkg.q4_append(torch.zeros(1, 1, 128), torch.zeros(1, 1, 128), torch.zeros(1, dtype=torch.int32), pool)
    with pytest.raises(ValueError):
        pkg.paged_release(*[torch.zeros(1, dtype=torch.int32)] * 5, page_size=16)
    with pytest.raises(ValueError):
        pkg.q4_pool(1, 1, 20, device="cpu")


def test_quantiser_restatement():
    """The scale is the smallest one that holds the maximum, and the stored value is off by at most half a step."""
    rng = np.random.default_rng(0)
    x = torch.from_numpy((rng.standard_normal((200, 128)) * 2.0 ** rng.integers(-14, 10, (200, 1))).astype(np.float16))
    y = U.q4_values(x)
    scales = U.scale_values()
    a = x.double().abs().reshape(200, 8, 16).amax(-1).numpy()
    s = scales[np.searchsorted(scales * 7.5, a)]
    assert np.all(7.5 * s >= a)
    lower = scales[np.maximum(np.searchsorted(scales, s) - 1, 0)]
    assert np.all((7.5 * lower < a) | (s == scales[0]))
    err = (y - x.double()).abs().reshape(200, 8, 16).amax(-1).numpy()
    assert np.all(err <= s / 2)
    assert torch.equal(y.half().double(), y) and torch.equal(y.bfloat16().double(), y)      # exact in both types


def test_paging_restatement_returns_every_page():
    lens, new, page = [5, 0, 40], [30, 17, 1], 16
    pg = U.Paging(lens, page, spare=8, max_pages=6)
    table, free = pg.table.copy(), pg.free.copy()
    starts, slots, lens2, pages2, head, status = U.reserve(lens, new, pg.pages, table, free, pg.head, page, 48)
    assert status == 0 and lens2 == [35, 17, 41] and len(set(slots)) == 48 and starts == [0, 30, 47, 48]
    pages3, head3 = U.release([0, 0, 0], pages2, table, free, head, page)
    assert pages3 == [0, 0, 0] and head3 == 0 and sorted(free) == sorted(pg.free)


def test_seen_keys_restatement():
    assert U.seen_keys(5, 2, 0, True, 0, 0).tolist() == [True] * 4 + [False]
    assert U.seen_keys(5, 2, 1, True, 1, 2).tolist() == [True, False, False, True, True]
    assert U.seen_keys(2, 4, 0, True, 0, 0).tolist() == [False, False]
    assert U.seen_keys(5, 9, 3, False, 0, 1).tolist() == [False] * 4 + [True]
