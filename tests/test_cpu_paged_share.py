"""Pages that several requests hold, without a GPU: refusals of the C entry points and the Python operators, and the
restatement that the GPU tests compare with."""
import ctypes
import random

import pytest
import torch

from share_util import Shared

P, Q = ctypes.c_void_p(4096), ctypes.c_void_p(8192)      # never dereferenced: the checks fail first


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg._native.load()


def _refused(pkg, status, text):
    assert status == pkg._native.DFLASH_ERR_INVALID
    assert text in pkg._native.last_error(), pkg._native.last_error()


def test_fork_refuses_bad_arguments(pkg, lib):
    def fork(src=P, dst=P, m=2, lens=P, n=4, page=16, ld=8, width=8, holders=P, num_pages=10, out=Q):
        return lib.dflash_paged_fork(src, dst, None, m, lens, P, n, page, P, ld, width, holders, num_pages, out, Q, None, None, None)

    for kw in (dict(src=None), dict(dst=None), dict(lens=None), dict(holders=None), dict(out=None)):
        _refused(pkg, fork(**kw), "NULL")
    _refused(pkg, fork(m=-1), "forks")
    _refused(pkg, fork(m=2049), "forks")
    _refused(pkg, fork(out=P), "must not be the inputs")
    _refused(pkg, fork(n=0), "n 0")
    _refused(pkg, fork(page=24), "page_size")
    _refused(pkg, fork(ld=7), "table_ld")
    _refused(pkg, fork(num_pages=-1), "num_pages")


def test_reserve_and_release_refuse_bad_arguments(pkg, lib):
    def reserve(lens=P, n=4, page=64, ld=8, holders=P, copies=Q, slots=P, num_slots=4, out=Q):
        return lib.dflash_paged_reserve_forked(lens, P, P, n, page, P, ld, 8, P, 10, P, holders, Q, slots, num_slots, out, Q, Q,
                                               copies, None, None, None)

    for kw in (dict(lens=None), dict(holders=None), dict(copies=None), dict(slots=None)):
        _refused(pkg, reserve(**kw), "NULL")
    _refused(pkg, reserve(num_slots=-1), "num_slots")
    _refused(pkg, reserve(out=P), "must not be the inputs")
    _refused(pkg, reserve(n=2049), "n 2049")
    _refused(pkg, reserve(page=8), "page_size")

    def release(keep=P, holders=P, out=Q, ld=8):
        return lib.dflash_paged_release_forked(keep, P, 4, 16, P, ld, 8, P, 10, P, holders, out, Q, None, None)

    _refused(pkg, release(keep=None), "NULL")
    _refused(pkg, release(holders=None), "NULL")
    _refused(pkg, release(out=P), "must not be the inputs")
    _refused(pkg, release(ld=1), "table_ld")


def test_page_copies_refuse_bad_arguments(pkg, lib):
    pools = (ctypes.c_void_p * 2)(4096, 8192)

    def copy(pools=pools, layers=2, num_pages=4, nkv=2, page=32, copies=P, n=3):
        return lib.dflash_q4_copy_pages(pools, layers, num_pages, nkv, page, copies, n, None)

    _refused(pkg, copy(pools=None), "NULL")
    _refused(pkg, copy(copies=None), "NULL")
    _refused(pkg, copy(pools=(ctypes.c_void_p * 2)(4096, None)), "NULL")
    _refused(pkg, copy(pools=(ctypes.c_void_p * 2)(4096, 8196)), "aligned")
    _refused(pkg, copy(layers=-1), "layers")
    _refused(pkg, copy(n=-1), "n -1")
    _refused(pkg, copy(page=20), "page_size")
    _refused(pkg, copy(nkv=0), "nkv")
    assert copy(n=0) == 0 and copy(layers=0) == 0


def test_python_operators_refuse_cpu_tensors(pkg):
    one = torch.zeros(1, dtype=torch.int32)
    table, holders = torch.zeros(1, 1, dtype=torch.int32), pkg.page_holders(4, device="cpu")
    with pytest.raises(ValueError):
        pkg.paged_fork(one, one, one, one, table, holders, 16)
    with pytest.raises(ValueError):
        pkg.paged_reserve_forked(one, one, one, table, one, one, holders, 16, 1)
    with pytest.raises(ValueError):
        pkg.paged_release_forked(one, one, table, one, one, holders, 16)
    with pytest.raises(ValueError):
        pkg.q4_copy_pages([pkg.q4_pool(1, 1, 16, device="cpu")], torch.zeros(1, 3, dtype=torch.int32))
    with pytest.raises(ValueError):
        pkg.page_holders(0, device="cpu")


def test_restatement_keeps_rows_apart():
    """No two requests ever write one row, and every page comes back."""
    rng = random.Random(0)
    for seed in range(30):
        s = Shared(7, 60, 16, 10)
        value = [dict() for _ in range(7)]        # slot -> the request's row there
        store = {}
        for step in range(40):
            if rng.random() < 0.4:
                src, dst = [rng.randrange(7) for _ in range(3)], rng.sample(range(7), 3)
                s.fork(src, dst)
            new = [rng.choice([0, 1, 20]) for _ in range(7)]
            s.release(s.lens)
            starts, slots, copies, served = s.reserve(new, sum(new))
            for a, b, r in copies:
                for i in range(r):
                    store[b * 16 + i] = store.get(a * 16 + i)
            real = [x for x in slots if x >= 0]
            assert len(set(real)) == len(real)
            owners = s.owners()
            for x in real:
                assert owners[x // 16] == 1
                store[x] = (step, x)
            s.lens = [0 if rng.random() < 0.2 else a for a in s.lens]
        s.release([0] * 7)
        assert s.head == 0 and sorted(s.free) == list(range(60))
