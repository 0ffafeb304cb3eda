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


def test_prefix_attention_refuses_bad_arguments(pkg, lib):
    def plan(table=P, ld=8, lens=P, n=4, max_rows=1, page=16, groups=P, g=2, own=Q, least=0):
        return lib.dflash_paged_prefix_plan(table, ld, 8, lens, None, n, max_rows, page, groups, g, 1, least, P, P, P, P, own, None)

    for kw in (dict(table=None), dict(lens=None), dict(groups=None), dict(own=None)):
        _refused(pkg, plan(**kw), "NULL")
    _refused(pkg, plan(ld=7), "table_ld")
    _refused(pkg, plan(n=0), "n 0")
    _refused(pkg, plan(max_rows=0), "max_rows")
    _refused(pkg, plan(max_rows=65537), "max_rows")
    _refused(pkg, plan(g=0), "groups")
    _refused(pkg, plan(g=2049), "groups")
    _refused(pkg, plan(own=P), "own_lens")
    _refused(pkg, plan(least=-1), "least")

    size = lib.dflash_q4_prefix_workspace_size
    assert size(100, 1, 8, 32, 8) >= 100 * 32 * 130 * 4 + lib.dflash_q4_attention_workspace_size(8, 32, 8)
    for bad in ((-1, 1, 8, 32, 8), (4, 0, 8, 32, 8), (4, 1, 0, 32, 8), (4, 1, 8, 7, 2), (4, 64, 1025, 8, 8), (2 ** 30, 1, 1, 8, 8)):
        assert size(*bad) == 0

    def attend(q=P, row=1024, ws=P, nbytes=1 << 40, starts=P, n=4, rows=4, max_rows=1, g=1, max_group=4, nq=8, nkv=2, scale=0.1,
               prefix=P, out=ctypes.c_void_p(1 << 30), page=16):
        return lib.dflash_q4_prefix_attention(q, row, 128, 0, P, 16, page, P, 8, 8, starts, n, rows, max_rows, P, prefix, P, g,
                                              max_group, P, P, nq, nkv, 1, scale, out, None, ws, nbytes, None)

    for kw in (dict(q=None), dict(ws=None), dict(prefix=None), dict(out=None)):
        _refused(pkg, attend(**kw), "NULL")
    _refused(pkg, attend(g=0), "groups")
    _refused(pkg, attend(max_group=0), "groups of 0")
    _refused(pkg, attend(max_group=2048, max_rows=64), "groups of 2048")
    _refused(pkg, attend(rows=3, starts=None), "without starts")
    _refused(pkg, attend(nq=7), "multiple")
    _refused(pkg, attend(scale=0.0), "positive")
    _refused(pkg, attend(row=1028), "strides")
    _refused(pkg, attend(page=20), "page_size")
    _refused(pkg, attend(ws=ctypes.c_void_p(4104)), "workspace")
    _refused(pkg, attend(nbytes=1000), "workspace too small")
    _refused(pkg, attend(out=P), "overlaps")
    assert attend(rows=0) == 0


def test_prefix_plan_refuses_bad_groups(pkg):
    table, lens = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    for groups in ([], [0, 4], [3, 2], [-1]):
        with pytest.raises(ValueError, match="groups"):
            pkg.paged_prefix_plan(table, lens, groups, 16)
    with pytest.raises(ValueError, match="max_group"):
        pkg.paged_prefix_plan(table, lens, lens, 16)
    with pytest.raises(ValueError):
        pkg.paged_prefix_plan(table, lens, [4], 16)          # tensors on the CPU
