"""Host side of the paged 4-bit cache without a GPU: what its kernels may rely
on, importing and building, and refusals at the ends of the ranges."""
import ctypes
import os

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


def _attend(lib, n=1, width=8, page=64, rows=1, max_rows=1, nq=2, nkv=2, window=0, starts=None, q=P, out=P, q_row=256):
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
