"""Host side of the paged 4-bit cache without a GPU: what its kernels may rely
on, importing and building, and refusals at the ends of the ranges."""
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
