"""Calls of the 4-bit weight operators that are refused before anything is launched."""
import hipgemm_b200 as hg

FAKE = 0x10000  # 16-byte aligned, never dereferenced: the checks fail before any CUDA call
INVALID = hg.HGEMM_ERR_INVALID_VALUE


def test_stalled_product_hook_argument_checks():
    def call(x=FAKE, ldx=64, q=FAKE, y=FAKE, m=24, n=32, k=64, group=64):
        return hg.lib().hgemm_debug_stalled_w4(x, ldx, q, FAKE, None, y, m, n, k, group, None)
    assert call(m=16) == call(k=0) == call(k=60) == call(ldx=68) == call(x=FAKE + 2) == INVALID  # another kernel's
    assert call(x=None) == call(q=None) == call(y=None) == call(group=48) == call(ldx=56) == INVALID
    assert call(q=FAKE + 8) == hg.HGEMM_ERR_ALIGNMENT
