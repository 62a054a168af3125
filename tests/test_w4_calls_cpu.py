"""Calls of the 4-bit weight operators that are refused before anything is launched."""
import types

import pytest

import hipgemm_b200 as hg
from hipgemm_b200 import w4

FAKE = 0x10000  # 16-byte aligned, never dereferenced: the checks fail before any CUDA call
INVALID = hg.HGEMM_ERR_INVALID_VALUE


def test_stalled_product_hook_argument_checks():
    def call(x=FAKE, ldx=64, q=FAKE, y=FAKE, m=24, n=32, k=64, group=64):
        return hg.lib().hgemm_debug_stalled_w4(x, ldx, q, FAKE, None, y, m, n, k, group, None)
    assert call(m=16) == call(k=0) == call(k=60) == call(ldx=68) == call(x=FAKE + 2) == INVALID  # another kernel's
    assert call(x=None) == call(q=None) == call(y=None) == call(group=48) == call(ldx=56) == INVALID
    assert call(q=FAKE + 8) == hg.HGEMM_ERR_ALIGNMENT


def test_a_stream_of_another_device_is_refused():
    """Every operator enters this context before it allocates or launches anything."""
    with pytest.raises(ValueError, match="stream is on cuda:1, the tensors are on cuda:0"):
        w4._context(0, types.SimpleNamespace(device_index=1, device_type=1, stream_id=0))
