"""Calls of the 4-bit weight operators that are refused before anything is launched."""
import ctypes
import types

import pytest
import torch

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


# x has 4 rows of 64 bf16, 80 apart; y 4 rows of 16: 128 bytes.  (Outputs that are not refused: test_w4_calls_gpu.py.)
@pytest.mark.parametrize("at", [0, 2, 126, 128, -126, 160, 3 * 160, 3 * 160 + 126])
def test_product_into_its_own_operand_is_refused(at):
    """CTAs would read what others have written."""
    assert hg.lib().hgemm_w4_gemm_tn(FAKE, 1, 80, FAKE * 16, FAKE * 32, None, FAKE + at, 4, 16, 64, 64, None) == INVALID


def test_product_into_a_gap_that_is_too_small_is_refused():
    for at, n in [(128, 9), (130, 8), (126, 8)]:  # the gap is 32 bytes, y two rows of n
        assert hg.lib().hgemm_w4_gemm_tn(FAKE, 1, 80, FAKE * 16, FAKE * 32, None, FAKE + at, 2, n, 64, 64, None) == INVALID


class _Weight(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("zeros", ctypes.c_void_p), ("group", ctypes.c_int)]


@pytest.mark.parametrize("t,at", [(65, 2), (65, -2), (100, 64 * 128), (100, -64 * 128)])
def test_experts_of_several_launches_into_their_own_operand_are_refused(t, at):
    """Rows of x that a later launch reads would have been written by an earlier one."""
    weight = _Weight(FAKE * 16, FAKE * 32, None, 64)
    w, x = ctypes.addressof(weight), FAKE * 4
    assert hg.lib().hgemm_w4_moe(x, 1, 64, FAKE * 48, FAKE * 49, t, 2, 8, 64, 32, w, w, w, x + at, FAKE * 50, 1 << 24,
                                 None) == INVALID


def test_operands_that_require_a_gradient_are_refused():
    """There is no backward pass, and a detached result would look like a constant."""
    w = hg.w4_pack(torch.zeros(32, 64, dtype=torch.uint8), torch.ones(32, 1), group=64)
    e = hg.w4_pack(torch.zeros(4, 32, 64, dtype=torch.uint8), torch.ones(4, 32, 1), group=64)
    x, ids, weights = torch.zeros(2, 64), torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, 1)
    xg, wg = x.clone().requires_grad_(), weights.clone().requires_grad_()
    calls = {"x": [lambda: hg.w4_gemm_tn(xg, w), lambda: hg.moe_route(xg, x, 1), lambda: hg.w4_moe(xg, ids, weights, e, e, e)],
             "router": [lambda: hg.moe_route(x, xg, 1)], "weights": [lambda: hg.w4_moe(x, ids, wg, e, e, e)]}
    for name, some in calls.items():
        for call in some:
            with pytest.raises(ValueError, match=f"{name} requires a gradient"):
                call()
            for off in (torch.no_grad(), torch.inference_mode()):
                with off, pytest.raises(ValueError, match="CUDA"):  # the next check: there is no GPU tensor here
                    call()


class _Fake:
    """What the wrapper's checks look at of a CUDA tensor."""

    def __init__(self, shape, dtype, stride=None):
        self.shape, self.dtype, self._stride = torch.Size(shape), dtype, stride
        self.dim, self.numel = lambda: len(shape), lambda: self.shape.numel()
        self.stride, self.get_device, self.is_contiguous = lambda: stride, lambda: 0, lambda: True


def _fake_weight(n, k, group=64, lead=(), q=None, scales=None, zeros=None):
    rb = -(-n // 16)
    return hg.W4Weight(_Fake(q or (*lead, rb, -(-k // 64), 512), torch.uint8),
                       _Fake(scales or (*lead, rb, -(-k // group), 8, 2), torch.bfloat16),
                       None if zeros is None else _Fake(zeros, torch.uint8), n, k, group)


def test_buffers_of_another_shape_with_as_many_elements_are_refused():
    w4._check_weight("w", _fake_weight(40, 200), 0, None)
    w4._check_weight("w", _fake_weight(40, 200, lead=(5,), zeros=(5, 3, 4, 8, 2)), 0, 5)
    for part, weight, count in [("q", _fake_weight(40, 200, q=(4, 3, 512)), None), ("q", _fake_weight(40, 200, q=(3, 512, 4)), None),
                                ("q", _fake_weight(40, 200, q=(1, 3, 4, 512)), None), ("scales", _fake_weight(40, 200, scales=(4, 3, 8, 2)), None),
                                ("scales", _fake_weight(40, 200, scales=(3, 4, 2, 8)), None),
                                ("zeros", _fake_weight(40, 200, zeros=(4, 3, 8, 2)), None),
                                ("q", _fake_weight(40, 200, lead=(5,), q=(3, 5, 4, 512)), 5),
                                ("scales", _fake_weight(40, 200, lead=(5,), scales=(15, 4, 8, 2)), 5)]:
        with pytest.raises(ValueError, match=rf"w\.{part} must be"):
            w4._check_weight("w", weight, 0, count)


def test_sizes_that_do_not_fit_an_int_are_refused():
    """They would be cut off on the way to the library: 2^32 + 64 columns would be 64."""
    for n, k in [(40, 2 ** 32 + 64), (2 ** 32 + 40, 64), (40, 2 ** 31), (-16, 64)]:
        with pytest.raises(ValueError, match="2\\^31"):
            w4._check_weight("w", _fake_weight(n, k), 0, None)
    for shape in [(2 ** 31, 64), (2, 2 ** 32 + 64)]:
        with pytest.raises(ValueError, match="2\\^31"):
            w4._check_rows("x", _Fake(shape, torch.bfloat16, (shape[1], 1)))
    assert w4._check_rows("x", _Fake((2 ** 31 - 1, 64), torch.bfloat16, (64, 1))) == (64, 1, 0)
