"""CPU checks of the 4-bit weight operators: sizes, the blocked layout, refusals before any launch."""
import ctypes

import pytest
import torch

import hipgemm_b200 as hg
from tests import w4_reference as ref

FAKE = 0x10000  # 16-byte aligned, never dereferenced: the checks fail before any CUDA call
INVALID, ALIGN, UNSUPPORTED = hg.HGEMM_ERR_INVALID_VALUE, hg.HGEMM_ERR_ALIGNMENT, hg.HGEMM_ERR_UNSUPPORTED


def test_buffer_sizes():
    L = hg.lib()
    for n, k in [(1, 1), (16, 64), (17, 65), (5120, 7168), (28672, 8192)]:
        assert L.hgemm_w4_q_bytes(n, k) == -(-n // 16) * -(-k // 64) * 512
        for group in (32, 64, 128):
            assert L.hgemm_w4_scales(n, k, group) == -(-n // 16) * -(-k // group) * 16
    assert L.hgemm_w4_q_bytes(0, 8) == L.hgemm_w4_q_bytes(8, 0) == L.hgemm_w4_scales(8, 8, 16) == 0
    # Sizes beyond 32 bits.
    assert L.hgemm_w4_q_bytes(1 << 20, 1 << 20) == 1 << 39
    assert L.hgemm_w4_moe_workspace_bytes(1, 8, 33, 1000) == 8 * (48 + 1008) * 4
    # At most 64 tokens or 512 pairs are held at a time.
    assert L.hgemm_w4_moe_workspace_bytes(1000, 8, 32, 16) == 512 * 48 * 4
    assert L.hgemm_w4_moe_workspace_bytes(1000, 3, 32, 16) == 64 * 3 * 48 * 4
    assert L.hgemm_w4_moe_workspace_bytes(0, 8, 32, 16) == L.hgemm_w4_moe_workspace_bytes(4, 17, 32, 16) == 0
    assert L.hgemm_w4_moe_workspace_bytes(4, 2, 0, 16) == L.hgemm_w4_moe_workspace_bytes(4, 2, 16, 0) == 0


@pytest.mark.parametrize("lead,n,k,group", [((), 1, 1, 32), ((), 16, 64, 64), ((), 37, 130, 128), ((3,), 20, 97, 32)])
@pytest.mark.parametrize("zero_point", [False, True])
def test_pack_puts_codes_where_the_header_says(lead, n, k, group, zero_point):
    gen = torch.Generator().manual_seed(n + k)
    codes, scales, zeros = ref.random_weight(gen, (*lead, n, k), group, zero_point)
    w = hg.w4_pack(codes, scales, zeros, group=group)
    assert w.q.numel() == (lead[0] if lead else 1) * hg.lib().hgemm_w4_q_bytes(n, k)
    assert w.scales.numel() == (lead[0] if lead else 1) * hg.lib().hgemm_w4_scales(n, k, group)
    assert w.experts == (lead[0] if lead else None)
    want = ref.values(codes, scales, zeros, group)
    for e in range(lead[0]) if lead else [None]:
        assert torch.equal(ref.lookup(w, e), want if e is None else want[e])


def test_pack_refusals():
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 1)
    with pytest.raises(ValueError, match="group"):
        hg.w4_pack(codes, scales, group=16)
    with pytest.raises(ValueError, match="uint8"):
        hg.w4_pack(codes.int(), scales, group=64)
    with pytest.raises(ValueError, match="scales"):
        hg.w4_pack(codes, torch.ones(4, 2), group=64)
    with pytest.raises(ValueError, match="0..15"):
        hg.w4_pack(codes + 16, scales, group=64)
    with pytest.raises(ValueError, match="zeros"):
        hg.w4_pack(codes, scales, torch.zeros(4, 1), group=64)
    with pytest.raises(ValueError, match="0..15"):
        hg.w4_pack(codes, scales, torch.full((4, 1), 16, dtype=torch.uint8), group=64)


@pytest.mark.parametrize("args,code", [
    ((FAKE, 0, -1, 8, 8, 32, FAKE, FAKE, None, None), INVALID),
    ((FAKE, 0, 1, -8, 8, 32, FAKE, FAKE, None, None), INVALID),
    ((FAKE, 0, 1, 8, 8, 48, FAKE, FAKE, None, None), INVALID),
    ((FAKE, 2, 1, 8, 8, 32, FAKE, FAKE, None, None), INVALID),
    ((None, 0, 1, 8, 8, 32, FAKE, FAKE, None, None), INVALID),
    ((FAKE, 0, 1, 8, 8, 32, None, FAKE, None, None), INVALID),
    ((FAKE, 0, 1, 8, 8, 32, FAKE, None, None, None), INVALID),
    ((FAKE + 2, 0, 1, 8, 8, 32, FAKE, FAKE, None, None), ALIGN),
    ((FAKE + 1, 1, 1, 8, 8, 32, FAKE, FAKE, None, None), ALIGN),
    ((FAKE, 0, 1, 8, 8, 32, FAKE + 8, FAKE, None, None), ALIGN),
    ((FAKE, 0, 1, 8, 8, 32, FAKE, FAKE + 2, None, None), ALIGN),
    ((FAKE, 0, 1, 8, 8, 32, FAKE, FAKE, FAKE + 1, None), ALIGN),
    ((None, 0, 0, 8, 8, 32, None, None, None, None), hg.HGEMM_OK),
    ((None, 0, 1, 0, 8, 32, None, None, None, None), hg.HGEMM_OK),
    ((None, 0, 1, 8, 0, 32, None, None, None, None), hg.HGEMM_OK),
])
def test_quantizer_argument_checks(args, code):
    assert hg.lib().hgemm_quantize_w4(*args) == code
    w, dt, count, n, k, group, q, s, z, stream = args
    assert hg.lib().hgemm_dequantize_w4(q, s, z, count, n, k, group, w, dt, stream) == code


@pytest.mark.parametrize("change,code", [
    (dict(M=-1), INVALID), (dict(N=-1), INVALID), (dict(K=-1), INVALID), (dict(group=16), INVALID), (dict(dt=3), INVALID),
    (dict(ldx=63), INVALID), (dict(x=None), INVALID), (dict(q=None), INVALID), (dict(s=None), INVALID), (dict(y=None), INVALID),
    (dict(x=FAKE + 1), ALIGN), (dict(y=FAKE + 1), ALIGN), (dict(q=FAKE + 4), ALIGN), (dict(s=FAKE + 2), ALIGN),
    (dict(z=FAKE + 1), ALIGN), (dict(M=0, x=None, y=None), hg.HGEMM_OK), (dict(N=0, q=None), hg.HGEMM_OK),
])
def test_linear_argument_checks(change, code):
    a = dict(x=FAKE, dt=1, ldx=64, q=FAKE, s=FAKE, z=None, y=FAKE, M=4, N=32, K=64, group=64) | change
    assert hg.lib().hgemm_w4_gemm_tn(a["x"], a["dt"], a["ldx"], a["q"], a["s"], a["z"], a["y"], a["M"], a["N"], a["K"],
                                     a["group"], None) == code


@pytest.mark.parametrize("change,code", [
    (dict(T=-1), INVALID), (dict(D=-1), INVALID), (dict(E=0), INVALID), (dict(k=0), INVALID), (dict(k=9), INVALID),
    (dict(dt=2), INVALID), (dict(E=1025), UNSUPPORTED), (dict(E=64, k=17), UNSUPPORTED), (dict(ldx=63), INVALID),
    (dict(x=None), INVALID), (dict(r=None), INVALID), (dict(ids=None), INVALID), (dict(w=None), INVALID),
    (dict(x=FAKE + 1), ALIGN), (dict(r=FAKE + 1), ALIGN), (dict(ids=FAKE + 2), ALIGN), (dict(w=FAKE + 2), ALIGN),
    (dict(T=0, x=None, ids=None), hg.HGEMM_OK),
])
def test_route_argument_checks(change, code):
    a = dict(x=FAKE, dt=1, ldx=64, r=FAKE, T=4, D=64, E=8, k=2, ids=FAKE, w=FAKE) | change
    assert hg.lib().hgemm_moe_route(a["x"], a["dt"], a["ldx"], a["r"], a["T"], a["D"], a["E"], a["k"], 1, a["ids"], a["w"],
                                    None) == code


class _Weight(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("zeros", ctypes.c_void_p), ("group", ctypes.c_int)]


@pytest.mark.parametrize("change,code", [
    (dict(T=-1), INVALID), (dict(D=-1), INVALID), (dict(F=-1), INVALID), (dict(E=0), INVALID), (dict(k=0), INVALID),
    (dict(dt=2), INVALID), (dict(E=1025), UNSUPPORTED), (dict(k=17), UNSUPPORTED), (dict(ldx=63), INVALID),
    (dict(x=None), INVALID), (dict(ids=None), INVALID), (dict(w=None), INVALID), (dict(out=None), INVALID),
    (dict(ws=None), INVALID), (dict(ws_bytes=100), INVALID), (dict(ws=FAKE + 8), ALIGN), (dict(x=FAKE + 1), ALIGN),
    (dict(out=FAKE + 1), ALIGN), (dict(ids=FAKE + 2), ALIGN), (dict(gate=(FAKE, FAKE, None, 16)), INVALID),
    (dict(up=(FAKE, FAKE, None, 32)), UNSUPPORTED), (dict(up=(FAKE, FAKE, FAKE, 64)), UNSUPPORTED),
    (dict(down=(None, FAKE, None, 64)), INVALID), (dict(down=(FAKE + 8, FAKE, None, 64)), ALIGN),
    (dict(T=0, x=None), hg.HGEMM_OK), (dict(D=0, x=None), hg.HGEMM_OK),
])
def test_moe_argument_checks(change, code):
    w = (FAKE, FAKE, None, 64)
    a = dict(x=FAKE, dt=1, ldx=64, ids=FAKE, w=FAKE, T=4, k=2, E=8, D=64, F=32, gate=w, up=w, down=w, out=FAKE, ws=FAKE,
             ws_bytes=1 << 20) | change
    structs = [_Weight(*a[n]) for n in ("gate", "up", "down")]
    assert hg.lib().hgemm_w4_moe(a["x"], a["dt"], a["ldx"], a["ids"], a["w"], a["T"], a["k"], a["E"], a["D"], a["F"],
                                 *map(ctypes.addressof, structs), a["out"], a["ws"], a["ws_bytes"], None) == code


def test_no_cpu_path():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    w = hg.w4_pack(torch.zeros(32, 64, dtype=torch.uint8), torch.ones(32, 1), group=64)
    e = hg.w4_pack(torch.zeros(4, 32, 64, dtype=torch.uint8), torch.ones(4, 32, 1), group=64)
    with pytest.raises(ValueError, match="CUDA"):
        hg.quantize_w4(x)
    with pytest.raises(ValueError, match="CUDA"):
        hg.dequantize_w4(w)
    with pytest.raises(ValueError, match="CUDA"):
        hg.w4_gemm_tn(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        hg.moe_route(x, x, 1)
    with pytest.raises(ValueError, match="CUDA"):
        hg.w4_moe(x, torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, 1), e, e, e)


@pytest.mark.parametrize("zero_point", [False, True])
def test_reference_quantizer_is_near_its_input(zero_point):
    """The reference itself: no element is off by more than half a step, and the scale's rounding."""
    w = torch.randn(33, 200, generator=torch.Generator().manual_seed(1))
    codes, s, z = ref.quantize(w, 64, zero_point)
    step = s.double().repeat_interleave(64, -1)[:, :200]
    # The scale is rounded by 2^-8 at most, 15 steps (or 7) long: the ends may be clamped by that much.
    assert bool(((ref.values(codes, s, z, 64) - w.double()).abs() <= step * (0.5 + 15 * 2.0 ** -8 + (0.5 if zero_point else 0))).all())
