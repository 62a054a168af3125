"""What the 4-bit weight operators keep of their operands: cases whose fp32 sums are exact or nearly
so, so that a value held in fewer bits on the way shows, against 64-bit values."""
import pytest
import torch

import hipgemm_b200 as hg
from tests import w4_reference as ref

pytestmark = pytest.mark.gpu


def _gen(*seed):
    return torch.Generator().manual_seed(sum(int(s) * m for s, m in zip(seed, (1, 1009, 100003, 7919, 31))))


def _pack(codes, scale, group, zero_point):
    """Codes around 8, one scale; zero_point: the same weight with zero points of 8."""
    groups = -(-codes.shape[-1] // group)
    scales = torch.full((*codes.shape[:-1], groups), scale)
    zeros = torch.full(scales.shape, 8, dtype=torch.uint8).cuda() if zero_point else None
    return hg.w4_pack(codes.cuda(), scales.cuda(), zeros, group=group), (codes.double() - 8) * scale


@pytest.mark.parametrize("t", [1, 9, 20])
@pytest.mark.parametrize("group,zero_point", [(32, False), (32, True), (64, False), (128, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_experts_keep_the_product_between_the_matrices(cuda_device, t, group, zero_point, dtype):
    """Pairs of hidden units that differ by about 2^-11 of themselves; each output is the difference of one pair."""
    gen = _gen(t, group)
    d, f = 64, 64
    gate, up, down = (torch.full(s, 8, dtype=torch.uint8) for s in ((1, f, d), (1, f, d), (1, d, f)))
    for p in range(f // 2):
        gate[0, 2 * p] = gate[0, 2 * p + 1] = torch.randint(4, 13, (d,), generator=gen, dtype=torch.uint8)
        up[0, 2 * p] = torch.randint(10, 16, (d,), generator=gen, dtype=torch.uint8)
        up[0, 2 * p + 1] = up[0, 2 * p]
        up[0, 2 * p + 1, 0] -= 1
    for n in range(d):
        down[0, n, 2 * (n % 32)], down[0, n, 2 * (n % 32) + 1] = 9, 7
    # x: multiples of 2^-4 below 1, the first element 2^-4: sums over gate and up are whole multiples of 2^-4 below
    # 2^9, exact in fp32 in any order.
    x = torch.randint(4, 16, (t, d), generator=gen).double() / 16
    x[:, 0] = 1 / 16
    (wg, g), (wu, u), (wd, _) = (_pack(c, s, group, zero_point) for c, s in ((gate, 2.0 ** -6), (up, 1.0), (down, 1.0)))
    a, b = x @ g[0].T, x @ u[0].T
    h = a * torch.sigmoid(a) * b
    want = (h[:, 0::2] - h[:, 1::2]).repeat(1, 2)
    size = (h[:, 0::2].abs() + h[:, 1::2].abs()).repeat(1, 2)
    assert bool((want.abs() <= size * 2.0 ** -10).all())  # both are 0 where the gate is
    # Both units of a pair have the same silu, off by a few roundings (2^-20 of the difference); each product is
    # rounded once (2^-24); the sum over down has at most 6 terms that are not 0.
    off = want.abs() * 2.0 ** -20 + size * (2.0 ** -24 + 6 * ref.ADD)
    got = hg.w4_moe(x.to(dtype).cuda(), torch.zeros(t, 1, dtype=torch.int32).cuda(), torch.ones(t, 1).cuda(), wg, wu, wd)
    ref.assert_close(got, want, off, dtype)


# ---- rows held in registers as whole numbers ------------------------------------------------------
#
# One or two rows, and any fp32 rows, of matrices that are large enough.

ROWS = [(1, torch.bfloat16), (2, torch.bfloat16), (1, torch.float32), (2, torch.float32), (3, torch.float32),
        (8, torch.float32), (11, torch.float32)]
ROW_IDS = [f"{m}-{str(t).split('.')[1]}" for m, t in ROWS]
TERMS = {torch.bfloat16: 1, torch.float32: 3}


@pytest.mark.parametrize("m,dtype", ROWS, ids=ROW_IDS)
@pytest.mark.parametrize("n,k,group,zero_point", [(5120, 1024, 128, False), (7100, 1100, 32, True), (2500, 4000, 64, True),
                                                  (4096, 2113, 128, True)])
def test_an_element_keeps_its_value_beside_any_other(cuda_device, m, n, k, group, zero_point, dtype):
    """Row r of W is 1 at column r % K and 0 elsewhere: y has the elements of x, whose magnitudes are far apart."""
    gen = _gen(m, n, k, group)
    row = torch.arange(n)
    zero = torch.randint(0, 15, (n, 1), generator=gen) if zero_point else torch.full((n, 1), 8)
    codes = zero.expand(n, k).clone()
    codes[row, row % k] += 1
    groups = -(-k // group)
    w = hg.w4_pack(codes.to(torch.uint8).cuda(), torch.ones(n, groups).cuda(),
                   zero.expand(n, groups).to(torch.uint8).contiguous().cuda() if zero_point else None, group=group)
    for lo, hi in [(0, 1), (-8, 8), (-24, 2), (-40, 20), (-50, 60)]:
        x = (torch.randn(m, k, generator=gen) * torch.exp2(torch.randint(lo, hi, (m, k), generator=gen).float())).to(dtype)
        got = hg.w4_gemm_tn(x.cuda(), w).cpu()
        want = x[:, row % k]
        if dtype == torch.bfloat16:
            assert torch.equal(got, want)
        else:
            # An element is held to 2^-20 of itself; five planes, put together in four additions.
            assert bool(((got.double() - want.double()).abs() <= want.double().abs() * (2.0 ** -20 + 4 * 2.0 ** -24)).all())


@pytest.mark.parametrize("m,dtype", ROWS, ids=ROW_IDS)
@pytest.mark.parametrize("zero_point", [False, True])
@pytest.mark.parametrize("size", [1.0e4, 1.0e5, 2.0 ** 20, 2.0 ** 40])
def test_an_outlier_that_no_weight_meets_costs_nothing(cuda_device, m, dtype, zero_point, size):
    gen = _gen(m, int(size) % 1000, 5)
    n, k, group = 5120, 2048, 64
    codes, scales, zeros = ref.random_weight(gen, (n, k), group, zero_point)
    at = torch.randint(0, k, (9,), generator=gen)
    codes[:, at] = 8 if zeros is None else zeros[:, at // group]
    w = hg.w4_pack(codes.cuda(), scales.cuda(), None if zeros is None else zeros.cuda(), group=group)
    values = ref.values(codes, scales, zeros, group)
    x = torch.randn(m, k, generator=gen)
    x[:, at] = size * torch.randn(m, 9, generator=gen)
    x = x.to(dtype)
    got = hg.w4_gemm_tn(x.cuda(), w)
    want, off = ref.linear(x, values, TERMS[dtype])
    ref.assert_close(got, want, off, dtype)
    # The same row among others, which another kernel takes for bf16: each is off by its bound at most.
    more = hg.w4_gemm_tn(torch.cat([x, x[:1], x[:1]]).cuda(), w)
    ref.assert_close(more[:m], want, off, dtype)
    bound = 2 * (off + ref.half_step(dtype) * (want.abs() + off))
    assert bool(((more[:m].cpu().double() - got.cpu().double()).abs() <= bound).all())


@pytest.mark.parametrize("m,dtype", ROWS, ids=ROW_IDS)
@pytest.mark.parametrize("n,k,group,zero_point", [(5120, 1024, 128, False), (7100, 1100, 32, True), (300, 20000, 64, False),
                                                  (300, 17000, 32, True)])
def test_weights_that_meet_the_small_elements_alone(cuda_device, m, n, k, group, zero_point, dtype):
    gen = _gen(m, n, k, 9)
    codes, scales, zeros = ref.random_weight(gen, (n, k), group, zero_point)
    x = (torch.randn(m, k, generator=gen) * torch.exp2(torch.randint(-30, 1, (1, k), generator=gen).float())).to(dtype)
    large = x.abs().amax(0) > 2.0 ** -20
    none = torch.full((n, k), 8, dtype=torch.uint8) if zeros is None else zeros.repeat_interleave(group, 1)[:, :k]
    codes = torch.where(large, none, codes)
    w = hg.w4_pack(codes.cuda(), scales.cuda(), None if zeros is None else zeros.cuda(), group=group)
    ref.assert_close(hg.w4_gemm_tn(x.cuda(), w), *ref.linear(x, ref.values(codes, scales, zeros, group), TERMS[dtype]), dtype)


# ---- range ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("m,dtype", [*ROWS, (5, torch.bfloat16), (12, torch.bfloat16), (40, torch.bfloat16), (70, torch.bfloat16)])
@pytest.mark.parametrize("n,k,group", [(5120, 1024, 128), (50, 256, 64), (4097, 1100, 32)])
def test_elements_up_to_the_documented_range(cuda_device, m, dtype, n, k, group):
    """Every code 15 steps from its zero point and every element just below 2^117, against a scale that brings the result
    back: no sum on the way is an infinity."""
    sign = (torch.arange(k) // group % 2 * 2 - 1).float()  # groups alternate: their scaled sums nearly cancel
    codes = torch.full((n, k), 15, dtype=torch.uint8)
    scales = torch.full((n, -(-k // group)), 2.0 ** -20)
    zeros = torch.zeros(n, -(-k // group), dtype=torch.uint8)
    w = hg.w4_pack(codes.cuda(), scales.cuda(), zeros.cuda(), group=group)
    x = (sign * 2.0 ** 117 * (1 - 2.0 ** -8)).expand(m, k).to(dtype)
    got = hg.w4_gemm_tn(x.cuda(), w)
    assert bool(got.isfinite().all())
    ref.assert_close(got, *ref.linear(x, ref.values(codes, scales, zeros, group), TERMS[dtype]), dtype)
    # Beyond it an infinity is one that the products' true sum leads to, never a NaN or a wrong number.
    got = hg.w4_gemm_tn((x.abs().double() * 4).to(dtype).cuda(), w).cpu()
    want = float(x.abs()[0, 0]) * 4 * 15 * 2.0 ** -20 * k
    assert bool(((got == float("inf")) | ((got.double() - want).abs() <= want * 2.0 ** -7)).all())


# ---- sums of fp32 rows ------------------------------------------------------------------------------


@pytest.mark.parametrize("m", [1, 3, 8, 20])
@pytest.mark.parametrize("group,zero_point", [(32, True), (64, False), (64, True), (128, False), (128, True)])
def test_one_group_of_fp32_is_rounded_twice(cuda_device, m, group, zero_point):
    """One group of elements in [1, 2) and steps of one sign: their first terms (8 bits, 2^-7 apart) times the steps add
    up to less than 2^12, exact in fp32 in any order."""
    gen = _gen(m, group)
    n, k = 64, group
    codes = torch.randint(8, 16, (n, k), generator=gen, dtype=torch.uint8)
    scales = torch.rand(n, 1, generator=gen).bfloat16() + 0.5
    zeros = torch.randint(0, 8, (n, 1), generator=gen, dtype=torch.uint8) if zero_point else None
    w = hg.w4_pack(codes.cuda(), scales.cuda(), None if zeros is None else zeros.cuda(), group=group)
    x = torch.rand(m, k, generator=gen) + 1
    want = x.double() @ ref.values(codes, scales, zeros, group).T
    # The other terms are below 2^-7 of x, in group / 8 additions; then two sums are added, and scaled: half a step each.
    bound = want * (2 * 2.0 ** -24 + group // 8 * ref.ADD * 2.0 ** -7)
    got = hg.w4_gemm_tn(x.cuda(), w).cpu().double()
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())
