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
