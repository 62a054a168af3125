"""Calls of the 4-bit weight operators that their documentation allows, or refuses, on tensors of the GPU."""
import pytest
import torch

import hipgemm_b200 as hg
from tests import w4_reference as ref

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _weight(gen, shape, group, zero_point=False):
    codes, scales, zeros = ref.random_weight(gen, shape, group, zero_point)
    cuda = [None if t is None else t.cuda() for t in (codes, scales, zeros)]
    return hg.w4_pack(*cuda, group=group), ref.values(codes, scales, zeros, group)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_product_beside_its_operand(cuda_device, dtype):
    """Into the gap between two rows of x, right before its first row and right behind its last."""
    gen = _gen(1)
    w, values = _weight(gen, (8, 64), 64)
    x = torch.randn(2, 64, generator=gen).to(dtype)
    for base, at in ((0, 64), (16, 0), (0, 144)):
        buf = torch.zeros(160, dtype=dtype, device="cuda")
        rows = buf[base:base + 144].as_strided((2, 64), (80, 1), base)
        rows.copy_(x)
        out = buf[at:at + 16].view(2, 8)
        ref.assert_close(hg.w4_gemm_tn(rows, w, out=out), *ref.linear(x, values, 3), dtype)
        assert torch.equal(rows.cpu(), x)
    square, _ = _weight(gen, (64, 64), 64)
    y = torch.randn(3, 64, generator=gen).to(dtype).cuda()
    with pytest.raises(hg.HgemmError) as err:
        hg.w4_gemm_tn(y, square, out=y)
    assert err.value.code == hg.HGEMM_ERR_INVALID_VALUE


def test_experts_into_their_operand(cuda_device):
    """out may be x itself, of any number of launches; of one launch it may lie anywhere."""
    gen = _gen(2)
    e, d, f, top_k = 6, 64, 48, 2
    (gate, g), (up, u), (down, dn) = (_weight(gen, s, 32) for s in ((e, f, d), (e, f, d), (e, d, f)))
    for t in (5, 64, 65, 200):
        x = torch.randn(t, d, generator=gen).bfloat16()
        ids = torch.stack([torch.randperm(e, generator=gen)[:top_k] for _ in range(t)]).int().cuda()
        weights = torch.softmax(torch.randn(t, top_k, generator=gen), 1).cuda()
        want = hg.w4_moe(x.cuda(), ids, weights, gate, up, down)
        y = x.cuda()
        assert hg.w4_moe(y, ids, weights, gate, up, down, out=y) is y and torch.equal(y, want)
        wide = torch.zeros(t, d + 8, dtype=torch.bfloat16, device="cuda")
        wide[:, :d] = x.cuda()
        out = wide.view(-1)[:t * d].view(t, d)
        assert torch.equal(hg.w4_moe(wide[:, :d], ids, weights, gate, up, down, out=out), want)
        buf = torch.zeros((t + 1) * d, dtype=torch.bfloat16, device="cuda")
        buf[:t * d] = x.cuda().view(-1)
        call = lambda: hg.w4_moe(buf[:t * d].view(t, d), ids, weights, gate, up, down, out=buf[d:].view(t, d))  # noqa: E731
        if t <= 64:
            assert torch.equal(call(), want)
        else:
            with pytest.raises(hg.HgemmError):
                call()
    want = ref.experts(x[:3], ids[:3].cpu(), weights[:3].cpu(), g, u, dn, 1)
    ref.assert_close(y[:3], *want, torch.bfloat16)
