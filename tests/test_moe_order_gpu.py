"""The order in which the router gives experts whose logits are close."""
import pytest
import torch

import hipgemm_b200 as hg

pytestmark = pytest.mark.gpu

# Sixteen products are summed in fp32 (16 additions, half a step of 2^-23 each), the rest in 64 bits; a little for
# what a rounding adds to the next one's operand.
OFF = 16.1 * 2.0 ** -24


def _near_rows(gen, e, d):
    """A token and rows that are orthogonal to it but for a common part and fp32's rounding: logits near 1."""
    x = torch.randn(1, d, generator=gen).double()
    z = torch.randn(e, d, generator=gen).double()
    z = z - (z @ x.T) / (x @ x.T) * x + x / (x @ x.T)
    return x.float(), z.float()


@pytest.mark.parametrize("t", [1, 16, 20])
@pytest.mark.parametrize("d,e,top_k", [(1000, 64, 8), (4096, 256, 16), (130, 33, 5)])
@pytest.mark.parametrize("spread", [0.0, 2.0 ** -22, 2.0 ** -18, 2.0 ** -10])
def test_logits_that_differ_by_a_few_steps(cuda_device, t, d, e, top_k, spread):
    """`spread`: what the logits of neighbours lie apart, of the sum of their products without signs."""
    gen = torch.Generator().manual_seed(d + e)
    x, router = _near_rows(gen, e, d)
    size = float((x.double().abs() @ router.double().abs().T).mean())
    steps = torch.randperm(e, generator=gen).double() * spread * size
    router = (router.double() + steps.view(-1, 1) * x.double() / (x.double() @ x.double().T)).float()
    x = x.expand(t, d) * torch.exp2(torch.arange(t).float() % 5).view(-1, 1)
    logits = x.double() @ router.double().T
    off = OFF * (x.double().abs() @ router.double().abs().T)
    ids, weights = hg.moe_route(x.cuda(), router.cuda(), top_k, renormalize=False)
    ids = ids.cpu().long()
    best, order = torch.sort(logits, dim=1, descending=True, stable=True)
    picked, bound = logits.gather(1, ids), 2 * off.amax(1, keepdim=True)
    assert bool(((picked - best[:, :top_k]).abs() <= bound).all())
    assert all(len(set(row)) == top_k for row in ids.tolist())
    # Where a rank is further than that from both neighbours, it is the expert's.
    gaps = best[:, :top_k] - best[:, 1:top_k + 1]
    before = torch.cat([torch.full((t, 1), torch.inf, dtype=torch.float64), gaps[:, :-1]], 1)
    alone = (gaps > bound) & (before > bound)
    assert torch.equal(ids[alone], order[:, :top_k][alone])
    assert spread < 2.0 ** -12 or bool(alone.any())
    # Each probability against its logit's: off by exp of the logits' errors and a few roundings of fp32, each of
    # them, below fp32's normal numbers, of half of 2^-149 (expf: two such steps; the division: one), whatever the
    # probability is: logits here lie up to hundreds apart.
    p = torch.softmax(logits, 1).gather(1, ids)
    assert bool(((weights.cpu().double() - p).abs() <= p * (torch.expm1(bound) + (e / 32 + 40) * 2.0 ** -23) + 3 * 2.0 ** -149).all())


@pytest.mark.parametrize("t", [1, 20])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_equal_rows_among_near_ones_keep_their_order(cuda_device, t, dtype):
    gen = torch.Generator().manual_seed(t)
    x, half = _near_rows(gen, 50, 777)
    router = torch.cat([half, half.flip(0), half]).to(dtype)  # rows i, 99 - i and 100 + i are equal
    ids, _ = hg.moe_route(x.expand(t, 777).to(dtype).cuda(), router.cuda(), 16)
    for row in ids.cpu().tolist():
        for r in range(0, 15, 3):
            i = row[r]
            assert i < 50 and row[r + 1:r + 3] == [99 - i, 100 + i]
        assert row[15] < 50
