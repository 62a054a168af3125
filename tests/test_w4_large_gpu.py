"""The 4-bit weight kernels that only large calls reach: experts whose row groups are split over two warps
instead of four, and quantiser and inverse on matrices of several waves of CTAs, whose loops reuse
their shared memory."""
import pytest
import torch

import hipgemm_b200 as hg
from tests import w4_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
TERMS = {torch.bfloat16: 1, torch.float32: 3}
HALF = 2.0 ** -24  # half a step of fp32


def _lookup(w, e):
    """Expert e of a stack in 64 bits, on its device, each code found by its place in the header's layout."""
    dev = w.q.device
    row, col = torch.arange(w.n, device=dev)[:, None], torch.arange(w.k, device=dev)[None, :]
    g, rr = row % 8, row // 8 % 2
    jg, t, jk, rk, half = col // 32 % 2, col // 8 % 4, col // 4 % 2, col // 2 % 2, col % 2
    byte = w.q[e][row // 16, col // 64, 16 * (4 * g + t) + 4 * (2 * jg + jk) + 2 * half + rk].long()
    at = (row // 16, col // w.group, g, rr)
    zero = 8 if w.zeros is None else w.zeros[e][at].long()
    return (((byte >> (4 * rr)) & 15) - zero).double() * w.scales[e][at].double()


def _stack(gen, e, n, k, group, zero_point):
    rb, kb, groups = -(-n // 16), -(-k // 64), -(-k // group)
    q = torch.randint(0, 256, (e, rb, kb, 512), dtype=torch.uint8, device="cuda", generator=gen)
    scales = (torch.rand(e, rb, groups, 8, 2, device="cuda", generator=gen) + 0.5) / (4.6 * k ** 0.5)
    zeros = torch.randint(0, 16, scales.shape, dtype=torch.uint8, device="cuda", generator=gen) if zero_point else None
    return hg.W4Weight(q, scales.bfloat16(), zeros, n, k, group)


def _linear(x, w, terms, group):
    """x @ w^T in 64 bits and the bound of its fp32 evaluation: a group's instructions (16 K and one term each), the
    groups, and the sums of up to 8 warps."""
    additions = group // 16 * terms + -(-w.shape[1] // group) + 8
    return x @ w.T, additions * ref.ADD * (x.abs() @ w.abs().T)


def _token(x, ids, weights, gate, up, down, terms):
    """One token's experts in 64 bits, and the bound."""
    out, off = 0.0, 0.0
    for e, weight in zip(ids.tolist(), weights.tolist()):
        g, dg = _linear(x, _lookup(gate, e), terms, gate.group)
        u, du = _linear(x, _lookup(up, e), terms, up.group)
        a = g * torch.sigmoid(g)
        # silu' is below 1.1; silu and the product round a few times.
        dh = 1.1 * dg * u.abs() + (a.abs() + 1.1 * dg) * du + (a * u).abs() * 16 * HALF
        wd = _lookup(down, e)
        y, dy = _linear(a * u, wd, 3, down.group)
        out = out + weight * y
        off = off + abs(weight) * (dh @ wd.abs().T + dy * (1 + 2.0 ** -10))
    return out, off * (1 + 2.0 ** -10) + (2 * len(ids) + 2) * ref.ADD * (out.abs() + off)


# t, experts, top_k, d, f: more than 2 (gate and up) and 4 (down) groups of rows an SM of 148.  The second has more than 8
# tokens an expert, which for bf16 takes two tiles of columns.
@pytest.mark.parametrize("t,e,top_k,d,f", [(32, 64, 6, 1300, 1000), (64, 16, 3, 4700, 1210)])
@pytest.mark.parametrize("group,zero_point", [(32, True), (64, False), (128, True), (128, False)])
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_experts_with_rows_split_over_two_warps(cuda_device, t, e, top_k, d, f, group, zero_point, dtype):
    sms = torch.cuda.get_device_properties(cuda_device).multi_processor_count
    assert e * -(-f // 64) >= 2 * sms and e * -(-d // 128) >= 4 * sms, "the case does not reach these kernels"
    gen = torch.Generator(device="cuda").manual_seed(t + group)
    gate, up = (_stack(gen, e, f, d, group, zero_point) for _ in range(2))
    down = _stack(gen, e, d, f, group, not zero_point)
    x = torch.randn(t, d, device="cuda", generator=gen).to(dtype)
    ids = torch.stack([torch.randperm(e, device="cuda", generator=gen)[:top_k] for _ in range(t)]).int()
    ids[1, 0] = -1
    weights = torch.softmax(torch.randn(t, top_k, device="cuda", generator=gen), 1)
    got = hg.w4_moe(x, ids, weights, gate, up, down)
    for i in (0, 1, t // 2, t - 1):
        keep = ids[i] >= 0
        want, off = _token(x[i].double(), ids[i][keep], weights[i][keep], gate, up, down, TERMS[dtype])
        ref.assert_close(got[i], want.cpu(), off.cpu(), dtype)
    assert torch.equal(hg.w4_moe(x, ids, weights, gate, up, down), got)


@pytest.mark.parametrize("n,k,dtype", [(4999, 5115, torch.float32), (6001, 4097, torch.bfloat16), (5000, 8192, torch.bfloat16),
                                       (7001, 4104, torch.float32)])
@pytest.mark.parametrize("group,zero_point", [(32, True), (64, False), (128, True)])
def test_quantize_matrices_of_several_waves(cuda_device, n, k, dtype, group, zero_point):
    gen = torch.Generator(device="cuda").manual_seed(n + group)
    w = torch.randn(n, k, device="cuda", generator=gen).to(dtype)
    groups = -(-k // group)
    x = torch.nn.functional.pad(w.double(), (0, groups * group - k)).view(n, groups, group)
    lo, hi = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
    s = ((hi - lo) / 15 if zero_point else torch.maximum(hi, -lo) / 7).float().bfloat16()
    s = torch.where(s == 0, torch.ones_like(s), s)
    z = (-lo / s.double()).round().clamp(0, 15) if zero_point else torch.full_like(lo, 8.0)
    codes = ((x / s.double()[..., None]).round() + z[..., None]).clamp(0, 15)
    want = ((codes - z[..., None]) * s.double()[..., None]).view(n, -1)[:, :k]
    got = hg.quantize_w4(w, group=group, zero_point=zero_point)
    packed = hg.w4_pack(codes.view(n, -1)[:, :k].to(torch.uint8), s, z.to(torch.uint8) if zero_point else None, group=group)
    assert torch.equal(got.scales, packed.scales)
    assert not zero_point or torch.equal(got.zeros, packed.zeros)
    assert torch.equal(_lookup(hg.W4Weight(*(None if v is None else v[None] for v in got[:3]), n, k, group), 0), want)
    for out in TYPES.values():
        assert torch.equal(hg.dequantize_w4(got, dtype=out), want.float().to(out))
