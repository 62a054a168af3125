"""The mixture-of-experts router and experts over 4-bit weights against plain 64-bit references
(w4_reference.py, where the bounds are derived)."""
import pytest
import torch

import hipgemm_b200 as hg
from tests import w4_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
TERMS = {torch.bfloat16: 1, torch.float32: 3}


def _gen(*seed):
    return torch.Generator().manual_seed(sum(int(s) * m for s, m in zip(seed, (1, 1009, 100003, 7919, 31))))


# ---- router ----------------------------------------------------------------------------------------


def _route_reference(x, router, top_k, renormalize):
    logits = x.double() @ router.double().T
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top_k]
    p = torch.softmax(logits, 1).gather(1, ids)
    return ids.int(), p / p.sum(1, keepdim=True) if renormalize else p, logits


@pytest.mark.parametrize("t,d,e,top_k", [(1, 64, 8, 2), (1, 1, 1, 1), (3, 100, 7, 7), (5, 33, 40, 4), (4, 2048, 128, 8),
                                         (17, 1000, 65, 16), (64, 512, 256, 8), (2, 40, 1024, 16), (130, 72, 33, 3)])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_route(cuda_device, t, d, e, top_k, renormalize, dtype):
    gen = _gen(t, d, e)
    x = torch.randn(t, d, generator=gen).to(dtype)
    router = (torch.randn(e, d, generator=gen) / d ** 0.5).to(dtype)
    ids, weights = hg.moe_route(x.cuda(), router.cuda(), top_k, renormalize=renormalize)
    want_ids, want, logits = _route_reference(x, router, top_k, renormalize)
    # Sums of 8 products in fp32 (8 additions, half a step each), the rest in 64 bits.
    off = 8 * 2.0 ** -24 * (x.double().abs() @ router.double().abs().T)
    picked = logits.gather(1, ids.cpu().long())
    near = (picked - logits.gather(1, want_ids.long())).abs() <= 2 * off.amax(1, keepdim=True)
    assert bool(near.all()), "an expert was chosen whose logit is not among the largest"
    for row in ids.cpu().tolist():
        assert len(set(row)) == top_k and all(0 <= i < e for i in row)
    # exp of a difference rounded to fp32 (2^-24 of at most 60), expf (2 steps of 2^-23), a sum over E / 32 + 5
    # additions and a division, with each of the two probabilities in it.
    rel = 2 * off.amax(1, keepdim=True) + 2 * (60 * 2.0 ** -24 + 2 * 2.0 ** -23 + (e / 32 + 8 + top_k) * 2.0 ** -24)
    p = torch.softmax(logits, 1).gather(1, ids.cpu().long())
    p = p / p.sum(1, keepdim=True) if renormalize else p
    assert bool(((weights.cpu().double() - p).abs() <= rel * p + 1e-30).all())
    assert bool((want > 0).all())


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_route_ties_go_to_the_lowest_index(cuda_device, dtype):
    gen = _gen(1)
    half = torch.randint(-4, 5, (40, 64), generator=gen).to(dtype)
    x = torch.randint(-4, 5, (9, 64), generator=gen).to(dtype)  # small whole numbers: sums are exact
    router = torch.cat([half, half, half[:5]])
    for top_k in (1, 4, 16):
        ids, weights = hg.moe_route(x.cuda(), router.cuda(), top_k)
        want_ids, want, _ = _route_reference(x, router, top_k, True)
        assert torch.equal(ids.cpu(), want_ids)
    ids, weights = hg.moe_route(torch.zeros_like(x).cuda(), router.cuda(), 3)
    assert torch.equal(ids.cpu(), torch.arange(3).int().expand(9, 3))
    assert torch.allclose(weights.cpu(), torch.full((9, 3), 1 / 3), rtol=1e-6)


def test_route_strides_and_nan(cuda_device):
    gen = _gen(2)
    router = torch.randn(20, 37, generator=gen)
    x = torch.randn(6, 37, generator=gen)
    buf = torch.full((6, 50), float("nan")).cuda()
    buf[:, 1:38] = x.cuda()
    ids, weights = hg.moe_route(buf[:, 1:38], router.cuda(), 5)
    assert torch.equal(ids.cpu(), _route_reference(x, router, 5, True)[0])
    # A NaN expert comes after all numbers; the token's probabilities are NaN, other tokens' are not.
    x[2, 3] = float("nan")
    ids, weights = hg.moe_route(x.cuda(), router.cuda(), 5)
    assert torch.equal(ids[2].cpu(), torch.arange(5).int()) and bool(weights[2].isnan().all())
    assert not bool(weights[[0, 1, 3, 4, 5]].isnan().any())
    assert hg.moe_route(x[:0].cuda(), router.cuda(), 2)[0].shape == (0, 2)


# ---- experts -----------------------------------------------------------------------------------------


def _stack(gen, shape, group, zero_point):
    codes, scales, zeros = ref.random_weight(gen, shape, group, zero_point)
    cuda = [None if t is None else t.cuda() for t in (codes, scales, zeros)]
    return hg.w4_pack(*cuda, group=group), ref.values(codes, scales, zeros, group)


def _layer(gen, e, d, f, group, zero_point, down_group=None, down_zero=None):
    parts = [_stack(gen, s, g, z) for s, g, z in [((e, f, d), group, zero_point), ((e, f, d), group, zero_point),
                                                  ((e, d, f), down_group or group, zero_point if down_zero is None else down_zero)]]
    return [p[0] for p in parts], [p[1] for p in parts]


def _tokens(gen, t, e, d, top_k, dtype):
    x = torch.randn(t, d, generator=gen).to(dtype)
    ids = torch.stack([torch.randperm(e, generator=gen)[:top_k] for _ in range(t)]).int()
    return x, ids, torch.softmax(torch.randn(t, top_k, generator=gen), 1)


def _check(x, ids, weights, packed, dense, **kw):
    got = hg.w4_moe(x.cuda(), ids.cuda(), weights.cuda(), *packed, **kw)
    assert got.shape == x.shape and got.dtype == x.dtype
    ref.assert_close(got, *ref.experts(x, ids, weights, *dense, TERMS[x.dtype]), x.dtype)
    return got


@pytest.mark.parametrize("t,e,top_k,d,f", [(1, 8, 2, 64, 64), (1, 1, 1, 1, 1), (2, 5, 5, 100, 33), (9, 4, 2, 72, 200),
                                           (3, 64, 8, 256, 80), (33, 3, 2, 130, 47), (64, 2, 1, 65, 16), (5, 17, 3, 520, 713),
                                           (20, 32, 16, 48, 40)])
@pytest.mark.parametrize("group,zero_point", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_experts(cuda_device, t, e, top_k, d, f, group, zero_point, dtype):
    gen = _gen(t, e, d, f, group)
    packed, dense = _layer(gen, e, d, f, group, zero_point)
    _check(*_tokens(gen, t, e, d, top_k, dtype), packed, dense)


def test_experts_of_other_groups_in_down(cuda_device):
    gen = _gen(11)
    for down_group, down_zero in [(32, False), (128, True), (64, True)]:
        packed, dense = _layer(gen, 6, 96, 80, 64, False, down_group, down_zero)
        _check(*_tokens(gen, 4, 6, 96, 2, torch.bfloat16), packed, dense)


def test_experts_more_tokens_than_one_launch(cuda_device):
    """Beyond 64 tokens, or 512 pairs, and all tokens at one expert."""
    gen = _gen(12)
    packed, dense = _layer(gen, 20, 64, 48, 32, True)
    for t, top_k in [(65, 2), (70, 8), (40, 16), (150, 1)]:
        x, ids, weights = _tokens(gen, t, 20, 64, top_k, torch.bfloat16)
        _check(x, ids, weights, packed, dense)
    x, ids, weights = _tokens(gen, 64, 20, 64, 2, torch.float32)
    ids[:, 0], ids[:, 1] = 7, 19
    _check(x, ids, weights, packed, dense)


def test_experts_invalid_and_repeated_ids(cuda_device):
    """Ids outside [0, E) add nothing, whatever their weight; an id twice counts with both weights."""
    gen = _gen(13)
    packed, dense = _layer(gen, 6, 80, 72, 32, False)
    x, ids, weights = _tokens(gen, 9, 6, 80, 4, torch.float32)
    ids[0] = -1
    ids[1] = torch.tensor([6, 2, -5, 2 ** 31 - 1])
    ids[2] = 3
    ids[3] = torch.tensor([1, 5, 1, 5])
    ids[4] = torch.tensor([0, -2 ** 31, 0, 6])
    got = _check(x, ids, weights, packed, dense)
    assert bool((got[0] == 0).all())
    # Weights and rows that do not count may hold anything.
    weights[0] = float("nan")
    x[0] = float("nan")
    again = hg.w4_moe(x.cuda(), ids.cuda(), weights.cuda(), *packed)
    assert torch.equal(again, got)
    ids[:] = -1
    assert bool((hg.w4_moe(x.cuda(), ids.cuda(), weights.cuda(), *packed) == 0).all())


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_experts_strides_guards_and_workspace(cuda_device, dtype):
    gen = _gen(14)
    t, e, top_k, d, f = 5, 6, 3, 72, 50
    packed, dense = _layer(gen, e, d, f, 32, True)
    x, ids, weights = _tokens(gen, t, e, d, top_k, dtype)
    for pad, at in [(8, 0), (5, 3)]:
        buf = torch.full((at + (t + 1) * (d + pad),), float("nan"), dtype=dtype).cuda()
        rows = buf[at:at + t * (d + pad)].view(t, d + pad)[:, :d]
        rows.copy_(x)
        out = torch.full((t + 2, d), -3.0, dtype=dtype).cuda()
        need = hg.lib().hgemm_w4_moe_workspace_bytes(t, top_k, d, f)
        ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8).cuda()  # NaN patterns
        got = hg.w4_moe(rows, ids.cuda(), weights.cuda(), *packed, out=out[1:-1], workspace=ws[:need])
        ref.assert_close(got, *ref.experts(x, ids, weights, *dense, TERMS[dtype]), dtype)
        assert bool((out[0] == -3).all()) and bool((out[-1] == -3).all()) and bool((ws[need:] == 0xFF).all())


def test_experts_infinity_stays_in_its_token(cuda_device):
    gen = _gen(15)
    packed, _ = _layer(gen, 4, 64, 50, 32, True)
    x, ids, weights = _tokens(gen, 6, 4, 64, 2, torch.bfloat16)
    clean = hg.w4_moe(x.cuda(), ids.cuda(), weights.cuda(), *packed)
    x[3, 5] = float("inf")
    got = hg.w4_moe(x.cuda(), ids.cuda(), weights.cuda(), *packed)
    keep = [0, 1, 2, 4, 5]
    assert torch.equal(got[keep], clean[keep]) and not bool(got[3].isfinite().all())


def test_experts_bits_depend_on_the_inputs_alone(cuda_device):
    """Repeated calls, two streams at once with a workspace each, and two graphs replayed in turn."""
    gen = _gen(16)
    packed, _ = _layer(gen, 16, 512, 256, 64, False)
    a = [v.cuda() for v in _tokens(gen, 24, 16, 512, 4, torch.bfloat16)]
    b = [v.cuda() for v in _tokens(gen, 3, 16, 512, 4, torch.bfloat16)]
    first = [hg.w4_moe(*v, *packed) for v in (a, b)]
    for _ in range(5):
        assert torch.equal(hg.w4_moe(*a, *packed), first[0]) and torch.equal(hg.w4_moe(*b, *packed), first[1])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = [[hg.w4_moe(*v, *packed, stream=s) for v, s in zip((a, b), streams)] for _ in range(10)]
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for pair in outs:
        assert torch.equal(pair[0], first[0]) and torch.equal(pair[1], first[1])
    graphs, held = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g, v in zip(graphs, (a, b)):
        with torch.cuda.graph(g):
            held.append(hg.w4_moe(*v, *packed))
    for _ in range(3):
        for h in held:
            h.zero_()
        for g in graphs:
            g.replay()
        assert torch.equal(held[0], first[0]) and torch.equal(held[1], first[1])


def test_a_layer_from_quantiser_to_output(cuda_device):
    """The operators as they are used together: weights quantised on the device, a projection, the
    router, the experts, in a graph that is replayed with other tokens."""
    gen = _gen(17)
    t, e, top_k, d, f = 4, 8, 2, 256, 192
    proj = hg.quantize_w4((torch.randn(d, d, generator=gen) / d ** 0.5).cuda(), group=64)
    gate, up = (hg.quantize_w4((torch.randn(e, f, d, generator=gen) / d ** 0.5).cuda(), group=32, zero_point=True) for _ in range(2))
    down = hg.quantize_w4((torch.randn(e, d, f, generator=gen) / f ** 0.5).cuda(), group=128)
    router = (torch.randn(e, d, generator=gen) / d ** 0.5).cuda()
    x = torch.empty(t, d).cuda()

    def layer():
        y = hg.w4_gemm_tn(x, proj)
        ids, weights = hg.moe_route(y, router, top_k)
        return y, ids, weights, hg.w4_moe(y, ids, weights, gate, up, down)

    x.copy_(torch.randn(t, d, generator=gen))
    layer()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = layer()
    dense = [torch.stack([ref.lookup(w, i) for i in range(e)]) for w in (gate, up, down)]
    for _ in range(3):
        x.copy_(torch.randn(t, d, generator=gen))
        graph.replay()
        y, ids, weights, out = (o.cpu() for o in outs)
        ref.assert_close(y, *ref.linear(x.cpu(), ref.lookup(proj), 3), torch.float32)
        want_ids, want, _ = _route_reference(y, router.cpu(), top_k, True)
        assert torch.equal(ids, want_ids) and torch.allclose(weights.double(), want, rtol=1e-5)
        ref.assert_close(out, *ref.experts(y, ids, weights, *dense, 3), torch.float32)


def test_wrapper_refusals(cuda_device):
    gen = _gen(18)
    (gate, up, down), _ = _layer(gen, 4, 64, 32, 32, False)
    x, ids, weights = (v.cuda() for v in _tokens(gen, 3, 4, 64, 2, torch.float32))
    call = hg.w4_moe
    with pytest.raises(ValueError, match="stack"):
        call(x, ids, weights, gate._replace(q=gate.q[0], scales=gate.scales[0]), up, down)
    with pytest.raises(ValueError, match="gate and up must be"):
        call(x, ids, weights, gate, up, gate)
    with pytest.raises(ValueError, match="ids"):
        call(x, ids.long(), weights, gate, up, down)
    with pytest.raises(ValueError, match="weights"):
        call(x, ids, weights[:, :1], gate, up, down)
    with pytest.raises(ValueError, match="down.q"):
        call(x, ids, weights, gate, up, down._replace(q=down.q[:2]))
    with pytest.raises(ValueError, match="out"):
        call(x, ids, weights, gate, up, down, out=torch.empty(3, 64, dtype=torch.bfloat16).cuda())
    with pytest.raises(hg.HgemmError) as err:
        call(x, ids, weights, gate, up, down, workspace=torch.empty(16, dtype=torch.uint8).cuda())
    assert err.value.code == hg.HGEMM_ERR_INVALID_VALUE
    with pytest.raises(hg.HgemmError) as err:
        hg.moe_route(x, torch.zeros(1100, 64).cuda(), 2)
    assert err.value.code == hg.HGEMM_ERR_UNSUPPORTED
    with pytest.raises(hg.HgemmError) as err:
        hg.moe_route(x, torch.zeros(4, 64).cuda(), 5)
    assert err.value.code == hg.HGEMM_ERR_INVALID_VALUE
    with pytest.raises(ValueError, match="router"):
        hg.moe_route(x, torch.zeros(4, 64, dtype=torch.bfloat16).cuda(), 2)
    with pytest.raises(ValueError, match="D mismatch"):
        hg.moe_route(x, torch.zeros(4, 63).cuda(), 2)
