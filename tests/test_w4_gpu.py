"""The 4-bit quantiser, its inverse and the product of a few rows with 4-bit weights, against plain
64-bit references (w4_reference.py, where the bounds are derived)."""
import pytest
import torch

import hipgemm_b200 as hg
from tests import w4_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
TERMS = {torch.bfloat16: 1, torch.float32: 3}


def _gen(*seed):
    return torch.Generator().manual_seed(sum(int(s) * m for s, m in zip(seed, (1, 1009, 100003, 7919, 31))))


def _weight(gen, shape, group, zero_point):
    codes, scales, zeros = ref.random_weight(gen, shape, group, zero_point)
    cuda = [None if t is None else t.cuda() for t in (codes, scales, zeros)]
    return hg.w4_pack(*cuda, group=group), ref.values(codes, scales, zeros, group)


# ---- quantiser and inverse --------------------------------------------------------------------


@pytest.mark.parametrize("n,k", [(1, 1), (1, 64), (16, 128), (17, 65), (5, 130), (40, 200), (129, 1032), (300, 4096)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zero_point", [False, True])
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_quantize_is_exact(cuda_device, n, k, group, zero_point, dtype):
    gen = _gen(n, k, group)
    w = (torch.randn(n, k, generator=gen) * torch.exp2(torch.randint(-30, 30, (n, 1), generator=gen).float())).to(dtype)
    codes, s, z = ref.quantize(w, group, zero_point)
    want = hg.w4_pack(codes, s, z, group=group)
    got = hg.quantize_w4(w.cuda(), group=group, zero_point=zero_point)
    assert (got.n, got.k, got.group) == (n, k, group)
    assert torch.equal(ref.lookup(got), ref.lookup(want))
    assert torch.equal(got.scales.cpu(), want.scales)
    if zero_point:
        assert torch.equal(got.zeros.cpu(), want.zeros)
    # Exact products in fp32, rounded once.
    for out in TYPES.values():
        assert torch.equal(hg.dequantize_w4(got, dtype=out).cpu(), ref.lookup(want).float().to(out))


@pytest.mark.parametrize("zero_point", [False, True])
def test_quantize_special_values(cuda_device, zero_point):
    w = torch.zeros(20, 128)
    w[1] = torch.linspace(-1e-42, 1e-42, 128)  # subnormal scale
    w[2] = torch.linspace(-3.4e38, 3.4e38, 128)
    w[3] = torch.randn(128, generator=_gen(1))
    w[3, 5] = float("nan")
    w[4, 7] = float("inf")
    w[4, 8] = 2.0
    w[5, 7] = -float("inf")
    w[6] = 1e-45
    w[7] = float("nan")
    w[8] = torch.arange(128) * 0.5 * 2.0 ** -4  # ties between two codes
    w[9] = -w[8]
    w[10] = torch.linspace(1.0, 2.0, 128)  # one sign only
    w[11] = 1e-39 * torch.randn(128, generator=_gen(2))
    w[12, :64] = 3.5
    w[12, 64:] = torch.arange(64) * 0.25
    w[13] = 2.0 ** -59 * torch.randn(128, generator=_gen(3))
    w[14] = 2.0 ** -62 * torch.randn(128, generator=_gen(4))
    w[15] = 2.0 ** 110 * torch.randn(128, generator=_gen(5))
    for group in (32, 64, 128):
        codes, s, z = ref.quantize(w, group, zero_point)
        got = hg.quantize_w4(w.cuda(), group=group, zero_point=zero_point)
        want = hg.w4_pack(codes, s, z, group=group)
        assert torch.equal(got.scales.cpu(), want.scales)
        assert zero_point is False or torch.equal(got.zeros.cpu(), want.zeros)
        assert torch.equal(ref.lookup(got), ref.lookup(want))


def test_quantize_stack_and_padding(cuda_device):
    """A stack is its matrices one by one; padding codes stand for 0, padding rows have scale 1."""
    w = torch.randn(5, 37, 100, generator=_gen(3)).cuda()
    for zero_point in (False, True):
        stack = hg.quantize_w4(w, group=32, zero_point=zero_point)
        for e in range(5):
            one = hg.quantize_w4(w[e], group=32, zero_point=zero_point)
            assert torch.equal(stack.q[e], one.q) and torch.equal(stack.scales[e], one.scales)
        assert torch.equal(hg.dequantize_w4(stack, torch.float32)[2], hg.dequantize_w4(one._replace(
            q=stack.q[2], scales=stack.scales[2], zeros=stack.zeros[2] if zero_point else None), torch.float32))
        padded = stack._replace(n=48, k=128)
        values = ref.lookup(padded, 1)
        assert bool((values[37:] == 0).all()) and bool((values[:, 100:] == 0).all())
        rows = padded.scales[1, 2].float().cpu()  # rows 32..47: [group][g][rr], row 32 + g + 8 rr
        assert bool((rows[:, 5:, 0] == 1).all()) and bool((rows[:, :, 1] == 1).all())


def test_quantize_reads_and_writes_nothing_else(cuda_device):
    """Unaligned input, and guard bytes around every output."""
    n, k, group = 35, 71, 64
    base = torch.full((n * k + 3,), float("nan")).cuda()
    w = torch.randn(n, k, generator=_gen(9))
    base[1:1 + n * k] = w.flatten().cuda()
    L, stream = hg.lib(), torch.cuda.current_stream().cuda_stream
    q_bytes, scales = L.hgemm_w4_q_bytes(n, k), L.hgemm_w4_scales(n, k, group)
    q = torch.full((q_bytes + 32,), 0xA5, dtype=torch.uint8).cuda()
    s = torch.full((scales + 4,), 77.0, dtype=torch.bfloat16).cuda()
    z = torch.full((scales + 4,), 0xA5, dtype=torch.uint8).cuda()
    assert L.hgemm_quantize_w4(base.data_ptr() + 4, 0, 1, n, k, group, q.data_ptr() + 16, s.data_ptr() + 4, z.data_ptr() + 2,
                               stream) == 0
    out = torch.full((n * k + 2,), -7.0).cuda()
    assert L.hgemm_dequantize_w4(q.data_ptr() + 16, s.data_ptr() + 4, z.data_ptr() + 2, 1, n, k, group, out.data_ptr() + 4, 0,
                                 stream) == 0
    torch.cuda.synchronize()
    codes, sc, zp = ref.quantize(w, group, True)
    assert torch.equal(out[1:-1].cpu().view(n, k).double(), ref.values(codes, sc, zp, group))
    assert float(out[0]) == float(out[-1]) == -7.0
    assert bool((q[:16] == 0xA5).all()) and bool((q[16 + q_bytes:] == 0xA5).all())
    assert bool((s[:2] == 77).all()) and bool((s[2 + scales:] == 77).all())
    assert bool((z[:2] == 0xA5).all()) and bool((z[2 + scales:] == 0xA5).all())


# ---- the product ---------------------------------------------------------------------------------


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65])
@pytest.mark.parametrize("n,k", [(48, 256), (17, 1), (1, 100), (33, 1000), (250, 2049)])
@pytest.mark.parametrize("group,zero_point", [(32, False), (64, True), (128, False)])
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_linear(cuda_device, m, n, k, group, zero_point, dtype):
    gen = _gen(m, n, k, group)
    w, values = _weight(gen, (n, k), group, zero_point)
    x = torch.randn(m, k, generator=gen).to(dtype)
    got = hg.w4_gemm_tn(x.cuda(), w)
    assert got.dtype == dtype and got.shape == (m, n)
    ref.assert_close(got, *ref.linear(x, values, TERMS[dtype]), dtype)


@pytest.mark.parametrize("group,zero_point", [(32, True), (128, True), (64, False)])
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 7168, 2048), (3, 5111, 1160), (1, 64, 8192), (16, 100, 28672), (24, 4096, 512)])
def test_linear_larger(cuda_device, m, n, k, group, zero_point, dtype):
    gen = _gen(m, n, k, 5)
    w, values = _weight(gen, (n, k), group, zero_point)
    x = torch.randn(m, k, generator=gen).to(dtype)
    ref.assert_close(hg.w4_gemm_tn(x.cuda(), w), *ref.linear(x, values, TERMS[dtype]), dtype)


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_linear_strides_and_guards(cuda_device, dtype):
    """Rows that are strided or start off 16 bytes; what lies between and behind them (NaN) is not
    read, what lies behind the output is left as it was."""
    gen = _gen(4)
    for k, pad, at in [(200, 8, 0), (200, 8, 8), (200, 3, 1), (77, 3, 2), (64, 0, 4), (33, 31, 0)]:
        w, values = _weight(gen, (50, k), 32, True)
        x = torch.randn(5, k, generator=gen).to(dtype)
        buf = torch.full((at + 6 * (k + pad),), float("nan"), dtype=dtype).cuda()
        rows = buf[at:at + 5 * (k + pad)].view(5, k + pad)[:, :k]
        rows.copy_(x)
        buf_out = torch.full((7, 50), -3.0, dtype=dtype).cuda()
        got = hg.w4_gemm_tn(rows, w, out=buf_out[1:6])
        ref.assert_close(got, *ref.linear(x, values, TERMS[dtype]), dtype)
        assert bool((buf_out[0] == -3).all()) and bool((buf_out[6] == -3).all())


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_linear_special_values(cuda_device, dtype):
    """Infinities and NaN reach their own row alone, and large, subnormal and zero elements keep their value."""
    gen = _gen(5)
    w, values = _weight(gen, (40, 96), 32, False)
    values[:, 3] = 0.0
    codes = torch.full((40, 96), 8, dtype=torch.uint8)
    codes[:, 4] = 9  # W[:, 4] = scale, the rest 0
    one = hg.w4_pack(codes.cuda(), torch.full((40, 3), 0.5).cuda(), group=32)
    x = torch.zeros(6, 96)
    x[0, 4] = float("inf")
    x[1, 4] = 3.0e38
    x[2, 4] = float("nan")
    x[3, 4] = -float("inf")
    x[4, 4] = 1.1
    x[5, 4] = 2.0 ** -120 * 1.0078125
    x = x.to(dtype)
    got = hg.w4_gemm_tn(x.cuda(), one).cpu()
    # 0 * inf is NaN, so the rows with an infinity are only defined where no other code meets it: all of them here.
    want = (x[:, 4].float() * 0.5).to(dtype)
    for i in range(6):
        if want[i].isnan():
            assert bool(got[i].isnan().all())
        else:
            assert bool((got[i] == want[i]).all()), (i, got[i, :4], want[i])


def test_linear_empty(cuda_device):
    w, _ = _weight(_gen(6), (40, 96), 32, False)
    assert hg.w4_gemm_tn(torch.empty(0, 96, dtype=torch.bfloat16).cuda(), w).shape == (0, 40)
    no_k = hg.W4Weight(torch.empty(3, 0, 512, dtype=torch.uint8).cuda(), torch.empty(3, 0, 8, 2, dtype=torch.bfloat16).cuda(),
                       None, 40, 0, 32)
    out = torch.full((3, 40), 5.0).cuda()
    assert bool((hg.w4_gemm_tn(torch.empty(3, 0).cuda(), no_k, out=out) == 0).all())
    no_n = hg.quantize_w4(torch.empty(0, 64).cuda(), group=32)
    assert hg.w4_gemm_tn(torch.ones(3, 64).cuda(), no_n).shape == (3, 0)
    assert hg.dequantize_w4(no_n).shape == (0, 64)


def test_linear_bits_depend_on_the_inputs_alone(cuda_device):
    """Repeated calls, another stream, a captured graph and its replays give the same bits; a row's
    result does not depend on the rows beside it within a tile of columns."""
    gen = _gen(7)
    for n, k, m in [(96, 8192, 3), (4096, 1024, 16), (333, 777, 40)]:
        w, _ = _weight(gen, (n, k), 64, True)
        x = torch.randn(m, k, generator=gen).to(torch.bfloat16).cuda()
        first = hg.w4_gemm_tn(x, w)
        for _ in range(5):
            assert torch.equal(hg.w4_gemm_tn(x, w), first)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        other = hg.w4_gemm_tn(x, w, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, first)
        flipped = hg.w4_gemm_tn(x.flip(0).contiguous(), w).flip(0)
        assert torch.equal(flipped, first)
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(first)
        with torch.cuda.graph(graph):
            hg.w4_gemm_tn(x, w, out=out)
        for _ in range(3):
            out.fill_(float("nan"))
            graph.replay()
            assert torch.equal(out, first)


def test_back_to_back_calls_see_each_other(cuda_device):
    """A chain of products without a wait between them: each reads what the one before wrote."""
    gen = _gen(8)
    w, values = _weight(gen, (512, 512), 64, False)
    x = torch.randn(4, 512, generator=gen).cuda()
    y, want = x, x.cpu().double()
    for _ in range(12):
        y = hg.w4_gemm_tn(y, w)
    for _ in range(12):
        want = want @ values.T
    # Each product is off by at most additions(512, 3) * 2^-22 of sums whose absolute values are below
    # sqrt(512) times the result's norm (Cauchy-Schwarz); 12 of them, in the 2-norm.
    assert float((y.cpu() - want).norm() / want.norm()) < 12 * ref.additions(512, 3) * ref.ADD * 512 ** 0.5 * 4


def test_wrapper_refusals(cuda_device):
    w, _ = _weight(_gen(9), (40, 96), 32, False)
    x = torch.zeros(2, 96).cuda()
    with pytest.raises(ValueError, match="K mismatch"):
        hg.w4_gemm_tn(x[:, :64].contiguous(), w)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        hg.w4_gemm_tn(x.half(), w)
    with pytest.raises(ValueError, match="2-D"):
        hg.w4_gemm_tn(x[:, ::2], w)
    with pytest.raises(ValueError, match="2-D"):
        hg.w4_gemm_tn(x[0], w)
    with pytest.raises(ValueError, match="overlapping"):
        hg.w4_gemm_tn(x[:1].expand(3, 96), w)
    with pytest.raises(ValueError, match="CUDA"):
        hg.w4_gemm_tn(x, w._replace(q=w.q.cpu()))
    with pytest.raises(ValueError, match="w.q"):
        hg.w4_gemm_tn(x, w._replace(q=w.q[:2]))
    with pytest.raises(ValueError, match="w.scales"):
        hg.w4_gemm_tn(x, w._replace(scales=w.scales.float()))
    with pytest.raises(ValueError, match="w.zeros"):
        hg.w4_gemm_tn(x, w._replace(zeros=w.scales))
    with pytest.raises(ValueError, match="group"):
        hg.w4_gemm_tn(x, w._replace(group=48))
    with pytest.raises(ValueError, match="out"):
        hg.w4_gemm_tn(x, w, out=torch.empty(2, 40, dtype=torch.bfloat16).cuda())
    with pytest.raises(ValueError, match="out"):
        hg.dequantize_w4(w, out=torch.empty(40, 96).cuda())
    with pytest.raises(ValueError, match="contiguous"):
        hg.quantize_w4(torch.zeros(4, 64).cuda().T)
    with pytest.raises(ValueError, match="group"):
        hg.quantize_w4(torch.zeros(4, 64).cuda(), group=100)
    with pytest.raises(TypeError):
        hg.quantize_w4(torch.zeros(4, 64, dtype=torch.float16).cuda())


# ---- the kernels that small matrices do not reach --------------------------------------------------
#
# One or two rows, and any fp32 rows, of matrices large enough hold x in registers as whole numbers;
# more than 16 bf16 rows go through the 5th-generation tensor cores.


def _planes_off(x, values):
    """What holding x as whole numbers may lose: half of the last place, 2^-21 of a power of two that is at most
    twice the largest of the row (bf16; fp32 2^-28), for every element."""
    last = 2.0 ** -21 if x.dtype == torch.bfloat16 else 2.0 ** -28
    return last * x.double().abs().amax(1, keepdim=True) * values.abs().sum(1)


@pytest.mark.parametrize("m,dtype", [(1, torch.bfloat16), (2, torch.bfloat16), (1, torch.float32), (2, torch.float32),
                                     (3, torch.float32), (8, torch.float32), (11, torch.float32)])
@pytest.mark.parametrize("n,k,group,zero_point", [(5120, 1024, 128, False), (7100, 1100, 32, True), (2500, 4000, 64, True),
                                                  (4096, 2113, 128, True), (300, 20000, 64, False)])
def test_linear_rows_in_registers(cuda_device, m, n, k, group, zero_point, dtype):
    gen = _gen(m, n, k, group, 3)
    w, values = _weight(gen, (n, k), group, zero_point)
    x = torch.randn(m, k, generator=gen).to(dtype)
    y, off = ref.linear(x, values, TERMS[dtype])
    got = hg.w4_gemm_tn(x.cuda(), w)
    ref.assert_close(got, y, off + _planes_off(x, values), dtype)
    assert torch.equal(hg.w4_gemm_tn(x.cuda(), w), got)


@pytest.mark.parametrize("m,dtype", [(1, torch.bfloat16), (2, torch.bfloat16), (2, torch.float32), (5, torch.float32),
                                     (24, torch.bfloat16), (40, torch.bfloat16)])
def test_linear_special_values_in_large_matrices(cuda_device, m, dtype):
    """Rows with infinities, NaN, the largest and the smallest numbers, and outliers, beside ordinary ones."""
    n, k = 5120, 1024
    gen = _gen(m, 77)
    codes, scales, _ = ref.random_weight(gen, (n, k), 64, False)
    codes[codes == 8] = 9  # no weight is 0: infinity times 0 would be NaN
    w, values = hg.w4_pack(codes.cuda(), scales.cuda(), group=64), ref.values(codes, scales, None, 64)
    kinds = [lambda r: r.__setitem__(5, float("inf")), lambda r: r.__setitem__(700, float("nan")),
             lambda r: r.mul_(2.0 ** 118), lambda r: r.mul_(2.0 ** -100), lambda r: r.__setitem__(3, -float("inf")),
             lambda r: r.__setitem__(9, 5000.0), lambda r: r.zero_(), lambda r: None]
    for first in range(len(kinds)):
        x = torch.randn(m, k, generator=gen)
        for i in range(min(m, 2)):
            kinds[(first + i) % len(kinds)](x[-1 - i])
        x = x.to(dtype)
        got = hg.w4_gemm_tn(x.cuda(), w).cpu()
        clean = torch.where(x.isfinite(), x, 0)
        y, off = ref.linear(clean, values, TERMS[dtype])
        for i in range(m):
            bad = x[i][~x[i].isfinite()]
            if bad.numel() == 0:
                ref.assert_close(got[i:i + 1], y[i:i + 1], (off + _planes_off(clean, values))[i:i + 1], dtype)
            elif bool(bad.isnan().any()):
                assert bool(got[i].isnan().all())
            else:
                want = x[i].double()[~x[i].isfinite()] * values[:, ~x[i].isfinite()]  # one infinity
                assert torch.equal(got[i].double(), want[:, 0])


@pytest.mark.parametrize("m", [17, 32, 33, 63, 64, 65, 130])
@pytest.mark.parametrize("n,k", [(128, 64), (1, 8), (100, 1000), (1000, 136), (513, 4104)])
@pytest.mark.parametrize("group,zero_point", [(32, True), (64, False), (128, True)])
def test_linear_many_rows(cuda_device, m, n, k, group, zero_point):
    gen = _gen(m, n, k, group, 9)
    w, values = _weight(gen, (n, k), group, zero_point)
    x = torch.randn(m, k, generator=gen).bfloat16()
    ref.assert_close(hg.w4_gemm_tn(x.cuda(), w), *ref.linear(x, values, 1), torch.bfloat16)
    assert hg.device_status() == 0


def test_linear_many_rows_strides_guards_and_graphs(cuda_device):
    """Rows that are strided (aligned, so that the tensor-core kernel takes them, and not), NaN between and behind
    them, rows of the output behind the last, a captured graph, another stream, and two streams at once."""
    gen = _gen(31)
    n, k = 700, 520
    w, values = _weight(gen, (n, k), 32, True)
    for m, pad, at in [(20, 8, 0), (40, 24, 8), (33, 3, 1), (70, 0, 0)]:
        x = torch.randn(m, k, generator=gen).bfloat16()
        buf = torch.full((at + (m + 1) * (k + pad),), float("nan"), dtype=torch.bfloat16).cuda()
        rows = buf[at:at + m * (k + pad)].view(m, k + pad)[:, :k]
        rows.copy_(x)
        out = torch.full((m + 2, n), -3.0, dtype=torch.bfloat16).cuda()
        first = hg.w4_gemm_tn(rows, w, out=out[1:-1]).clone()
        ref.assert_close(first, *ref.linear(x, values, 1), torch.bfloat16)
        assert bool((out[0] == -3).all()) and bool((out[-1] == -3).all())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            hg.w4_gemm_tn(rows, w, out=out[1:-1])
        for _ in range(3):
            out[1:-1].fill_(float("nan"))
            graph.replay()
            assert torch.equal(out[1:-1], first)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        got = [[hg.w4_gemm_tn(rows, w, stream=s) for s in streams] for _ in range(8)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, first) for pair in got for g in pair)
    assert hg.device_status() == 0


def test_a_call_for_each_kernel_in_a_row(cuda_device):
    """Products of 1, 2, 5, 16 and 48 rows one after the other on one stream, each on the one before's output."""
    gen = _gen(41)
    size = 2048
    w, values = _weight(gen, (size, size), 128, False)
    x = torch.randn(48, size, generator=gen).bfloat16().cuda()
    outs = []
    for m in (48, 16, 5, 2, 1):
        x = hg.w4_gemm_tn(x[:m], w)
        outs.append(x)
    torch.cuda.synchronize()
    for before, got in zip(outs, outs[1:]):
        y = before[:got.shape[0]].cpu()
        want, off = ref.linear(y, values, 1)
        ref.assert_close(got, want, off + _planes_off(y, values), torch.bfloat16)
