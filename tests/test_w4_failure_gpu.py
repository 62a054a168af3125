"""The failure path of the 4-bit product on the tensor cores, without a fault.  hgemm_debug_stalled_w4 never
reports the first step of x as copied, so that every bounded wait of the kernel's roles expires after its limit
(about 2 s).  The kernel records a role-coded status, drains, frees tensor memory and returns; the context stays
usable: an ordinary product right afterwards is correct and leaves the status clear."""
import time

import pytest
import torch

import hipgemm_b200 as hg
from tests import w4_reference as ref

pytestmark = pytest.mark.gpu

# role << 8 | site: flush (sums ready), unpacking and x copy (stage free), MMA (stage full, accumulator free).
WAIT_SITES = {0x0401, 0x0501, 0x0601, 0x0701, 0x0703}


# One CTA a row group, and clusters that split K; 32 and 64 columns.
@pytest.mark.parametrize("m,n,k,group", [(24, 200, 512, 64), (24, 200, 4096, 32), (64, 200, 4096, 128)])
def test_bounded_waits_expire_and_the_context_survives(cuda_device, m, n, k, group):
    gen = torch.Generator().manual_seed(m + k)
    codes, scales, _ = ref.random_weight(gen, (n, k), group, False)
    w = hg.w4_pack(codes.cuda(), scales.cuda(), group=group)
    x = torch.randn(m, k, generator=gen).bfloat16()
    xd, y = x.cuda(), torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    want, off = ref.linear(x, ref.values(codes, scales, None, group), 1)
    hg.device_status()  # clears any earlier word
    ref.assert_close(hg.w4_gemm_tn(xd, w), want, off, torch.bfloat16)
    torch.cuda.synchronize()
    began = time.perf_counter()
    rc = hg.lib().hgemm_debug_stalled_w4(xd.data_ptr(), k, w.q.data_ptr(), w.scales.data_ptr(), None, y.data_ptr(), m, n, k, group,
                                         torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    elapsed = time.perf_counter() - began
    assert rc == hg.HGEMM_OK
    status = hg.device_status()  # read and cleared
    assert status in WAIT_SITES, hex(status)
    assert 1.0 < elapsed < 60.0, elapsed
    ref.assert_close(hg.w4_gemm_tn(xd, w), want, off, torch.bfloat16)
    assert hg.device_status() == 0
