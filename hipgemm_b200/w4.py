"""Torch-facing wrappers for 4-bit weights with group scales and the mixture-of-experts layer
over them (a few tokens at a time: decoding).

    w = quantize_w4(W, group=128)              # (N, K) or (E, N, K) -> W4Weight
    y = w4_gemm_tn(x, w)                       # y[M,N] = x[M,K] . W[N,K]^T
    ids, p = moe_route(x, router, top_k=8)     # router: product, softmax, top-k
    y = w4_moe(x, ids, p, gate, up, down)      # the chosen experts' gated products

The buffers' layout is in include/hipgemm_b200.h; the reference (nirw4nna/hipgemm) has no
counterpart.  Every function works on the tensors' device, on `stream` or torch's current one,
and can be captured into a CUDA graph after one call on the device.  Inference only: the products,
the router and the experts refuse operands that require a gradient unless gradients are off.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from ._lib import check
from .gemm import _fn, _get_device, _stream_handle

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_GROUPS = (32, 64, 128)
_MOST = 2 ** 31 - 1  # the C functions' sizes are ints, and ctypes cuts larger ones off without a word


class W4Weight(NamedTuple):
    """A 4-bit weight, or a stack of E of them: blocked codes q ((E,) row blocks, K blocks, 512)
    uint8, scales ((E,) row blocks, groups, 8, 2) bfloat16, zeros (the same shape, uint8) or None,
    and the matrix's n rows, k columns and group size."""
    q: torch.Tensor
    scales: torch.Tensor
    zeros: torch.Tensor | None
    n: int
    k: int
    group: int

    @property
    def experts(self) -> int | None:
        """E of a stack, None for one matrix."""
        return self.q.shape[0] if self.q.dim() == 4 else None


def _dtype_code(name: str, t: torch.Tensor) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    return code


def _check_weight(name: str, w: W4Weight, dev: int, count: int | None) -> None:
    """Types, sizes and place of a weight's buffers; `count` experts, or one matrix (None)."""
    # A few cheap tests in the common case (this wrapper's host time adds to every launch of a small
    # product); anything else takes the detailed ones, which raise the specific error.
    q, s, z, n, k, group = w
    if group in _GROUPS and 0 <= n <= _MOST and 0 <= k <= _MOST:
        rb = (n + 15) // 16
        if count is None:
            blocks, groups = (rb, (k + 63) // 64, 512), (rb, (k + group - 1) // group, 8, 2)
        else:
            blocks, groups = (count, rb, (k + 63) // 64, 512), (count, rb, (k + group - 1) // group, 8, 2)
        if (q.shape == blocks and s.shape == groups and q.dtype is torch.uint8 and s.dtype is torch.bfloat16
                and q.is_contiguous() and s.is_contiguous() and q.get_device() == dev >= 0 and s.get_device() == dev
                and (z is None or (z.shape == groups and z.dtype is torch.uint8 and z.is_contiguous() and z.get_device() == dev))):
            return
    _check_weight_in_detail(name, w, dev, count)


def _check_weight_in_detail(name: str, w: W4Weight, dev: int, count: int | None) -> None:
    q, s, z, n, k, group = w
    if group not in _GROUPS:
        raise ValueError(f"{name}.group must be 32, 64 or 128, got {group}")
    if not 0 <= n <= _MOST or not 0 <= k <= _MOST:
        raise ValueError(f"{name} is {n} x {k}: sizes have to be below 2^31")
    rb, lead = -(-n // 16), () if count is None else (count,)
    shape = (*lead, rb, -(-k // 64), 512)
    if q.dtype != torch.uint8 or q.shape != shape or not q.is_contiguous():
        raise ValueError(f"{name}.q must be a contiguous uint8 tensor of shape {shape}")
    shape = (*lead, rb, -(-k // group), 8, 2)
    if s.dtype != torch.bfloat16 or s.shape != shape or not s.is_contiguous():
        raise ValueError(f"{name}.scales must be a contiguous bfloat16 tensor of shape {shape}")
    if z is not None and (z.dtype != torch.uint8 or z.shape != shape or not z.is_contiguous()):
        raise ValueError(f"{name}.zeros must be a contiguous uint8 tensor of shape {shape}")
    raise ValueError(f"{name} must be on the same CUDA device as the other tensors (there is no CPU path)")


def _check_rows(name: str, x: torch.Tensor) -> tuple[int, int, int]:
    """Row stride (elements), type code and device index of a 2-D fp32 or bf16 CUDA tensor with contiguous rows."""
    dev = x.get_device()
    if dev < 0:
        raise ValueError(f"{name} must be on a CUDA device (there is no CPU path)")
    if x.dim() != 2:
        raise ValueError(f"{name} must be a 2-D tensor with contiguous, non-overlapping rows")
    ld, one = x.stride()
    rows, columns = x.shape
    if rows > _MOST or columns > _MOST:
        raise ValueError(f"{name} is {rows} x {columns}: sizes have to be below 2^31")
    if (columns > 1 and one != 1) or (rows > 1 and ld < columns):
        raise ValueError(f"{name} must be a 2-D tensor with contiguous, non-overlapping rows")
    dt = _DTYPES.get(x.dtype)
    return ld, _dtype_code(name, x) if dt is None else dt, dev


def _check_no_gradient(**tensors: torch.Tensor) -> None:
    """These operators have no backward pass: a result that is cut off from its operands must not look like one
    that is not."""
    if torch.is_grad_enabled():
        for name, t in tensors.items():
            if t.requires_grad:
                raise ValueError(f"{name} requires a gradient, which this operator does not give: detach it, or call under torch.no_grad()")


class _on:
    """Device `dev` and, for torch's allocations, `stream` (the stream that the kernels run on: memory
    freed on another one must not be handed out while it is in use) made current for a call."""

    def __init__(self, dev: int, stream: torch.cuda.Stream | None):
        self.parts = [torch.cuda.device(dev)] if stream is None else [torch.cuda.device(dev), torch.cuda.stream(stream)]

    def __enter__(self):
        for part in self.parts:
            part.__enter__()

    def __exit__(self, *exc):
        for part in reversed(self.parts):
            part.__exit__(*exc)
        return False


class _Nothing:
    def __enter__(self):
        pass

    def __exit__(self, *exc):
        return False


_nothing = _Nothing()


def _context(dev: int, stream: torch.cuda.Stream | None):
    """A context for a call on `dev` and `stream`; none where both are current already."""
    if stream is None:
        if _get_device is not None and _get_device() == dev:
            return _nothing
    elif stream.device_index != dev:
        # The kernel would run there, on pointers into another device's memory.
        raise ValueError(f"stream is on cuda:{stream.device_index}, the tensors are on cuda:{dev}")
    return _on(dev, stream)


def w4_pack(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *, group: int) -> W4Weight:
    """Codes made elsewhere -> the blocked layout, on the codes' device (layout only, any device).
    codes: (N, K) or (E, N, K) uint8, 0..15; scales: (..., N, ceil(K / group)), rounded to
    bfloat16; zeros: the same shape, uint8 0..15, or None (code 8 stands for 0)."""
    if codes.dtype != torch.uint8 or codes.dim() not in (2, 3):
        raise ValueError("codes must be an (N, K) or (E, N, K) uint8 tensor")
    if group not in _GROUPS:
        raise ValueError(f"group must be 32, 64 or 128, got {group}")
    *lead, n, k = codes.shape
    rb, kb, groups = -(-n // 16), -(-k // 64), -(-k // group)
    for name, t in (("scales", scales), ("zeros", zeros)):
        if t is not None and (t.shape != (*lead, n, groups) or t.device != codes.device):
            raise ValueError(f"{name} must have shape {(*lead, n, groups)} and be on the codes' device")
    if zeros is not None and zeros.dtype != torch.uint8:
        raise ValueError("zeros must be uint8")
    for name, t in (("codes", codes), ("zeros", zeros)):
        if t is not None and t.numel() and int(t.max()) > 15:
            raise ValueError(f"{name} must be 0..15")
    r = len(lead)
    c = torch.nn.functional.pad(codes, (0, kb * 64 - k, 0, rb * 16 - n))
    c = c.reshape(*lead, rb, 2, 8, kb, 2, 4, 2, 2, 2)  # rb rr g kb jg t jk rk half
    c = c.permute(*range(r), r, r + 3, r + 2, r + 5, r + 4, r + 6, r + 8, r + 7, r + 1)  # rb kb g t jg jk half rk rr
    q = (c[..., 0] | (c[..., 1] << 4)).reshape(*lead, rb, kb, 512).contiguous()

    def blocked(t, fill):
        t = torch.nn.functional.pad(t, (0, 0, 0, rb * 16 - n), value=fill)
        t = t.reshape(*lead, rb, 2, 8, groups)
        return t.permute(*range(r), r, r + 3, r + 2, r + 1).contiguous()

    return W4Weight(q, blocked(scales.to(torch.bfloat16), 1.0), None if zeros is None else blocked(zeros, 0), n, k, group)


def quantize_w4(w: torch.Tensor, group: int = 128, zero_point: bool = False,
                stream: torch.cuda.Stream | None = None) -> W4Weight:
    """4-bit quantisation on the GPU (hgemm_quantize_w4) of an (N, K) matrix or an (E, N, K) stack,
    fp32 or bf16: one bf16 scale per row and `group` K, and with zero_point one zero point."""
    if not w.is_cuda or not w.is_contiguous() or w.dim() not in (2, 3):
        raise ValueError("w must be a contiguous (N, K) or (E, N, K) CUDA tensor (there is no CPU path)")
    dt = _dtype_code("w", w)
    if group not in _GROUPS:
        raise ValueError(f"group must be 32, 64 or 128, got {group}")
    *lead, n, k = w.shape
    if max(w.shape) > _MOST:
        raise ValueError(f"w is {tuple(w.shape)}: sizes have to be below 2^31")
    rb, dev = -(-n // 16), w.get_device()
    with _context(dev, stream):
        q = w.new_empty((*lead, rb, -(-k // 64), 512), dtype=torch.uint8)
        scales = w.new_empty((*lead, rb, -(-k // group), 8, 2), dtype=torch.bfloat16)
        zeros = w.new_empty(scales.shape, dtype=torch.uint8) if zero_point else None
        rc = _fn("hgemm_quantize_w4")(w.data_ptr(), dt, lead[0] if lead else 1, n, k, group, q.data_ptr(),
                                      scales.data_ptr(), zeros.data_ptr() if zero_point else None,
                                      _stream_handle(stream, dev))
    check(rc, "hgemm_quantize_w4")
    return W4Weight(q, scales, zeros, n, k, group)


def dequantize_w4(w: W4Weight, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
                  stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """The values of a 4-bit weight, (N, K) or (E, N, K): (code - zero) * scale, rounded once."""
    dev, count = w.q.get_device(), w.experts
    if dev < 0:
        raise ValueError("w must be on a CUDA device (there is no CPU path)")
    _check_weight("w", w, dev, count)
    shape = (w.n, w.k) if count is None else (count, w.n, w.k)
    with _context(dev, stream):
        if out is None:
            out = w.q.new_empty(shape, dtype=dtype)
        elif out.shape != shape or out.dtype != dtype or not out.is_contiguous() or out.get_device() != dev:
            raise ValueError(f"out must be a contiguous {dtype} tensor of shape {shape} on w's device")
        rc = _fn("hgemm_dequantize_w4")(w.q.data_ptr(), w.scales.data_ptr(), None if w.zeros is None else w.zeros.data_ptr(),
                                        1 if count is None else count, w.n, w.k, w.group, out.data_ptr(),
                                        _dtype_code("out", out), _stream_handle(stream, dev))
    check(rc, "hgemm_dequantize_w4")
    return out


def w4_gemm_tn(x: torch.Tensor, w: W4Weight, out: torch.Tensor | None = None, *,
               stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """y[M,N] = x[M,K] @ W[N,K]^T for a few rows of x (fp32 or bf16, rows may be strided); y has x's
    type, sums are fp32 (hgemm_w4_gemm_tn).  out may not overlap x.  From about 16 rows of a large W
    on fp8_gemm_tn is faster, from 64 on a bf16 product with dequantize_w4's values."""
    if x.requires_grad:
        _check_no_gradient(x=x)
    ldx, dt, dev = _check_rows("x", x)
    _check_weight("w", w, dev, None)
    m, k = x.shape
    if k != w.k:
        raise ValueError(f"K mismatch: x is {tuple(x.shape)}, w is {w.n} x {w.k}")
    with _context(dev, stream):
        if out is None:
            out = x.new_empty((m, w.n))
        elif out.shape != (m, w.n) or out.dtype != x.dtype or not out.is_contiguous() or out.get_device() != dev:
            raise ValueError("out must be a contiguous (M, N) tensor of x's type on x's device")
        rc = _fn("hgemm_w4_gemm_tn")(x.data_ptr(), dt, ldx, w.q.data_ptr(), w.scales.data_ptr(),
                                     None if w.zeros is None else w.zeros.data_ptr(), out.data_ptr(), m, w.n, k, w.group,
                                     _stream_handle(stream, dev))
    if rc:
        check(rc, "hgemm_w4_gemm_tn")
    return out


def moe_route(x: torch.Tensor, router: torch.Tensor, top_k: int, *, renormalize: bool = True,
              stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The router of a mixture of experts (hgemm_moe_route): softmax(x[T,D] @ router[E,D]^T) and per
    token the top_k largest: ids (T, top_k) int32, largest first, and their probabilities (T,
    top_k) float32, which add up to 1 with renormalize.  E <= 1024, top_k <= 16."""
    if x.requires_grad or router.requires_grad:
        _check_no_gradient(x=x, router=router)
    ldx, dt, dev = _check_rows("x", x)
    if router.dtype != x.dtype or router.dim() != 2 or not router.is_contiguous() or router.get_device() != dev:
        raise ValueError("router must be a contiguous (E, D) tensor of x's type on x's device")
    t, d = x.shape
    e = router.shape[0]
    if top_k > _MOST:
        raise ValueError("top_k has to be below 2^31")
    if router.shape[1] != d:
        raise ValueError(f"D mismatch: x is {tuple(x.shape)}, router is {tuple(router.shape)}")
    with _context(dev, stream):
        ids = x.new_empty((t, max(top_k, 0)), dtype=torch.int32)
        weights = x.new_empty((t, max(top_k, 0)), dtype=torch.float32)
        rc = _fn("hgemm_moe_route")(x.data_ptr(), dt, ldx, router.data_ptr(), t, d, e, top_k, bool(renormalize),
                                    ids.data_ptr(), weights.data_ptr(), _stream_handle(stream, dev))
    if rc:
        check(rc, "hgemm_moe_route")
    return ids, weights


def w4_moe(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, gate: W4Weight, up: W4Weight, down: W4Weight,
           out: torch.Tensor | None = None, *, workspace: torch.Tensor | None = None,
           stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """The experts of a mixture for a few tokens (hgemm_w4_moe), in three kernels:
    out[t] = sum_j weights[t,j] * down_e(silu(gate_e x[t]) * (up_e x[t])), e = ids[t,j].
    x (T, D) fp32 or bf16, ids (T, top_k) int32 and weights (T, top_k) float32 as moe_route gives
    them (ids outside [0, E) add nothing), gate and up (E, F, D), down (E, D, F).  out may be x.
    workspace: hgemm_w4_moe_workspace_bytes(T, top_k, D, F) bytes that no other running call uses,
    else allocated by torch."""
    if x.requires_grad or weights.requires_grad:
        _check_no_gradient(x=x, weights=weights)
    ldx, dt, dev = _check_rows("x", x)
    t, d = x.shape
    e, f = gate.experts, gate.n
    if e is None:
        raise ValueError("gate must be a stack of experts, (E, F, D)")
    _check_weight("gate", gate, dev, e)
    _check_weight("up", up, dev, e)
    _check_weight("down", down, dev, e)
    if gate.k != d or up.n != f or up.k != d or down.n != d or down.k != f:
        raise ValueError(f"x is {tuple(x.shape)}, gate {e} x {f} x {gate.k}, up {up.n} x {up.k}, down {down.n} x {down.k}: "
                         "gate and up must be (E, F, D), down (E, D, F)")
    if ids.dtype != torch.int32 or ids.dim() != 2 or ids.shape[0] != t or not ids.is_contiguous() or ids.get_device() != dev:
        raise ValueError("ids must be a contiguous (T, top_k) int32 tensor on x's device")
    top_k = ids.shape[1]
    if (weights.dtype != torch.float32 or weights.shape != ids.shape or not weights.is_contiguous()
            or weights.get_device() != dev):
        raise ValueError("weights must be a contiguous (T, top_k) float32 tensor on x's device")
    with _context(dev, stream):
        if out is None:
            out = x.new_empty((t, d))
        elif out.shape != (t, d) or out.dtype != x.dtype or not out.is_contiguous() or out.get_device() != dev:
            raise ValueError("out must be a contiguous (T, D) tensor of x's type on x's device")
        if workspace is None:
            workspace = x.new_empty(_fn("hgemm_w4_moe_workspace_bytes")(t, top_k, d, f), dtype=torch.uint8)
        elif workspace.get_device() != dev or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous tensor on x's device")
        # Three hgemm_w4_weight: q, scales, zeros, group.
        packed = (ctypes.c_uint64 * 12)(
            gate.q.data_ptr(), gate.scales.data_ptr(), 0 if gate.zeros is None else gate.zeros.data_ptr(), gate.group,
            up.q.data_ptr(), up.scales.data_ptr(), 0 if up.zeros is None else up.zeros.data_ptr(), up.group,
            down.q.data_ptr(), down.scales.data_ptr(), 0 if down.zeros is None else down.zeros.data_ptr(), down.group)
        at = ctypes.addressof(packed)
        rc = _fn("hgemm_w4_moe")(x.data_ptr(), dt, ldx, ids.data_ptr(), weights.data_ptr(), t, top_k, e, d, f, at, at + 32,
                                 at + 64, out.data_ptr(), workspace.data_ptr(),
                                 workspace.numel() * workspace.element_size(), _stream_handle(stream, dev))
    if rc:
        check(rc, "hgemm_w4_moe")
    return out
