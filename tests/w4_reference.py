"""Plain 64-bit references of the 4-bit weight operators, and what their results may be off by."""
import math

import torch

# One addition in fp32 by a tensor core or an FMA: half a step (2^-24) if rounded, a whole one (2^-23)
# if truncated; twice that, as one instruction adds several products.
ADD = 2.0 ** -22


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def lookup(w, index=None):
    """The matrix of a W4Weight in 64 bits (on the CPU), each code found by its place in the layout
    that the header describes."""
    q, s, z = (None if t is None else t.cpu() for t in (w.q, w.scales, w.zeros))
    if index is not None:
        q, s, z = q[index], s[index], None if z is None else z[index]
    row, col = torch.arange(w.n)[:, None], torch.arange(w.k)[None, :]
    g, rr = row % 8, row // 8 % 2
    jg, t, jk, rk, half = col // 32 % 2, col // 8 % 4, col // 4 % 2, col // 2 % 2, col % 2
    byte = q[row // 16, col // 64, 16 * (4 * g + t) + 4 * (2 * jg + jk) + 2 * half + rk].long()
    code = (byte >> (4 * rr)) & 15
    at = (row // 16, col // w.group, g, rr)
    return (code - (8 if z is None else z[at].long())).double() * s[at].double()


def quantize(w, group, zero_point):
    """codes (N, K), scales (N, groups) bf16, zeros (N, groups) or None of one CPU matrix."""
    n, k = w.shape
    groups = -(-k // group)
    x = torch.nn.functional.pad(w.double(), (0, groups * group - k)).view(n, groups, group)
    known = torch.where(x.isnan(), 0.0, x)
    lo, hi = known.amin(-1).clamp(max=0), known.amax(-1).clamp(min=0)
    s = (hi - lo) / 15 if zero_point else torch.maximum(hi, -lo) / 7
    s = s.float().to(torch.bfloat16).clamp(max=torch.finfo(torch.bfloat16).max)
    s = torch.where(s == 0, torch.ones_like(s), s)
    sd = s.double()
    z = (-lo / sd).round().clamp(0, 15) if zero_point else torch.full_like(sd, 8.0)
    c = (x / sd[..., None]).round()
    c = (torch.where(c.isnan(), 0.0, c) + z[..., None]).clamp(0, 15)
    return c.view(n, -1)[:, :k].to(torch.uint8), s, z.to(torch.uint8) if zero_point else None


def random_weight(gen, shape, group, zero_point, scale=None):
    """Random codes, scales and zeros (CPU, row-major) of an (N, K) or (E, N, K) weight."""
    *lead, n, k = shape
    groups = -(-k // group)
    codes = torch.randint(0, 16, (*lead, n, k), generator=gen, dtype=torch.uint8)
    scales = (torch.rand(*lead, n, groups, generator=gen) + 0.5) / (4.6 * math.sqrt(k)) if scale is None else scale
    zeros = torch.randint(0, 16, (*lead, n, groups), generator=gen, dtype=torch.uint8) if zero_point else None
    return codes, scales.to(torch.bfloat16), zeros


def values(codes, scales, zeros, group):
    """(code - zero) * scale in 64 bits."""
    k = codes.shape[-1]
    s = scales.double().repeat_interleave(group, -1)[..., :k]
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(group, -1)[..., :k]
    return (codes.double() - z) * s


def additions(k, terms):
    """The longest chain of additions behind a sum over K: the terms' products of one 64-K part (four
    instructions each), the parts, 8 warps and 8 CTAs."""
    return 4 * terms + -(-k // 64) + 16


def linear(x, w, terms):
    """x @ w^T in 64 bits and the bound of its fp32 evaluation."""
    x = x.double()
    return x @ w.T, additions(w.shape[1], terms) * ADD * (x.abs() @ w.abs().T)


def experts(x, ids, weights, gate, up, down, terms):
    """The experts' sum in 64 bits (dense stacks gate, up, down) and the bound of its evaluation."""
    t, d = x.shape
    out, off = torch.zeros(t, d, dtype=torch.float64), torch.zeros(t, d, dtype=torch.float64)
    for i in range(t):
        for j in range(ids.shape[1]):
            e = int(ids[i, j])
            if not 0 <= e < gate.shape[0]:
                continue
            g, dg = linear(x[i:i + 1], gate[e], terms)
            u, du = linear(x[i:i + 1], up[e], terms)
            a = g * torch.sigmoid(g)
            h = a * u
            # silu' is below 1.1; silu and the product round a few times (16 half steps); h is kept in two bf16: what
            # the first (truncated: off by a step, 2^-7) leaves is rounded by half a step, 2^-8.
            dh = 1.1 * dg * u.abs() + (a.abs() + 1.1 * dg) * du + h.abs() * (16 * 2.0 ** -24 + 2.0 ** -15)
            y, dy = linear(h, down[e], 2)
            w = float(weights[i, j])
            out[i] += w * y[0]
            off[i] += abs(w) * (dh @ down[e].abs().T + dy * (1 + 2.0 ** -10))[0]
    # The pairs' sums: one more addition each for the weight and the sum, at most 2 * top_k + 16.
    return out, off * (1 + 2.0 ** -10) + (2 * ids.shape[1] + 16) * ADD * (out.abs() + off)


def assert_close(got, ref, off, dtype):
    got = got.detach().cpu().double()
    bound = off + half_step(dtype) * (ref.abs() + off) + 2.0 ** -126
    bad = (got - ref).abs() > bound
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - ref).abs() / bound).max()):.3g} of the bound"
