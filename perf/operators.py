"""What is measured of the 4-bit weight operators: cases, inputs, plain torch forms and 64-bit values.

Kinds of case:
    quantise  a weight matrix to 4-bit codes with group scales, and back to values
    linear    a few rows of activations times such a matrix
    route     the router of a mixture of experts: product, softmax, top-k
    experts   the chosen experts' gated products, summed with the router's weights

Blocked codes: (row blocks of 16, K blocks of 64, 512 bytes).  Byte 16 * (4 g + t) + 4 * j + b of a block holds,
with j = 2 * jg + jk and b = 2 * half + rk, the codes of k = 32 jg + 8 t + 4 jk + 2 rk + half in rows g (low
nibble) and g + 8 (high nibble).  Scales and zero points: (row blocks, groups, 8, 2), row g + 8 * last index.
"""
import math

import torch

own = False

DEVICE = "cuda"


# ---- cases ------------------------------------------------------------------------------------


def listed():
    return [
        # One attention projection of a small model, converted at load time.
        {"name": "quantise 512x2048", "kind": "quantise", "n": 512, "k": 2048, "group": 32, "zeros": True, "type": "bf16"},
        # A matrix whose sides divide by nothing, kept in fp32.
        {"name": "quantise 4999x5115", "kind": "quantise", "n": 4999, "k": 5115, "group": 64, "zeros": False, "type": "f32"},
        # The largest FFN matrix of the GEMM benchmark.
        {"name": "quantise 28672x8192", "kind": "quantise", "n": 28672, "k": 8192, "group": 128, "zeros": False, "type": "bf16"},
        # Decoding one token: the smallest product of the GEMM benchmark's shapes.
        {"name": "linear 1x7168x2048", "kind": "linear", "m": 1, "n": 7168, "k": 2048, "group": 128, "zeros": False, "type": "bf16"},
        # Three fp32 rows and odd sides.
        {"name": "linear 3x5111x7163", "kind": "linear", "m": 3, "n": 5111, "k": 7163, "group": 32, "zeros": True, "type": "f32"},
        # A small decode batch against the FFN matrix.
        {"name": "linear 16x28672x8192", "kind": "linear", "m": 16, "n": 28672, "k": 8192, "group": 128, "zeros": True, "type": "bf16"},
        # A large decode batch against a square projection.
        {"name": "linear 64x8192x8192", "kind": "linear", "m": 64, "n": 8192, "k": 8192, "group": 64, "zeros": False, "type": "bf16"},
        # The router for one token.
        {"name": "route 1x2048x128", "kind": "route", "t": 1, "d": 2048, "e": 128, "top": 8, "type": "bf16", "norm": True},
        # The router for a decode batch of a wide model.
        {"name": "route 64x7168x256", "kind": "route", "t": 64, "d": 7168, "e": 256, "top": 8, "type": "f32", "norm": False},
        # One token through eight of 64 experts.
        {"name": "experts 1 of 64", "kind": "experts", "t": 1, "e": 64, "top": 8, "d": 2048, "f": 1024, "group": 128, "zeros": False, "type": "bf16"},
        # Odd sides, fp32, a few tokens that share experts.
        {"name": "experts 5 of 17", "kind": "experts", "t": 5, "e": 17, "top": 3, "d": 1000, "f": 713, "group": 32, "zeros": True, "type": "f32"},
        # A decode batch that reaches nearly every expert of a large layer.
        {"name": "experts 32 of 64", "kind": "experts", "t": 32, "e": 64, "top": 6, "d": 4096, "f": 2048, "group": 128, "zeros": False, "type": "bf16"},
    ]


def _size(rng, lo, hi):
    """A size spread over its logarithm; about half of them are multiples of 64."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 64:
        v -= v % 64
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(["quantise", "linear", "linear", "route", "experts", "experts"])
    type_ = rng.choice(["bf16", "bf16", "f32"])
    group, zeros = rng.choice([32, 64, 128]), rng.random() < 0.5
    if kind == "quantise":
        return {"kind": kind, "n": _size(rng, 256, 28672), "k": _size(rng, 512, 8192 if type_ == "bf16" else 4096),
                "group": group, "zeros": zeros, "type": type_}
    if kind == "linear":
        # fp32 rows cost three products each: fewer of them.
        return {"kind": kind, "m": _size(rng, 1, 64 if type_ == "bf16" else 16), "n": _size(rng, 512, 16384),
                "k": _size(rng, 512, 8192), "group": group, "zeros": zeros, "type": type_}
    if kind == "route":
        e = _size(rng, 8, 256)
        return {"kind": kind, "t": _size(rng, 1, 64), "d": _size(rng, 256, 7168), "e": e, "top": rng.randint(1, min(8, e)),
                "type": type_, "norm": rng.random() < 0.5}
    e = _size(rng, 4, 64)
    return {"kind": kind, "t": _size(rng, 1, 32 if type_ == "bf16" else 8), "e": e, "top": rng.randint(1, min(6, e)), "d": _size(rng, 256, 4096),
            "f": _size(rng, 256, 2048), "group": group, "zeros": zeros, "type": type_}


# ---- inputs -----------------------------------------------------------------------------------


def _dtype(case):
    return torch.bfloat16 if case["type"] == "bf16" else torch.float32


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _weight(gen, lead, n, k, group, zeros):
    """Codes of normally distributed weights, scales that give them a standard deviation near 1 / sqrt(k)."""
    rb, kb, groups = -(-n // 16), -(-k // 64), -(-k // group)
    mid = 7.5 if zeros else 8.0

    def nibbles():
        c = torch.empty(*lead, rb, kb, 512, device=DEVICE)
        return c.normal_(mid, 2.6, generator=gen).round_().clamp_(0 if zeros else 1, 15).to(torch.uint8)

    q = nibbles() | (nibbles() << 4)
    scales = torch.empty(*lead, rb, groups, 8, 2, device=DEVICE).uniform_(0.7, 1.3, generator=gen) / (2.6 * math.sqrt(k))
    z = torch.randint(5, 11, (*lead, rb, groups, 8, 2), device=DEVICE, generator=gen, dtype=torch.uint8) if zeros else None
    return q, scales.to(torch.bfloat16), z, n, k, group


def prepare(case, seed):
    gen, kind, dtype = _generator(seed), case["kind"], _dtype(case)

    def normal(*shape, std=1.0):
        return torch.empty(*shape, device=DEVICE).normal_(0.0, std, generator=gen)

    if kind == "quantise":
        w = normal(case["n"], case["k"], std=1 / math.sqrt(case["k"])).to(dtype)
        return {"case": case, "w": w}
    if kind == "linear":
        x = normal(case["m"], case["k"]).to(dtype)
        return {"case": case, "x": x, "w": _weight(gen, (), case["n"], case["k"], case["group"], case["zeros"])}
    x = normal(case["t"], case["d"]).to(dtype)
    if kind == "route":
        return {"case": case, "x": x, "router": normal(case["e"], case["d"], std=1 / math.sqrt(case["d"])).to(dtype)}
    t, e, d, f = case["t"], case["e"], case["d"], case["f"]
    logits = normal(t, e, std=1.5)
    top, ids = torch.topk(logits, case["top"], dim=1)
    more = (case["group"], case["zeros"])
    return {"case": case, "x": x, "ids": ids.to(torch.int32), "weights": torch.softmax(top, 1),
            "gate": _weight(gen, (e,), f, d, *more), "up": _weight(gen, (e,), f, d, *more),
            "down": _weight(gen, (e,), d, f, *more)}


# ---- one pass ---------------------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import hipgemm_b200 as hg
    case = state["case"]
    kind = case["kind"]
    if kind == "quantise":
        w = hg.quantize_w4(state["w"], group=case["group"], zero_point=case["zeros"])
        out = {"values": hg.dequantize_w4(w, dtype=state["w"].dtype), "scales": w.scales}
        return dict(out, zeros=w.zeros) if case["zeros"] else out
    if kind == "linear":
        return hg.w4_gemm_tn(state["x"], hg.W4Weight(*state["w"]))
    if kind == "route":
        return hg.moe_route(state["x"], state["router"], case["top"], renormalize=case["norm"])
    return hg.w4_moe(state["x"], state["ids"], state["weights"], hg.W4Weight(*state["gate"]), hg.W4Weight(*state["up"]),
                     hg.W4Weight(*state["down"]))


def _rows(blocked, n):
    """Per-row group data (row blocks, groups, 8, 2) -> (n, groups)."""
    *lead, rb, groups, _, _ = blocked.shape
    r = len(lead)
    return blocked.permute(*range(r), r, r + 3, r + 2, r + 1).reshape(*lead, rb * 16, groups)[..., :n, :]


def _values(weight):
    """The fp32 matrix (or stack of them) that a blocked weight stands for."""
    q, scales, zeros, n, k, group = weight
    *lead, rb, kb, _ = q.shape
    r = len(lead)
    v = q.view(*lead, rb, kb, 8, 4, 2, 2, 2, 2)  # g t jg jk half rk
    v = torch.stack([v & 15, v >> 4], -1)  # ... rr
    order = [r, r + 8, r + 2, r + 1, r + 4, r + 3, r + 5, r + 7, r + 6]  # rb rr g kb jg t jk rk half
    codes = v.permute(*range(r), *order).reshape(*lead, rb * 16, kb * 64)[..., :n, :k].float()
    s = _rows(scales, n).float().repeat_interleave(group, -1)[..., :k]
    if zeros is None:
        return (codes - 8) * s
    return (codes - _rows(zeros, n).float().repeat_interleave(group, -1)[..., :k]) * s


def _plain_quantise(w, group, zeros):
    n, k = w.shape
    rb, groups = -(-n // 16), -(-k // group)
    # 64 bits: codes next to the border between two steps, scales next to that between two bf16 numbers.
    x = torch.nn.functional.pad(w.double(), (0, groups * group - k)).view(n, groups, group)
    top = torch.finfo(torch.bfloat16).max
    if zeros:
        lo, hi = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
        s = (hi - lo) / 15
    else:
        s = x.abs().amax(-1) / 7
    s = s.float().to(torch.bfloat16).clamp(max=top)
    s = torch.where(s == 0, torch.ones_like(s), s)
    sd = s.double()[..., None]
    if zeros:
        z = (-lo[..., None] / sd).round().clamp(0, 15)
        c = (x / sd).round().add(z).clamp(0, 15) - z
    else:
        c = (x / sd).round().clamp(-8, 7)
    values = (c * sd).view(n, -1)[:, :k].to(w.dtype)

    def blocked(v, fill):  # (n, groups) -> (row blocks, groups, 8, 2)
        v = torch.nn.functional.pad(v, (0, 0, 0, rb * 16 - n), value=fill)
        return v.view(rb, 2, 8, groups).permute(0, 3, 2, 1).contiguous()

    out = {"values": values, "scales": blocked(s, 1)}
    return dict(out, zeros=blocked(z[..., 0].to(torch.uint8), 0)) if zeros else out


def _run_plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "quantise":
        return _plain_quantise(state["w"], case["group"], case["zeros"])
    x = state["x"]
    if kind == "linear":
        return (x.float() @ _values(state["w"]).T).to(x.dtype)
    if kind == "route":
        logits = x.double() @ state["router"].double().T  # 64 bits: values next to the border of the top-k
        order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :case["top"]]
        p = torch.softmax(logits, 1).gather(1, order)
        if case["norm"]:
            p = p / p.sum(1, keepdim=True)
        return order.to(torch.int32), p.float()
    # Experts: every (token, expert) pair with its own matrices, or, where there are more pairs than experts, every
    # expert on every token with the weights of the pairs that were not chosen at zero.
    ids, t, e = state["ids"].long(), case["t"], case["e"]
    if ids.numel() <= e:
        picked = [_values((w[0][ids.view(-1)], w[1][ids.view(-1)], None if w[2] is None else w[2][ids.view(-1)], *w[3:]))
                  for w in (state["gate"], state["up"], state["down"])]
        xs = x.float().repeat_interleave(case["top"], 0)[..., None]
        g, u = picked[0] @ xs, picked[1] @ xs
        y = (picked[2] @ (g * torch.sigmoid(g) * u))[..., 0].view(t, case["top"], -1)
        return (y * state["weights"][..., None]).sum(1).to(x.dtype)
    mix = torch.zeros(t, e, device=DEVICE).scatter_add_(1, ids, state["weights"])
    g = x.float() @ _values(state["gate"]).transpose(1, 2)
    u = x.float() @ _values(state["up"]).transpose(1, 2)
    y = (g * torch.sigmoid(g) * u) @ _values(state["down"]).transpose(1, 2)
    return (y * mix.T[..., None]).sum(0).to(x.dtype)


# ---- work and 64-bit values -------------------------------------------------------------------


def _weight_bytes(n, k, group, zeros):
    return n * k / 2 + n * -(-k // group) * (3 if zeros else 2)


def work(case):
    size = 2 if case["type"] == "bf16" else 4
    kind = case["kind"]
    if kind == "quantise":
        n, k = case["n"], case["k"]
        return {"bytes": 2 * n * k * size + 2 * _weight_bytes(n, k, case["group"], case["zeros"]), "flops": 4 * n * k}
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": _weight_bytes(n, k, case["group"], case["zeros"]) + m * (n + k) * size, "flops": 2 * m * n * k}
    t, e, d = case["t"], case["e"], case["d"]
    if kind == "route":
        return {"bytes": (t + e) * d * size + t * case["top"] * 8, "flops": 2 * t * e * d}
    f, top = case["f"], case["top"]
    reached = e * (1 - (1 - top / e) ** t)  # experts that at least one token is sent to
    one = 2 * _weight_bytes(f, d, case["group"], case["zeros"]) + _weight_bytes(d, f, case["group"], case["zeros"])
    return {"bytes": reached * one + 2 * t * d * size + t * top * 8, "flops": 6 * t * top * d * f}


def _exact_values(weight, index=None):
    """The matrix in 64 bits, each entry looked up by its place in the blocked layout."""
    q, scales, zeros, n, k, group = weight
    if index is not None:
        q, scales, zeros = q[index], scales[index], None if zeros is None else zeros[index]
    row, col = torch.arange(n, device=DEVICE)[:, None], torch.arange(k, device=DEVICE)[None, :]
    c = col % 64
    byte = 16 * (4 * (row % 8) + (c % 32) // 8) + 4 * (2 * (c // 32) + (c % 8) // 4) + 2 * (c % 2) + (c % 4) // 2
    code = (q[row // 16, col // 64, byte].long() >> (4 * ((row % 16) // 8))) & 15
    at = (row // 16, col // group, row % 8, (row % 16) // 8)
    return (code - (8 if zeros is None else zeros[at].long())).double() * scales[at].double()


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantise":
        w, group = state["w"].double(), case["group"]
        n, k = w.shape
        rb, groups = -(-n // 16), -(-k // group)
        values, scales = torch.empty_like(w), torch.ones(rb * 16, groups, dtype=torch.float64, device=DEVICE)
        for j in range(groups):
            part = w[:, j * group:(j + 1) * group]
            high, low = part.max(1).values, part.min(1).values
            if case["zeros"]:
                low, high = low.minimum(torch.zeros_like(low)), high.maximum(torch.zeros_like(high))
                s = ((high - low) / 15).to(torch.bfloat16).double()
                z = (-low / s).round().clamp(0, 15)[:, None]
                values[:, j * group:(j + 1) * group] = ((part / s[:, None]).round().add(z).clamp(0, 15) - z) * s[:, None]
            else:
                s = (torch.maximum(high, -low) / 7).to(torch.bfloat16).double()
                values[:, j * group:(j + 1) * group] = (part / s[:, None]).round().clamp(-8, 7) * s[:, None]
            scales[:n, j] = s
        row = torch.arange(rb * 16, device=DEVICE).view(rb, 2, 8).transpose(1, 2)  # (row block, g, half)
        out = {"values": values, "scales": scales[row].permute(0, 3, 1, 2).contiguous()}
        return dict(out, zeros=None) if case["zeros"] else out
    x = state["x"].double()
    if kind == "linear":
        return torch.einsum("mk,nk->mn", x, _exact_values(state["w"]))
    if kind == "route":
        logits = torch.stack([(row * state["router"].double()).sum(1) for row in x])
        p = (logits - logits.max(1, keepdim=True).values).exp()
        best = p.topk(case["top"], 1).values
        return None, best / (best if case["norm"] else p).sum(1, keepdim=True)
    out = torch.zeros(case["t"], case["d"], dtype=torch.float64, device=DEVICE)
    ids = state["ids"].long()
    for expert in ids.unique().tolist():
        token, slot = (ids == expert).nonzero(as_tuple=True)
        xs = x[token]
        g = torch.einsum("td,fd->tf", xs, _exact_values(state["gate"], expert))
        u = torch.einsum("td,fd->tf", xs, _exact_values(state["up"], expert))
        y = torch.einsum("tf,df->td", g / (1 + (-g).exp()) * u, _exact_values(state["down"], expert))
        out.index_add_(0, token, y * state["weights"][token, slot].double()[:, None])
    return out
