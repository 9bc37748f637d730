"""Rotary positions and attention over packed documents from their definitions, in 64 bits on the CPU, with the error bounds that the
tests use.  Written document by document; gradients through autograd."""
import math

import torch

LOG2E = 1.4426950408889634
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # a rounding is off by at most half a step, relative to the value


def offsets(lengths, device="cuda"):
    return torch.tensor([0] + list(lengths)).cumsum(0).to(torch.int32).to(device)


def rotary(x, positions, inv_freq, sections, interleaved=False, inverse=False):
    x, pairs = x.double().cpu(), inv_freq.numel()
    positions = positions.cpu().reshape(x.shape[0], -1)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    angle = positions[:, axis].double() * inv_freq.double().cpu()
    c, s = angle.cos()[:, None], angle.sin()[:, None] * (-1 if inverse else 1)
    y = x.clone()
    first = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    second = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    return y


def attention(q, k, v, q_len, k_len=None, causal=False, prefix=None, slopes=None, cap=0.0, scale=0.125, d_out=None, seen_only=False):
    """dict of 64-bit out, stats (maximum in units of ln 2, sum), and with `d_out` d_q, d_k, d_v, d_slopes; rows of no document: 0.
    `seen_only`: keys that no row of a group sees do not enter at all (they may hold NaN)."""
    k_len = list(q_len if k_len is None else k_len)
    q, k, v = (t.detach().double().cpu().clone().requires_grad_(d_out is not None) for t in (q, k, v))
    slopes = None if slopes is None else slopes.detach().double().cpu().clone().requires_grad_(d_out is not None)
    heads, group = q.shape[1], q.shape[1] // k.shape[1]
    out, stats = torch.zeros_like(q).detach(), torch.zeros(*q.shape[:2], 2, dtype=torch.float64)
    stats[..., 0] = -math.inf
    total, a, b = 0.0, 0, 0
    big, top_dp, sum_dp, weight = 0.0, 0.0, 0.0, torch.zeros(k.shape[0], k.shape[1], dtype=torch.float64)  # weight: what each key weighs in all rows together
    for doc, (n, m) in enumerate(zip(q_len, k_len)):
        for i in range(n):
            p = i + m - n
            last = m if not causal else min(m, max(p + 1, int(prefix[doc]) if prefix is not None else 0))
            if last <= 0:
                continue
            for h in range(heads):
                qi, ks, vs = q[a + i, h], k[b:b + last, h // group], v[b:b + last, h // group]
                score = ks @ qi * scale
                big = max(big, float((ks.detach().abs() @ qi.detach().abs()).max()) * scale if not seen_only else 0.0)
                if cap:
                    score = cap * torch.tanh(score / cap)
                if slopes is not None:
                    score = score - slopes[h] * (p - torch.arange(last)).abs()
                p_row = torch.softmax(score, 0)
                weight[b:b + last, h // group] += p_row.detach()
                y = p_row @ vs
                out[a + i, h] = y.detach()
                top = score.max().detach()
                stats[a + i, h, 0] = top * LOG2E
                stats[a + i, h, 1] = torch.exp(score.detach() - top).sum()
                if d_out is not None:
                    g = d_out[a + i, h].double().cpu()
                    top_dp = max(top_dp, float((vs.detach() @ g).abs().max()))
                    sum_dp = max(sum_dp, float((vs.detach().abs() @ g.abs()).max()))
                    total = total + (y * d_out[a + i, h].double().cpu()).sum()
        a, b = a + n, b + m
    got = {"out": out, "stats": stats, "big": big, "weight": weight, "top_dp": top_dp, "sum_dp": sum_dp}
    if d_out is not None:
        leaves = [q, k, v] + ([slopes] if slopes is not None else [])
        grads = torch.autograd.grad(total, leaves, allow_unused=True) if torch.is_tensor(total) else [None] * len(leaves)
        for name, leaf, g in zip(("d_q", "d_k", "d_v", "d_slopes"), leaves, grads):
            got[name] = torch.zeros_like(leaf) if g is None else g
    return got


def score_error(ref, keys, slopes=None, scale=0.125, cap=0.0):
    """How far a score may be off, in fp32: 64 products and sums of it (64 + 2 roundings of terms whose absolute values sum up to
    `big`), the bias (3 roundings of slope * distance, the exponent's change of units among them), tanh (2 ulp of cap or score)."""
    bias = float(slopes.abs().max()) * keys if slopes is not None else 0.0
    return 2.0 ** -24 * (68 * ref["big"] + 4 * bias + 8 * (min(cap, ref["big"]) if cap else 0.0) + 8)


def out_bound(ref, v, dtype, keys, ds):
    """|out - exact| elementwise: weights off by 2 ds each (numerator and sum), `keys` additions in fp32, bf16: every weight rounded;
    the output rounded."""
    top = float(v.double().abs().max()) if v.numel() else 0.0
    inner = (2 * ds + (keys + 8) * 2.0 ** -24 + (HALF[dtype] if dtype == torch.bfloat16 else 0.0)) * top
    return inner + HALF[dtype] * ref["out"].abs() + 1e-30


def grad_bounds(ref, q, k, v, d_out, dtype, keys, ds, cap=0.0, slopes=None, scale=0.125):
    """Elementwise bounds of d_q, d_k, d_v, d_slopes.  A weight is off by 2 ds of itself (bf16: and rounded once more in a product);
    dP = dO.v and D = dO.O are sums of 64 products, D of the result's own error too; dS = P (dP - D), bf16: rounded."""
    e, h = 2.0 ** -24, HALF[dtype] if dtype == torch.bfloat16 else 0.0
    top = lambda t: float(t.double().abs().max()) if t.numel() else 0.0  # noqa: E731
    rows = q.shape[0] * q.shape[1]
    length = float(d_out.double().abs().sum(-1).max()) if rows else 0.0
    both = ref["top_dp"]                                          # |dP| at most, hence |D| as well (a mean of dP)
    far_out = float(out_bound(ref, v, dtype, keys, ds).max()) * length if rows else 0.0
    weight = 2 * ds + 8 * e
    off = 2 * weight * both + 136 * e * ref["sum_dp"] + (32 * e * both if cap else 0.0)
    one = off + far_out + 2 * h * both                            # error of dS over P
    out = {
        "d_q": scale * top(k) * (one + keys * e * 2 * both) + HALF[dtype] * ref["d_q"].abs() + 1e-30,
        "d_k": (scale * top(q) * (one + rows * e * 2 * both) * ref["weight"])[..., None] + HALF[dtype] * ref["d_k"].abs() + 1e-30,
        "d_v": (top(d_out) * (weight + h + rows * e) * ref["weight"])[..., None] + HALF[dtype] * ref["d_v"].abs() + 1e-30,
    }
    if slopes is not None:  # every factor in fp32; a head's rows are summed in 64 bits
        out["d_slopes"] = torch.full((q.shape[1],), q.shape[0] * keys * 2 * (off + (keys + 8) * e * 2 * both), dtype=torch.float64)
    return out
