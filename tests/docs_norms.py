"""Attention over packed documents and its gradients from their formulas, in 64 bits on the CPU, with places to plant a mistake; the cases whose
results are compared in the 2-norm, and how far they may be off there.

A rounding to bf16 is off by at most u = 2^-8 of the value, u / sqrt 3 in the root mean square; independent ones of terms that do not cancel add up in
the norm, so r of them leave sqrt(r / 3) u, and a quarter more is allowed for the terms that do.  A result counts
    out, d_v   2: the weights in front of the product, itself
    d_q, d_k   3: dS in front of the product, D (where it comes from a rounded `out`), itself
    d_slopes   none: every factor is held in fp32
fp32 (normal q, k, v, d_out; scale 1 / 8): a score is a sum of 64 products of size 1, partial sums of up to 16: 64 half steps of at most 2^-24 x 16, 74 in the
root mean square, an eighth of that behind the scale, and two more for the exponent: a weight is off by 10 x 2^-24 or so, out and d_v by as much; 16 are
allowed.  dP and D are such sums too: sqrt 3 times as much in d_q and d_k, 32 allowed; 64 for d_slopes, a sum over rows of either sign."""
import math

import torch

U = 2.0 ** -8
TOLERANCE = {torch.bfloat16: {"out": 1.25 * math.sqrt(2 / 3) * U, "d_v": 1.25 * math.sqrt(2 / 3) * U, "d_q": 1.25 * U, "d_k": 1.25 * U, "d_slopes": 64 * 2.0 ** -24},
             torch.float32: {"out": 16 * 2.0 ** -24, "d_v": 16 * 2.0 ** -24, "d_q": 32 * 2.0 ** -24, "d_k": 32 * 2.0 ** -24, "d_slopes": 64 * 2.0 ** -24}}

_g = torch.Generator().manual_seed(1)
SHORT = torch.randint(0, 71, (22,), generator=_g).tolist() + [70, 0, 1]
OTHER = torch.randint(0, 71, (22,), generator=_g).tolist() + [1, 70, 0]
# name: query lengths, key lengths, query heads, key heads, masks; which key heads are compared
CASES = {
    # waves that take turns over the keys, shared key heads, every mask there is
    "turns": ([160, 40, 200], None, 6, 2, dict(causal=True, prefix=120, slopes=0.2), None),
    "turns, capped": ([160, 40, 200], None, 4, 2, dict(cap=4.0), None),
    # ... whose rows are cut into parts for the keys' gradients (one key head for many rows)
    "parts of rows": ([300, 1, 219], None, 6, 1, dict(causal=True, cap=9.0, slopes=0.02), None),
    # ... whose keys are cut into parts (few rows over many keys)
    "parts of keys": ([3, 1, 5], [700, 900, 1333], 6, 2, dict(causal=True, slopes=0.01), None),
    # a wave alone with its rows or keys
    "alone": (SHORT, None, 48, 24, dict(causal=True, cap=3.0), [0, 23]),
    "alone, other keys": (SHORT, OTHER, 30, 30, dict(causal=True, prefix=50, slopes=0.3), [0, 29]),
    # four waves that share tiles; in the order of their ways
    "shared, fp32": ([300, 17, 129, 0, 64, 250], None, 352, 352, dict(causal=True, slopes=0.05), [0, 351]),
    "shared, bf16": ([300, 17, 129, 0, 64, 250], None, 144, 144, dict(causal=True, cap=20.0), [0, 143]),
    "uneven": ([37, 400, 0, 5, 500, 129, 1], None, 44, 22, dict(causal=True, prefix=300, slopes=0.1), [0, 21]),
    # rows whose weight lies on few keys
    "few keys": ([2, 3, 1, 5, 4, 7, 8, 6] * 12, None, 4, 4, dict(), None),
    "steep": ([300, 100], None, 4, 2, dict(causal=True, slopes=2.0), None),
}


def inputs(case, dtype, mean=0.0):
    """q, k, v, d_out and the masks of a case, on the CPU; `mean`: added to every value of v."""
    q_len, k_len, heads, kv_heads, masks, _ = CASES[case]
    g = torch.Generator().manual_seed(len(case))
    rows, keys = sum(q_len), sum(k_len or q_len)
    make = lambda n, h, m=0.0: (torch.randn(n, h, 64, generator=g) + m).to(dtype)  # noqa: E731
    q, k, v, d_out = make(rows, heads), make(keys, kv_heads), make(keys, kv_heads, mean), make(rows, heads)
    how = {n: masks[n] for n in ("causal", "cap") if n in masks}
    if "prefix" in masks:
        how["prefix"] = torch.randint(-3, masks["prefix"], (len(q_len),), generator=g, dtype=torch.int32)
    if "slopes" in masks:
        how["slopes"] = masks["slopes"] * (0.5 + torch.rand(heads, generator=g))
    return q, k, v, d_out, how


def definition(q, k, v, d_out, q_len, k_len=None, causal=False, prefix=None, slopes=None, cap=0.0, scale=0.125, mistake=None):
    """{out, d_q, d_k, d_v, d_slopes} in 64 bits.  `mistake`: what a kernel could get wrong, planted here."""
    dtype = q.dtype
    q, k, v, d_out = (t.detach().double().cpu() for t in (q, k, v, d_out))
    group, heads = q.shape[1] // k.shape[1], q.shape[1]
    if mistake == "the bias":
        slopes = None if slopes is None else torch.zeros_like(slopes)
    got = {"out": torch.zeros_like(q), "d_q": torch.zeros_like(q), "d_k": torch.zeros_like(k), "d_v": torch.zeros_like(v),
           "d_slopes": torch.zeros(heads, dtype=torch.float64)}
    a = b = 0
    for doc, (n, m) in enumerate(zip(q_len, q_len if k_len is None else k_len)):
        i, j = torch.arange(n)[:, None] + (m - n), torch.arange(m)[None]
        seen = torch.ones(n, m, dtype=torch.bool)
        if causal:
            seen = j <= i + (1 if mistake == "a key too many" else 0)
            if prefix is not None and mistake != "the prefix":
                seen = seen | (j < int(prefix[doc]))
        if mistake == "the last key" and m > 1:
            seen = seen & (j < m - 1)
        for h in range(heads if n and m else 0):
            qs, ks, vs, go = q[a:a + n, h], k[b:b + m, h // group], v[b:b + m, h // group], d_out[a:a + n, h]
            score = qs @ ks.t() * scale
            bent = torch.tanh(score / cap) if cap else None
            score = cap * bent if cap else score
            far = (i - j).abs().double()
            if slopes is not None:
                score = score - float(slopes[h]) * far
            score = score.masked_fill(~seen, -math.inf)
            some = seen.any(1, keepdim=True)
            p = torch.softmax(score.masked_fill(~some, 0.0), 1) * some
            out = p @ vs
            dp = go @ vs.t()
            D = (p * dp).sum(1, keepdim=True)
            if mistake == "D":
                D = torch.zeros_like(D)
            if mistake == "D from the rounded out":
                D = (go * out.to(dtype).double()).sum(1, keepdim=True)
            ds = p * (dp - D)
            if mistake == "a row" and n > 1:
                ds[n // 2], p[n // 2] = 0, 0
            got["d_slopes"][h] -= (ds * far).sum()
            if cap and mistake != "the cap's slope":
                ds = ds * (1 - bent * bent)
            got["out"][a:a + n, h] = out
            got["d_q"][a:a + n, h] = scale * ds @ ks
            if mistake != "the other heads of a group" or h % group == 0:
                got["d_k"][b:b + m, h // group] += scale * ds.t() @ qs
                got["d_v"][b:b + m, h // group] += p.t() @ go
        a, b = a + n, b + m
    if slopes is None:
        del got["d_slopes"]
    return got


def off(got, want):
    """How far a result is off, in the 2-norm, relative to its own."""
    want = want.double().cpu()
    return float((got.double().cpu() - want).norm() / want.norm())


def compared(case):
    """(key heads, query heads) that are compared."""
    _, _, heads, kv_heads, _, some = CASES[case]
    some = list(range(kv_heads)) if some is None else some
    group = heads // kv_heads
    return some, [h * group + g for h in some for g in range(group)]


def of_some(case, q, k, v, d_out, how):
    """A case's definition (a partial function of its mistake) for the heads that are compared."""
    kv, heads = compared(case)
    how = dict(how)
    if "slopes" in how:
        how["slopes"] = how["slopes"][heads]
    return lambda mistake=None: definition(q[:, heads], k[:, kv], v[:, kv], d_out[:, heads], *CASES[case][:2], mistake=mistake, **how)
