"""What the video-token operators are measured on: rotary positions with several axes, attention over packed documents, and
attention with its gradients.  `run` makes the framework's own calls where `own` is true; otherwise it computes the same values
from elementary torch operations, in 32 bits (the angles of the rotation in 64), rounded once at the end."""
import math
import random

import torch

own = False

HEAD = 64
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
LOG2E = 1.4426950408889634


# ------------------------------------------------------------------------------------------------------------- the cases
def _rotary(name, dtype, clips, frames, side, heads, interleaved=False, gradient=False, start=0):
    return {"name": name, "op": "rotary", "dtype": dtype, "clips": clips, "frames": frames, "side": side, "heads": heads,
            "interleaved": interleaved, "gradient": gradient, "start": start}


def _attention(name, dtype, docs, q_min, q_max, heads, kv_heads=0, k_min=0, k_max=0, causal=False, prefix=0, slopes=False,
               cap=0.0, train=False, mix=1):
    """`k_max` = 0: the keys are the queries' own rows; `prefix`: the longest prefix that every row of a document sees."""
    return {"name": name, "op": "train" if train else "attention", "dtype": dtype, "docs": docs, "q_min": q_min, "q_max": q_max,
            "heads": heads, "kv_heads": kv_heads or heads, "k_min": k_min, "k_max": k_max, "causal": causal, "prefix": prefix,
            "slopes": slopes, "cap": cap, "mix": mix}


def listed():
    return [
        # one frame of 14 x 14 patches: q and k of 12 heads rotated in front of a single image's attention (latency)
        _rotary("rotary_one_frame", "f32", 1, 1, 14, 24),
        # a training batch of 64 clips of 8 frames, q and k of 12 heads
        _rotary("rotary_clips", "bf16", 64, 8, 14, 24),
        # the gradient of the same in the type the framework trains in, of a stream that has run for days (far positions)
        _rotary("rotary_gradient", "f32", 37, 5, 14, 24, interleaved=True, gradient=True, start=9_000_011),
        # one caption of the text tower (latency)
        _attention("attention_one_caption", "f32", 1, 77, 77, 8, causal=True),
        # a batch of captions packed without their padding
        _attention("attention_captions", "bf16", 512, 4, 77, 8, causal=True, mix=3),
        # every token of a clip sees every other: 16 frames of 14 x 14 patches
        _attention("attention_clips", "bf16", 3, 3136, 3136, 12),
        # one new token for each of 24 sequences that are being written, over what they hold so far
        _attention("attention_next_token", "bf16", 24, 1, 1, 12, 4, k_min=300, k_max=12000, causal=True, slopes=True, mix=5),
        # frames in front of captions: the frames (the prefix) are seen by all, the caption reads backwards; capped scores
        _attention("attention_prefix", "f32", 7, 210, 1300, 12, causal=True, prefix=1200, slopes=True, cap=30.0, mix=7),
        # training: packed captions in the type the framework trains in
        _attention("train_captions", "f32", 256, 4, 77, 8, causal=True, train=True, mix=11),
        # training: clips of 4 to 8 frames, capped scores
        _attention("train_clips", "bf16", 6, 784, 1568, 12, cap=50.0, train=True, mix=13),
        # training: frames in front of captions, heads that share keys, a bias by distance whose slopes are learnt
        _attention("train_prefix", "f32", 9, 61, 900, 8, 2, causal=True, prefix=700, slopes=True, train=True, mix=17),
        # training: one long stream of tokens
        _attention("train_long", "bf16", 1, 7777, 7777, 8, 2, causal=True, train=True, mix=19),
    ]


def _spread(rng, low, high):
    """A whole number between `low` and `high`, spread over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    dtype = rng.choice(["bf16", "f32"])
    op = rng.choice(["rotary", "attention", "attention", "train", "train"])
    if op == "rotary":
        side, frames, heads = rng.randint(7, 24), rng.randint(1, 16), rng.randint(1, 24)
        most = max(1, int((100_000_000 if dtype == "bf16" else 50_000_000) // (side * side * frames * heads * HEAD)))
        return {k: v for k, v in _rotary("", dtype, _spread(rng, 1, min(most, 64)), frames, side, heads, rng.random() < 0.5,
                                         rng.random() < 0.5, rng.choice([0, _spread(rng, 1, 10_000_000)])).items() if k != "name"}
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4])
    causal = rng.random() < 0.6
    most = 100_000_000 if dtype == "f32" else 200_000_000  # score entries of the padded batch
    if op == "attention" and rng.random() < 0.4:  # few queries over many keys
        q_max, k_max = rng.choice([1, 1, rng.randint(2, 9)]), _spread(rng, 64, 12000)
        docs = _spread(rng, 1, max(1, min(32, 250_000 // k_max)))
        lengths = dict(docs=docs, q_min=rng.randint(1, q_max), q_max=q_max, k_min=rng.randint(1, k_max), k_max=k_max)
    else:
        q_max = _spread(rng, 1, 3200)
        docs = _spread(rng, 1, max(1, min(512, int(most // (heads * q_max * q_max)), 25_000 // q_max)))
        lengths = dict(docs=docs, q_min=rng.randint(0, q_max), q_max=q_max)
    return {k: v for k, v in _attention("", dtype, heads=heads, kv_heads=kv_heads, causal=causal,
                                        prefix=_spread(rng, 1, 1200) if causal and rng.random() < 0.4 else 0, slopes=rng.random() < 0.4,
                                        cap=rng.choice([0.0, 0.0, 30.0, 50.0]), train=op == "train", mix=rng.randint(100, 1_000_000),
                                        **lengths).items() if k != "name"}


def _lengths(case):
    """(query rows, key rows, prefix) of each document."""
    r = random.Random(case["mix"])
    q = [r.randint(case["q_min"], case["q_max"]) for _ in range(case["docs"])]
    q[r.randrange(len(q))] = case["q_max"]
    k = q
    if case["k_max"]:
        k = [max(a, r.randint(case["k_min"], case["k_max"])) for a in q]
    return q, k, [r.randint(0, case["prefix"]) for _ in q]


def _sections(pairs):
    """The pairs of a head's dimensions that turn with time, height and width."""
    a = pairs // 4
    return (a, (pairs - a) // 2, pairs - a - (pairs - a) // 2)


# ------------------------------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(t)

    s = dict(case)
    if case["op"] == "rotary":
        n, f, a = case["clips"], case["frames"], case["side"]
        grid = torch.meshgrid(torch.arange(f), torch.arange(a), torch.arange(a), indexing="ij")
        one = torch.stack([x.reshape(-1) for x in grid], 1)
        positions = one.repeat(n, 1)
        positions[:, 0] += case["start"] + torch.arange(n).repeat_interleave(f * a * a) * f
        pairs = HEAD // 2
        rows = positions.shape[0]
        qkv = normal(rows, (case["heads"] + case["heads"] // 2) * HEAD)  # q | k | v of the fused projection: q and k are turned
        s.update(x=qkv[:, :case["heads"] * HEAD].view(rows, case["heads"], HEAD), positions=positions.to(torch.int32).cuda(),
                 inv_freq=(100.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float().cuda(), sections=_sections(pairs))
        s["axis"] = torch.repeat_interleave(torch.arange(3), torch.tensor(s["sections"])).cuda()
        return s
    q_len, k_len, prefix = _lengths(case)
    offsets = lambda n: torch.tensor([0] + n).cumsum(0).to(torch.int32).cuda()  # noqa: E731
    hq, hk = case["heads"], case["kv_heads"]
    rows, keys = sum(q_len), sum(k_len)
    if case["k_max"]:
        q, kv = normal(rows, hq, HEAD), normal(keys, 2, hk, HEAD)
        k, v = kv[:, 0], kv[:, 1]
    else:
        qkv = normal(rows, (hq + 2 * hk) * HEAD)  # the fused projection's rows: q | k | v
        q, k, v = (x.view(rows, -1, HEAD) for x in qkv.split([hq * HEAD, hk * HEAD, hk * HEAD], 1))
    s.update(q=q, k=k, v=v, q_offsets=offsets(q_len), k_offsets=offsets(k_len) if case["k_max"] else None,
             q_max=max(q_len), k_max_=max(k_len), prefix_=torch.tensor(prefix, dtype=torch.int32).cuda() if case["prefix"] else None,
             slopes_=(2.0 ** (-8.0 * (torch.arange(hq) + 1) / hq)).float().cuda() if case["slopes"] else None)
    if case["op"] == "train":
        s["d_out"] = normal(rows, hq, HEAD)
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    if s["op"] == "rotary":
        return _own_rotary(s) if own else _plain_rotary(s)
    return _own_attention(s) if own else _plain_attention(s)


def _own_rotary(s):
    from fitclip_amd import ops
    return ops.rotary(s["x"], s["positions"], s["inv_freq"], s["sections"], interleaved=s["interleaved"], inverse=s["gradient"])


def _own_attention(s):
    from fitclip_amd import ops
    how = dict(k_offsets=s["k_offsets"], causal=s["causal"], prefix=s["prefix_"], slopes=s["slopes_"], cap=s["cap"])
    out, stats = ops.attention_docs(s["q"], s["k"], s["v"], s["q_offsets"], **how)
    if s["op"] == "attention":
        return out, stats
    return (out, stats) + ops.attention_docs_backward(s["d_out"], s["q"], s["k"], s["v"], out, stats, s["q_offsets"],
                                                      slope_grad=s["slopes"], **how)


def _plain_rotary(s):
    x, pairs = s["x"].float(), HEAD // 2
    angle = s["positions"][:, s["axis"]].double() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if s["gradient"]:
        sin = -sin
    if s["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2).to(s["x"].dtype)
    a, b = x[..., :pairs], x[..., pairs:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(s["x"].dtype)


def _plain_attention(s):
    q, k, v = s["q"], s["k"], s["v"]
    t, scale, cap = q.dtype, HEAD ** -0.5, s["cap"]
    q_off = s["q_offsets"].long()
    k_off = q_off if s["k_offsets"] is None else s["k_offsets"].long()
    docs, hq, hk, lq, lk = q_off.numel() - 1, q.shape[1], k.shape[1], s["q_max"], s["k_max_"]
    group = hq // hk

    def padded(x, off, most):  # packed rows -> [docs, heads, rows, HEAD]
        at = (off[:-1, None] + torch.arange(most, device=x.device)).clamp_(max=x.shape[0] - 1)
        return x.float()[at].permute(0, 2, 1, 3).contiguous()

    def grouped(x, off, most):  # ... with the heads that share keys side by side: [docs, kv heads, group * rows, HEAD]
        return padded(x, off, most).view(docs, hk, group * most, HEAD)

    qp, kp, vp = grouped(q, q_off, lq), padded(k, k_off, lk), padded(v, k_off, lk)
    raw = (qp @ kp.transpose(-1, -2).contiguous()).mul_(scale)
    raw = raw.view(docs, hk, group, lq, lk)
    bent = torch.tanh(raw / cap) if cap else None
    score = cap * bent if cap else raw
    n_q, n_k = q_off.diff()[:, None], k_off.diff()[:, None]
    row, col = torch.arange(lq, device=q.device)[None], torch.arange(lk, device=q.device)
    place = row + n_k - n_q  # a document's last query stands at its last key
    last = n_k.expand(docs, lq)
    if s["causal"]:
        seen = place + 1 if s["prefix_"] is None else torch.maximum(place + 1, s["prefix_"].long()[:, None])
        last = torch.minimum(last, seen)
    hidden = ((col >= last[..., None]) | (row >= n_q)[..., None])[:, None, None]
    if s["slopes"]:
        far = (place[..., None] - col).abs().float()[:, None, None]
        slope = s["slopes_"].view(1, hk, group, 1, 1)
        score = score - slope * far
    score = score.masked_fill(hidden, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = p.view(docs, hk, group * lq, lk) @ vp

    def packed(x, off, rows):  # [docs, heads, rows, ...] -> the packed rows
        at = torch.arange(rows, device=x.device)
        doc = torch.searchsorted(off, at, right=True) - 1
        return x[doc, :, at - off[doc]]

    stats = torch.cat([top * LOG2E, total], -1).view(docs, hq, lq, 2)
    got = (packed(out.view(docs, hq, lq, HEAD), q_off, q.shape[0]).to(t), packed(stats, q_off, q.shape[0]))
    if s["op"] == "attention":
        return got
    do = grouped(s["d_out"], q_off, lq) * (row < n_q)[:, None, None].expand(docs, hk, group, lq).reshape(docs, hk, group * lq, 1)
    flat = p.view(docs, hk, group * lq, lk)
    dv = flat.transpose(-1, -2).contiguous() @ do
    dp = (do @ vp.transpose(-1, -2).contiguous()).view(docs, hk, group, lq, lk)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    more = ()
    if s["slopes"]:
        more = (-(ds * far).double().sum((0, 3, 4)).float().reshape(hq),)
    if cap:
        ds = ds * (1 - bent * bent)
    ds = ds.reshape(docs, hk, group * lq, lk) * scale
    dq, dk = ds @ kp, ds.transpose(-1, -2).contiguous() @ qp
    return got + (packed(dq.view(docs, hq, lq, HEAD), q_off, q.shape[0]).to(t), packed(dk, k_off, k.shape[0]).to(t),
                  packed(dv, k_off, v.shape[0]).to(t)) + more


# ---------------------------------------------------------------------------------------------------- what it cannot do without
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "rotary":
        rows = case["clips"] * case["frames"] * case["side"] ** 2
        values = rows * case["heads"] * HEAD
        return {"bytes": 2 * size * values + 12 * rows, "flops": 3 * values}
    q_len, k_len, prefix = _lengths(case)
    hq, hk = case["heads"], case["kv_heads"]
    pairs = 0
    for a, b, p in zip(q_len, k_len, prefix):
        if not case["causal"]:
            pairs += a * b
        else:
            pairs += sum(min(b, max(i + b - a + 1, p)) for i in range(a))
    rows, keys = sum(q_len) * hq * HEAD, sum(k_len) * hk * HEAD
    stats = 8 * sum(q_len) * hq
    if case["op"] == "attention":
        return {"bytes": size * 2 * (rows + keys) + stats, "flops": 4 * HEAD * pairs * hq}
    return {"bytes": size * (4 * rows + 4 * keys) + stats, "flops": 12 * HEAD * pairs * hq}


# ------------------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        x, pairs = s["x"].double(), HEAD // 2
        lo = [0]
        for n in s["sections"]:
            lo.append(lo[-1] + n)
        angle = torch.cat([s["positions"][:, i, None].double() * s["inv_freq"][None, lo[i]:lo[i + 1]].double() for i in range(3)], 1)
        turn = torch.polar(torch.ones_like(angle), -angle if case["gradient"] else angle)[:, None]
        if case["interleaved"]:
            return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:2], pairs, 2)) * turn).reshape(x.shape)
        y = torch.complex(x[..., :pairs].contiguous(), x[..., pairs:].contiguous()) * turn
        return torch.cat([y.real, y.imag], -1)
    q_len, k_len, prefix = _lengths(case)
    train = case["op"] == "train"
    hq, hk = case["heads"], case["kv_heads"]
    q, k, v = (s[n].double().requires_grad_(train) for n in "qkv")
    slopes = None if s["slopes_"] is None else s["slopes_"].double().requires_grad_(train)
    out, stats = torch.zeros_like(q).detach(), torch.zeros(*q.shape[:2], 2, dtype=torch.float64, device=q.device)
    grads = [torch.zeros_like(x).detach() for x in (q, k, v)]
    d_slopes = torch.zeros(hq, dtype=torch.float64, device=q.device)
    a = b = 0
    for n, m, pre in zip(q_len, k_len, prefix):
        if n and m:
            for head in range(hk):  # one group of heads at a time: a long document's scores stay small enough
                mine = slice(head * (hq // hk), (head + 1) * (hq // hk))
                qs, ks, vs = q[a:a + n, mine], k[b:b + m, head], v[b:b + m, head]
                score = torch.matmul(qs.transpose(0, 1), ks.t()) * HEAD ** -0.5
                if case["cap"]:
                    score = case["cap"] * torch.tanh(score / case["cap"])
                i = torch.arange(n, device=q.device)[:, None] + (m - n)
                j = torch.arange(m, device=q.device)[None]
                if slopes is not None:
                    score = score - slopes[mine, None, None] * (i - j).abs()
                if case["causal"]:
                    score = score.masked_fill((j > i) & (j >= pre), -math.inf)
                rows = (score > -math.inf).any(-1, keepdim=True)
                p = torch.softmax(score.masked_fill(~rows, 0.0), -1) * rows
                y = torch.matmul(p, vs).transpose(0, 1)
                out[a:a + n, mine] = y.detach()
                top = score.detach().amax(-1)
                stats[a:a + n, mine, 0] = top.t() * LOG2E
                stats[a:a + n, mine, 1] = torch.exp(score.detach() - top.masked_fill(top == -math.inf, 0.0)[..., None]).sum(-1).t()
                if train:
                    leaves = [qs, ks, vs] + ([] if slopes is None else [slopes])
                    got = torch.autograd.grad(y, leaves, s["d_out"][a:a + n, mine].double())
                    grads[0][a:a + n, mine] = got[0]
                    grads[1][b:b + m, head] = got[1]
                    grads[2][b:b + m, head] = got[2]
                    if slopes is not None:
                        d_slopes += got[3]
        a, b = a + n, b + m
    if not train:
        return out, stats
    return (out, stats, *grads) + ((d_slopes,) if slopes is not None else ())
