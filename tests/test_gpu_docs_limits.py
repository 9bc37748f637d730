"""GPU: attention over packed documents at the edges of what it takes, against 64-bit references on the CPU (docs_reference.py)."""
import math
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, str(Path(__file__).resolve().parent))
import docs_reference as R  # noqa: E402
from fitclip_amd import ops  # noqa: E402

DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16]
# (query lengths, key lengths, heads): waves that take turns over the keys, the same with the key range cut into parts, a wave alone with its
# rows, waves that share tiles of keys (fp32: more than eight workgroups per compute unit)
SHAPES = {"turns": ([40, 20], None, 2), "parts": ([1, 2], [900, 1100], 2), "alone": ([40, 20] * 60, None, 24), "shared": ([300, 200, 300], None, 352)}


def _rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("how", ["infinite keys", "products beyond the range", "a bias beside them"])
def test_rows_whose_scores_are_all_minus_infinity(dtype, shape, how):
    """The first document's scores are -inf throughout: its rows are 0 with stats (-inf, 0), its gradients 0, in every shape of a workgroup, and
    the other documents' results are what they are without it."""
    q_len, k_len, heads = SHAPES[shape]
    rows, keys = sum(q_len), sum(k_len or q_len)
    q, k, v = _rand(rows, heads, 64, seed=1).abs().to(dtype), _rand(keys, heads, 64, seed=2, dtype=dtype), _rand(keys, heads, 64, seed=3, dtype=dtype)
    d_out = _rand(rows, heads, 64, seed=4, dtype=dtype)
    m, n = q_len[0], (k_len or q_len)[0]
    off = (R.offsets(q_len), None if k_len is None else R.offsets(k_len))
    slopes = dict(slopes=torch.full((heads,), 0.01, device=DEV)) if how == "a bias beside them" else {}
    clean = ops.attention_docs(q, k, v, *off, causal=True, **slopes)
    clean += ops.attention_docs_backward(d_out, q, k, v, *clean, *off, causal=True, slope_grad=bool(slopes), **slopes)
    if how == "products beyond the range":
        q[:m], k[:n] = 1e20, -1e20
    else:
        k[:n, :, 5] = -math.inf
    out, stats = ops.attention_docs(q, k, v, *off, causal=True, **slopes)
    assert (out[:m] == 0).all() and (stats[:m, :, 0] == -math.inf).all() and (stats[:m, :, 1] == 0).all()
    grads = ops.attention_docs_backward(d_out, q, k, v, out, stats, *off, causal=True, slope_grad=bool(slopes), **slopes)
    assert not grads[0][:m].any() and not grads[1][:n].any() and not grads[2][:n].any()
    assert all(torch.isfinite(g).all() for g in grads)
    # rows that met an infinite key in a tile of theirs are formed again key by key, with weights in fp32: in another order, and without a bf16
    # weight's rounding (three of them at most: its own and both results'; gradients eight, with those of D and dS).  A score is off by 64 products
    # and sums of terms that add up to 10 at most in either way, a weight by twice that, a gradient's two factors by that each: 4 x 2 x 68 x 10
    for got, want, start, roundings in ((out, clean[0], m, 3), (grads[0], clean[2], m, 8), (grads[1], clean[3], n, 8), (grads[2], clean[4], n, 8)):
        got, want = got[start:].double(), want[start:].double()
        assert float((got - want).abs().max()) <= (roundings * R.HALF[dtype] + 5440 * 2.0 ** -24) * float(want.abs().max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("scale,size,slopes", [(1e30, 1.0, False), (1e12, 1.0, False), (0.125, 1e5, False), (1e30, 1.0, True)])
def test_scores_so_large_that_one_key_has_all_the_weight(dtype, shape, scale, size, slopes):
    """Scores of up to 1e31, the largest of a row (beyond 2^24 in units of ln 2) 100 and more above the others, whatever the rounding of the products:
    the result is that key's value and its gradient the sum of the rows' that chose it, and q and k get no gradient at all."""
    q_len, k_len, heads = SHAPES[shape]
    rows, keys = sum(q_len), sum(k_len or q_len)
    q, k, v = (size * _rand(rows, heads, 64, seed=11)).to(dtype), (size * _rand(keys, heads, 64, seed=12)).to(dtype), _rand(keys, heads, 64, seed=13, dtype=dtype)
    d_out = _rand(rows, heads, 64, seed=14, dtype=dtype)
    off = (R.offsets(q_len), None if k_len is None else R.offsets(k_len))
    how = dict(scale=scale, causal=True) | (dict(slopes=torch.full((heads,), 0.5, device=DEV)) if slopes else {})
    out, stats = ops.attention_docs(q, k, v, *off, **how)
    d_q, d_k, d_v = ops.attention_docs_backward(d_out, q, k, v, out, stats, *off, **how)[:3]
    want_v, sizes = torch.zeros(keys, heads, 64, dtype=torch.float64), torch.zeros(keys, heads, 64, dtype=torch.float64)
    a = b = 0
    plain = torch.zeros(rows, heads, dtype=torch.bool)  # rows whose choice no rounding can change
    chosen = torch.zeros(rows, heads, dtype=torch.long)
    for n, m in zip(q_len, k_len or q_len):
        x, y = q[a:a + n].cpu().double().transpose(0, 1), k[b:b + m].cpu().double().transpose(0, 1)
        hidden = torch.arange(m)[None] > torch.arange(n)[:, None] + (m - n)
        score = (x @ y.transpose(1, 2).contiguous() * scale).masked_fill(hidden, -math.inf)
        sure = 4 * 68 * 2.0 ** -24 * scale * (x.abs() @ y.abs().transpose(1, 2).contiguous()).amax(-1) + 100 + 0.5 * m
        top = score.topk(2, -1)
        plain[a:a + n] = ((top.values[..., 0] - top.values[..., -1] > sure) & (top.values[..., 0].abs() > 1.2e7)).t()
        chosen[a:a + n] = top.indices[..., 0].t() + b
        a, b = a + n, b + m
    assert plain.float().mean() > 0.9  # (a check of the inputs)
    at = chosen[..., None].expand(-1, -1, 64)
    picked = v.cpu().gather(0, at)
    # beyond 2^30 formed again, with a weight of 1: exact.  Below, the weight is 2^x, x up to 2^-25 of the score, over a sum of the same: fp32 a
    # reciprocal's and a product's rounding, bf16 the weight's in front of the product (1 needs none, 2^x does; the sum keeps it in fp32: 2^-8 of the
    # result) and the result's own (2^-8 of itself)
    again = plain & (stats[..., 0].abs() >= 2.0 ** 30).cpu()
    assert torch.equal(out.cpu()[again], picked[again])
    loose = 4 * 2.0 ** -24 if dtype == torch.float32 else 2 * 2.0 ** -8 + 2.0 ** -16
    assert ((out.cpu().double() - picked.double()).abs() <= loose * picked.double().abs())[plain].all()
    assert not d_q.cpu()[plain].any()
    d_out64 = d_out.cpu().double()
    want_v.scatter_add_(0, at, d_out64)
    sizes.scatter_add_(0, at, d_out64.abs())
    sure_keys = torch.ones(keys, heads, dtype=torch.bool)  # keys of documents and heads in which every row's choice is plain
    a = b = 0
    for n, m in zip(q_len, k_len or q_len):
        sure_keys[b:b + m] = plain[a:a + n].all(0)
        a, b = a + n, b + m
    assert sure_keys.any()
    assert not d_k.cpu()[sure_keys].any()
    bound = R.HALF[dtype] * want_v.abs() + rows * 2.0 ** -24 * sizes  # a sum of up to `rows` terms in fp32, rounded once
    assert ((d_v.cpu().double() - want_v).abs() <= bound)[sure_keys].all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_weights_of_large_scores_add_up_to_one(dtype, shape):
    """Scores of 2^16 to 2^26 (on both sides of what a maximum rounded to 24 bits can do), several keys of comparable weight: whatever each weight is, a row's add up
    to 1, so a document's d_v adds up to its d_out."""
    q_len, k_len, heads = SHAPES[shape]
    rows, keys = sum(q_len), sum(k_len or q_len)
    off = (R.offsets(q_len), None if k_len is None else R.offsets(k_len))
    for large in (2.0 ** 8, 2.0 ** 9, 2.0 ** 10, 2.0 ** 13):  # scores of large^2 x 8 / 8
        q, k = _rand(rows, heads, 64, seed=21, dtype=dtype), _rand(keys, heads, 64, seed=22, dtype=dtype)
        q[..., :8], k[..., :8] = large, large
        v, d_out = _rand(keys, heads, 64, seed=23, dtype=dtype), _rand(rows, heads, 64, seed=24, dtype=dtype)
        out, stats = ops.attention_docs(q, k, v, *off)
        d_q, d_k, d_v = ops.attention_docs_backward(d_out, q, k, v, out, stats, *off)
        assert all(torch.isfinite(t).all() for t in (out, d_q, d_k, d_v))
        a = b = 0
        for n, m in zip(q_len, k_len or q_len):
            got, want = d_v[b:b + m].double().sum(0), d_out[a:a + n].double().sum(0)
            # d_v's rounding; bf16: the weights' in front of the product, half a step of the maximum's size in log2 units in the exponent
            # (2^-7 ln 2 at 2^17, at most); sums of n and m terms in fp32, exponents of up to 64 in
            # units of 2^-24 on both sides
            terms = d_out[a:a + n].double().abs().sum(0)
            bound = R.HALF[dtype] * (d_v[b:b + m].double().abs().sum(0) + terms) + ((2.0 ** -7 if dtype == torch.bfloat16 else 0) + (n + m + 256) * 2.0 ** -24) * terms
            assert ((got - want).abs() <= bound).all(), (large, float(((got - want).abs() / bound).max()))
            a, b = a + n, b + m


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("far", [2.0 ** 8, 2.0 ** 14, 2.0 ** 18])
def test_weights_of_near_and_far_rows_over_the_same_keys(dtype, shape, far):
    """Every third row's scores are 2^12 or so, the others' 2^20 to 2^30: near rows, formed with far ones' keys, keep weights that add up to 1, so that a
    document's d_v adds up to its d_out."""
    q_len, k_len, heads = SHAPES[shape]
    rows, keys = sum(q_len), sum(k_len or q_len)
    off = (R.offsets(q_len), None if k_len is None else R.offsets(k_len))
    q, k = _rand(rows, heads, 64, seed=25, dtype=dtype), _rand(keys, heads, 64, seed=26, dtype=dtype)
    q[..., :8], k[..., :8] = 2.0 ** 6, 2.0 ** 6
    q[torch.arange(rows, device=DEV) % 3 != 0] *= far
    v, d_out = _rand(keys, heads, 64, seed=27, dtype=dtype), _rand(rows, heads, 64, seed=28, dtype=dtype)
    out, stats = ops.attention_docs(q, k, v, *off)
    d_q, d_k, d_v = ops.attention_docs_backward(d_out, q, k, v, out, stats, *off)
    assert all(torch.isfinite(t).all() for t in (out, d_q, d_k, d_v))
    a = b = 0
    for n, m in zip(q_len, k_len or q_len):
        got, want = d_v[b:b + m].double().sum(0), d_out[a:a + n].double().sum(0)
        terms = d_out[a:a + n].double().abs().sum(0)
        # d_v's and the weights' rounding, sums of n and m terms; a near row's scores (2^12, of terms of 2^15 and some 2^9 in all) in two orders of 64
        # products: each is off by 64 half steps of 2^15 x 2^-24 / 8 at most, in the exponent
        bound = R.HALF[dtype] * (d_v[b:b + m].double().abs().sum(0) + terms) + (2 * 64 * 2.0 ** -12 + (n + m + 256) * 2.0 ** -24) * terms
        assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())
        a, b = a + n, b + m


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale,cap", [(1.0, 1e6), (1.0, 1e8), (1.0, 1e10), (1.0, 1e14), (1.0, 1e20), (1e-20, 30.0), (1e-25, 1.0), (1e-30, 1e8)])
def test_caps_far_above_the_scale(dtype, scale, cap):
    """Scores of a quarter of the cap, where it bends them by 2 %, for quotients scale / cap down to 1e-38: powers of the quotient leave fp32."""
    rows, heads = 33, 2
    size = (0.25 * cap / scale / 64) ** 0.5  # all products positive: `big` of the error bound is the score itself
    q, k = ((size * (0.9 + 0.1 * torch.rand(rows, heads, 64, generator=torch.Generator().manual_seed(s)))).to(dtype).to(DEV) for s in (31, 32))
    v, d_out = _rand(rows, heads, 64, seed=33, dtype=dtype), _rand(rows, heads, 64, seed=34, dtype=dtype)
    out, stats = ops.attention_docs(q, k, v, R.offsets([rows]), cap=cap, scale=scale)
    ref = R.attention(q, k, v, [rows], cap=cap, scale=scale)
    ds = R.score_error(ref, rows, cap=cap, scale=scale)
    want = ref["stats"][..., 0]
    assert ((stats[..., 0].double().cpu() - want).abs() <= R.LOG2E * ds + 2.0 ** -23 * want.abs()).all()
    assert torch.isfinite(out).all()
    grads = ops.attention_docs_backward(d_out, q, k, v, out, stats, R.offsets([rows]), cap=cap, scale=scale)
    assert all(torch.isfinite(g).all() for g in grads)
    # whatever each weight is, a row's add up to 1
    bound = R.HALF[dtype] * (grads[2].double().abs().sum(0) + d_out.double().abs().sum(0)) + ((2.0 ** -7 if dtype == torch.bfloat16 else 0) + 400 * 2.0 ** -24) * d_out.double().abs().sum(0)
    assert ((grads[2].double().sum(0) - d_out.double().sum(0)).abs() <= bound).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale,cap", [(1e-30, 1e30), (1e-36, 30.0), (1e-20, 1e20), (1e-10, 1e29)])
def test_small_scores_under_far_caps(dtype, scale, cap):
    """Scores of up to 4 or so from a small scale and large products, below the cap by up to 29 powers of ten."""
    q_len = [40, 3]
    size = (1 / scale) ** 0.5 / 4
    q, k = (size * _rand(43, 2, 64, seed=35)).to(dtype), (size * _rand(43, 2, 64, seed=36)).to(dtype)
    v, d_out = _rand(43, 2, 64, seed=37, dtype=dtype), _rand(43, 2, 64, seed=38, dtype=dtype)
    out, stats = ops.attention_docs(q, k, v, R.offsets(q_len), causal=True, cap=cap, scale=scale)
    ref = R.attention(q, k, v, q_len, causal=True, cap=cap, scale=scale)
    ds = R.score_error(ref, 40, scale=scale, cap=cap)
    assert ((out.double().cpu() - ref["out"]).abs() <= R.out_bound(ref, v, dtype, 40, ds)).all()
    assert float(ref["stats"][..., 1].max()) > 2 and float((stats[..., 0].double().cpu() - ref["stats"][..., 0]).abs().max()) <= R.LOG2E * ds + 2.0 ** -20
    # (30 is no far cap: it bends a score of 4 by 0.6 %, so the weights are those of the definition with its cap, not those without one)
    ref = R.attention(q, k, v, q_len, causal=True, cap=cap, scale=scale, d_out=d_out)
    d_v = ops.attention_docs_backward(d_out, q, k, v, out, stats, R.offsets(q_len), causal=True, cap=cap, scale=scale)[2]
    bound = R.grad_bounds(ref, q, k, v, d_out, dtype, 40, ds, cap, scale=scale)["d_v"]
    assert ((d_v.double().cpu() - ref["d_v"]).abs() <= bound).all()


def test_rotary_of_more_rows_than_a_launch_has_workgroups_of_sixteen():
    rows, last = (1 << 28) + 5, 37
    x = torch.zeros(rows, 1, 16, dtype=torch.bfloat16, device=DEV)
    x[-last:] = _rand(last, 1, 16, seed=41, dtype=torch.bfloat16)
    x[:last] = _rand(last, 1, 16, seed=42, dtype=torch.bfloat16)
    ends = torch.cat([x[:last], x[-last:]]).clone()
    positions = torch.arange(rows, dtype=torch.int32, device=DEV)
    inv_freq = _rand(8, seed=43).abs()
    assert ops.rotary(x, positions, inv_freq, out=x) is x
    want = R.rotary(ends, torch.cat([positions[:last], positions[-last:]]), inv_freq, (8,))
    got = torch.cat([x[:last], x[-last:]]).double().cpu()
    # two products and their sum in fp32 with cos and sin good to 2^-22 (2 ulp, and an angle of 2^28 turns from a 64-bit product), rounded once
    assert ((got - want).abs() <= R.HALF[torch.bfloat16] * want.abs() + 8 * 2.0 ** -22 * ends.double().abs().max().cpu()).all()
    assert not x[last:-last].any()
