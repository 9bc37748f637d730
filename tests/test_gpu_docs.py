"""GPU: rotary positions and attention over packed documents (fc_rotary, fc_attention_docs) against 64-bit references on the CPU, at
the sizes and masks where they can go wrong.  Bounds: docs_reference.py."""
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


def _rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _within(name, got, want, bound):
    got, want = got.double().cpu(), want.double().cpu()
    assert got.shape == want.shape
    assert torch.isfinite(got).all(), name
    worst = ((got - want).abs() / bound).max() if got.numel() else torch.tensor(0.0)
    print(f"{name}: worst error over its bound {float(worst):.3f}", flush=True)
    assert float(worst) <= 1, (name, float(worst), float((got - want).abs().max()))


# ------------------------------------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,dim,sections", [(1, 1, 64, (8, 12, 12)), (196, 24, 64, (8, 12, 12)), (77, 3, 64, (32,)),
                                                     (1025, 5, 64, (0, 16)), (2051, 2, 16, (3, 4, 1)), (33, 7, 256, (40, 40, 40)),
                                                     (18001, 1, 64, (8, 12, 12))])
def test_rotary(dtype, interleaved, rows, heads, dim, sections):
    x = _rand(rows, heads, dim, seed=1, dtype=dtype)
    pairs = sum(sections)
    g = torch.Generator().manual_seed(2)
    positions = torch.randint(-5, 10_000_000, (rows, len(sections)), generator=g, dtype=torch.int32).to(DEV)
    inv_freq = (100.0 ** (-torch.arange(pairs) / pairs)).float().to(DEV)
    y = ops.rotary(x, positions, inv_freq, sections, interleaved=interleaved)
    want = R.rotary(x, positions, inv_freq, sections, interleaved)
    # cos and sin off by an ulp of 1 (the angle in turns is exact to 2^-25, times 2 pi) each and the two products' roundings
    bound = x.double().abs().max().cpu() * 16 * 2.0 ** -24 + R.HALF[dtype] * want.abs()
    _within("rotary", y, want, bound)
    back = ops.rotary(y, positions, inv_freq, sections, interleaved=interleaved, inverse=True)
    _within("inverse", back, R.rotary(y, positions, inv_freq, sections, interleaved, inverse=True),
            y.double().abs().max().cpu() * 16 * 2.0 ** -24 + R.HALF[dtype] * x.double().abs().max().cpu() * 2)
    assert torch.equal(back[..., 2 * pairs:], x[..., 2 * pairs:])


@pytest.mark.parametrize("dtype", TYPES)
def test_rotary_turns_q_and_k_of_a_fused_projection_in_place(dtype):
    rows, heads = 333, 6
    qkv = _rand(rows, 3 * heads * 64, seed=3, dtype=dtype)
    kept = qkv.clone()
    positions = torch.arange(rows * 2, dtype=torch.int32).view(rows, 2).to(DEV)
    inv_freq = torch.rand(32, generator=torch.Generator().manual_seed(4)).to(DEV)
    qk = qkv[:, :2 * heads * 64].view(rows, 2 * heads, 64)
    want = ops.rotary(qk, positions, inv_freq, (20, 12))
    assert ops.rotary(qk, positions, inv_freq, (20, 12), out=qk) is qk
    assert torch.equal(qk, want) and torch.equal(qkv[:, 2 * heads * 64:], kept[:, 2 * heads * 64:])


def test_rotary_is_its_own_gradient_by_differences():
    rows, heads = 9, 2
    x, dy = _rand(rows, heads, 64, seed=5), _rand(rows, heads, 64, seed=6)
    positions = torch.arange(rows, dtype=torch.int32).to(DEV)
    inv_freq = torch.rand(16, generator=torch.Generator().manual_seed(7)).to(DEV)
    dx = ops.rotary(dy, positions, inv_freq, inverse=True)
    for step in (1.0, 64.0):  # the rotation is linear: differences of any width are exact up to rounding
        e = torch.zeros_like(x)
        e[4, 1, 3] = step
        diff = ((ops.rotary(x + e, positions, inv_freq) - ops.rotary(x, positions, inv_freq)).double() * dy.double()).sum() / step
        # 128 values of up to 64, each rounded in the two results and in the angle's cos and sin
        assert abs(float(diff) - float(dx[4, 1, 3])) < 128 * 2.0 ** -24 * 64 * float(dy.abs().max())


# ---------------------------------------------------------------------------------------------------------------- attention
def _operands(q_rows, k_rows, heads, kv_heads, dtype, seed=0, layout="apart"):
    if layout == "fused":
        qkv = _rand(q_rows, (heads + 2 * kv_heads) * 64, seed=seed, dtype=dtype)
        q, k, v = (t.view(q_rows, -1, 64) for t in qkv.split([heads * 64, kv_heads * 64, kv_heads * 64], 1))
        return q, k, v
    if layout == "heads first":  # [heads, rows, 64] memory
        make = lambda n, h, s: _rand(h, n, 64, seed=s, dtype=dtype).transpose(0, 1)  # noqa: E731
    else:
        make = lambda n, h, s: _rand(n, h, 64, seed=s, dtype=dtype)  # noqa: E731
    return make(q_rows, heads, seed), make(k_rows, kv_heads, seed + 1), make(k_rows, kv_heads, seed + 2)


def _check_forward(q, k, v, q_len, k_len=None, **how):
    q_off = R.offsets(q_len)
    k_off = None if k_len is None else R.offsets(k_len)
    out, stats = ops.attention_docs(q, k, v, q_off, k_off, **how)
    how.pop("out", None)
    ref = R.attention(q, k, v, q_len, k_len, **how)
    keys = max(list(q_len if k_len is None else k_len) + [0])
    ds = R.score_error(ref, keys, how.get("slopes"), cap=how.get("cap", 0.0))
    covered = sum(q_len)
    _within("out", out[:covered], ref["out"][:covered], R.out_bound(ref, v, q.dtype, keys, ds)[:covered])
    got, want = stats.double().cpu()[:covered], ref["stats"][:covered]
    empty = want[..., 1] == 0
    assert torch.equal(got[..., 0] == -math.inf, empty) and (got[..., 1][empty] == 0).all() and (out[:covered].cpu()[empty] == 0).all()
    if (~empty).any():
        _within("stats max", got[..., 0][~empty], want[..., 0][~empty], R.LOG2E * ds + 2.0 ** -23 * want[..., 0][~empty].abs() + 1e-30)
        _within("stats sum", got[..., 1][~empty], want[..., 1][~empty], (2 * ds + (keys + 8) * 2.0 ** -24) * want[..., 1][~empty])
    return out, stats


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_len", [[1], [2], [31], [32], [33], [64], [65], [127, 1], [130], [0, 5, 0, 0, 3, 0], [1] * 70,
                                   [20, 0, 77, 4, 33, 1, 64], [197, 50], [0] * 100 + [7] + [0] * 90 + [3, 30], [3] * 62, [2] * 63,
                                   ([1, 0, 2] * 800)[:2300]])
def test_attention_of_documents(dtype, causal, q_len):
    q, k, v = _operands(sum(q_len), sum(q_len), 2, 2, dtype, seed=len(q_len), layout="fused")
    _check_forward(q, k, v, q_len, causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (6, 2), (12, 4), (5, 5)])
@pytest.mark.parametrize("layout", ["apart", "heads first"])
def test_attention_head_layouts(dtype, heads, kv_heads, layout):
    q_len = [23, 1, 40]
    q, k, v = _operands(64, 64, heads, kv_heads, dtype, seed=heads, layout=layout)
    _check_forward(q, k, v, q_len, causal=True, slopes=torch.rand(heads, generator=torch.Generator().manual_seed(1)).to(DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0, 2.0, 30.0])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("prefix", [False, True])
def test_attention_masks_caps_and_biases(dtype, cap, slopes, prefix):
    q_len = [45, 7, 0, 61, 12]
    q, k, v = _operands(125, 125, 4, 2, dtype, seed=9, layout="fused")
    pre = torch.tensor([20, 100, 3, 0, -4], dtype=torch.int32, device=DEV) if prefix else None
    _check_forward(q, k, v, q_len, causal=True, prefix=pre, cap=cap, slopes=torch.tensor([0.5, 0.0, 2.0, 0.01], device=DEV) if slopes else None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_len,k_len", [([1], [1]), ([1], [900]), ([1, 1, 1], [40, 700, 1]), ([3, 0, 5], [700, 9, 333]), ([1], [0]),
                                         ([4, 2], [2, 9]), ([40, 3], [7, 900]), ([1] * 40, list(range(1, 80, 2)))])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_of_few_rows_over_many_keys(dtype, q_len, k_len, causal):
    """Splits over the keys among them (few rows, mean length above 512); more queries than keys: causal rows that see nothing."""
    q, k, v = _operands(sum(q_len), sum(k_len), 6, 2, dtype, seed=3)
    _check_forward(q, k, v, q_len, k_len, causal=causal)


# enough rows for waves that work alone (a mean below 160), and for 128 rows that share a tile of keys (6 or 8 tiles of 128 rows a head: more
# than eight, bf16 three, workgroups per compute unit)
MANY = [(torch.float32, 352, [300, 17, 129, 0, 64, 250]), (torch.bfloat16, 144, [300, 17, 129, 0, 64, 250]),
        (torch.float32, 352, [600, 17, 129, 0, 250]), (torch.bfloat16, 144, [600, 17, 129, 0, 250])]


@pytest.mark.parametrize("dtype,heads,q_len", MANY)
def test_attention_four_wave_tiles(dtype, heads, q_len):
    """Enough rows that 128 of them share a tile of keys, in documents that end inside tiles."""
    rows, most = sum(q_len), max(q_len)
    q, k, v = _operands(rows, rows, heads, heads, dtype, seed=4, layout="fused")
    for causal in (False, True):
        out, stats = ops.attention_docs(q, k, v, R.offsets(q_len), causal=causal, cap=20.0)
        some = [0, 31, heads - 1]  # (the reference is slow: three heads of them)
        ref = R.attention(q[:, some], k[:, some], v[:, some], q_len, causal=causal, cap=20.0)
        ds = R.score_error(ref, most, cap=20.0)
        _within("out", out[:, some], ref["out"], R.out_bound(ref, v, dtype, most, ds))
        alone = [ops.attention_docs(q[:, h:h + 1], k[:, h:h + 1], v[:, h:h + 1], R.offsets(q_len), causal=causal, cap=20.0)[0] for h in some]
        for h, other in zip(some, alone):  # single waves form the same sums up to the order of the tiles
            _within("one head", other, ref["out"][:, some.index(h):some.index(h) + 1], R.out_bound(ref, v, dtype, most, ds)[:, :1])


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_rows_behind_the_last_document(dtype):
    q, k, v = _operands(90, 90, 2, 2, dtype, seed=5)
    q_off = R.offsets([10, 31])
    poison = torch.full_like(q, 7.0)
    out, stats = ops.attention_docs(q, k, v, q_off, out=poison)
    assert out is poison and (out[41:] == 7).all() and not (out[:41] == 7).all()
    own, own_stats = ops.attention_docs(q, k, v, q_off)
    assert torch.equal(own[:41], out[:41]) and (own[41:] == 0).all()
    for s in (stats, own_stats):
        assert (s[41:, :, 0] == -math.inf).all() and (s[41:, :, 1] == 0).all()
    nothing, s = ops.attention_docs(q, k, v, R.offsets([]))
    assert (nothing == 0).all() and (s[..., 1] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("k_len", [None, [90, 700]])
def test_attention_values_behind_a_mask_reach_nobody(dtype, bad, k_len):
    """Keys that a row does not see may hold anything: another document's, a later one's, one of no document."""
    q_len = [30, 50]
    keys = sum(k_len or q_len)
    q, k, v = _operands(80, keys + 5, 2, 1, dtype, seed=6)
    q_off, k_off = R.offsets(q_len), R.offsets(k_len or q_len)
    clean = ops.attention_docs(q, k, v, q_off, k_off, causal=True)
    for who in (k, v):
        kept = who.clone()
        who[(k_len or q_len)[0] - 1] = bad          # the first document's last key: only its last row sees it
        who[keys - 1, :, 5] = bad                   # the last key of all, in one dimension
        who[keys:] = bad                            # of no document
        out, stats = ops.attention_docs(q, k, v, q_off, k_off, causal=True)
        reached = torch.zeros(80, dtype=torch.bool, device=DEV)
        reached[29] = reached[79] = True
        fine = lambda t: torch.isfinite(t)  # noqa: E731
        assert fine(out[~reached]).all() and fine(stats[~reached]).all()
        scale = float(v[torch.isfinite(v)].abs().max())
        # the second pass adds in another order and keeps its weights in fp32: a rounding of them apart
        assert float((out[~reached].double() - clean[0][~reached].double()).abs().max()) <= 3 * R.HALF[dtype] * scale + 700 * 2.0 ** -24 * scale
        if math.isnan(bad) or who is v:  # (an infinite key may score -inf and weigh nothing)
            assert not fine(out[29]).all() and not fine(out[79]).all()
        who.copy_(kept)


# ---------------------------------------------------------------------------------------------------------------- gradients
def _check_gradients(q, k, v, q_len, k_len=None, seed=50, ref=None, **how):
    d_out = _rand(*q.shape, seed=seed, dtype=q.dtype)
    q_off, k_off = R.offsets(q_len), None if k_len is None else R.offsets(k_len)
    out, stats = ops.attention_docs(q, k, v, q_off, k_off, **how)
    slopes = how.get("slopes")
    grads = ops.attention_docs_backward(d_out, q, k, v, out, stats, q_off, k_off, slope_grad=slopes is not None, **how)
    ref = ref or R.attention(q, k, v, q_len, k_len, d_out=d_out, **how)
    keys = max(list(q_len if k_len is None else k_len) + [0])
    ds = R.score_error(ref, keys, slopes, cap=how.get("cap", 0.0))
    bounds = R.grad_bounds(ref, q, k, v, d_out, q.dtype, keys, ds, how.get("cap", 0.0), slopes)
    for name, got in zip(("d_q", "d_k", "d_v", "d_slopes"), grads):
        _within(name, got, ref[name], bounds[name])
    again = ops.attention_docs_backward(d_out, q, k, v, out, stats, q_off, k_off, slope_grad=slopes is not None, **how)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    return grads, ref, bounds


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_len", [[1], [2], [31], [32], [33], [65], [127, 1], [0, 5, 0, 0, 3, 0], [1] * 70, [20, 0, 77, 4, 33, 1, 64],
                                   [0] * 100 + [7] + [0] * 90 + [3, 30], [3] * 62, [2] * 63, ([1, 0, 2] * 800)[:2300]])
def test_gradients_of_documents(dtype, causal, q_len):
    q, k, v = _operands(sum(q_len), sum(q_len), 2, 2, dtype, seed=len(q_len), layout="fused")
    grads, _, _ = _check_gradients(q, k, v, q_len, causal=causal)
    if max(q_len) == 1:  # one key: its weight is 1 whatever the score
        assert not grads[0].any() and not grads[1].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(3, 1), (6, 2), (5, 5)])
@pytest.mark.parametrize("layout", ["apart", "heads first"])
def test_gradients_of_shared_heads(dtype, heads, kv_heads, layout):
    q, k, v = _operands(64, 64, heads, kv_heads, dtype, seed=heads, layout=layout)
    _check_gradients(q, k, v, [23, 1, 40], causal=True, slopes=torch.rand(heads, generator=torch.Generator().manual_seed(1)).to(DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0, 2.0, 30.0])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("prefix", [False, True])
def test_gradients_of_masks_caps_and_biases(dtype, cap, slopes, prefix):
    q_len = [45, 7, 0, 61, 12]
    q, k, v = _operands(125, 125, 4, 2, dtype, seed=9, layout="fused")
    pre = torch.tensor([20, 100, 3, 0, -4], dtype=torch.int32, device=DEV) if prefix else None
    _check_gradients(q, k, v, q_len, causal=True, prefix=pre, cap=cap, slopes=torch.tensor([0.5, 0.0, 2.0, 0.01], device=DEV) if slopes else None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_len,k_len", [([1], [900]), ([1, 1, 1], [40, 700, 1]), ([3, 0, 5], [70, 9, 333]), ([1], [0]), ([4, 2], [2, 9]),
                                         ([40, 3], [7, 300]), ([100, 30], [1, 1]), ([0, 0], [5, 60])])
@pytest.mark.parametrize("causal", [False, True])
def test_gradients_of_other_numbers_of_keys(dtype, q_len, k_len, causal):
    q, k, v = _operands(sum(q_len), sum(k_len), 6, 2, dtype, seed=3)
    _check_gradients(q, k, v, q_len, k_len, causal=causal)


@pytest.mark.parametrize("dtype,heads,q_len", MANY)
def test_gradients_four_wave_tiles(dtype, heads, q_len):
    rows, most = sum(q_len), max(q_len)
    q, k, v = _operands(rows, rows, heads, heads, dtype, seed=4, layout="fused")
    d_out = _rand(rows, heads, 64, seed=5, dtype=dtype)
    for causal in (False, True):
        out, stats = ops.attention_docs(q, k, v, R.offsets(q_len), causal=causal)
        grads = ops.attention_docs_backward(d_out, q, k, v, out, stats, R.offsets(q_len), causal=causal)
        some = [0, heads - 1]
        ref = R.attention(q[:, some], k[:, some], v[:, some], q_len, causal=causal, d_out=d_out[:, some])
        bounds = R.grad_bounds(ref, q[:, some], k[:, some], v[:, some], d_out[:, some], dtype, most, R.score_error(ref, most))
        for name, got in zip(("d_q", "d_k", "d_v"), grads):
            _within(name, got[:, some], ref[name], bounds[name])


def _some_heads(q, k, v, d_out, q_len, k_len, kv_heads, **how):
    """The reference of the given key heads' query heads alone (it is slow), with what to take of the operators' results."""
    group = q.shape[1] // k.shape[1]
    heads = [h * group + g for h in kv_heads for g in range(group)]
    if how.get("slopes") is not None:
        how["slopes"] = how["slopes"][heads]
    keys, (q, k, v, d_out) = max(k_len or q_len), (q[:, heads], k[:, kv_heads], v[:, kv_heads], d_out[:, heads])
    ref = R.attention(q, k, v, q_len, k_len, d_out=d_out, **how)
    ds = R.score_error(ref, keys, how.get("slopes"), cap=how.get("cap", 0.0))
    return ref, R.out_bound(ref, v, q.dtype, keys, ds), R.grad_bounds(ref, q, k, v, d_out, q.dtype, keys, ds, how.get("cap", 0.0), how.get("slopes")), heads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,cross,how", [(24, 24, False, {}), (48, 24, False, dict(causal=True, cap=3.0)),
                                                      (30, 30, True, dict(causal=True, slopes=True, prefix=True)),
                                                      (27, 27, True, dict(cap=20.0, slopes=True))])
def test_many_short_documents(dtype, heads, kv_heads, cross, how):
    """More than two waves per compute unit, each alone with its rows or keys: documents of 0 to 70 tokens."""
    g = torch.Generator().manual_seed(31)
    q_len = torch.randint(0, 71, (22,), generator=g).tolist() + [70, 0, 1]
    k_len = torch.randint(0, 71, (22,), generator=g).tolist() + [1, 70, 0] if cross else None
    how = dict(how)
    if how.get("prefix"):
        how["prefix"] = torch.randint(-3, 60, (25,), generator=g, dtype=torch.int32).to(DEV)
    if how.get("slopes"):
        how["slopes"] = (0.3 * torch.rand(heads, generator=g)).to(DEV)
    q, k, v = _operands(sum(q_len), sum(k_len or q_len), heads, kv_heads, dtype, seed=32, layout="apart" if cross else "fused")
    d_out = _rand(*q.shape, seed=35, dtype=dtype)
    q_off, k_off = R.offsets(q_len), R.offsets(k_len) if cross else None
    out, stats = ops.attention_docs(q, k, v, q_off, k_off, **how)
    grads = ops.attention_docs_backward(d_out, q, k, v, out, stats, q_off, k_off, slope_grad="slopes" in how, **how)
    some = [0, kv_heads - 1]
    ref, out_bound, bounds, of = _some_heads(q, k, v, d_out, q_len, k_len, some, **how)
    _within("out", out[:, of], ref["out"], out_bound)
    for name, got, which in zip(("d_q", "d_k", "d_v"), grads, (of, some, some)):
        _within(name, got[:, which], ref[name], bounds[name])
    if "slopes" in how:
        _within("d_slopes", grads[3][of], ref["d_slopes"], bounds["d_slopes"])


@pytest.mark.parametrize("dtype", TYPES)
def test_many_short_documents_with_values_behind_masks(dtype):
    """NaN and infinities of keys that a row does not see reach nobody, where a wave works alone."""
    q_len = [29, 40, 3, 64] * 6
    rows, heads = sum(q_len), 24
    q, k, v = _operands(rows, rows, heads, heads, dtype, seed=33, layout="fused")
    off, d_out = R.offsets(q_len), _rand(rows, heads, 64, seed=34, dtype=dtype)
    some, start = [0, 23], 29 + 40  # (start: the third document, of three rows)
    ref, out_bound, bounds, _ = _some_heads(q, k, v, d_out, q_len, None, some, causal=True)
    k[start + 1], v[start + 1] = math.nan, math.inf  # seen by the document's last two rows alone
    out, stats = ops.attention_docs(q, k, v, off, causal=True)
    grads = ops.attention_docs_backward(d_out, q, k, v, out, stats, off, causal=True)
    reached = torch.zeros(rows, dtype=torch.bool, device=DEV)
    reached[start + 1:start + 3] = True
    assert not torch.isfinite(out[reached]).all() and torch.isfinite(stats[~reached]).all()
    own = reached.clone()
    own[start] = True  # keys that a reached row sees
    for name, got, bound, kept in (("out", out, out_bound, ~reached), ("d_q", grads[0], bounds["d_q"], ~reached),
                                   ("d_k", grads[1], bounds["d_k"], ~own), ("d_v", grads[2], bounds["d_v"], ~own)):
        kept = kept.cpu()
        _within(name, got[:, some].cpu()[kept], ref[name].cpu()[kept], bound.cpu().expand(rows, len(some), 64)[kept])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [False, True])
def test_gradients_of_few_keys_with_many_rows(dtype, bad):
    """One key head of six query heads: the rows of a key are cut into parts."""
    q_len, heads = [300, 1, 219], 6
    rows = sum(q_len)
    q, k, v = _operands(rows, rows, heads, 1, dtype, seed=13, layout="fused")
    how = dict(causal=True, cap=9.0, slopes=torch.full((heads,), 0.02, device=DEV))
    if not bad:
        _check_gradients(q, k, v, q_len, **how)
        return
    q_off, d_out = R.offsets(q_len), _rand(rows, heads, 64, seed=14, dtype=dtype)
    out, stats = ops.attention_docs(q, k, v, q_off, **how)
    clean = ops.attention_docs_backward(d_out, q, k, v, out, stats, q_off, **how)
    d_out[299] = math.nan  # the first document's last row: sees all of its keys, and no other
    got = ops.attention_docs_backward(d_out, q, k, v, out, stats, q_off, **how)
    assert not torch.isfinite(got[2][:300]).any() and torch.isfinite(got[0][:299]).all()
    for a, b in zip(got, clean):
        assert torch.isfinite(a[300:]).all()
        # done again key by key, with weights in fp32
        assert float((a[300:].double() - b[300:].double()).abs().max()) <= 8 * R.HALF[dtype] * float(b.double().abs().max()) + 1e-4


def test_gradients_by_differences():
    """Central differences of the 64-bit forward against the kernels' gradients."""
    q_len, how = [5, 14], dict(causal=True, cap=3.0, prefix=torch.tensor([2, 9], dtype=torch.int32, device=DEV),
                               slopes=torch.tensor([0.3, 0.05], device=DEV))
    q, k, v = _operands(19, 19, 2, 1, torch.float32, seed=21)
    grads, ref, bounds = _check_gradients(q, k, v, q_len, seed=50, **how)
    d_out = _rand(*q.shape, seed=50).double().cpu()
    ops64 = {"d_q": q.double().cpu(), "d_k": k.double().cpu(), "d_v": v.double().cpu(), "d_slopes": how["slopes"].double().cpu()}
    step = 1e-4

    def loss(x):
        return float((R.attention(x["d_q"], x["d_k"], x["d_v"], q_len, **(how | {"slopes": x["d_slopes"]}))["out"] * d_out).sum())
    for name, got in zip(ops64, grads):
        flat = got.double().cpu().reshape(-1)
        for at in (0, flat.numel() // 2, flat.numel() - 1):
            moved = []
            for sign in (step, -step):
                x = {n: t.clone() for n, t in ops64.items()}
                x[name].view(-1)[at] += sign
                moved.append(loss(x))
            # truncation: step^2 times a third derivative of order 100; rounding of the 64-bit sums: 1e-13 / step
            assert abs((moved[0] - moved[1]) / (2 * step) - float(flat[at])) <= float(bounds[name].reshape(-1)[at]) + 1e-5


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_go_into_the_columns_of_a_fused_projection(dtype):
    rows, heads = 90, 2
    q, k, v = _operands(rows, rows, heads, heads, dtype, seed=5, layout="fused")
    q_off, d_out = R.offsets([10, 31]), _rand(rows, heads, 64, seed=6, dtype=dtype)
    out, stats = ops.attention_docs(q, k, v, q_off)
    own = ops.attention_docs_backward(d_out, q, k, v, out, stats, q_off)
    assert all((g[41:] == 0).all() for g in own)
    d_qkv = torch.full((rows, 3 * heads * 64), 7.0, dtype=dtype, device=DEV)
    into = [t.view(rows, heads, 64) for t in d_qkv.split(heads * 64, 1)]
    got = ops.attention_docs_backward(d_out, q, k, v, out, stats, q_off, d_q=into[0], d_k=into[1], d_v=into[2])
    assert all(a.data_ptr() == b.data_ptr() and torch.equal(a[:41], c[:41]) for a, b, c in zip(got, into, own))
    assert (d_qkv[41:] == 7).all()
    part = ops.attention_docs_backward(d_out, q, k, v, out, stats, q_off, d_k=into[1])
    assert (part[0][41:] == 0).all() and (part[1][41:] == 7).all() and (part[2][41:] == 0).all()
    none = ops.attention_docs_backward(d_out, q, k, v, out, stats, R.offsets([]), slopes=torch.ones(heads, device=DEV), slope_grad=True)
    assert not any(g.any() for g in none)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_gradients_of_what_nobody_sees(dtype, bad):
    """NaN and infinities in rows and keys of other documents, of later keys and of no document reach no gradient that does not see them."""
    q_len, rows = [30, 50], 85
    q, k, v = _operands(rows, rows, 2, 1, dtype, seed=6)
    d_out = _rand(rows, 2, 64, seed=7, dtype=dtype)
    q_off = R.offsets(q_len)
    out, stats = ops.attention_docs(q, k, v, q_off, causal=True)
    clean = ops.attention_docs_backward(d_out, q, k, v, out, stats, q_off, causal=True)
    for who in (q, k, v, d_out):
        kept = who.clone()
        who[0] = bad    # the first document's first row / key: its whole document may be reached, the second one may not
        who[80:] = bad  # of no document
        o2, s2 = ops.attention_docs(q, k, v, q_off, causal=True)
        got = ops.attention_docs_backward(d_out, q, k, v, o2, s2, q_off, causal=True)
        for a, b in zip(got, clean):
            assert torch.isfinite(a[30:]).all()
            # the second pass adds in another order and keeps its weights in fp32
            assert float((a[30:].double() - b[30:].double()).abs().max()) <= 8 * R.HALF[dtype] * float(b.double().abs().max()) + 1e-4
        who.copy_(kept)
    # a later row's dO reaches its own gradients and what it sees, no earlier row's d_q
    d_out[29] = bad
    got = ops.attention_docs_backward(d_out, q, k, v, out, stats, q_off, causal=True)
    assert torch.isfinite(got[0][:29]).all() and torch.isfinite(got[0][30:]).all() and not torch.isfinite(got[2][:30]).all()
    assert all(torch.isfinite(g[30:]).all() for g in got)


def test_a_block_of_video_tokens_forward_backward_and_captured():
    """Rotary positions on q and k in place, attention over packed clips, its gradients, and the rotation taken back: against autograd in
    64 bits, and replayed from a captured graph."""
    frames, side, heads = [2, 5, 3], 3, 2
    rows = sum(frames) * side * side
    q_len = [f * side * side for f in frames]
    place = torch.cat([torch.stack(torch.meshgrid(torch.arange(f), torch.arange(side), torch.arange(side), indexing="ij"), -1).view(-1, 3)
                       for f in frames]).to(torch.int32).to(DEV)
    inv_freq = (100.0 ** (-torch.arange(32) / 32)).to(DEV)
    src = _rand(rows, 3 * heads * 64, seed=31)
    d_out = _rand(rows, heads, 64, seed=32)
    q_off = R.offsets(q_len)
    D = heads * 64

    def block(qkv):
        qk = qkv[:, :2 * D].view(rows, 2 * heads, 64)
        ops.rotary(qk, place, inv_freq, (8, 12, 12), out=qk)
        q, k, v = (t.view(rows, heads, 64) for t in qkv.split(D, 1))
        out, stats = ops.attention_docs(q, k, v, q_off, cap=20.0)
        d_qkv = torch.empty_like(qkv)
        d_q, d_k, d_v = (t.view(rows, heads, 64) for t in d_qkv.split(D, 1))
        ops.attention_docs_backward(d_out, q, k, v, out, stats, q_off, cap=20.0, d_q=d_q, d_k=d_k, d_v=d_v)
        d_qk = d_qkv[:, :2 * D].view(rows, 2 * heads, 64)
        ops.rotary(d_qk, place, inv_freq, (8, 12, 12), inverse=True, out=d_qk)
        return out, d_qkv

    out, d_qkv = block(src.clone())
    x = src.double().cpu()
    turned = torch.cat([R.rotary(x[:, :2 * D].view(rows, 2 * heads, 64), place, inv_freq, (8, 12, 12)).reshape(rows, 2 * D), x[:, 2 * D:]], 1)
    q, k, v = (t.reshape(rows, heads, 64) for t in turned.split(D, 1))
    ref = R.attention(q, k, v, q_len, d_out=d_out, cap=20.0)
    ds = R.score_error(ref, 45, cap=20.0) + 2.0 ** -24 * 64 * ref["big"]  # q and k carry the rotation's own error: 32 ulp of each
    _within("out", out, ref["out"], R.out_bound(ref, v, torch.float32, 45, ds))
    bounds = R.grad_bounds(ref, q, k, v, d_out, torch.float32, 45, ds, cap=20.0)
    back = [R.rotary(ref[n], place, inv_freq, (8, 12, 12), inverse=True) for n in ("d_q", "d_k")]
    for n, got, want in zip(("d_q", "d_k", "d_v"), d_qkv.split(D, 1), back + [ref["d_v"]]):
        # turned back: a value takes both of its pair's errors, and the rotation's own
        bound = 2 * bounds[n].max() + 32 * 2.0 ** -24 * want.abs().max()
        _within(n, got.reshape(rows, heads, 64), want, bound)

    side_stream = torch.cuda.Stream()
    side_stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side_stream):
        buf = src.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side_stream):
            got = block(buf)
        for turn in range(3):
            buf.copy_(src)
            for t in got:
                t.zero_()
            graph.replay()
            eager = block(src.clone())
            side_stream.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, eager)) and torch.equal(got[0], out) and torch.equal(got[1], d_qkv)
    torch.cuda.current_stream().wait_stream(side_stream)


def test_attention_on_another_stream_and_in_a_graph():
    q_len, k_len = [1, 1, 1], [300, 2000, 5]
    q, k, v = _operands(3, 2305, 6, 2, torch.bfloat16, seed=8)
    q_off, k_off = R.offsets(q_len), R.offsets(k_len)
    eager = ops.attention_docs(q, k, v, q_off, k_off, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.attention_docs(q, k, v, q_off, k_off, causal=True)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, other))
        graphs = []
        for _ in range(2):  # two captured graphs: each has its own workspace
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                got = ops.attention_docs(q, k, v, q_off, k_off, causal=True)
            graphs.append((graph, got))
        for turn in range(3):
            k_off.copy_(R.offsets([300 - turn, 2000, 5 + turn]))  # lengths are read on the device: a replay follows them
            want = ops.attention_docs(q, k, v, q_off, k_off, causal=True)
            for graph, got in graphs:
                for t in got:
                    t.zero_()
                graph.replay()
            side.synchronize()
            for _, got in graphs:
                assert all(torch.equal(a, b) for a, b in zip(want, got))
    torch.cuda.current_stream().wait_stream(side)


def test_attention_agrees_with_the_fixed_length_operator():
    n, S, heads = 3, 77, 8
    for dtype in TYPES:
        qkv = _rand(n * S, 3 * heads * 64, seed=11, dtype=dtype)
        fixed = ops.attention(qkv, n, S, heads, causal=True).view(n * S, heads, 64)
        q, k, v = (t.view(n * S, heads, 64) for t in qkv.split(heads * 64, 1))
        packed, _ = ops.attention_docs(q, k, v, R.offsets([S] * n), causal=True)
        ref = R.attention(q, k, v, [S] * n, causal=True)
        bound = R.out_bound(ref, v, dtype, S, R.score_error(ref, S))
        _within("fixed", fixed, ref["out"], bound)
        _within("packed", packed, ref["out"], bound)


def test_attention_offsets_beyond_32_bits():
    """A cache whose last keys lie more than 2^32 bytes behind its first."""
    keys = (1 << 32) // 128 // 8 + 1000  # 8 key heads of 128 bytes
    cache = torch.empty(keys, 8, 64, dtype=torch.bfloat16, device=DEV)
    cache[:64] = _rand(64, 8, 64, seed=1, dtype=torch.bfloat16)
    cache[-700:] = _rand(700, 8, 64, seed=2, dtype=torch.bfloat16)
    q = _rand(2, 8, 64, seed=3, dtype=torch.bfloat16)
    k_off = torch.tensor([keys - 700, keys - 300, keys], dtype=torch.int32, device=DEV)
    out, _ = ops.attention_docs(q, cache, cache, R.offsets([1, 1]), k_off)
    tail = cache[-700:].clone()
    ref = R.attention(q, tail, tail, [1, 1], [400, 300])
    _within("far", out, ref["out"], R.out_bound(ref, tail, torch.bfloat16, 400, R.score_error(ref, 400)))


@pytest.mark.parametrize("dtype", TYPES)
def test_extreme_caps_scales_and_slopes(dtype):
    q_len = [40, 3, 33]
    q, k, v = _operands(76, 76, 2, 2, dtype, seed=60)
    # a cap so small that its reciprocal leaves fp32: every score is 0 up to 1e-35, the weights are equal
    flat = R.attention(torch.zeros_like(q), k, v, q_len, causal=True)
    even = R.out_bound(flat, v, dtype, 40, 2.0 ** -24)
    for how in (dict(cap=1e-36), dict(scale=1e-36), dict(cap=1e30, scale=1e-36)):
        out, stats = ops.attention_docs(q, k, v, R.offsets(q_len), causal=True, **how)
        _within(str(how), out, flat["out"], even)
        grads = ops.attention_docs_backward(torch.ones_like(out), q, k, v, out, stats, R.offsets(q_len), causal=True, **how)
        assert all(torch.isfinite(g).all() for g in grads)
    # a slope so steep that every query sees its own place alone (weights below 2^-1000 beside 1)
    out, stats = ops.attention_docs(q, k, v, R.offsets(q_len), slopes=torch.tensor([1e4, 3e30], device=DEV))
    assert torch.equal(out, v) and (stats[..., 1] == 1).all()
    # slopes of the other sign: the first key is the farthest, and alone (distances within a document differ by one)
    out, _ = ops.attention_docs(q, k, v, R.offsets(q_len), causal=True, slopes=torch.full((2,), -1e5, device=DEV))
    firsts = torch.tensor([0] * 40 + [40] * 3 + [43] * 33, device=DEV)
    assert torch.equal(out, v[firsts])


@pytest.mark.parametrize("dtype", TYPES)
def test_no_queries_or_no_rows_at_all(dtype):
    k = _rand(70, 2, 64, seed=61, dtype=dtype)
    q = torch.empty(0, 4, 64, dtype=dtype, device=DEV)
    slopes = torch.ones(4, device=DEV)
    for keys, docs in ((k, 3), (k[:0], 3), (k[:0], 0)):
        q_off = torch.zeros(docs + 1, dtype=torch.int32, device=DEV)
        k_off = R.offsets([30, 0, 40]) if len(keys) else q_off
        out, stats = ops.attention_docs(q, keys, keys, q_off, k_off, slopes=slopes)
        assert out.shape == (0, 4, 64) and stats.shape == (0, 4, 2)
        d_q, d_k, d_v, d_slopes = ops.attention_docs_backward(out, q, keys, keys, out, stats, q_off, k_off, slopes=slopes, slope_grad=True)
        assert d_q.shape == q.shape and (d_k == 0).all() and (d_v == 0).all() and (d_slopes == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_into_its_own_queries(dtype):
    """out may be q: each row is read by the workgroup that writes it, before it does (splits over the keys among them)."""
    for q_len, k_len in (([40, 77, 3], None), ([1, 2], [900, 1100])):
        q, k, v = _operands(sum(q_len), sum(k_len or q_len), 6, 2, dtype, seed=62)
        offs = (R.offsets(q_len), None if k_len is None else R.offsets(k_len))
        want, stats = ops.attention_docs(q, k, v, *offs, causal=True)
        got, own = ops.attention_docs(q, k, v, *offs, causal=True, out=q)
        assert got is q and torch.equal(got, want) and torch.equal(own, stats)


def test_calls_on_two_streams_at_once():
    """Scratch is each call's own: splits and row tables of calls that overlap in time."""
    q_len, k_len = [1] * 6, [700, 2000, 1, 900, 1500, 40]
    sets = []
    for seed in (70, 71):
        q, k, v = _operands(6, sum(k_len), 6, 2, torch.bfloat16, seed=seed)
        sets.append((q, k, v, _rand(6, 6, 64, seed=seed + 5, dtype=torch.bfloat16)))
    offs = (R.offsets(q_len), R.offsets(k_len))

    def both(q, k, v, d_out):
        out, stats = ops.attention_docs(q, k, v, *offs, causal=True)
        return (out, stats) + ops.attention_docs_backward(d_out, q, k, v, out, stats, *offs, causal=True)
    want = [both(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(both(*s))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0, 50.0])
def test_results_in_the_norm(dtype, cap):
    """Errors of single values may reach their bounds; all of them together may not: in the 2-norm they add up like noise.  A result's
    roundings (bf16: its own, its weights', d_out and out as the gradient reads them: 4 of at most 2^-8, a third of that in the mean square, and
    twice as much where differences dP - D take something away) stay below 6 x 2^-8 of the norm; fp32 sums of up to 400 terms below 400 x 2^-24."""
    q_len = [160, 40, 200]
    q, k, v = _operands(400, 400, 4, 2, dtype, seed=80, layout="fused")
    d_out = _rand(400, 4, 64, seed=81, dtype=dtype)
    out, stats = ops.attention_docs(q, k, v, R.offsets(q_len), causal=True, cap=cap)
    grads = ops.attention_docs_backward(d_out, q, k, v, out, stats, R.offsets(q_len), causal=True, cap=cap)
    ref = R.attention(q, k, v, q_len, causal=True, cap=cap, d_out=d_out)
    for name, got in (("out", out), ("d_q", grads[0]), ("d_k", grads[1]), ("d_v", grads[2])):
        want = ref[name].to(DEV).double()
        far = float((got.double() - want).norm() / want.norm())
        assert far <= (6 * R.HALF[dtype] if dtype == torch.bfloat16 else 400 * 2.0 ** -24), (name, far)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,how", [(22, 22, {}), (44, 22, dict(causal=True, slopes=True)), (26, 26, dict(causal=True, prefix=True, cap=8.0))])
def test_uneven_documents_in_the_order_of_their_ways(dtype, heads, kv_heads, how):
    """More than two workgroups per compute unit take their tiles longest way first, those that reach into the next document before all: every
    tile exactly once, rows in front of the first and behind the last document among them."""
    g = torch.Generator().manual_seed(90)
    q_len = [37, 400, 0, 5, 500, 129, 1]
    n, lead, rows = sum(q_len), 5, sum(q_len) + 5 + 60
    how = dict(how)
    if how.get("prefix"):
        how["prefix"] = torch.randint(-3, 300, (7,), generator=g, dtype=torch.int32).to(DEV)
    if how.get("slopes"):
        how["slopes"] = (0.1 * torch.rand(heads, generator=g)).to(DEV)
    q, k, v = _operands(rows, rows, heads, kv_heads, dtype, seed=91)
    d_out, off = _rand(rows, heads, 64, seed=92, dtype=dtype), R.offsets(q_len) + lead
    out, stats = ops.attention_docs(q, k, v, off, **how)
    grads = ops.attention_docs_backward(d_out, q, k, v, out, stats, off, slope_grad="slopes" in how, **how)
    own = slice(lead, lead + n)
    some = [0, kv_heads - 1]
    ref, out_bound, bounds, of = _some_heads(q[own], k[own], v[own], d_out[own], q_len, None, some, **how)
    _within("out", out[own][:, of], ref["out"], out_bound)
    for name, got, which in zip(("d_q", "d_k", "d_v"), grads, (of, some, some)):
        _within(name, got[own][:, which], ref[name], bounds[name])
        assert (got[:lead] == 0).all() and (got[lead + n:] == 0).all()
    assert (out[:lead] == 0).all() and (out[lead + n:] == 0).all() and (stats[lead + n:, :, 1] == 0).all() and (stats[:lead, :, 1] == 0).all()
    if "slopes" in how:
        _within("d_slopes", grads[3][of], ref["d_slopes"], bounds["d_slopes"])


@pytest.mark.parametrize("dtype", TYPES)
def test_thousands_of_documents_and_runs_of_empty_ones(dtype):
    """The search for a row's (key's) document in more than 2048 of them, with more empty ones in a row than a wave looks at in one step."""
    q_len = [3] * 300 + [0] * 200 + [2, 0, 0, 1] * 400 + [0] * 70 + [5] * 100 + [0] * 65
    rows = sum(q_len)
    q, k, v = _operands(rows, rows, 9, 9, dtype, seed=95, layout="fused")
    d_out, off = _rand(rows, 9, 64, seed=96, dtype=dtype), R.offsets(q_len)
    out, stats = ops.attention_docs(q, k, v, off, causal=True)
    grads = ops.attention_docs_backward(d_out, q, k, v, out, stats, off, causal=True)
    ref, out_bound, bounds, _ = _some_heads(q, k, v, d_out, q_len, None, [4], causal=True)
    _within("out", out[:, [4]], ref["out"], out_bound)
    for name, got in zip(("d_q", "d_k", "d_v"), grads):
        _within(name, got[:, [4]], ref[name], bounds[name])
    one, one_stats = ops.attention_docs(q[:, 4:5], k[:, 4:5], v[:, 4:5], off, causal=True)  # (few workgroups: another shape)
    _within("one head", one, ref["out"], out_bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,heads", [(70, 3), (3000, 8)])
def test_queries_without_any_keys(dtype, rows, heads):
    q, none = _rand(rows, heads, 64, seed=97, dtype=dtype), torch.empty(0, heads, 64, dtype=dtype, device=DEV)
    q_off, k_off = R.offsets([rows // 2, 0, rows - rows // 2]), torch.zeros(4, dtype=torch.int32, device=DEV)
    out, stats = ops.attention_docs(q, none, none, q_off, k_off, causal=True)
    assert (out == 0).all() and (stats[..., 0] == -math.inf).all() and (stats[..., 1] == 0).all()
    d_q, d_k, d_v = ops.attention_docs_backward(torch.ones_like(q), q, none, none, out, stats, q_off, k_off, causal=True)
    assert (d_q == 0).all() and d_k.shape == d_v.shape == none.shape
