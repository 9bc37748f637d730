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
                                   [20, 0, 77, 4, 33, 1, 64], [197, 50]])
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


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_four_wave_tiles(dtype):
    """Enough rows that 128 of them share a tile of keys, in documents that end inside tiles."""
    q_len = [300, 17, 129, 0, 64, 250]
    rows = sum(q_len)
    heads = 64  # 6 tiles of 128 rows x 64 heads: more than one workgroup per compute unit
    q, k, v = _operands(rows, rows, heads, heads, dtype, seed=4, layout="fused")
    for causal in (False, True):
        out, stats = ops.attention_docs(q, k, v, R.offsets(q_len), causal=causal, cap=20.0)
        some = [0, 31, 63]  # (the reference is slow: three heads of them)
        ref = R.attention(q[:, some], k[:, some], v[:, some], q_len, causal=causal, cap=20.0)
        ds = R.score_error(ref, 300, cap=20.0)
        _within("out", out[:, some], ref["out"], R.out_bound(ref, v, dtype, 300, ds))
        alone = [ops.attention_docs(q[:, h:h + 1], k[:, h:h + 1], v[:, h:h + 1], R.offsets(q_len), causal=causal, cap=20.0)[0] for h in some]
        for h, other in zip(some, alone):  # single waves form the same sums up to the order of the tiles
            _within("one head", other, ref["out"][:, some.index(h):some.index(h) + 1], R.out_bound(ref, v, dtype, 300, ds)[:, :1])


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
