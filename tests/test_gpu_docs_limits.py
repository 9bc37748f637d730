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
