"""CPU: that the bounds which the packed-document attention's results are held to in the 2-norm would not let a mistake pass."""
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))
import docs_norms as N  # noqa: E402
import docs_reference as R  # noqa: E402

# mistake: the results that it reaches
ALL = ("out", "d_q", "d_k", "d_v")
MISTAKES = {"D": ("d_q", "d_k"), "the cap's slope": ("d_q", "d_k"), "the prefix": ALL, "the bias": ALL, "a key too many": ALL, "the last key": ALL,
            "a row": ("d_q", "d_k", "d_v", "d_slopes"), "the other heads of a group": ("d_k", "d_v")}


def _applies(mistake, case):
    q_len, k_len, heads, kv_heads, masks, _ = N.CASES[case]
    return {"the cap's slope": "cap" in masks, "the prefix": "prefix" in masks, "the bias": "slopes" in masks, "a key too many": "causal" in masks,
            "the other heads of a group": heads > kv_heads}.get(mistake, True)


@pytest.mark.parametrize("case", ["turns", "turns, capped", "alone, other keys", "few keys"])
def test_the_formulas_are_those_of_the_reference(case):
    q, k, v, d_out, how = N.inputs(case, torch.float32)
    kv, heads = N.compared(case)
    got = N.of_some(case, q, k, v, d_out, how)()
    if "slopes" in how:
        how["slopes"] = how["slopes"][heads]
    want = R.attention(q[:, heads], k[:, kv], v[:, kv], *N.CASES[case][:2], d_out=d_out[:, heads], **how)
    for name, t in got.items():
        assert N.off(t, want[name]) < 1e-12, name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", N.CASES)
def test_a_term_left_out_is_beyond_the_bounds(case, dtype):
    make = N.of_some(case, *N.inputs(case, dtype))
    want = make()
    for mistake, reached in MISTAKES.items():
        if not _applies(mistake, case):
            continue
        got = make(mistake)
        for name in reached:
            if name in want:
                assert N.off(got[name], want[name]) > 2 * N.TOLERANCE[dtype][name], (mistake, name)
    for name, t in want.items():
        assert N.off(torch.zeros_like(t), t) > 2 * N.TOLERANCE[dtype][name]


@pytest.mark.parametrize("case", ["few keys", "steep"])
def test_a_d_from_a_rounded_result_is_beyond_the_bounds_of_rows_with_few_keys(case):
    make = N.of_some(case, *N.inputs(case, torch.bfloat16, mean=16.0))
    want, got = make(), make("D from the rounded out")
    assert all(N.off(got[name], want[name]) > 2 * N.TOLERANCE[torch.bfloat16][name] for name in ("d_q", "d_k"))
