"""GPU: results of the packed-document attention in the 2-norm, in every shape of a workgroup, against the formulas in 64 bits (docs_norms.py: the cases,
the bounds and why; test_docs_norms.py: what they would not let pass)."""
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, str(Path(__file__).resolve().parent))
import docs_norms as N  # noqa: E402
import docs_reference as R  # noqa: E402
from fitclip_amd import ops  # noqa: E402


def _results(case, q, k, v, d_out, how):
    q_len, k_len = N.CASES[case][:2]
    q, k, v, d_out = (t.cuda() for t in (q, k, v, d_out))
    how = {n: x.cuda() if torch.is_tensor(x) else x for n, x in how.items()}
    off = (R.offsets(q_len), None if k_len is None else R.offsets(k_len))
    out, stats = ops.attention_docs(q, k, v, *off, **how)
    grads = ops.attention_docs_backward(d_out, q, k, v, out, stats, *off, slope_grad="slopes" in how, **how)
    kv, heads = N.compared(case)
    return {n: t[heads] if n == "d_slopes" else t[:, kv if n in ("d_k", "d_v") else heads]
            for n, t in zip(("out", "d_q", "d_k", "d_v", "d_slopes"), (out, *grads))}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", N.CASES)
def test_results_in_the_norm(case, dtype):
    q, k, v, d_out, how = N.inputs(case, dtype)
    got, want = _results(case, q, k, v, d_out, how), N.of_some(case, q, k, v, d_out, how)()
    far = {n: N.off(got[n], want[n]) / N.TOLERANCE[dtype][n] for n in want}
    print(f"{case} {dtype}: " + ", ".join(f"{n} {x:.2f}" for n, x in far.items()), flush=True)
    assert set(got) == set(want) and max(far.values()) <= 1, far


@pytest.mark.parametrize("case", ["few keys", "steep"])
def test_rows_with_few_keys_take_d_from_their_weights(case):
    """Values around 16: D = dO.out from a rounded `out` is off by more than what it is taken from is worth."""
    q, k, v, d_out, how = N.inputs(case, torch.bfloat16, mean=16.0)
    got, want = _results(case, q, k, v, d_out, how), N.of_some(case, q, k, v, d_out, how)()
    far = {n: N.off(got[n], want[n]) / N.TOLERANCE[torch.bfloat16][n] for n in ("out", "d_q", "d_k", "d_v")}
    print(f"{case}: " + ", ".join(f"{n} {x:.2f}" for n, x in far.items()), flush=True)
    assert max(far.values()) <= 1, far
