"""CPU: calls of the rotary and packed-document operators at the edges of what they take, in Python and behind the C ABI (no launch is reached)."""
import pytest
import torch

from fitclip_amd import _lib, ops

OFF = torch.tensor([0, 8], dtype=torch.int32)


def test_out_may_be_q_itself_and_no_other_view_of_it():
    """A workgroup writes rows of `out` while others still read rows of q: only a row of its own may be written where it was read."""
    rows, heads = 8, 2
    buf = torch.zeros(rows + 1, heads, 64)
    first = torch.zeros(heads, rows, 64)
    k, v = torch.zeros(rows, heads, 64), torch.zeros(rows, heads, 64)
    wide = torch.zeros(rows, 3 * heads * 64)
    fused = wide[:, :heads * 64].view(rows, heads, 64)
    for q, out in ((buf[:-1], buf[1:]), (buf[1:], buf[:-1]),                                    # a row further
                   (fused, wide[:, 64:64 + heads * 64].view(rows, heads, 64)),                  # a head further
                   (fused, wide.view(-1)[:rows * heads * 64].view(rows, heads, 64)),            # the same place, other strides
                   (first.transpose(0, 1), first.view(rows, heads, 64))):                       # heads first, and rows first
        with pytest.raises(ValueError, match="out overlaps q"):
            ops.attention_docs(q, k, v, OFF, out=out)
    for q, out in ((buf[1:], buf[1:]), (fused, fused), (fused, wide[:, heads * 64:2 * heads * 64].view(rows, heads, 64)),
                   (buf[:1], buf.view(-1)[:128].view(1, heads, 64))):                           # itself; beside it; one row, whatever its stride says
        off, kv = (OFF, k) if q.shape[0] == rows else (torch.tensor([0, 1], dtype=torch.int32), k[:1])
        with pytest.raises(_lib.FitclipHipError, match="no CPU fallback"):  # every check before the device's has passed
            ops.attention_docs(q, kv, kv, off, out=out)


def _c_docs(**change):
    fields = dict(kind=0, docs=1, q_heads=4, kv_heads=2, causal=0, fill=0, scale=0.125, cap=0.0, q_rows=8, k_rows=8, q=4096, k=4096, v=4096,
                  q_row=256, q_head=64, k_row=128, k_head=64, v_row=128, v_head=64, q_offsets=4096, k_offsets=4096)
    return _lib.fc_docs(**(fields | change))


def test_the_c_entry_takes_q_as_out_with_its_strides_alone():
    lib = _lib.load()
    for change in (dict(out_row=512), dict(out_head=128)):
        a = dict(out=4096, out_row=256, out_head=64) | change
        assert lib.fc_attention_docs(_c_docs(), *a.values(), 4096, None, 0, None) == -1 and b"in place" in lib.fc_last_error()


@pytest.mark.parametrize("how", [dict(cap=1e-50), dict(cap=2.0 ** -150), dict(scale=1e-46), dict(cap=float("nan")), dict(cap=float("inf"))])
def test_caps_and_scales_that_float32_cannot_hold(how):
    """A cap that is rounded to 0 would be none at all."""
    q = torch.zeros(8, 2, 64)
    with pytest.raises(ValueError, match="scale must be positive"):
        ops.attention_docs(q, q, q, OFF, **how)
    with pytest.raises(_lib.FitclipHipError, match="no CPU fallback"):
        ops.attention_docs(q, q, q, OFF, cap=2.0 ** -149, scale=2.0 ** -149)


def test_the_c_entries_refuse_negative_strides_of_results_and_d_out():
    """d_out's row stride goes into 32-bit offsets: a negative one would read far outside."""
    lib = _lib.load()
    d = _c_docs()
    for change in (dict(row=-256), dict(head=-64)):
        a = dict(out=8192, row=256, head=64) | change
        assert lib.fc_attention_docs(d, *a.values(), 4096, None, 0, None) == -1 and b"negative" in lib.fc_last_error()
    for at in range(5):  # out, d_out, d_q, d_k, d_v
        for which in (0, 1):
            strides = [[256, 64], [256, 64], [256, 64], [128, 64], [128, 64]]
            strides[at][which] *= -1
            o, g, q, k, v = strides
            assert lib.fc_attention_docs_backward(d, 4096, *o, 4096, 4096, *g, 4096, *q, 4096, *k, 4096, *v, None, 4096, 1 << 30, None) == -1
            assert b"negative" in lib.fc_last_error(), lib.fc_last_error()


def test_rotary_refuses_rows_beyond_a_launch():
    import ctypes
    lib = _lib.load()
    assert lib.fc_rotary(1, 8192, 16, 16, 4096, 1, 4096, (ctypes.c_int32 * 1)(8), 8, 0, 0, 4096, 16, 16, 1 << 35, 1, 16, None) == -1
    assert b"rows" in lib.fc_last_error()
