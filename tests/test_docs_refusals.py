"""CPU: what the rotary and packed-document operators refuse, in Python and behind the C ABI (no launch is reached)."""
import ctypes

import pytest
import torch

from fitclip_amd import _lib, ops


def _qkv(rows=8, heads=4, kv_heads=2, dtype=torch.float32):
    return torch.zeros(rows, heads, 64, dtype=dtype), torch.zeros(rows, kv_heads, 64, dtype=dtype), torch.zeros(rows, kv_heads, 64, dtype=dtype)


OFF = torch.tensor([0, 8], dtype=torch.int32)


@pytest.mark.parametrize("change,error,match", [
    (dict(q=torch.zeros(8, 4, 32)), ValueError, r"\[rows, heads, 64\]"),
    (dict(q=torch.zeros(8, 256)), ValueError, r"\[rows, heads, 64\]"),
    (dict(q=torch.zeros(8, 4, 64, dtype=torch.float64)), TypeError, "float32 or bfloat16"),
    (dict(k=torch.zeros(8, 2, 64, dtype=torch.bfloat16)), TypeError, "k must be"),
    (dict(q=torch.zeros(8, 4, 128)[..., ::2]), ValueError, "contiguous"),
    (dict(q=torch.zeros(8, 5, 64)), ValueError, "a multiple is needed"),
    (dict(v=torch.zeros(8, 4, 64)), ValueError, "same shape"),
    (dict(q_offsets=OFF.long()), TypeError, "q_offsets"),
    (dict(q_offsets=OFF[:0]), ValueError, "docs"),
    (dict(k_offsets=torch.zeros(3, dtype=torch.int32)), ValueError, "k_offsets"),
    (dict(q=torch.zeros(9, 4, 64)), ValueError, "k_offsets is needed"),
    (dict(prefix=torch.zeros(1, dtype=torch.int32)), ValueError, "causal"),
    (dict(prefix=torch.zeros(2, dtype=torch.int32), causal=True), ValueError, "prefix"),
    (dict(slopes=torch.zeros(2)), ValueError, "slopes"),
    (dict(slopes=torch.zeros(4, dtype=torch.float64)), TypeError, "slopes"),
    (dict(cap=-1.0), ValueError, "cap"),
    (dict(cap=float("nan")), ValueError, "cap"),
    (dict(scale=0.0), ValueError, "scale"),
    (dict(scale=float("inf")), ValueError, "scale"),
    (dict(scale=2e30), ValueError, "1e30"),
    (dict(cap=2e30), ValueError, "1e30"),
    (dict(), _lib.FitclipHipError, "no CPU fallback"),
])
def test_attention_refuses(change, error, match):
    q, k, v = _qkv()
    how = dict(q=q, k=k, v=v, q_offsets=OFF) | change
    with pytest.raises(error, match=match):
        ops.attention_docs(**how)


def test_written_tensors_may_not_overlap_themselves():
    x = torch.zeros(8, 4, 64)
    for bad in (torch.zeros(1, 4, 64).expand(8, 4, 64), torch.zeros(8, 1, 64).expand(8, 4, 64), torch.zeros(8 * 256).as_strided((8, 4, 64), (128, 64, 1)),
                torch.zeros(8, 4, 64, dtype=torch.bfloat16), torch.zeros(7, 4, 64)):
        with pytest.raises((ValueError, TypeError)):
            ops._written(bad, "out", x)
    for fine in (torch.zeros(8, 12, 64)[:, 4:8], torch.zeros(4, 8, 64).transpose(0, 1), torch.zeros(8, 4, 80)[..., :64]):
        ops._written(fine, "out", x)


def test_results_may_not_overlap_operands():
    qkv = torch.zeros(8, 3 * 128)
    q, k, v = (x.view(8, 2, 64) for x in qkv.split(128, 1))
    first = torch.zeros(3, 4, 9, 64)
    a, b, c = (x.transpose(0, 1) for x in first)            # heads first, one block behind the other
    mixed = torch.zeros(4, 3, 9, 64)
    d, e, f = (mixed[:, i].transpose(0, 1) for i in range(3))  # ... in turns
    for one, two in ((q, k), (q, v), (v, k), (a, b), (c, a), (d, e), (f, d), (q, a), (q[:0], q), (q[:4], q[4:]), (q[:, :1], q[:, 1:])):
        assert not ops._meet(one, two) and not ops._meet(two, one)
    shifted = qkv[:, 64:192].view(8, 2, 64)
    for one, two in ((q, q), (q, shifted), (shifted, k), (q[:5], q[4:]), (a, first[0, 1:].transpose(0, 1)), (d, mixed[:, 0, 1:].transpose(0, 1)),
                     (q, qkv.view(-1)[1300:1300 + 128 * 8].view(8, 2, 64))):
        assert ops._meet(one, two) and ops._meet(two, one)
    off = OFF
    with pytest.raises(ValueError, match="out overlaps k"):
        ops.attention_docs(q, k, v, off, out=k)
    with pytest.raises(ValueError, match="out overlaps v"):
        ops.attention_docs(q, k, v, off, out=v)
    out, stats = torch.zeros(8, 2, 64), torch.zeros(8, 2, 2)
    for given, match in ((dict(d_q=q), "d_q overlaps q"), (dict(d_k=v), "d_k overlaps v"), (dict(d_v=out), "d_v overlaps out"),
                         (dict(d_k=torch.zeros(8, 2, 64), d_q=shifted), "d_q overlaps")):
        with pytest.raises(ValueError, match=match):
            ops.attention_docs_backward(torch.zeros(8, 2, 64), q, k, v, out, stats, off, **given)
    one = torch.zeros(8, 2, 64)
    with pytest.raises(ValueError, match="d_k overlaps d_v"):
        ops.attention_docs_backward(torch.zeros(8, 2, 64), q, k, v, out, stats, off, d_k=one, d_v=one)
    positions, inv_freq = torch.zeros(8, dtype=torch.int32), torch.zeros(32)
    with pytest.raises(ValueError, match="overlaps"):
        ops.rotary(q, positions, inv_freq, out=shifted)


@pytest.mark.parametrize("change,error,match", [
    (dict(x=torch.zeros(8, 64)), ValueError, "rows, heads, dim"),
    (dict(x=torch.zeros(8, 2, 64, dtype=torch.float16)), TypeError, "float32 or bfloat16"),
    (dict(positions=torch.zeros(8, 2)), TypeError, "positions"),
    (dict(positions=torch.zeros(7, 3, dtype=torch.int32)), ValueError, "positions"),
    (dict(positions=torch.zeros(8, 4, dtype=torch.int32)), ValueError, "positions"),
    (dict(inv_freq=torch.zeros(2, 16)), ValueError, "inv_freq"),
    (dict(sections=(8, 8, 8)), ValueError, "sections"),
    (dict(sections=(16, 16)), ValueError, "sections"),
    (dict(sections=None), ValueError, "sections"),
    (dict(out=torch.zeros(8, 2, 32)), ValueError, "out"),
    (dict(), _lib.FitclipHipError, "no CPU fallback"),
])
def test_rotary_refuses(change, error, match):
    how = dict(x=torch.zeros(8, 2, 64), positions=torch.zeros(8, 3, dtype=torch.int32), inv_freq=torch.zeros(32), sections=(8, 12, 12)) | change
    with pytest.raises(error, match=match):
        ops.rotary(**how)


def _c_docs(**change):
    fields = dict(kind=0, docs=1, q_heads=4, kv_heads=2, causal=0, fill=0, scale=0.125, cap=0.0, q_rows=8, k_rows=8, q=4096, k=4096, v=4096,
                  q_row=256, q_head=64, k_row=128, k_head=64, v_row=128, v_head=64, q_offsets=4096, k_offsets=4096)
    return _lib.fc_docs(**(fields | change))


@pytest.mark.parametrize("change,match", [
    (dict(kind=2), b"element kind"), (dict(docs=-1), b"negative"), (dict(kv_heads=0), b"multiple"), (dict(q_heads=5), b"multiple"),
    (dict(q_rows=1 << 30), b"2\\^31"), (dict(k_rows=1 << 31), b"2\\^31"), (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale"),
    (dict(cap=-1.0), b"cap"), (dict(prefix=4096), b"causal"), (dict(q=None), b"null"), (dict(q_offsets=None), b"null"), (dict(v=None), b"null"),
    (dict(scale=2e30), b"1e30"), (dict(cap=2e30), b"1e30"), (dict(q_row=-256), b"negative"), (dict(v_head=-64), b"negative"),
    (dict(q_row=1 << 23), b"32 MiB"), (dict(k_row=1 << 23), b"32 MiB"), (dict(v_row=1 << 23), b"32 MiB"),
    (dict(k=4104), b"16-byte"), (dict(q_row=258), b"16-byte"), (dict(v_head=2), b"16-byte"),
])
def test_the_c_entry_refuses(change, match):
    import re
    lib = _lib.load()
    d = _c_docs(**change)
    assert lib.fc_attention_docs(d, 4096, 256, 64, 4096, None, 0, None) == -1
    assert re.search(match, lib.fc_last_error()), lib.fc_last_error()
    assert lib.fc_attention_docs_scratch_bytes(d) == 0


def test_the_c_entry_checks_struct_outputs_and_scratch():
    lib = _lib.load()
    d = _c_docs()
    d.struct_size -= 8
    assert lib.fc_attention_docs(d, 4096, 256, 64, 4096, None, 0, None) == -1 and b"struct_size" in lib.fc_last_error()
    assert lib.fc_attention_docs(None, 4096, 256, 64, 4096, None, 0, None) == -1
    d = _c_docs()
    assert lib.fc_attention_docs(d, None, 256, 64, 4096, None, 0, None) == -1 and b"output" in lib.fc_last_error()
    assert lib.fc_attention_docs(d, 4100, 256, 64, 4096, None, 0, None) == -1 and b"16-byte" in lib.fc_last_error()
    assert lib.fc_attention_docs(d, 4096, 257, 64, 4096, None, 0, None) == -1
    few = _c_docs(q_rows=1, k_rows=100_000)  # split over the keys: scratch is needed
    need = lib.fc_attention_docs_scratch_bytes(few)
    assert need > 0 and need % 264 == 0
    assert lib.fc_attention_docs(few, 4096, 256, 64, 4096, None, 0, None) == -3
    assert lib.fc_attention_docs(few, 4096, 256, 64, 4096, 4096, need - 1, None) == -3
    assert lib.fc_attention_docs(_c_docs(docs=0), 4096, 256, 64, 4096, None, 0, None) == 0   # nothing to do
    assert lib.fc_attention_docs(_c_docs(q_rows=0), None, 256, 64, None, None, 0, None) == 0
    assert ctypes.sizeof(_lib.fc_docs) == d.struct_size


@pytest.mark.parametrize("change,match", [
    (dict(kind=5), b"kind"), (dict(dim=60), b"dimensions"), (dict(dim=512), b"dimensions"), (dict(pairs=30), b"pairs"), (dict(pairs=36), b"pairs"),
    (dict(axes=4), b"axes"), (dict(axes=2), b"sections"), (dict(x=None), b"null"), (dict(x=4100), b"16-byte"), (dict(x_row=70), b"16-byte"),
    (dict(rows=-1), b"rows"), (dict(out=8192, out_row=192), b"strides"),
])
def test_the_c_rotary_refuses(change, match):
    lib = _lib.load()
    a = dict(kind=1, x=8192, x_row=128, x_head=64, positions=4096, axes=3, inv_freq=4096, sections=(ctypes.c_int32 * 3)(8, 12, 12), pairs=32,
             interleaved=0, inverse=0, out=4096, out_row=128, out_head=64, rows=8, heads=2, dim=64, st=None) | change
    assert lib.fc_rotary(*a.values()) == -1
    assert match in lib.fc_last_error(), lib.fc_last_error()


@pytest.mark.parametrize("change,error,match", [
    (dict(d_out=torch.zeros(8, 2, 64)), ValueError, "d_out"),
    (dict(out=torch.zeros(8, 4, 64, dtype=torch.bfloat16)), TypeError, "out"),
    (dict(stats=torch.zeros(8, 4)), ValueError, "stats"),
    (dict(stats=torch.zeros(8, 4, 2, dtype=torch.float64)), ValueError, "stats"),
    (dict(slope_grad=True), ValueError, "slopes"),
    (dict(d_k=torch.zeros(8, 4, 64)), ValueError, "d_k"),
    (dict(d_v=torch.zeros(1, 2, 64).expand(8, 2, 64)), ValueError, "overlap"),
    (dict(), _lib.FitclipHipError, "no CPU fallback"),
])
def test_gradients_refuse(change, error, match):
    q, k, v = _qkv()
    how = dict(d_out=torch.zeros(8, 4, 64), q=q, k=k, v=v, out=torch.zeros(8, 4, 64), stats=torch.zeros(8, 4, 2), q_offsets=OFF) | change
    with pytest.raises(error, match=match):
        ops.attention_docs_backward(**how)


def test_the_c_gradients_refuse():
    lib = _lib.load()

    def call(d, out=4096, d_k=4096, dq_row=256, d_slopes=None, scratch=4096, n=1 << 30):
        return lib.fc_attention_docs_backward(d, out, 256, 64, 4096, 4096, 256, 64, 4096, dq_row, 64, d_k, 128, 64, 4096, 128, 64, d_slopes, scratch, n, None)
    d = _c_docs()
    need = lib.fc_attention_docs_backward_scratch_bytes(d)
    assert need > 0 and lib.fc_attention_docs_backward_scratch_bytes(_c_docs(kind=9)) == 0
    assert call(d, out=None) == -1 and b"null" in lib.fc_last_error()
    assert call(d, d_k=None) == -1 and b"null" in lib.fc_last_error()
    assert call(d, dq_row=258) == -1 and b"16-byte" in lib.fc_last_error()
    assert call(d, d_slopes=4096) == -1 and b"slopes" in lib.fc_last_error()
    assert call(d, n=need - 1) == -3 and call(d, scratch=None) == -3
    assert call(_c_docs(docs=0), scratch=None) == 0
    bad = _c_docs()
    bad.struct_size = 16
    assert call(bad) == -1 and b"struct_size" in lib.fc_last_error()
