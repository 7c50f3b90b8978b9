"""Argument checks of the paged-cache, rotary-table and sampling entry points,
which answer before any device call (no GPU), and the numpy cache formats that
the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import paged_ref

A = 1 << 20   # an aligned address that no check follows


def kv(qk, **over):
    d = dict(type=qk.I8, kv_heads=8, head_dim=128, page_rows=64, pages=10, key=A, value=A, key_scale=A, value_scale=A)
    return qk.qk_paged_kv(**(d | over))


def batch(qk, **over):
    d = dict(page_table=A, table_rows=4, table_stride=8, seqs=A, n_seqs=4, n_tokens=4, max_count=1, max_rows=500)
    return qk.qk_paged_batch(**(d | over))


def write(qk, cache=None, b=None, **over):
    d = dict(q=A, ldq=4096, q_out=A, ldq_out=4096, k=A, ldk=1024, v=A, ldv=1024, heads=32, cosine=A, sine=A,
             positions=500, rot_dim=128, half=0, stream=None) | over
    return qk.lib().qk_rope_paged_write(ctypes.byref(cache or kv(qk)), ctypes.byref(b or batch(qk)), *d.values())


def read(qk, cache=None, b=None, **over):
    d = dict(key_out=A, ldk=1024, value_out=A, ldv=1024, stream=None) | over
    return qk.lib().qk_paged_read_f32(ctypes.byref(cache or kv(qk)), ctypes.byref(b or batch(qk)), *d.values())


def attend(qk, cache=None, b=None, **over):
    d = dict(q=A, ldq=4096, out=A, ldout=4096, heads=32, scale=0.0, workspace=A, nbytes=1 << 20, stream=None) | over
    return qk.lib().qk_paged_attention_f32(ctypes.byref(cache or kv(qk)), ctypes.byref(b or batch(qk)), *d.values())


KV_BAD = [(dict(type=12), "TYPE"), (dict(head_dim=80), "LIMIT"), (dict(head_dim=0), "LIMIT"),
          (dict(page_rows=48), "LIMIT"), (dict(page_rows=8), "LIMIT"), (dict(page_rows=2048), "LIMIT"),
          (dict(pages=0), "INVALID_ARG"), (dict(pages=1 << 31), "INVALID_ARG"), (dict(kv_heads=0), "INVALID_ARG"),
          (dict(key=None), "INVALID_ARG"), (dict(value_scale=None), "INVALID_ARG"), (dict(value=A + 8), "ALIGN"),
          (dict(key_scale=A + 4), "ALIGN")]
BATCH_BAD = [(dict(n_seqs=-1), "INVALID_ARG"), (dict(n_tokens=-1), "INVALID_ARG"), (dict(page_table=None), "INVALID_ARG"),
             (dict(seqs=None), "INVALID_ARG"), (dict(table_rows=0), "INVALID_ARG"), (dict(table_stride=0), "INVALID_ARG"),
             (dict(max_count=0), "INVALID_ARG"), (dict(max_rows=0), "INVALID_ARG"),
             (dict(max_rows=0x7FFFFFFF), "INVALID_ARG"), (dict(n_seqs=65536), "LIMIT"), (dict(seqs=A + 4), "ALIGN")]


@pytest.mark.parametrize("call", [write, read, attend])
@pytest.mark.parametrize("over,status", KV_BAD)
def test_cache_refusals(qk, call, over, status):
    assert call(qk, cache=kv(qk, **over)) == getattr(qk, "QK_ERR_" + status)
    assert qk.lib().qk_last_error()


@pytest.mark.parametrize("call", [write, read, attend])
@pytest.mark.parametrize("over,status", BATCH_BAD)
def test_batch_refusals(qk, call, over, status):
    assert call(qk, b=batch(qk, **over)) == getattr(qk, "QK_ERR_" + status)


@pytest.mark.parametrize("over,status", [
    (dict(rot_dim=7), "INVALID_ARG"), (dict(rot_dim=130), "INVALID_ARG"), (dict(rot_dim=-2), "INVALID_ARG"),
    (dict(half=2), "INVALID_ARG"), (dict(k=None), "INVALID_ARG"), (dict(q=None), "INVALID_ARG"),
    (dict(cosine=None), "INVALID_ARG"), (dict(heads=12), "INVALID_ARG"), (dict(heads=0), "INVALID_ARG"),
    (dict(ldk=1020), "INVALID_ARG"), (dict(ldq=4092), "INVALID_ARG"), (dict(ldq_out=4100), "INVALID_ARG"),
    (dict(q=A + 4), "ALIGN"), (dict(ldv=1026), "ALIGN")])
def test_write_refusals(qk, over, status):
    """(ldq_out=4100: in place with two strides.)"""
    assert write(qk, **over) == getattr(qk, "QK_ERR_" + status)


def test_too_many_rows(qk):
    b = batch(qk, max_count=1 << 30, max_rows=1 << 30, n_tokens=1 << 30)
    assert write(qk, b=b, cache=kv(qk, head_dim=64, kv_heads=4096), q=None, q_out=None, rot_dim=64, ldk=1 << 18,
                 ldv=1 << 18) == qk.QK_ERR_LIMIT
    assert attend(qk, b=b) == qk.QK_ERR_LIMIT
    b = batch(qk, max_count=1 << 27, max_rows=1 << 27, n_tokens=1 << 27)   # 2^32 threads
    assert write(qk, b=b) == qk.QK_ERR_LIMIT and read(qk, b=b) == qk.QK_ERR_LIMIT and attend(qk, b=b) == qk.QK_ERR_LIMIT


@pytest.mark.parametrize("over,status", [
    (dict(key_out=None, value_out=None), "INVALID_ARG"), (dict(ldk=1020), "INVALID_ARG"), (dict(ldv=1026), "ALIGN"),
    (dict(value_out=A + 8), "ALIGN")])
def test_read_refusals(qk, over, status):
    assert read(qk, **over) == getattr(qk, "QK_ERR_" + status)


@pytest.mark.parametrize("over,status", [
    (dict(heads=12), "INVALID_ARG"), (dict(heads=0), "INVALID_ARG"), (dict(scale=float("nan")), "INVALID_ARG"),
    (dict(scale=float("inf")), "INVALID_ARG"), (dict(q=None), "INVALID_ARG"), (dict(out=None), "INVALID_ARG"),
    (dict(ldq=4092), "INVALID_ARG"), (dict(ldout=4098), "ALIGN"), (dict(out=A + 4), "ALIGN"),
    (dict(workspace=A + 8), "ALIGN")])
def test_attention_refusals(qk, over, status):
    assert attend(qk, **over) == getattr(qk, "QK_ERR_" + status)


def test_empty_calls_are_no_ops(qk):
    """No sequence, or no token: nothing is launched, whatever the pointers."""
    for b in (batch(qk, n_seqs=0), batch(qk, n_tokens=0)):
        assert write(qk, b=b) == 0 and read(qk, b=b) == 0 and attend(qk, b=b) == 0
    assert qk.lib().qk_rope_tables_f32(10000.0, 64, None, None, 0, 0, None, None, None) == 0
    assert qk.lib().qk_sample_rows_f32(None, 5, 5, 0, *[None] * 8, 0, None) == 0


@pytest.mark.parametrize("over,status", [
    (dict(theta=0.0), "INVALID_ARG"), (dict(theta=float("nan")), "INVALID_ARG"), (dict(rot_dim=63), "LIMIT"),
    (dict(rot_dim=514), "LIMIT"), (dict(first_pos=-1), "INVALID_ARG"), (dict(positions=-1), "INVALID_ARG"),
    (dict(first_pos=0x7FFFFFF0), "LIMIT"), (dict(positions=(1 << 30) + 1), "LIMIT"), (dict(cosine=None), "INVALID_ARG")])
def test_table_refusals(qk, over, status):
    d = dict(theta=10000.0, rot_dim=64, scaling=None, freq_factors=None, first_pos=0, positions=100, cosine=A, sine=A,
             stream=None) | over
    assert qk.lib().qk_rope_tables_f32(*d.values()) == getattr(qk, "QK_ERR_" + status)


@pytest.mark.parametrize("over,status", [
    (dict(type=9), "TYPE"), (dict(factor=0.0), "INVALID_ARG"), (dict(factor=float("inf")), "INVALID_ARG"),
    (dict(type=2, original_context=0.0), "INVALID_ARG"), (dict(type=2, high_freq_factor=1.0), "INVALID_ARG"),
    (dict(type=3, beta_slow=0.0), "INVALID_ARG"), (dict(type=3, beta_fast=0.5), "INVALID_ARG"),
    (dict(type=3, attention_factor=float("nan")), "INVALID_ARG")])
def test_scaling_refusals(qk, over, status):
    s = qk.qk_rope_scaling(**(dict(type=1, factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                   original_context=8192.0, beta_fast=32.0, beta_slow=1.0, attention_factor=0.0) | over))
    got = qk.lib().qk_rope_tables_f32(10000.0, 64, ctypes.byref(s), None, 0, 100, A, A, None)
    assert got == getattr(qk, "QK_ERR_" + status)


@pytest.mark.parametrize("over,status", [
    (dict(n=0), "INVALID_ARG"), (dict(ldv=999), "INVALID_ARG"), (dict(rows=-1), "INVALID_ARG"),
    (dict(n=(1 << 19) + 1, ldv=1 << 20), "LIMIT"), (dict(rows=65536), "LIMIT"), (dict(logits=None), "INVALID_ARG"),
    (dict(uniform=None), "INVALID_ARG"), (dict(out=None), "INVALID_ARG"), (dict(workspace=A + 16), "ALIGN")])
def test_sample_refusals(qk, over, status):
    d = dict(logits=A, n=1000, ldv=1000, rows=4, temperature=None, top_k=None, top_p=None, min_p=None, uniform=A,
             out=A, prob=None, workspace=A, nbytes=1 << 30, stream=None) | over
    assert qk.lib().qk_sample_rows_f32(*d.values()) == getattr(qk, "QK_ERR_" + status)


def test_attention_workspace_query(qk):
    ask = lambda b, *a: qk.lib().qk_paged_attention_workspace_bytes(ctypes.byref(b), *a)
    assert ask(batch(qk, max_rows=1), 32, 8, 128) == 0
    assert ask(batch(qk, n_seqs=0), 32, 8, 128) == 0
    assert ask(batch(qk), 12, 8, 128) == 0
    assert ask(batch(qk, max_rows=100000, n_seqs=1, n_tokens=1), 32, 8, 128) > 0


def test_wrappers_refuse_host_tensors(qk):
    """What the Python functions are given is checked before the library is asked."""
    import torch
    x = torch.zeros(4, 128)
    with pytest.raises(qk.QKError, match="GPU tensor"):
        qk.PagedKV(qk.F16, torch.zeros(2, 1, 16, 64, dtype=torch.float16), torch.zeros(2, 1, 16, 64, dtype=torch.float16))
    with pytest.raises(qk.QKError, match="not F16"):
        qk.PagedKV(qk.Q4_K, x, x)
    with pytest.raises(qk.QKError, match="GPU tensor"):
        qk.sample_rows(x, torch.zeros(4), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(qk.QKError, match="GPU tensor"):
        qk.rope_tables(10000.0, 64, x, x)


def test_float8_values_and_rows():
    """The oracle's float8 table against its own rounding, and the row formats'
    corners: a full row, a zero row, a tiny one, one that is not finite."""
    v = paged_ref.E4M3
    assert v[0x7E] == 448 and v[1] == 2.0 ** -9 and v[0x38] == 1 and np.isnan(v[0x7F])
    row = np.zeros((1, 256), dtype=np.float32)
    row[0, :254] = v[[b for b in range(256) if b & 127 != 127]]
    codes, scale, value = paged_ref.encode(row, "e4m3")
    assert scale[0] == 1 and np.array_equal(value, row.astype(np.float64))
    for kind in ("i8", "e4m3"):
        _, s, x = paged_ref.encode(np.array([[0.0] * 4, [2.0 ** -101] * 4, [np.nan, 1, 2, 3]], dtype=np.float32), kind)
        assert s[0] == s[1] == 1 and np.isnan(s[2]) and not x[:2].any() and np.isnan(x[2]).all()
    _, s, x = paged_ref.encode(np.array([[127.0, 0.5, 1.5, -2.5]], dtype=np.float32), "i8")
    assert s[0] == 1 and x[0].tolist() == [127, 0, 2, -2]


@pytest.mark.parametrize("over", [
    dict(q_out=A + 16),                                        # a few values on
    dict(q_out=A + 4 * 4096 + 16, k=4 * A, v=4 * A),           # a row and a few values on
    dict(q_out=A - 4 * 4096 + 16, k=4 * A, v=4 * A),
    dict(q=2 * A, q_out=4 * A, k=4 * A + 4 * (4096 - 4), v=8 * A),   # q_out's last values
    dict(q=2 * A, q_out=4 * A, k=8 * A, v=4 * A - 4 * 1020),   # and its first
    dict(q=2 * A, q_out=4 * A, ldq_out=5120, k=4 * A + 4 * 4096, ldk=5000, v=8 * A),   # other strides: from the second row on
])
def test_write_refuses_overlaps(qk, over):
    """q_out may be q, and nothing else of q, k or v (sizes are floats: q rows of
    4096, k and v rows of 1024, four tokens)."""
    assert write(qk, **over) == qk.QK_ERR_INVALID_ARG
    assert b"overlaps" in qk.lib().qk_last_error()


def test_read_attention_and_tables_refuse_overlaps(qk):
    assert read(qk) == read(qk, value_out=A + 4 * 1020) == read(qk, value_out=A + 16 * 1023, ldv=2048) == qk.QK_ERR_INVALID_ARG
    assert b"overlaps" in qk.lib().qk_last_error()
    assert attend(qk, out=A + 16) == attend(qk, ldout=4100) == attend(qk, out=A - 16 * 4000, ldout=4100) == qk.QK_ERR_INVALID_ARG
    assert b"overlaps" in qk.lib().qk_last_error()
    assert qk.lib().qk_rope_tables_f32(10000.0, 64, None, None, 0, 100, A, A + 4 * 3199, None) == qk.QK_ERR_INVALID_ARG


def test_wrappers_refuse_what_an_int_does_not_hold(qk):
    """ctypes would pass the lower 32 bits on."""
    for call in (lambda: qk.sample_workspace_bytes(1000, 2 ** 32 + 1), lambda: qk.sample_workspace_bytes(2 ** 32 + 1000, 1)):
        with pytest.raises(qk.QKError, match="beyond"):
            call()


def test_wrappers_refuse_a_stream_of_another_device(qk):
    torch = qk._torch()

    class Stream:
        device, cuda_stream = torch.device("cuda", 1), 0

    def launched(*args):
        raise AssertionError("launched")
    with pytest.raises(qk.QKError, match="stream of cuda:1"):
        qk._launch(torch.device("cuda", 0), Stream, launched)
