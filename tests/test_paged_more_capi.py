"""Argument checks of 4-bit caches, attention terms and page pools, which answer
before any device call (no GPU), and the numpy forms that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import paged_more_ref as ref
from test_paged_capi import A, BATCH_BAD, KV_BAD, batch, kv, read, write


def attend(qk, cache=None, b=None, terms=None, **over):
    d = dict(q=A, ldq=4096, out=A, ldout=4096, heads=32, scale=0.0) | over
    t = qk.qk_attention_terms(**(dict(cap=0.0, window=0, slopes=None, prefix=None) | (terms or {})))
    return qk.lib().qk_paged_attention_terms_f32(ctypes.byref(cache or kv(qk)), ctypes.byref(b or batch(qk)), *d.values(),
                                                 ctypes.byref(t), A, 1 << 20, None)


def pool(qk, layers=None, **over):
    d = dict(page_table=A, table_rows=4, table_stride=8, refs=A, pages=10, page_rows=64, layers=None, n_layers=0)
    p = qk.qk_page_pool(**(d | over))
    if layers is not None:
        p.layers, p.n_layers = (qk.qk_paged_kv * len(layers))(*layers), len(layers)
    return p


BIG = 1 << 30


def resize(qk, p=None, **over):
    d = dict(begins=None, lengths=A, missing=A, workspace=A, nbytes=BIG, stream=None) | over
    return qk.lib().qk_pages_resize(ctypes.byref(p or pool(qk)), *d.values())


def fork(qk, p=None, **over):
    d = dict(parents=A, lengths=A, missing=A, workspace=A, nbytes=BIG, stream=None) | over
    return qk.lib().qk_pages_fork(ctypes.byref(p or pool(qk)), *d.values())


def compact(qk, p=None, **over):
    d = dict(moved=A, workspace=A, nbytes=BIG, stream=None) | over
    return qk.lib().qk_pages_compact(ctypes.byref(p or pool(qk)), *d.values())


def status(qk, name):
    return getattr(qk, "QK_ERR_" + name)


@pytest.mark.parametrize("over,name", [(dict(key_scale=None), "INVALID_ARG"), (dict(head_dim=80), "LIMIT"),
                                       (dict(value=A + 8), "ALIGN"), (dict(value_scale=A + 8), "ALIGN")])
def test_4_bit_cache_refusals(qk, over, name):
    for call in (write, read, attend):
        assert call(qk, cache=kv(qk, type=qk.I4, **over)) == status(qk, name)


def test_4_bit_calls_without_tokens(qk):
    b = batch(qk, n_tokens=0)
    for call in (write, read, attend):
        assert call(qk, cache=kv(qk, type=qk.I4), b=b) == 0


@pytest.mark.parametrize("over,name", KV_BAD)
def test_cache_refusals(qk, over, name):
    assert attend(qk, cache=kv(qk, **over)) == status(qk, name)


@pytest.mark.parametrize("over,name", BATCH_BAD)
def test_batch_refusals(qk, over, name):
    assert attend(qk, b=batch(qk, **over)) == status(qk, name)


@pytest.mark.parametrize("terms,name", [
    (dict(cap=-1.0), "INVALID_ARG"), (dict(cap=float("nan")), "INVALID_ARG"), (dict(cap=float("inf")), "INVALID_ARG"),
    (dict(cap=2.0 ** -65), "INVALID_ARG"), (dict(cap=2.0 ** 65), "INVALID_ARG"), (dict(window=-1), "INVALID_ARG"),
    (dict(slopes=A + 2), "ALIGN"), (dict(prefix=A + 1), "ALIGN")])
def test_term_refusals(qk, terms, name):
    assert attend(qk, terms=terms) == status(qk, name)
    assert qk.lib().qk_last_error()


def test_workspace_of_a_window(qk):
    """As of the rows that it leaves; without one as of the call without terms."""
    size = lambda window, **over: qk.lib().qk_paged_attention_terms_workspace_bytes(
        ctypes.byref(batch(qk, max_rows=100000, **over)), 32, 8, 128, window)
    plain = qk.lib().qk_paged_attention_workspace_bytes(ctypes.byref(batch(qk, max_rows=100000)), 32, 8, 128)
    assert size(0) == plain >= size(4096) > size(1000) > 0
    assert size(100) == 0 and size(-1) == 0 and size(2 ** 31 - 1) == plain


@pytest.mark.parametrize("call", [resize, fork, compact])
@pytest.mark.parametrize("over,name", [
    (dict(page_table=None), "INVALID_ARG"), (dict(refs=None), "INVALID_ARG"), (dict(table_rows=0), "INVALID_ARG"),
    (dict(table_stride=0), "INVALID_ARG"), (dict(pages=0), "INVALID_ARG"), (dict(pages=(1 << 30) + 1), "LIMIT"),
    (dict(page_rows=48), "LIMIT"), (dict(page_rows=8), "LIMIT"), (dict(table_rows=1 << 24), "LIMIT"),
    (dict(table_rows=1 << 16, table_stride=(1 << 14) + 1), "LIMIT"), (dict(refs=A + 4), "ALIGN"),
    (dict(page_table=A + 2), "ALIGN"), (dict(n_layers=-1), "INVALID_ARG"), (dict(n_layers=2), "INVALID_ARG")])
def test_pool_refusals(qk, call, over, name):
    p = pool(qk, **over)
    assert call(qk, p) == status(qk, name)
    assert qk.lib().qk_pages_workspace_bytes(ctypes.byref(p)) == 0


@pytest.mark.parametrize("call", [resize, fork, compact])
def test_layer_refusals(qk, call):
    for over, name in ((dict(pages=11), "SHAPE"), (dict(page_rows=32), "SHAPE"), (dict(type=3), "TYPE"), (dict(key=None), "INVALID_ARG"),
                       (dict(kv_heads=4096, page_rows=64, head_dim=256, type=qk.I8), None)):
        got = call(qk, pool(qk, [kv(qk), kv(qk, **over)]), nbytes=4)
        assert got == (status(qk, name) if name else status(qk, "INVALID_ARG"))   # (then: of the workspace)
    wide = kv(qk, kv_heads=4096, page_rows=1024, head_dim=256)
    assert call(qk, pool(qk, [wide], page_rows=1024)) == status(qk, "LIMIT")


@pytest.mark.parametrize("call", [resize, fork, compact])
def test_workspace_refusals(qk, call):
    need = qk.lib().qk_pages_workspace_bytes(ctypes.byref(pool(qk)))
    assert need > 0
    assert call(qk, workspace=None) == status(qk, "INVALID_ARG")
    assert call(qk, nbytes=need - 1) == status(qk, "INVALID_ARG")
    assert call(qk, workspace=A + 4) == status(qk, "ALIGN")


def test_row_refusals(qk):
    assert resize(qk, lengths=None) == status(qk, "INVALID_ARG")
    assert resize(qk, begins=A + 1) == status(qk, "ALIGN") and resize(qk, lengths=A + 2) == status(qk, "ALIGN")
    assert resize(qk, missing=A + 2) == status(qk, "ALIGN")
    assert fork(qk, parents=None) == status(qk, "INVALID_ARG") and fork(qk, lengths=None) == status(qk, "INVALID_ARG")
    assert fork(qk, parents=A + 2) == status(qk, "ALIGN") and compact(qk, moved=A + 2) == status(qk, "ALIGN")


def test_copy_refusals(qk):
    def copy(layers, n_layers=None, source=A, target=A, n=3):
        array = (qk.qk_paged_kv * max(len(layers), 1))(*layers)
        return qk.lib().qk_pages_copy(array, len(layers) if n_layers is None else n_layers, source, target, n, None)

    assert copy([kv(qk)], n=-1) == status(qk, "INVALID_ARG") and copy([kv(qk)], n_layers=-1) == status(qk, "INVALID_ARG")
    assert copy([kv(qk)], source=None) == status(qk, "INVALID_ARG") and copy([kv(qk)], target=A + 2) == status(qk, "ALIGN")
    assert copy([kv(qk), kv(qk, pages=11)]) == status(qk, "SHAPE") and copy([kv(qk, type=3)]) == status(qk, "TYPE")
    assert copy([kv(qk)], n=0) == 0 and copy([], source=None) == 0


# ------------------------------------------------------- the numpy forms --

@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_4_bit_rows(qk, hd):
    """Codes within 7, every value within half a step, the row's largest within 2^-12
    of itself, and all of them fp32 numbers."""
    rng = np.random.default_rng(hd)
    x = (rng.standard_normal((200, hd)) * np.exp(rng.uniform(-80, 80, (200, 1)))).astype(np.float32)
    codes, entries, value = ref.encode4(x)
    scale = entries[..., :4].copy().view(np.float32)[..., 0].astype(np.float64)
    step = np.repeat(entries[..., 4:] * scale[:, None], hd // 4, -1)
    top = np.abs(x).max(-1).astype(np.float64)
    none = top < 2.0 ** -100   # zeros
    assert none.any() and not codes[none].any()
    codes, value, x, step, scale, top = (a[~none] for a in (codes, value, x, step, scale, top))
    assert (np.abs(value - x) <= step / 2 * (1 + 1e-12)).all()
    assert np.array_equal(value.astype(np.float32), value)
    assert (1785 * scale >= top).all() and (1785 * scale <= top * (1 + 2.0 ** -12)).all()
    assert (np.abs(value).max(-1) >= top * (1 - 2.0 ** -12)).all()
    nibbles = np.stack([codes & 15, codes >> 4])
    assert not (nibbles == 8).any()


def test_pages_by_hand():
    p = ref.Pages(3, 4, 8, 16, [np.arange(8)])
    assert p.resize([40, 16, 0]) == 0 and p.table.tolist() == [[0, 1, 2, -1], [3, -1, -1, -1], [-1] * 4]
    assert p.fork([-1, -1, 0], [0, 0, 40]) == 0 and p.table[2].tolist() == [0, 1, 4, -1]
    assert p.refs.tolist() == [2, 2, 1, 1, 1, 0, 0, 0] and p.contents[0][4] == 2
    assert p.resize([0, -1, -1]) == 0 and p.refs.tolist() == [1, 1, 0, 1, 1, 0, 0, 0]
    assert p.compact() == 1 and p.table[2].tolist() == [0, 1, 2, -1] and p.contents[0][2] == 2
    assert p.resize([-1, 200, -1]) == 13 - 4 and p.table[1].tolist() == [3, 4, 5, 6]
