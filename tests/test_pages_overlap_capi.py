"""Page pool calls refuse a number returned, a table, counts or a workspace that share
memory with other arguments: rows read their lengths while others write."""
import ctypes

import pytest

T, R, W, L, B, N = (0x10000 * i for i in range(1, 7))   # table, refs, workspace, lengths, begins or parents, number


def pool(qk, **over):
    d = dict(page_table=T, table_rows=6, table_stride=8, refs=R, pages=100, page_rows=64, layers=None, n_layers=0)
    return qk.qk_page_pool(**(d | over))


def call(qk, name, p, **over):
    d = dict(first=B, lengths=L, number=N, workspace=W) | over
    args = (d["number"],) if name == "compact" else (d["first"], d["lengths"], d["number"])
    return getattr(qk.lib(), "qk_pages_" + name)(ctypes.byref(p), *args, d["workspace"], 1 << 30, None)


def text(qk):
    return qk.lib().qk_last_error().decode()


@pytest.mark.parametrize("name", ["resize", "fork"])
@pytest.mark.parametrize("over", [dict(number=L), dict(number=L + 20), dict(number=B + 8), dict(number=T + 188), dict(number=R + 396),
                                  dict(lengths=T + 4), dict(first=T - 4), dict(lengths=R + 396), dict(first=R - 20),
                                  dict(number=W + 64), dict(lengths=W - 20), dict(workspace=L - 16), dict(workspace=T + 176)])
def test_rows_and_numbers(qk, name, over):
    assert call(qk, name, pool(qk), **over) == qk.QK_ERR_INVALID_ARG and "overlaps" in text(qk)


@pytest.mark.parametrize("name", ["resize", "fork", "compact"])
@pytest.mark.parametrize("pool_over,over", [(dict(refs=T + 176), {}), (dict(refs=T - 16), {}), ({}, dict(number=T)),
                                            ({}, dict(number=W)), ({}, dict(workspace=R + 384)), ({}, dict(workspace=R - 16))])
def test_pools(qk, name, pool_over, over):
    assert call(qk, name, pool(qk, **pool_over), **over) == qk.QK_ERR_INVALID_ARG and "overlaps" in text(qk)


@pytest.mark.gpu
def test_what_is_only_read_may_be_the_same(qk, torch_gpu):
    from test_gpu_pages import Both

    import numpy as np
    b = Both(qk, torch_gpu, np.random.default_rng(0), 6, 4, 30, 16)
    rows = b.i32([64, 17, 0, 5, 32, -1])
    qk.pages_resize(b.pool, rows, begins=rows, missing=b.number, workspace=b.ws)
    b.check(b.ref.resize(rows.cpu().numpy(), rows.cpu().numpy()))
    qk.pages_fork(b.pool, rows, rows, missing=b.number, workspace=b.ws)
    b.check(b.ref.fork(rows.cpu().numpy(), rows.cpu().numpy()))
    with pytest.raises(qk.QKError):
        qk.pages_resize(b.pool, rows, missing=rows[:1], workspace=b.ws)
