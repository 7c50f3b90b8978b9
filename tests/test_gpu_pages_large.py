"""qk_pages_resize, qk_pages_fork and qk_pages_compact over pools of millions of pages and
tables of thousands of rows, where what a workgroup counts is a segment of several
thousand pages and row sums are carried on; against array operations in numpy."""
import numpy as np
import pytest

from conftest import to_dev

pytestmark = pytest.mark.gpu


def resize(table, refs, page_rows, lengths, begins=None):
    entry, stride = np.arange(table.shape[1]), table.shape[1]
    have, change = (table >= 0) & (table < len(refs)), (lengths >= 0)[:, None]
    first = np.zeros(len(lengths), np.int64) if begins is None else np.maximum(begins, 0) // page_rows
    last = -(-lengths.astype(np.int64) // page_rows)
    want = (entry >= first[:, None]) & (entry < last[:, None])
    drop, need = have & ~want & change, want & ~have & change
    refs -= np.bincount(table[drop], minlength=len(refs)).astype(np.int32)
    table[drop] = -1
    free = np.flatnonzero(refs == 0)[: need.sum()]
    given = np.full(need.sum(), -1, dtype=np.int32)
    given[: len(free)] = free
    table[need] = given   # in order of rows and entries
    refs[free] = 1
    return len(given) - len(free) + int(np.maximum(last - np.maximum(first, stride), 0)[lengths >= 0].sum())


def fork(table, refs, page_rows, parents, lengths):
    rows, stride = table.shape
    old, free = table.copy(), np.flatnonzero(refs == 0)
    taken = missing = 0
    for c in np.flatnonzero((parents >= 0) & (parents < rows) & (parents != np.arange(rows))):
        full, part = divmod(max(int(lengths[c]), 0), page_rows)
        new = np.where(np.arange(stride) < full, old[parents[c]], -1).astype(np.int32)
        new[(new < 0) | (new >= len(refs))] = -1
        if part and full < stride and 0 <= old[parents[c], full] < len(refs):
            new[full] = free[taken] if taken < len(free) else -1
            missing += taken >= len(free)
            taken += 1
        held = old[c][(old[c] >= 0) & (old[c] < len(refs))]
        np.subtract.at(refs, held, 1)
        np.add.at(refs, new[new >= 0], 1)
        table[c] = new
    return missing


def compact(table, refs):
    live = int((refs > 0).sum())
    movers, holes = np.flatnonzero(refs[live:] > 0) + live, np.flatnonzero(refs[:live] == 0)
    to = np.arange(len(refs), dtype=np.int32)
    to[movers] = holes
    refs[holes], refs[movers] = refs[movers], 0
    have = (table >= 0) & (table < len(refs))
    table[have] = to[table[have]]
    return len(movers)


class Both:
    def __init__(self, qk, t, table, pages, page_rows):
        self.qk, self.t, self.table, self.page_rows = qk, t, table, page_rows
        self.refs = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
        self.pool = qk.PagePool(to_dev(t, table), to_dev(t, self.refs), page_rows)
        self.ws = t.full((qk.pages_workspace_bytes(self.pool),), 0xFF, dtype=t.uint8, device="cuda")
        self.number = t.full((1,), -7, dtype=t.int32, device="cuda")

    def i32(self, a):
        return None if a is None else to_dev(self.t, a.astype(np.int32))

    def check(self, number):
        self.t.cuda.synchronize()
        assert int(self.number) == number
        assert np.array_equal(self.pool.page_table.cpu().numpy(), self.table)
        assert np.array_equal(self.pool.refs.cpu().numpy(), self.refs)

    def resize(self, lengths, begins=None):
        self.qk.pages_resize(self.pool, self.i32(lengths), begins=self.i32(begins), missing=self.number, workspace=self.ws)
        self.check(resize(self.table, self.refs, self.page_rows, lengths, begins))

    def fork(self, parents, lengths):
        self.qk.pages_fork(self.pool, self.i32(parents), self.i32(lengths), missing=self.number, workspace=self.ws)
        self.check(fork(self.table, self.refs, self.page_rows, parents, lengths))

    def compact(self):
        self.qk.pages_compact(self.pool, moved=self.number, workspace=self.ws)
        self.check(compact(self.table, self.refs))


# Held rows of all rows: the pool is more than four fifths full, so that the first free
# pages lie in the middle of a segment, and what the call gives reaches over many.
@pytest.mark.parametrize("rows,stride,pages,held", [(2800, 1000, 3000017, 2600), (5000, 30, 140001, 4300), (1025, 1100, 1 << 20, 900),
                                                    (1100, 1100, (1 << 20) + 1, 930), (70, 9000, 600000, 64)])
@pytest.mark.parametrize("front", [False, True])
def test_large_pools(qk, torch_gpu, rows, stride, pages, held, front):
    """Pages held anywhere, or the pool's first ones."""
    rng = np.random.default_rng(rows + front)
    table = np.full((rows, stride), -1, dtype=np.int32)
    order = np.arange(pages) if front else rng.permutation(pages)
    table[:held] = order[: held * stride].reshape(held, stride)
    table = table[rng.permutation(rows)]
    b = Both(qk, torch_gpu, table, pages, 16)
    new = np.flatnonzero(table[:, 0] < 0)
    lengths = np.full(rows, -1)
    lengths[new] = rng.integers(0, stride * 16 + 1, len(new))
    lengths[rng.random(rows) < 0.01] = 100
    b.resize(lengths)
    lengths = np.where(rng.random(rows) < 0.1, rng.integers(0, stride * 16 + 1, rows), -1)
    b.resize(lengths, lengths - 3000)
    parents = np.where(rng.random(rows) < 0.05, rng.integers(0, rows, rows), -1)
    b.fork(parents, rng.integers(0, stride * 16 + 1, rows))
    b.compact()
    b.resize(np.full(rows, stride * 16 + 20))   # more than there are
    b.resize(np.where(np.arange(rows) % 2, -1, 0))
    b.compact()
