"""qk_pages_resize, qk_pages_fork, qk_pages_compact and qk_pages_copy against the
same, entry by entry, in numpy: tables, counts and contents are equal."""
import numpy as np
import pytest

import paged_more_ref as ref
from conftest import to_dev

pytestmark = pytest.mark.gpu


class Both:
    """A pool on the GPU and in numpy, the same calls to both."""

    def __init__(self, qk, t, rng, rows, stride, pages, page_rows, kinds=(), kvh=1, hd=64):
        self.qk, self.t = qk, t
        self.layers = []
        for kind in kinds:
            kv = qk.PagedKV.empty(getattr(qk, kind), pages, kvh, page_rows, hd)
            self.layers.append(kv)
        self.parts = [x for kv in self.layers for x in (kv.key, kv.value, kv.key_scale, kv.value_scale) if x is not None]
        for x in self.parts:
            raw = to_dev(t, rng.integers(0, 256, x.numel() * x.element_size(), dtype=np.uint8))
            x.view(t.uint8).view(-1).copy_(raw)
        self.pool = qk.PagePool.empty(rows, stride, pages, page_rows, self.layers)
        self.ref = ref.Pages(rows, stride, pages, page_rows, [x.view(t.uint8).cpu().numpy() for x in self.parts])
        self.ws = t.full((qk.pages_workspace_bytes(self.pool),), 0xFF, dtype=t.uint8, device="cuda")
        self.number = t.full((1,), -7, dtype=t.int32, device="cuda")

    def i32(self, a):
        return None if a is None else to_dev(self.t, np.asarray(a, dtype=np.int32))

    def resize(self, lengths, begins=None):
        self.qk.pages_resize(self.pool, self.i32(lengths), begins=self.i32(begins), missing=self.number, workspace=self.ws)
        self.check(self.ref.resize(lengths, begins))

    def fork(self, parents, lengths):
        self.qk.pages_fork(self.pool, self.i32(parents), self.i32(lengths), missing=self.number, workspace=self.ws)
        self.check(self.ref.fork(parents, lengths))

    def compact(self):
        self.qk.pages_compact(self.pool, moved=self.number, workspace=self.ws)
        self.check(self.ref.compact())

    def check(self, number):
        self.t.cuda.synchronize()
        assert int(self.number) == number
        assert np.array_equal(self.pool.page_table.cpu().numpy(), self.ref.table)
        assert np.array_equal(self.pool.refs.cpu().numpy(), self.ref.refs)
        assert self.consistent()
        for x, want in zip(self.parts, self.ref.contents):
            assert np.array_equal(x.view(self.t.uint8).cpu().numpy(), want)

    def consistent(self):
        t = self.ref.table
        held = t[(t >= 0) & (t < len(self.ref.refs))]
        return np.array_equal(np.bincount(held, minlength=len(self.ref.refs)), self.ref.refs)


@pytest.mark.parametrize("rows,stride,pages,page_rows", [(1, 1, 1, 16), (3, 5, 9, 16), (40, 17, 500, 32), (7, 300, 1500, 64),
                                                         (300, 9, 2000, 128), (5, 700, 20001, 16)])
def test_sequences_come_and_go(qk, torch_gpu, rows, stride, pages, page_rows):
    """Rows grow, shrink, end, drop what a window left behind, beyond the table and
    beyond the pool; some stay."""
    rng = np.random.default_rng(rows)
    b = Both(qk, torch_gpu, rng, rows, stride, pages, page_rows)
    most = stride * page_rows
    for step in range(6):
        lengths = rng.integers(0, most + 1, rows)
        lengths[rng.random(rows) < 0.2] = -1
        lengths[rng.random(rows) < 0.2] = 0
        if step == 3:
            lengths[rng.random(rows) < 0.3] = most + 3 * page_rows + 1
        begins = None if step % 2 else (lengths - rng.integers(0, most + 1, rows)).clip(-5, None)
        b.resize(lengths, begins)
    b.resize(np.full(rows, most))
    b.resize(np.zeros(rows))
    assert not b.ref.refs.any()


def test_lengths_at_page_ends(qk, torch_gpu):
    b = Both(qk, torch_gpu, np.random.default_rng(0), 8, 4, 40, 16)
    for lengths in ([0, 1, 15, 16, 17, 31, 32, 33], [1, 16, 17, 0, 64, 48, 49, 2 ** 31 - 1], [-1, -2 ** 31, 0, 1, 2, 3, 4, 5]):
        b.resize(lengths)
    b.resize([64] * 8, [0, 1, 15, 16, 17, 63, 64, 2 ** 31 - 1])


def test_entries_that_name_no_page(qk, torch_gpu):
    """They count as absent: taken where a row needs them, else left."""
    t = torch_gpu
    b = Both(qk, t, np.random.default_rng(0), 3, 6, 12, 16)
    b.resize([96, 40, 20])
    for r, e, v in ((0, 2, 12), (1, 5, 2 ** 31 - 1), (2, 4, -9)):
        p = b.ref.table[r, e]
        if 0 <= p < 12:
            b.ref.refs[p] -= 1
        b.ref.table[r, e] = v
    b.pool.page_table.copy_(b.i32(b.ref.table))
    b.pool.refs.copy_(b.i32(b.ref.refs))
    b.resize([96, 16, -1])
    b.fork([1, -1, 0], [96, 0, 90])
    b.compact()


@pytest.mark.parametrize("kinds", [(), ("F16",), ("I8", "I4"), ("F8_E4M3", "F16", "I4")])
def test_forks(qk, torch_gpu, kinds):
    """One prompt's continuations, forks of forks, lengths at and inside pages, rows
    that are replaced, exchanged and kept."""
    rng = np.random.default_rng(len(kinds))
    b = Both(qk, torch_gpu, rng, 12, 7, 70, 16, kinds, kvh=2)
    b.resize([100, 33, 64, 0, 1, 16] + [0] * 6)
    b.fork([-1] * 6 + [0, 0, 1, 2, 4, 3], [0] * 6 + [100, 97, 33, 64, 1, 50])
    b.fork([0, 2, 1, 3, 6, 12, -1, 7, 7, 7, 99, -3], [100, 64, 33, 5, 31, 1, 1, 97, 96, 80, 4, 4])   # 1 and 2 exchange
    b.fork([1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 0], [1000] * 12)   # all take the next one's place, lengths beyond the rows
    b.resize([0] * 6 + [-1] * 6)
    b.fork([6] * 6 + [-1] * 6, [-5, 0, 1, 15, 16, 17] + [0] * 6)
    b.resize([0] * 12)
    assert not b.ref.refs.any()


def test_fork_without_free_pages(qk, torch_gpu):
    """Shared pages need none; the last part of one is missing, lowest rows first served."""
    b = Both(qk, torch_gpu, np.random.default_rng(1), 6, 4, 5, 16, ("I8",))
    b.resize([50, 0, 0, 0, 0, 0])
    b.fork([-1, 0, 0, 0, 0, 0], [0, 50, 48, 50, 17, 1])


@pytest.mark.parametrize("kinds", [(), ("I4",), ("F16", "I8")])
@pytest.mark.parametrize("rows,stride,pages", [(6, 5, 40), (30, 40, 1300), (3, 4, 20000)])
def test_compaction(qk, torch_gpu, kinds, rows, stride, pages):
    """After sequences ended, with forks that share pages; twice; an empty pool."""
    if kinds and pages > 5000:
        pytest.skip("a pool as large as this is looked over without contents")
    rng = np.random.default_rng(rows)
    b = Both(qk, torch_gpu, rng, rows, stride, pages, 16, kinds)
    b.compact()
    b.resize(rng.integers(1, stride * 16 + 1, rows))
    b.compact()   # nothing moves
    b.fork([0 if r == rows - 1 else -1 for r in range(rows)], [stride * 8 + 3] * rows)
    b.resize([0 if r % 2 == 0 else -1 for r in range(rows)])
    b.compact()
    b.compact()
    b.resize(rng.integers(0, stride * 16 + 1, rows))
    b.compact()
    b.resize([0] * rows)
    b.compact()
    # The last pages alone.
    b.ref.table[0, 0], b.ref.table[1, 1], b.ref.table[2, 2] = pages - 1, pages - 2, pages - 1
    b.ref.refs[[pages - 1, pages - 2]] = 2, 1
    b.pool.page_table.copy_(b.i32(b.ref.table))
    b.pool.refs.copy_(b.i32(b.ref.refs))
    b.compact()


@pytest.mark.parametrize("kind,kvh,hd,page_rows", [("F16", 8, 128, 64), ("I8", 1, 64, 16), ("I4", 3, 96, 16), ("I4", 8, 256, 128)])
def test_copies(qk, torch_gpu, kind, kvh, hd, page_rows):
    """Many pages, pairs that name none, a page onto itself; more layers than one
    launch takes."""
    t = torch_gpu
    rng = np.random.default_rng(kvh)
    layers, pages = 40 if kvh == 1 else 2, 61
    b = Both(qk, t, rng, 1, 1, pages, page_rows, (kind,) * layers, kvh, hd)
    order = rng.permutation(pages)
    src, dst = order[:30].copy(), order[30:60].copy()
    src[3], dst[4], src[5], dst[6] = -1, pages, 2 ** 31 - 1, -8
    dst[7] = src[7]
    qk.pages_copy(b.layers, b.i32(src), b.i32(dst))
    qk.pages_copy(b.layers, b.i32([]), b.i32([]))
    for s, d in zip(src, dst):
        if 0 <= s < pages and 0 <= d < pages:
            for a in b.ref.contents:
                a[d] = a[s]
    for x, want in zip(b.parts, b.ref.contents):
        assert np.array_equal(x.view(t.uint8).cpu().numpy(), want)


def test_captured_step(qk, torch_gpu):
    """Resize, fork and compaction in one graph, replayed with new lengths."""
    t = torch_gpu
    rng = np.random.default_rng(2)
    b = Both(qk, t, rng, 8, 6, 60, 16, ("I4", "F16"), kvh=2)
    lengths, parents, forked = (t.zeros(8, dtype=t.int32, device="cuda") for _ in range(3))

    def step():
        qk.pages_resize(b.pool, lengths, missing=b.number, workspace=b.ws)
        qk.pages_fork(b.pool, parents, forked, workspace=b.ws)
        qk.pages_compact(b.pool, workspace=b.ws)

    side = t.cuda.Stream()
    with t.cuda.stream(side):
        step()   # of an empty pool
    side.synchronize()
    b.ref.resize(np.zeros(8)), b.ref.fork(np.zeros(8, int), np.zeros(8)), b.ref.compact()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        step()
    for _ in range(5):
        n = [rng.integers(-10, 97, 8), rng.integers(-4, 8, 8), rng.integers(0, 97, 8)]
        for dev, a in zip((lengths, parents, forked), n):
            dev.copy_(b.i32(a))
        graph.replay()
        missing = b.ref.resize(n[0])
        b.ref.fork(n[1], n[2])
        b.ref.compact()
        b.check(missing)


def test_other_stream(qk, torch_gpu):
    """A call on a stream that is not current."""
    t = torch_gpu
    b = Both(qk, t, np.random.default_rng(2), 8, 6, 60, 16, ("I8",))
    lengths = b.i32([90, 17, 0, 1, 16, 40, 3, 96])
    t.cuda.synchronize()
    side = t.cuda.Stream()
    qk.pages_resize(b.pool, lengths, missing=b.number, workspace=b.ws, stream=side)
    side.synchronize()
    b.check(b.ref.resize([90, 17, 0, 1, 16, 40, 3, 96]))
