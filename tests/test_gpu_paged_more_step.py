"""Page pools, 4-bit rows and attention with terms as a serving step uses them
together: prompts written into pages that the pool gives, forked, continued token by
token, compacted; against numpy in 64 bits."""
import numpy as np
import pytest

import paged_more_ref as ref
from conftest import rel_l2, to_dev

pytestmark = pytest.mark.gpu
HEADS, KVH, HD, PR, LAYERS = 8, 2, 64, 16, 2
TOL = 4e-6   # as in the tests of attention with terms


class Server:
    """A pool of two layers on the GPU, and the rows of every sequence in numpy."""

    def __init__(self, qk, t, type, rows=8, pages=60, stride=10):
        self.qk, self.t = qk, t
        self.layers = [qk.PagedKV.empty(type, pages, KVH, PR, HD) for _ in range(LAYERS)]
        for kv in self.layers:
            for x in (kv.key, kv.value, kv.key_scale, kv.value_scale):
                if x is not None:
                    x.view(t.uint8).fill_(0xFF)   # what nobody wrote is not a number
        self.pool = qk.PagePool.empty(rows, stride, pages, PR, self.layers)
        self.ws = t.empty(qk.pages_workspace_bytes(self.pool), dtype=t.uint8, device="cuda")
        self.missing = t.zeros(1, dtype=t.int32, device="cuda")
        self.rows = [[np.zeros((0, 2, KVH, HD)) for _ in range(rows)] for _ in range(LAYERS)]   # of each layer and table row

    def i32(self, a):
        return to_dev(self.t, np.asarray(a, dtype=np.int32))

    def resize(self, lengths):
        self.qk.pages_resize(self.pool, self.i32(lengths), missing=self.missing, workspace=self.ws)
        assert int(self.missing) == 0

    def values(self, x):
        """What rows of the cache keep of x [n, KVH, HD]."""
        return ref.encode4(x)[2] if self.layers[0].type == self.qk.I4 else x.astype(np.float16).astype(np.float64)

    def step(self, rng, seqs, **terms):
        """New tokens (table row, count) of each sequence through all layers; every layer's outputs."""
        t, qk = self.t, self.qk
        pos = [len(self.rows[0][r]) for r, _ in seqs]
        lengths = np.full(self.pool.rows, -1)
        for (r, c), p in zip(seqs, pos):
            lengths[r] = p + c
        self.resize(lengths)
        first = np.concatenate([[0], np.cumsum([c for _, c in seqs])])
        n = int(first[-1])
        desc = [[first[i], c, pos[i], r] for i, (r, c) in enumerate(seqs)]
        batch = qk.PagedBatch(self.pool.page_table, self.i32(desc), n, max(c for _, c in seqs),
                              max(p + c for p, (_, c) in zip(pos, seqs)))
        ws = t.empty(max(1, qk.paged_attention_workspace_bytes(batch, HEADS, KVH, HD, window=terms.get("window", 0))),
                     dtype=t.uint8, device="cuda")
        dev = {k: to_dev(t, v) if isinstance(v, np.ndarray) else v for k, v in terms.items()}
        for layer, kv in enumerate(self.layers):
            q, k, v = (rng.standard_normal((n, w * HD)).astype(np.float32) for w in (HEADS, KVH, KVH))
            out = t.full((n, HEADS * HD), np.nan, device="cuda")
            qk.rope_paged_write(kv, batch, None, None, to_dev(t, k), to_dev(t, v), None, None, 0, rot_dim=0)
            qk.paged_attention(kv, batch, to_dev(t, q), out, HEADS, workspace=ws, **dev)
            kk, vv = self.values(k.reshape(n, KVH, HD)), self.values(v.reshape(n, KVH, HD))
            want = np.zeros((n, HEADS, HD))
            for i, (r, c) in enumerate(seqs):
                new = np.stack([kk[first[i]:first[i + 1]], vv[first[i]:first[i + 1]]], 1)
                self.rows[layer][r] = np.concatenate([self.rows[layer][r], new])
                all_ = self.rows[layer][r]
                at = np.arange(len(all_))
                for j in range(c):
                    p = pos[i] + j
                    seen = at <= p
                    if "prefix" in terms:
                        seen = seen | (at < terms["prefix"][i])
                    if terms.get("window"):
                        seen = seen & (p - at < terms["window"])
                    for h in range(HEADS):
                        s = all_[seen, 0, h * KVH // HEADS] @ q[first[i] + j, h * HD:(h + 1) * HD].astype(np.float64) / np.sqrt(HD)
                        if terms.get("cap"):
                            s = terms["cap"] * np.tanh(s / terms["cap"])
                        if "slopes" in terms:
                            s = s - terms["slopes"][h] * np.abs(p - at[seen])
                        w = np.exp(s - s.max())
                        want[first[i] + j, h] = w @ all_[seen, 1, h * KVH // HEADS] / w.sum()
            assert rel_l2(out.cpu().numpy(), want.reshape(n, -1)) < TOL

    def fork(self, parents, lengths):
        self.qk.pages_fork(self.pool, self.i32(parents), self.i32(lengths), missing=self.missing, workspace=self.ws)
        assert int(self.missing) == 0
        old = [list(x) for x in self.rows]
        for c, p in enumerate(parents):
            if 0 <= p != c:
                for layer in range(LAYERS):
                    self.rows[layer][c] = old[layer][p][: lengths[c]]

    def end(self, rows):
        lengths = np.full(self.pool.rows, -1)
        lengths[list(rows)] = 0
        self.resize(lengths)
        for layer in self.rows:
            for r in rows:
                layer[r] = layer[r][:0]


@pytest.mark.parametrize("type", ["I4", "F16"])
def test_serving(qk, torch_gpu, type):
    """Prompts (one whose first rows see each other), three continuations of each, some
    dropped, the pool compacted, and on."""
    rng = np.random.default_rng(1)
    s = Server(qk, torch_gpu, getattr(qk, type))
    slopes = np.exp2(-np.arange(1, HEADS + 1)).astype(np.float32)
    s.step(rng, [(0, 70), (1, 33)], prefix=np.array([40, 0], np.int32))
    s.step(rng, [(0, 1), (1, 1)], cap=10.0)
    s.fork([-1, -1, 0, 0, 1, 1, -1, -1], [0, 0, 71, 64, 34, 20, 0, 0])
    for _ in range(3):
        s.step(rng, [(r, 1) for r in (3, 0, 5, 1, 2, 4)], window=40, slopes=slopes)
    s.end([0, 4])
    s.step(rng, [(6, 50), (2, 1)])
    s.fork([2, -1, -1, -1, -1, 6, -1, 2], [74, 0, 0, 0, 0, 49, 0, 60])
    held = int((s.pool.refs > 0).sum())
    qk.pages_compact(s.pool, workspace=s.ws)
    assert (s.pool.refs[:held] > 0).all() and not s.pool.refs[held:].any()
    s.step(rng, [(r, 1) for r in (0, 1, 2, 3, 5, 6, 7)], cap=20.0, window=64)
    s.step(rng, [(7, 30), (5, 2)])
    s.end(range(8))
    assert not s.pool.refs.any() and (s.pool.page_table == -1).all()


def test_captured_decoding(qk, torch_gpu):
    """A decoding step as a graph: rows' pages, the write, attention with terms; replayed
    with lengths that the device holds, against the same calls one by one."""
    t = torch_gpu
    rng = np.random.default_rng(2)
    n, pages = 3, 40
    make = lambda: qk.PagedKV.empty(qk.I4, pages, KVH, PR, HD)
    slopes = to_dev(t, np.exp2(-np.arange(1, HEADS + 1)).astype(np.float32))
    sides = []
    for _ in range(2):
        kv = make()
        pool = qk.PagePool.empty(n, 8, pages, PR, [kv])
        seqs = t.tensor([[i, 1, 0, i] for i in range(n)], dtype=t.int32, device="cuda")
        batch = qk.PagedBatch(pool.page_table, seqs, n, 1, 8 * PR)
        ws = t.empty(qk.pages_workspace_bytes(pool), dtype=t.uint8, device="cuda")
        aws = t.empty(max(1, qk.paged_attention_workspace_bytes(batch, HEADS, KVH, HD, window=50)), dtype=t.uint8, device="cuda")
        lengths = t.zeros(n, dtype=t.int32, device="cuda")
        q, k, v = (t.zeros(n, w * HD, device="cuda") for w in (HEADS, KVH, KVH))
        out = t.zeros(n, HEADS * HD, device="cuda")

        def step(pool=pool, lengths=lengths, ws=ws, kv=kv, batch=batch, q=q, k=k, v=v, out=out, aws=aws):
            qk.pages_resize(pool, lengths, workspace=ws)
            qk.rope_paged_write(kv, batch, None, None, k, v, None, None, 0, rot_dim=0)
            qk.paged_attention(kv, batch, q, out, HEADS, workspace=aws, cap=15.0, window=50, slopes=slopes)

        sides.append((step, pool, seqs, lengths, (q, k, v), out))
    side = t.cuda.Stream()
    with t.cuda.stream(side):
        sides[0][0]()   # (of no rows' pages: nothing is written)
    side.synchronize()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        sides[0][0]()
    at = np.array([0, 15, 60])
    for i in range(6):
        x = [to_dev(t, rng.standard_normal(y.shape).astype(np.float32)) for y in sides[0][4]]
        for j, (step, pool, seqs, lengths, ins, out) in enumerate(sides):
            for y, new in zip(ins, x):
                y.copy_(new)
            seqs[:, 2] = to_dev(t, at.astype(np.int32))
            lengths.copy_(to_dev(t, (at + 1).astype(np.int32)))
            if i == 0:   # rows before the first token of each sequence: absent ones' pages given, and zeros in them
                qk.pages_resize(pool, lengths, workspace=t.empty(qk.pages_workspace_bytes(pool), dtype=t.uint8, device="cuda"))
                for kv_part in (pool.layers[0].key, pool.layers[0].value, pool.layers[0].key_scale, pool.layers[0].value_scale):
                    kv_part.zero_()
            graph.replay() if j == 0 else step()
            t.cuda.synchronize()
        assert t.equal(sides[0][5], sides[1][5]) and t.isfinite(sides[0][5]).all()
        assert t.equal(sides[0][1].page_table, sides[1][1].page_table)
        at = at + 1


def test_two_calls_at_once(qk, torch_gpu):
    """Attention with terms on two streams, each with a workspace of its own."""
    t = torch_gpu
    rng = np.random.default_rng(3)
    pool = ref.Pool(rng, "i4", 2, 128, 32, [(1, 3000), (1, 500), (2, 1500)])
    q = rng.standard_normal((pool.n, 8 * 128)).astype(np.float32)
    kv, batch = pool.dev(qk, t)
    nb = qk.paged_attention_workspace_bytes(batch, 8, 2, 128)
    qd = to_dev(t, q)
    want = [pool.attention(q, 8), pool.attention(q, 8, cap=5.0)]
    streams, outs = [t.cuda.Stream() for _ in range(2)], [t.empty_like(qd) for _ in range(2)]
    spaces = [t.empty(nb, dtype=t.uint8, device="cuda") for _ in range(2)]
    t.cuda.synchronize()
    for _ in range(5):
        for i, terms in enumerate(({}, dict(cap=5.0))):
            qk.paged_attention(kv, batch, qd, outs[i], 8, workspace=spaces[i], stream=streams[i], **terms)
    t.cuda.synchronize()
    for out, w in zip(outs, want):
        assert rel_l2(out.cpu().numpy(), w) < TOL


def test_wrapper_refusals(qk, torch_gpu):
    """Tensors of another type, shape or size, and what is no layer of the pool."""
    t = torch_gpu
    kv = qk.PagedKV.empty(qk.I4, 6, 2, 16, 64)
    assert tuple(kv.key.shape) == (6, 2, 16, 32) and kv.head_dim == 64 and tuple(kv.key_scale.shape) == (6, 2, 16, 8)
    with pytest.raises(qk.QKError):
        qk.PagedKV(qk.I4, kv.key, kv.value)
    with pytest.raises(qk.QKError):
        qk.PagedKV(qk.I4, kv.key, kv.value, t.zeros(6, 2, 16, device="cuda"), t.zeros(6, 2, 16, device="cuda"))
    with pytest.raises(qk.QKError):
        qk.PagedKV(qk.I4, kv.key.view(t.int8), kv.value.view(t.int8), kv.key_scale, kv.value_scale)
    pool = qk.PagePool.empty(3, 4, 6, 16, [kv])
    ws = t.empty(qk.pages_workspace_bytes(pool), dtype=t.uint8, device="cuda")
    ok = t.zeros(3, dtype=t.int32, device="cuda")
    qk.pages_resize(pool, ok, workspace=ws)
    for bad in (ok.long(), ok[:2], ok.cpu(), t.zeros(6, dtype=t.int32, device="cuda")[::2]):
        with pytest.raises(qk.QKError):
            qk.pages_resize(pool, bad, workspace=ws)
        with pytest.raises(qk.QKError):
            qk.pages_fork(pool, ok, bad, workspace=ws)
    with pytest.raises(qk.QKError):
        qk.pages_resize(pool, ok, workspace=ws[:-4])
    with pytest.raises(qk.QKError):
        qk.pages_compact(pool, moved=ok, workspace=ws)
    with pytest.raises(qk.QKError):
        qk.pages_workspace_bytes(qk.PagePool.empty(3, 4, 7, 16, [kv]))
    with pytest.raises(qk.QKError):
        qk.pages_copy([kv], ok, ok[:2])
    batch = qk.PagedBatch(pool.page_table, t.zeros(1, 4, dtype=t.int32, device="cuda"), 1, 1, 16)
    q, out = t.zeros(1, 256, device="cuda"), t.zeros(1, 256, device="cuda")
    for terms in (dict(slopes=t.zeros(3, device="cuda")), dict(prefix=ok), dict(cap=-1.0), dict(window=-2),
                  dict(slopes=t.zeros(4, device="cuda", dtype=t.float64)), dict(window=1 << 31)):
        with pytest.raises(qk.QKError):
            qk.paged_attention(kv, batch, q, out, 4, **terms)


def test_a_row_cut_back_into_a_shared_page(qk, torch_gpu):
    """Forked again from one that holds the page, it goes on without touching it."""
    rng = np.random.default_rng(4)
    s = Server(qk, torch_gpu, qk.I4)
    s.step(rng, [(0, 64)])
    s.fork([-1, 0] + [-1] * 6, [0, 64] + [0] * 6)
    s.step(rng, [(1, 5), (0, 1)])
    s.resize([-1, 40] + [-1] * 6)
    for layer in s.rows:
        layer[1] = layer[1][:40]
    assert int((s.pool.refs > 1).sum()) == 3   # 40 rows of the prompt's 64, in pages of 16
    s.fork([-1, 0] + [-1] * 6, [0, 40] + [0] * 6)
    assert int((s.pool.refs > 1).sum()) == 2
    s.step(rng, [(1, 30), (0, 1)])
    s.step(rng, [(0, 1), (1, 1)], window=50)
