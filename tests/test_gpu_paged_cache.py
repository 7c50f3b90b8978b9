"""qk_rope_paged_write and qk_paged_read_f32 against numpy in 64 bits: codes,
scales and rotated queries bit for bit, rows of every kind and position, and
what must be left alone."""
import numpy as np
import pytest

import paged_ref
from conftest import to_dev

pytestmark = pytest.mark.gpu
KINDS = ["f16", "i8", "e4m3"]
LAYOUTS = [(8, 2, 64), (6, 6, 96), (12, 4, 128), (3, 1, 256)]


def tables(rng, positions, rot):
    a = rng.uniform(-np.pi, np.pi, (positions, rot // 2))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def bits(a):
    a = np.ascontiguousarray(a)
    return a.view({1: np.uint8, 2: np.uint16, 4: np.uint32}[a.dtype.itemsize])


def codes_of(t):
    """A pool's stored bits."""
    import torch
    return bits(t.view({1: torch.uint8, 2: torch.int16}[t.element_size()]).cpu().numpy())


def run(qk, t, pool, q, k, v, cos, sin, heads, rot, half, **over):
    kv, batch = pool.dev(qk, t, **over)
    n = batch.n_tokens
    dev = lambda a: None if a is None else to_dev(t, a)
    qo = None if q is None else t.full((n, q.shape[1]), np.nan, device="cuda")
    qk.rope_paged_write(kv, batch, dev(q), qo, dev(k), dev(v), dev(cos), dev(sin), heads, rot_dim=rot, half=half)
    back = [t.full((n, k.shape[1]), 7.0, device="cuda") for _ in range(2)]
    qk.paged_read(kv, batch, *back)
    t.cuda.synchronize()
    return kv, None if qo is None else qo.cpu().numpy(), [b.cpu().numpy() for b in back]


def check(qk, t, pool, q, k, v, cos, sin, heads, rot, half, skip=(), unwritten=(), **over):
    """Every row of the pool and every query against the oracle; the sequences
    of skip leave everything as it was, those of unwritten are read as they
    were."""
    before = [[None if a is None else a.copy() for a in p[:2]] for p in (pool.key, pool.value)]
    kv, qo, back = run(qk, t, pool, q, k, v, cos, sin, heads, rot, half, **over)
    n, hd, kvh = len(k), pool.hd, pool.kvh
    pos = np.zeros(n, dtype=int)
    live = np.zeros(n, dtype=bool)
    for i, (first, count, p, _) in enumerate(pool.seqs):
        if i not in skip + unwritten:
            pos[first:first + count] = np.arange(p, p + count)
            live[first:first + count] = True
    rows = lambda x: x.reshape(n, -1, hd)
    c, s = (np.zeros((n, 0), np.float32),) * 2 if not rot else (cos[pos % len(cos)], sin[pos % len(cos)])
    if q is not None:
        want = paged_ref.rotate(rows(q), c, s, rot, half).reshape(n, -1)
        assert np.array_equal(bits(qo[live]), bits(want[live]))
        assert np.isnan(qo[~live]).all()
    new = [paged_ref.encode(paged_ref.rotate(rows(k), c, s, rot, half), pool.kind), paged_ref.encode(rows(v), pool.kind)]
    for (codes, scale), (wc, ws, wv), old, got, gscale, b in zip(before, new, (pool.key[2], pool.value[2]),
                                                                 (kv.key, kv.value), (kv.key_scale, kv.value_scale),
                                                                 back):
        expect = np.full((n, kvh, hd), 7.0)
        for i, (first, count, p, tab) in enumerate(pool.seqs):
            for j in range(count if i not in skip else 0):
                page, slot = pool.table[tab, (p + j) // pool.page_rows], (p + j) % pool.page_rows
                if not 0 <= page < pool.pages:
                    expect[first + j] = 0
                    continue
                if i in unwritten:
                    expect[first + j] = old[page, :, slot]
                    continue
                codes[page, :, slot] = wc[first + j]
                if ws is not None:
                    scale[page, :, slot] = ws[first + j]
                expect[first + j] = wv[first + j]
        assert np.array_equal(codes_of(got), bits(codes))
        if scale is not None:
            assert np.array_equal(gscale.cpu().numpy(), scale, equal_nan=True)
        # code * scale, rounded once.
        assert np.array_equal(b, expect.astype(np.float32).reshape(n, -1), equal_nan=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hd", LAYOUTS)
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("page_rows", [16, 128])
def test_ragged_batch(qk, torch_gpu, kind, heads, kvh, hd, half, page_rows):
    """Single tokens, chunks that start and end inside pages, a fresh sequence."""
    rng = np.random.default_rng(hd + page_rows)
    pool = paged_ref.Pool(rng, kind, kvh, hd, page_rows, [(1, 0), (1, 700), (37, 13), (130, 0), (5, 123)])
    cos, sin = tables(rng, 701, hd)
    q, k, v = (rng.standard_normal((pool.n, w * hd)).astype(np.float32) for w in (heads, kvh, kvh))
    check(qk, torch_gpu, pool, q, k, v, cos, sin, heads, hd, half)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rot", [0, 2, 6, 32, 44, 48, 64])
@pytest.mark.parametrize("half", [False, True])
def test_partly_rotated_heads(qk, torch_gpu, kind, rot, half):
    rng = np.random.default_rng(rot)
    pool = paged_ref.Pool(rng, kind, 2, 64, 32, [(9, 3), (1, 50)])
    cos, sin = tables(rng, 60, rot) if rot else (None, None)
    q, k, v = (rng.standard_normal((pool.n, w * 64)).astype(np.float32) for w in (4, 2, 2))
    check(qk, torch_gpu, pool, q, k, v, cos, sin, 4, rot, half)


@pytest.mark.parametrize("kind", KINDS)
def test_values_at_the_formats_corners(qk, torch_gpu, kind):
    """Ties of the rounding, rows of zeros, of tiny and of huge values, a value
    that alone fills the range, and rows that hold what is not finite."""
    rng = np.random.default_rng(5)
    pool = paged_ref.Pool(rng, kind, 1, 64, 16, [(24, 0)])
    x = np.zeros((24, 64), dtype=np.float32)
    x[1, 0], x[1, 1:] = 127, np.arange(-31, 32) + 0.5          # i8 ties
    x[2, 0], x[2, 1:] = 448, np.linspace(0, 0.05, 63)           # e4m3 subnormals
    x[3] = paged_ref.E4M3[np.arange(64)] + paged_ref.E4M3[np.arange(1, 65)]   # e4m3 ties at scale 2 ...
    x[3, 0] = 896
    x[4] = 2.0 ** -101
    x[5] = rng.standard_normal(64) * 2.0 ** -98
    x[6] = rng.standard_normal(64) * 1e37
    x[7], x[7, 5] = 1, np.nan
    x[8], x[8, 63] = 1, np.inf
    x[9], x[9, 0] = 1, -np.inf
    x[10, 7] = -3e38
    x[11, 7] = 450   # just past 448: the next scale
    x[12, :] = 2.0 ** -100
    x[13, ::2] = -0.0
    x[14] = 65519
    x[15] = 65504
    x[16:] = rng.standard_normal((8, 64)) * np.exp(rng.standard_normal((8, 64)) * 4)
    if kind == "f16":
        x[6] /= 1e35
        x[10, 7] = -3e3
    check(qk, torch_gpu, pool, None, x, x[::-1].copy(), None, None, 1, 0, False)


@pytest.mark.parametrize("kind", KINDS)
def test_absent_pages_and_left_out_sequences(qk, torch_gpu, kind):
    """Table entries outside the pool write nothing and read zeros; sequences
    that do not fit what the batch says are left out whole."""
    rng = np.random.default_rng(9)
    seqs = [(20, 10), (3, 0), (4, 40), (2, 0), (1, 90), (6, 0)]
    pool = paged_ref.Pool(rng, kind, 2, 64, 16, seqs, table_extra=0)
    pool.table[0, 1] = pool.pages            # rows 16 .. 31 of the first
    pool.table[1, 0] = -5
    pool.table[5, 0] = 2 ** 31 - 1
    cos, sin = tables(rng, 60, 64)
    q, k, v = (rng.standard_normal((pool.n, w * 64)).astype(np.float32) for w in (4, 2, 2))
    # The fourth has a table row that is not there, the fifth reaches beyond
    # the tables (position 90 of 60).
    pool.seqs[3, 3] = len(seqs)
    check(qk, torch_gpu, pool, q, k, v, cos, sin, 4, 64, False, skip=(3,), unwritten=(4,))


@pytest.mark.parametrize("change,skip", [
    (dict(max_count=19), (0,)), (dict(max_rows=43), (2,)), (dict(n_tokens=28), (2,))])
def test_bounds_of_the_batch(qk, torch_gpu, change, skip):
    rng = np.random.default_rng(2)
    pool = paged_ref.Pool(rng, "i8", 2, 64, 16, [(20, 10), (5, 0), (4, 40)])
    n = change.get("n_tokens", pool.n)
    q, k, v = (rng.standard_normal((n, w * 64)).astype(np.float32) for w in (4, 2, 2))
    cos, sin = tables(rng, 60, 64)
    check(qk, torch_gpu, pool, q, k, v, cos, sin, 4, 64, False, skip=skip, **change)


@pytest.mark.parametrize("field,value", [(0, -1), (1, 0), (1, -3), (2, -1), (3, -1), (2, 2 ** 31 - 2), (0, 2 ** 31 - 2)])
def test_bad_descriptors(qk, torch_gpu, field, value):
    rng = np.random.default_rng(2)
    pool = paged_ref.Pool(rng, "i8", 1, 64, 16, [(4, 10), (5, 0)])
    n = pool.n
    pool.seqs[0, field] = value
    cos, sin = tables(rng, 60, 64)
    q, k, v = (rng.standard_normal((n, 64)).astype(np.float32) for _ in range(3))
    check(qk, torch_gpu, pool, q, k, v, cos, sin, 1, 64, False, skip=(0,))


def test_strides_and_in_place(qk, torch_gpu):
    """q, k and v as slices of one fused buffer, q rotated in place, outputs
    with room between their rows."""
    t = torch_gpu
    rng = np.random.default_rng(4)
    heads, kvh, hd = 4, 2, 64
    pool = paged_ref.Pool(rng, "i8", kvh, hd, 16, [(7, 3), (1, 20)])
    cos, sin = tables(rng, 21, hd)
    fused = rng.standard_normal((pool.n, (heads + 2 * kvh) * hd + 4)).astype(np.float32)
    q, k, v = np.split(fused[:, :-4], [heads * hd, (heads + kvh) * hd], 1)
    kv, batch = pool.dev(qk, t)
    f = to_dev(t, fused)
    qd, kd, vd = f[:, : heads * hd], f[:, heads * hd: (heads + kvh) * hd], f[:, (heads + kvh) * hd: -4]
    qk.rope_paged_write(kv, batch, qd, qd, kd, vd, to_dev(t, cos), to_dev(t, sin), heads)
    wide = t.full((pool.n, 2, kvh * hd + 8), 7.0, device="cuda")
    qk.paged_read(kv, batch, wide[:, 0, : kvh * hd], wide[:, 1, : kvh * hd])
    pos = np.r_[3:10, 20]
    rows = lambda x: x.reshape(pool.n, -1, hd)
    got = f.cpu().numpy()
    assert np.array_equal(bits(got[:, : heads * hd]),
                          bits(paged_ref.rotate(rows(q), cos[pos], sin[pos], hd, False).reshape(pool.n, -1)))
    assert np.array_equal(got[:, heads * hd:], fused[:, heads * hd:])
    w = wide.cpu().numpy()
    for i, x in enumerate((paged_ref.rotate(rows(k), cos[pos], sin[pos], hd, False), rows(v))):
        want = paged_ref.encode(x, "i8")[2].astype(np.float32).reshape(pool.n, -1)
        assert np.array_equal(w[:, i, : kvh * hd], want)
    assert (w[:, :, kvh * hd:] == 7).all()
    only = t.empty(pool.n, kvh * hd, device="cuda")
    qk.paged_read(kv, batch, None, only)
    assert np.array_equal(only.cpu().numpy(), w[:, 1, : kvh * hd])
    qk.paged_read(kv, batch, only, None)
    assert np.array_equal(only.cpu().numpy(), w[:, 0, : kvh * hd])


def test_pages_beyond_2_to_the_31_bytes(qk, torch_gpu):
    """A pool of 5 GB: its last pages' rows lie beyond 32-bit offsets."""
    t = torch_gpu
    pages, rows, kvh, hd = 20000, 128, 8, 128
    kv = qk.PagedKV.empty(qk.I8, pages, kvh, rows, hd)
    table = t.tensor([[pages - 1, 3, pages - 7]], dtype=t.int32, device="cuda")
    seqs = t.tensor([[0, 300, 50, 0]], dtype=t.int32, device="cuda")
    batch = qk.PagedBatch(table, seqs, 300, 300, 350)
    rng = np.random.default_rng(8)
    k, v = (rng.standard_normal((300, kvh * hd)).astype(np.float32) for _ in range(2))
    qk.rope_paged_write(kv, batch, None, None, to_dev(t, k), to_dev(t, v), None, None, 1, rot_dim=0)
    back = [t.empty(300, kvh * hd, device="cuda") for _ in range(2)]
    qk.paged_read(kv, batch, *back)
    for b, x in zip(back, (k, v)):
        assert np.array_equal(b.cpu().numpy(), paged_ref.encode(x.reshape(300, kvh, hd), "i8")[2].astype(np.float32).reshape(300, -1))
    q = rng.standard_normal((300, kvh * hd)).astype(np.float32)
    # Rows 0 .. 49 were never written: those of the sequence without them.
    seqs2 = t.tensor([[0, 300, 0, 0]], dtype=t.int32, device="cuda")
    kv2, out = kv, t.empty(300, kvh * hd, device="cuda")
    qk.rope_paged_write(kv2, qk.PagedBatch(table, seqs2, 300, 300, 300), None, None, to_dev(t, k), to_dev(t, v), None, None, 1, rot_dim=0)
    qk.paged_attention(kv2, qk.PagedBatch(table, seqs2, 300, 300, 300), to_dev(t, q), out, kvh)
    ek, ev = (paged_ref.encode(x.reshape(300, kvh, hd), "i8")[2] for x in (k, v))
    for tok in (0, 130, 299):
        for h in (0, 7):
            s = ek[: tok + 1, h] @ q[tok, h * hd:(h + 1) * hd].astype(np.float64) / np.sqrt(hd)
            p = np.exp(s - s.max())
            want = p @ ev[: tok + 1, h] / p.sum()
            assert np.abs(out[tok, h * hd:(h + 1) * hd].cpu().numpy() - want).max() < 2e-5


def test_refusals(qk, torch_gpu):
    t = torch_gpu
    kv = qk.PagedKV.empty(qk.I8, 4, 2, 16, 64)
    table = t.zeros(1, 4, dtype=t.int32, device="cuda")
    batch = qk.PagedBatch(table, t.tensor([[0, 1, 0, 0]], dtype=t.int32, device="cuda"), 1, 1, 1)
    x = t.zeros(1, 128, device="cuda")
    with pytest.raises(qk.QKError, match="shape"):
        qk.paged_read(kv, batch, t.zeros(2, 128, device="cuda"), x)
    with pytest.raises(qk.QKError, match="float32"):
        qk.paged_read(kv, batch, x.half(), x)
    with pytest.raises(qk.QKError, match="null pointer"):
        qk.paged_read(kv, batch, None, None)
    with pytest.raises(qk.QKError, match="scales belong"):
        qk.PagedKV(qk.I8, kv.key, kv.value)
    with pytest.raises(qk.QKError, match="shape"):
        qk.PagedKV(qk.I8, kv.key, kv.value[:2], kv.key_scale, kv.value_scale)
    with pytest.raises(qk.QKError, match="int8"):
        qk.PagedKV(qk.I8, kv.key.half(), kv.value.half(), kv.key_scale, kv.value_scale)
    with pytest.raises(qk.QKError, match="head_dim"):
        qk.paged_read(qk.PagedKV.empty(qk.F16, 4, 2, 16, 80), batch, t.zeros(1, 160, device="cuda"), None)
    with pytest.raises(qk.QKError, match="int32"):
        qk.PagedBatch(table.long(), batch.seqs, 1, 1, 1)
    with pytest.raises(qk.QKError, match="expected"):
        qk.PagedBatch(table, batch.seqs[:, :3].contiguous(), 1, 1, 1)
    with pytest.raises(qk.QKError, match="16-byte"):
        qk.paged_read(kv, batch, t.zeros(129, device="cuda")[1:].view(1, 128), None)
    with pytest.raises(qk.QKError, match="contiguous"):
        qk.paged_read(kv, batch, t.zeros(1, 256, device="cuda")[:, ::2], None)


def test_queries_beside_their_rotation(qk, torch_gpu):
    """q and q_out as the two halves of one buffer's rows, and k and v behind."""
    t = torch_gpu
    rng = np.random.default_rng(11)
    heads, kvh, hd = 4, 2, 64
    pool = paged_ref.Pool(rng, "f16", kvh, hd, 16, [(7, 3), (1, 20)])
    cos, sin = tables(rng, 21, hd)
    kv, batch = pool.dev(qk, t)
    w, kw = heads * hd, kvh * hd
    f = to_dev(t, rng.standard_normal((pool.n, 2 * w + 2 * kw)).astype(np.float32))
    before = f.cpu().numpy()
    qk.rope_paged_write(kv, batch, f[:, :w], f[:, w: 2 * w], f[:, 2 * w: 2 * w + kw], f[:, 2 * w + kw:], to_dev(t, cos), to_dev(t, sin), heads)
    got, pos = f.cpu().numpy(), np.r_[3:10, 20]
    want = paged_ref.rotate(before[:, :w].reshape(pool.n, -1, hd), cos[pos], sin[pos], hd, False).reshape(pool.n, -1)
    assert np.array_equal(bits(got[:, w: 2 * w]), bits(want))
    assert np.array_equal(got[:, :w], before[:, :w]) and np.array_equal(got[:, 2 * w:], before[:, 2 * w:])
    with pytest.raises(qk.QKError, match="overlaps"):
        qk.rope_paged_write(kv, batch, f[:, :w], f[:, hd: w + hd], f[:, 2 * w: 2 * w + kw], f[:, 2 * w + kw:], to_dev(t, cos), to_dev(t, sin), heads)


def test_sizes_beyond_an_int(qk, torch_gpu):
    """Bounds and strides whose lower 32 bits would be fine are refused; a single
    row has no stride to refuse."""
    t = torch_gpu
    kv = qk.PagedKV.empty(qk.F16, 4, 2, 16, 64)
    table, seqs = t.zeros(1, 4, dtype=t.int32, device="cuda"), t.tensor([[0, 2, 0, 0]], dtype=t.int32, device="cuda")
    for sizes in ((2 ** 32 + 2, 2, 2), (2, 2 ** 32 + 2, 2), (2, 2, 2 ** 32 + 2)):
        with pytest.raises(qk.QKError, match="beyond"):
            qk.PagedBatch(table, seqs, *sizes)
    batch = qk.PagedBatch(table, seqs, 2, 2, 2)
    far = t.empty(2 ** 32 + 256, device="cuda")      # 17 GB, never touched
    with pytest.raises(qk.QKError, match="apart"):
        qk.paged_read(kv, batch, far.as_strided((2, 128), (2 ** 32 + 128, 1)), None)
    with pytest.raises(qk.QKError, match="beyond"):
        qk.rope_tables(1e4, 64, t.empty(2, 32, device="cuda"), t.empty(2, 32, device="cuda"), first_pos=2 ** 32)
    one = qk.PagedBatch(table, t.tensor([[0, 1, 0, 0]], dtype=t.int32, device="cuda"), 1, 1, 1)
    odd = t.full((1, 131), 7.0, device="cuda")
    kv.key.zero_()
    qk.paged_read(kv, one, odd[:, :128], None)
    assert not odd[:, :128].any() and (odd[:, 128:] == 7).all()
    qk.paged_read(kv, one, far.as_strided((1, 128), (2 ** 32 + 128, 1)), None)
    assert not far[:128].any()
