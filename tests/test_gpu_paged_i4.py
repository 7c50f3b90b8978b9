"""4-bit paged rows: qk_rope_paged_write and qk_paged_read_f32 bit for bit, and
qk_paged_attention_f32 over them, against numpy in 64 bits."""
import numpy as np
import pytest

import paged_more_ref as ref
import paged_ref
from conftest import rel_l2, to_dev

pytestmark = pytest.mark.gpu
LAYOUTS = [(8, 2, 64), (6, 6, 96), (12, 4, 128), (3, 1, 256)]
# As of the other row types (a score is within 3e-6 of itself, as is an average of
# values by its weights): codes times multipliers are whole numbers, exact operands,
# and the rest of the arithmetic is the same.
TOL = 3e-6
PAIRS = 3 << 22   # of a query row and a cache row: from there on chunks have a kernel of their own


def bits(a):
    return np.ascontiguousarray(a).view(np.uint32)


def write(qk, t, pool, k, v):
    """k and v written as the batch's rows: (PagedKV, the rows read back)."""
    kv, batch = pool.dev(qk, t)
    qk.rope_paged_write(kv, batch, None, None, to_dev(t, k), to_dev(t, v), None, None, 0, rot_dim=0)
    back = [t.full((pool.n, k.shape[1]), 7.0, device="cuda") for _ in range(2)]
    qk.paged_read(kv, batch, *back)
    t.cuda.synchronize()
    return kv, [b.cpu().numpy() for b in back]


def check_written(qk, t, pool, k, v):
    kv, back = write(qk, t, pool, k, v)
    for x, old, got, entries, b in ((k, pool.key, kv.key, kv.key_scale, back[0]),
                                    (v, pool.value, kv.value, kv.value_scale, back[1])):
        codes, scales = old[0].copy(), old[1].copy()
        wc, ws, wv = ref.encode4(x.reshape(pool.n, pool.kvh, pool.hd))
        for first, count, p, tab in pool.seqs:
            for j in range(count):
                page, slot = pool.table[tab, (p + j) // pool.page_rows], (p + j) % pool.page_rows
                codes[page, :, slot], scales[page, :, slot] = wc[first + j], ws[first + j]
        assert np.array_equal(got.cpu().numpy(), codes)
        got_e = entries.cpu().numpy()
        nan = np.isnan(np.ascontiguousarray(scales[..., :4]).view(np.float32))[..., 0]
        assert np.array_equal(got_e[~nan], scales[~nan]) and np.array_equal(got_e[nan][..., 4:], scales[nan][..., 4:])
        assert np.isnan(np.ascontiguousarray(got_e[..., :4]).view(np.float32)[..., 0][nan]).all()
        with np.errstate(over="raise"):   # a value as written is an fp32 number
            assert np.array_equal(b, wv.astype(np.float32).reshape(pool.n, -1), equal_nan=True)
        fine = np.isfinite(wv)
        assert np.array_equal(wv.astype(np.float32)[fine].astype(np.float64), wv[fine])


@pytest.mark.parametrize("heads,kvh,hd", LAYOUTS)
@pytest.mark.parametrize("page_rows", [16, 128])
def test_rows_of_a_ragged_batch(qk, torch_gpu, heads, kvh, hd, page_rows):
    """Normal values, a quarter far above the others, one far below, values on
    the grid and between two of it."""
    rng = np.random.default_rng(hd + page_rows)
    pool = ref.Pool(rng, "i4", kvh, hd, page_rows, [(1, 0), (1, 700), (37, 13), (130, 0), (5, 123)])
    k, v = (rng.standard_normal((pool.n, kvh * hd)).astype(np.float32) for _ in range(2))
    k[3:9, : hd // 4] *= 1000
    k[9:12, hd // 4: hd // 2] *= 1e-4
    v[5:30] = rng.integers(-14, 15, v[5:30].shape) * 0.5   # steps of 1 where the largest is 7: ties
    v[5:30, ::hd] = 7
    v[30:60] *= np.exp(rng.uniform(-60, 60, (30, 1))).astype(np.float32)
    check_written(qk, torch_gpu, pool, k, v)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_rows_at_the_ends_of_the_range(qk, torch_gpu, hd):
    """Zeros, rows below and above 2^-100, next to fp32's largest, not finite."""
    rng = np.random.default_rng(hd)
    pool = ref.Pool(rng, "i4", 1, hd, 16, [(12, 3)])
    k, v = (rng.standard_normal((pool.n, hd)).astype(np.float32) for _ in range(2))
    k[0] = 0
    k[1] *= np.float32(2.0 ** -110)
    k[2] = 0
    k[2, 5] = 2.0 ** -100
    k[3, 7] = np.inf
    k[4, hd - 1] = np.nan
    k[5] *= np.float32(1e38) / np.abs(k[5]).max()
    k[6, 1] = ref.FMAX
    k[7, hd // 2] = -ref.FMAX
    v[0] = -0.0
    v[1] = ref.FMAX
    v[2, -1] = -np.inf
    v[3] = np.nextafter(np.float32(2.0 ** -100), np.float32(0))
    v[4] = 1785.0
    v[5] = np.nextafter(np.float32(1785.0), np.float32(2000))
    v[6] = np.nextafter(np.float32(1785.0), np.float32(0))
    check_written(qk, torch_gpu, pool, k, v)


def test_rotated_rows(qk, torch_gpu):
    """Rotation, queries and 4-bit rows in one call, and pages that are absent."""
    t = torch_gpu
    rng = np.random.default_rng(1)
    pool = ref.Pool(rng, "i4", 2, 96, 16, [(20, 10), (1, 60)])
    pool.table[0, 1] = -1
    a = rng.uniform(-np.pi, np.pi, (61, 22))
    cos, sin = np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)
    q, k, v = (rng.standard_normal((pool.n, w * 96)).astype(np.float32) for w in (4, 2, 2))
    kv, batch = pool.dev(qk, t)
    out, kb, vb = t.empty(pool.n, 384, device="cuda"), t.empty(pool.n, 192, device="cuda"), t.empty(pool.n, 192, device="cuda")
    qk.rope_paged_write(kv, batch, to_dev(t, q), out, to_dev(t, k), to_dev(t, v), to_dev(t, cos), to_dev(t, sin), 4,
                        rot_dim=44, half=True)
    qk.paged_read(kv, batch, kb, vb)
    pos = np.r_[10:30, 60]
    turn = lambda x: paged_ref.rotate(x.reshape(pool.n, -1, 96), cos[pos], sin[pos], 44, True)
    assert np.array_equal(bits(out.cpu().numpy()), bits(turn(q).reshape(pool.n, -1)))
    gone = (pos >= 16) & (pos < 32) & (np.arange(pool.n) < 20)
    for got, x in ((kb, turn(k)), (vb, v.reshape(pool.n, 2, 96))):
        want = ref.encode4(x)[2].astype(np.float32).reshape(pool.n, -1)
        want[gone] = 0
        assert np.array_equal(got.cpu().numpy(), want)


# ----------------------------------------------------------- attention --

@pytest.fixture(params=["own bound", "wide bound"])
def wide(request):
    """max_rows as the batch has it, and so large that what is chosen by it is what
    long contexts take."""
    return request.param == "wide bound"


def attend(qk, t, pool, q, heads, wide=False, workspace=True, scale=0.0):
    over = {"max_rows": max(pool.max_rows, -(-PAIRS // (pool.n * heads)))} if wide else {}
    kv, batch = pool.dev(qk, t, **over)
    out = t.full((batch.n_tokens, heads * pool.hd), np.nan, device="cuda")
    nb = qk.paged_attention_workspace_bytes(batch, heads, pool.kvh, pool.hd) if workspace else 0
    ws = t.full((nb,), 0xFF, dtype=t.uint8, device="cuda") if nb else None   # stale partials are not numbers
    qk.paged_attention(kv, batch, to_dev(t, q), out, heads, scale=scale, workspace=ws)
    t.cuda.synchronize()
    return out.cpu().numpy()


def queries(rng, pool, heads):
    return rng.standard_normal((pool.n, heads * pool.hd)).astype(np.float32)


@pytest.mark.parametrize("heads,kvh,hd", [(32, 8, 64), (6, 6, 64), (16, 2, 96), (5, 1, 96), (20, 4, 128), (20, 1, 128),
                                          (8, 1, 256), (4, 2, 256)])
@pytest.mark.parametrize("seqs", [[(1, n - 1) for n in (1, 2, 15, 16, 17, 31, 32, 33, 64, 127, 129, 400)], [(70, 0)],
                                  [(3, 90), (33, 31), (1, 64), (64, 0)]], ids=["decode", "fresh", "mixed"])
def test_attention(qk, torch_gpu, heads, kvh, hd, seqs, wide):
    """Single tokens and chunks, lengths around tiles and pages, unused rows not
    finite."""
    rng = np.random.default_rng(hd + len(seqs))
    pool = ref.Pool(rng, "i4", kvh, hd, 16 if hd == 96 else 64, seqs)
    pool.poison(pool.unused())
    q = queries(rng, pool, heads)
    assert rel_l2(attend(qk, torch_gpu, pool, q, heads, wide), pool.attention(q, heads)) < TOL


@pytest.mark.parametrize("heads,kvh,hd,count,pos", [(32, 8, 64, 1, 5000), (8, 1, 256, 3, 4000), (16, 2, 96, 2, 3001),
                                                    (8, 2, 128, 300, 1200), (8, 8, 64, 517, 300), (16, 2, 96, 150, 1500),
                                                    (8, 1, 256, 130, 1700)])
def test_long_rows_and_chunks(qk, torch_gpu, heads, kvh, hd, count, pos, wide):
    """Rows split over workgroups, and long chunks: a few tokens against the
    oracle, all of them against the call without a workspace (one split)."""
    rng = np.random.default_rng(pos)
    pool = ref.Pool(rng, "i4", kvh, hd, 128, [(count, pos)])
    pool.poison(pool.unused())
    q = queries(rng, pool, heads)
    got = attend(qk, torch_gpu, pool, q, heads, wide)
    assert rel_l2(got, attend(qk, torch_gpu, pool, q, heads, wide, workspace=False)) < TOL
    k, v, _ = pool.rows(0, pos + count)
    for i in sorted({0, count // 3, count - 1}):
        for h in (0, heads - 1):
            s = k[: pos + i + 1, h * kvh // heads] @ q[i, h * hd:(h + 1) * hd].astype(np.float64) / np.sqrt(hd)
            p = np.exp(s - s.max())
            assert rel_l2(got[i, h * hd:(h + 1) * hd], p @ v[: pos + i + 1, h * kvh // heads] / p.sum()) < 2 * TOL


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("seqs", [[(1, 200), (1, 40)], [(300, 5)]], ids=["decode", "chunk"])
def test_every_code_and_multiplier(qk, torch_gpu, hd, seqs, wide):
    """Rows that no writer made: all sixteen codes, multipliers 1 to 255, scales
    over 2^20."""
    rng = np.random.default_rng(hd)
    pool = ref.Pool(rng, "i4", 2, hd, 32, seqs)
    for part in (pool.key, pool.value):
        part[0] = rng.integers(0, 256, part[0].shape, dtype=np.uint8)
        part[1] = rng.integers(1, 256, part[1].shape, dtype=np.uint8)
        top = 2.0 ** -11 if part is pool.key else 1.0   # scores of a few
        scale = (top * np.exp2(rng.uniform(-10, 0 if part is pool.key else 10, part[1].shape[:3]))).astype(np.float32)
        part[1][..., :4] = scale[..., None].view(np.uint8)
        part[2] = ref.decode4(part[0], part[1])
    q = queries(rng, pool, 4) * np.float32(0.1)
    assert rel_l2(attend(qk, torch_gpu, pool, q, 4, wide), pool.attention(q, 4)) < TOL


@pytest.mark.parametrize("seqs", [[(1, 200), (1, 40)], [(300, 5)]], ids=["decode", "chunk"])
def test_absent_pages_and_rows_that_are_not_finite(qk, torch_gpu, seqs, wide):
    """Absent pages take no part; a row with a scale that is not a number makes the
    tokens that see it not finite, and no other."""
    rng = np.random.default_rng(4)
    pool = ref.Pool(rng, "i4", 2, 128, 16, seqs)
    pool.table[0, 1] = -1
    pool.poison(pool.unused())
    q = queries(rng, pool, 8)
    want = pool.attention(q, 8)
    assert rel_l2(attend(qk, torch_gpu, pool, q, 8, wide), want) < TOL
    first, count, pos, tab = pool.seqs[0]
    row = pos + count // 2   # of the first sequence: the tokens from there on see it
    pool.value[1][pool.table[tab, row // 16], :, row % 16, :4] = np.full(1, np.nan, np.float32).view(np.uint8)
    got = attend(qk, torch_gpu, pool, q, 8, wide)
    bad = np.zeros(pool.n, bool)
    bad[first + row - pos: first + count] = True
    assert not np.isfinite(got[bad]).any()
    assert rel_l2(got[~bad], want[~bad]) < TOL if (~bad).any() else True


def test_rows_of_large_values(qk, torch_gpu, wide):
    """Keys next to fp32's largest with queries as small, values likewise."""
    rng = np.random.default_rng(9)
    big = lambda *s: (rng.standard_normal(s) * 1e37).astype(np.float32)
    pool = ref.Pool(rng, "i4", 2, 64, 16, [(1, 300), (90, 20)], draw=big)
    q = queries(rng, pool, 4) * np.float32(1e-37)
    assert rel_l2(attend(qk, torch_gpu, pool, q, 4, wide), pool.attention(q, 4)) < TOL
