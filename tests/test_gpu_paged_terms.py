"""qk_paged_attention_terms_f32 against softmax attention in 64 bits: scores capped by
a tanh, biased by distance, of a window, of a prefix, over every cache type."""
import numpy as np
import pytest

import paged_more_ref as ref
from conftest import rel_l2, to_dev

pytestmark = pytest.mark.gpu
KINDS = ["f16", "i8", "e4m3", "i4"]
# Without terms 3e-6.  A capped score is within 3 * 2^-24 of itself more (the quotient,
# the polynomial or the exponential, the product), of a few units; a bias within 2 *
# 2^-24 of itself, of the scores that have weight again a few: 1e-6 together.
TOL = 4e-6
PAIRS = 3 << 22


@pytest.fixture(params=["own bound", "wide bound"])
def wide(request):
    """max_rows as the batch has it, and so large that what is chosen by it is what
    long contexts take."""
    return request.param == "wide bound"


def run(qk, t, pool, q, heads, wide=False, workspace=True, scale=0.0, **terms):
    over = {"max_rows": max(pool.max_rows, -(-PAIRS // (pool.n * heads)))} if wide else {}
    kv, batch = pool.dev(qk, t, **over)
    out = t.full((batch.n_tokens, heads * pool.hd), np.nan, device="cuda")
    nb = qk.paged_attention_workspace_bytes(batch, heads, pool.kvh, pool.hd, window=terms.get("window", 0)) if workspace else 0
    ws = t.full((nb,), 0xFF, dtype=t.uint8, device="cuda") if nb else None
    dev = {k: to_dev(t, v) if isinstance(v, np.ndarray) else v for k, v in terms.items()}
    qk.paged_attention(kv, batch, to_dev(t, q), out, heads, scale=scale, workspace=ws, **dev)
    t.cuda.synchronize()
    return out.cpu().numpy()


def queries(rng, pool, heads, gain=1.0):
    return (gain * rng.standard_normal((pool.n, heads * pool.hd))).astype(np.float32)


def slopes(heads):
    return np.exp2(-8 * np.arange(1, heads + 1) / heads).astype(np.float32)


SEQS = {"decode": [(1, n - 1) for n in (1, 2, 16, 17, 33, 64, 129, 400)], "chunk": [(150, 0)],
        "mixed": [(3, 90), (33, 31), (1, 64), (64, 0), (1, 300)]}
TERMS = {"cap": dict(cap=5.0), "wide cap": dict(cap=50.0), "window": dict(window=40), "one row": dict(window=1),
         "alibi": dict(slopes=True), "prefix": dict(prefix=[50, 0, 70, 1, 10 ** 6, -5, 33, 64]),
         "all": dict(cap=8.0, window=75, slopes=True, prefix=[60, 20, 10, 100, 3, 0, 2, 90])}


def of(terms, heads, seqs):
    t = dict(terms)
    if "slopes" in t:
        t["slopes"] = slopes(heads)
    if "prefix" in t:
        t["prefix"] = np.array(t["prefix"][: len(seqs)], dtype=np.int32)
    return t


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 64), (5, 5, 96), (16, 4, 128), (6, 1, 256)])
@pytest.mark.parametrize("seqs", SEQS)
@pytest.mark.parametrize("terms", TERMS)
def test_terms(qk, torch_gpu, kind, heads, kvh, hd, seqs, terms, wide):
    rng = np.random.default_rng(hd + len(terms))
    s = SEQS[seqs]
    pool = ref.Pool(rng, kind, kvh, hd, 16 if hd in (96, 128) else 64, s)
    pool.poison(pool.unused())
    q = queries(rng, pool, heads, 4.0 if "cap" in terms else 1.0)   # scores of up to 15: on both sides of 0.55 caps
    t = of(TERMS[terms], heads, s)
    tol = TOL * (4 if "cap" in terms else 1)   # scores four times as large
    assert rel_l2(run(qk, torch_gpu, pool, q, heads, wide, **t), pool.attention(q, heads, **t)) < tol


@pytest.mark.parametrize("kind", ["f16", "i4"])
@pytest.mark.parametrize("count,pos", [(1, 5000), (3, 3999), (200, 3000)])
@pytest.mark.parametrize("window", [1, 31, 64, 1000, 4096, 2 ** 31 - 1])
def test_windows_of_long_contexts(qk, torch_gpu, kind, count, pos, window, wide):
    """Rows before the window may hold anything (their pages may be gone); splits lie
    in the window."""
    rng = np.random.default_rng(window % 1000 + pos)
    pool = ref.Pool(rng, kind, 2, 64, 32, [(count, pos)])
    gone = max(0, pos - window + 1) // 32
    pool.table[0, :gone] = -1
    pool.poison(pool.unused())
    q = queries(rng, pool, 8)
    got = run(qk, torch_gpu, pool, q, 8, wide, window=window)
    assert rel_l2(got, run(qk, torch_gpu, pool, q, 8, wide, workspace=False, window=window)) < TOL
    some = sorted({0, count // 2, count - 1})
    k, v, _ = pool.rows(0, pos + count)
    for i in some:
        lo = max(0, pos + i - window + 1)
        for h in (0, 7):
            s = k[lo: pos + i + 1, h // 4] @ q[i, h * 64:(h + 1) * 64].astype(np.float64) / 8
            p = np.exp(s - s.max())
            assert rel_l2(got[i, h * 64:(h + 1) * 64], p @ v[lo: pos + i + 1, h // 4] / p.sum()) < 2 * TOL


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("seqs", ["decode", "chunk"])
def test_no_terms_are_the_plain_call(qk, torch_gpu, kind, seqs, wide):
    rng = np.random.default_rng(2)
    pool = ref.Pool(rng, kind, 2, 128, 32, SEQS[seqs])
    q = queries(rng, pool, 4)
    plain = run(qk, torch_gpu, pool, q, 4, wide)
    n = len(SEQS[seqs])
    far = run(qk, torch_gpu, pool, q, 4, wide, window=10 ** 6, prefix=np.zeros(n, np.int32), slopes=np.zeros(4, np.float32))
    assert rel_l2(far, plain) < 1e-6   # other splits, the same sums
    assert np.array_equal(run(qk, torch_gpu, pool, q, 4, wide, cap=0.0, window=0), plain)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("seqs", ["decode", "chunk"])
def test_masked_rows_may_hold_anything(qk, torch_gpu, kind, seqs, wide):
    """Rows behind a window that are not finite reach no token; one inside it does."""
    rng = np.random.default_rng(3)
    s = [(1, 200), (1, 90)] if seqs == "decode" else [(40, 100)]
    pool = ref.Pool(rng, kind, 2, 64, 16, s)
    q = queries(rng, pool, 4)
    t = dict(window=30, cap=20.0)
    want = pool.attention(q, 4, **t)
    mask = np.zeros((pool.pages, 16), bool)
    for first, count, pos, tab in pool.seqs:
        for r in range(pos - 30 + 1):
            mask[pool.table[tab, r // 16], r % 16] = True
    keep = [[None if x is None else x.copy() for x in p] for p in (pool.key, pool.value)]
    pool.poison(mask)
    assert rel_l2(run(qk, torch_gpu, pool, q, 4, wide, **t), want) < 4 * TOL
    pool.key, pool.value = keep
    mask[:] = False
    first, count, pos, tab = pool.seqs[0]
    row = pos + count // 2 - 5   # in the window of the sequence's tokens from row - pos to row - pos + 29
    mask[pool.table[tab, row // 16], row % 16] = True
    pool.poison(mask)
    got = run(qk, torch_gpu, pool, q, 4, wide, **t)
    at = np.arange(pool.n)
    sees = (at >= first) & (at < first + count) & (row <= pos + at - first) & (pos + at - first - row < 30)
    assert sees.any() and not np.isfinite(got[sees]).any()
    assert rel_l2(got[~sees], want[~sees]) < 4 * TOL


@pytest.mark.parametrize("kind", ["f16", "i4"])
@pytest.mark.parametrize("seqs", ["decode", "chunk", "mixed"])
def test_prefixes_at_the_ends_of_the_range(qk, torch_gpu, kind, seqs, wide):
    """The least and the largest number: no prefix, and all rows that there are."""
    rng = np.random.default_rng(7)
    s = SEQS[seqs]
    pool = ref.Pool(rng, kind, 2, 64, 16, s)
    pool.poison(pool.unused())
    q = queries(rng, pool, 8)
    for window in (0, 2 ** 31 - 1):
        t = dict(prefix=np.array([(-2 ** 31, 2 ** 31 - 1, -1)[i % 3] for i in range(len(s))], dtype=np.int32), window=window)
        assert rel_l2(run(qk, torch_gpu, pool, q, 8, wide, **t), pool.attention(q, 8, **t)) < TOL


def test_rows_that_see_nothing(qk, torch_gpu, wide):
    """A window of which every page is absent: zeros."""
    rng = np.random.default_rng(5)
    pool = ref.Pool(rng, "i8", 2, 64, 16, [(1, 100), (1, 50)])
    pool.table[0, 4:7] = -1   # rows 64 to 111
    q = queries(rng, pool, 4)
    got = run(qk, torch_gpu, pool, q, 4, wide, window=20, slopes=slopes(4))
    want = pool.attention(q, 4, window=20, slopes=slopes(4))
    assert not got[0].any() and not want[0].any() and rel_l2(got, want) < TOL


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("seqs", ["decode", "chunk"])
def test_scores_far_beyond_the_cap(qk, torch_gpu, kind, seqs, wide):
    """Scores of thousands come to the cap, to equal weights where all of a row's do;
    a negative scale turns them."""
    rng = np.random.default_rng(6)
    pool = ref.Pool(rng, kind, 2, 64, 16, SEQS[seqs])
    q = queries(rng, pool, 4, 300.0)
    for scale in (1.0, -1.0):
        got = run(qk, torch_gpu, pool, q, 4, wide, scale=scale, cap=3.0)
        # Of scores of thousands an error of 3e-6 of them moves those near 0 alone,
        # whose share of all is 1e-3 (|s| < 3 of 2400): 1e-3 * 0.01.
        assert rel_l2(got, pool.attention(q, 4, scale=scale, cap=3.0)) < 2e-5


def test_large_keys(qk, torch_gpu, wide):
    """Key scales above 2^96 (their tiles have units of their own)."""
    rng = np.random.default_rng(9)
    for kind in ("i8", "e4m3", "i4"):
        pool = ref.Pool(rng, kind, 2, 64, 16, [(1, 300), (90, 20)], draw=lambda *s: (rng.standard_normal(s) * 1e36).astype(np.float32))
        q = queries(rng, pool, 4) * np.float32(1e-36)
        t = dict(cap=10.0, window=100, slopes=slopes(4))
        assert rel_l2(run(qk, torch_gpu, pool, q, 4, wide, **t), pool.attention(q, 4, **t)) < TOL


@pytest.mark.parametrize("kind", ["i8", "e4m3", "i4"])
@pytest.mark.parametrize("seqs", ["decode", "chunk", "mixed"])
@pytest.mark.parametrize("terms", ["window", "all"])
def test_values_far_apart(qk, torch_gpu, kind, seqs, terms, wide):
    """Value rows 2^60 apart: each token's own, by the rows that it sees.  A product of
    weight and value is within the score's error of itself (or 2^-32 of the token's
    largest), and few of them make up a token's sum: three times TOL of each head's."""
    rng = np.random.default_rng(11)
    s = SEQS[seqs]
    pool = ref.Pool(rng, kind, 2, 64, 16, s)
    pool.value = list((ref.encode4 if kind == "i4" else lambda x: ref.paged_ref.encode(x, kind))(
        (rng.standard_normal((pool.pages, 2, 16, 64)) * np.exp2(rng.uniform(-30, 30, (pool.pages, 1, 16, 1)))).astype(np.float32)))
    q = queries(rng, pool, 8)
    t = of(TERMS[terms], 8, s)
    got, want = run(qk, torch_gpu, pool, q, 8, wide, **t).reshape(-1, 64), pool.attention(q, 8, **t).reshape(-1, 64)
    norm = np.linalg.norm(want, axis=1)
    assert (np.linalg.norm(got - want, axis=1) <= 3 * TOL * norm).all()


@pytest.mark.parametrize("kind", ["f16", "i8", "i4"])
@pytest.mark.parametrize("heads", [8, 16])
def test_rows_apart_in_place_and_left_out(qk, torch_gpu, kind, heads):
    """Strided queries and outputs, outputs in the queries' place, a sequence that does
    not fit the batch and tokens of none: as they were."""
    t = torch_gpu
    rng = np.random.default_rng(12)
    pool = ref.Pool(rng, kind, 2, 64, 16, [(1, 40), (1, 300), (1, 0), (1, 90)])
    q = queries(rng, pool, heads)
    terms = dict(cap=10.0, window=200)
    want = pool.attention(q, heads, **terms)
    pool.seqs[1, 2] = 2 ** 31 - 2   # its position
    kv, batch = pool.dev(qk, t, max_rows=400, n_tokens=6)
    big = t.full((6, heads * 64 + 12), 7.0, device="cuda")
    rows = big[:, 4: 4 + heads * 64]
    rows[:4] = to_dev(t, q)
    out = t.full((6, heads * 64 + 8), np.nan, device="cuda")[:, : heads * 64]
    ws = t.full((qk.paged_attention_workspace_bytes(batch, heads, 2, 64, window=200),), 0xFF, dtype=t.uint8, device="cuda")
    qk.paged_attention(kv, batch, rows, out, heads, workspace=ws, **terms)
    got = out.cpu().numpy()
    assert rel_l2(got[[0, 2, 3]], want[[0, 2, 3]]) < TOL and np.isnan(got[[1, 4, 5]]).all()
    qk.paged_attention(kv, batch, rows, rows, heads, workspace=ws, **terms)
    assert np.array_equal(rows.cpu().numpy()[[0, 2, 3]], got[[0, 2, 3]])
    assert np.array_equal(rows.cpu().numpy()[1], q[1]) and (rows[4:] == 7).all()
    assert (big[:, :4] == 7).all() and (big[:, 4 + heads * 64:] == 7).all()
