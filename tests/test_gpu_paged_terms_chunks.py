"""qk_paged_attention_terms_f32 where chunks of a prompt have a kernel of their own: with
windows that hide rows, prefixes, caps and slopes, for sequences of many query rows beside
those of few.  Every test first asserts, by the rule that chooses, that it gets there."""
import numpy as np
import pytest

import paged_more_ref as ref
from conftest import rel_l2, to_dev

pytestmark = pytest.mark.gpu
KINDS = ["f16", "i8", "e4m3", "i4"]
TOL = 4e-6   # as in the tests of terms: a score's errors, in units of a few
# Single tokens, chunks from the first row on, over a few rows and over many; 16 or more
# chunk workgroups a KV head.
SEQS = [(150, 0), (1, 1200), (160, 63), (131, 64), (155, 1100), (3, 500), (160, 640), (129, 17), (150, 1023)]
LAYOUTS = [(32, 8, 64), (40, 8, 128), (48, 12, 96)]


def chunks(pool, heads, window=0, **terms):
    """Whether the call's sequences of more than 64 query rows a KV head take the chunk kernel."""
    rows = pool.max_count * (heads // pool.kvh)
    cache = min(pool.max_rows, window + pool.max_count + 62) if window else pool.max_rows
    units = -(-rows // 128) * pool.kvh * len(pool.seqs)
    return rows > 64 and pool.hd <= 128 and (units >= 256 or pool.n * heads * cache >= 3 << 22)


def attention(pool, q, heads, scale=None, cap=0.0, window=0, slopes=None, prefix=None):
    """Softmax attention in 64 bits, a (sequence, head) at a time."""
    hd = pool.hd
    scale = 1 / np.sqrt(hd) if scale is None else scale
    out = np.full((pool.n, heads, hd), np.nan)
    for i, (first, count, pos, t) in enumerate(pool.seqs):
        k, v, present = pool.rows(t, pos + count)
        p, r = pos + np.arange(count)[:, None], np.arange(pos + count)
        seen = r <= p
        if prefix is not None:
            seen = seen | (r < int(prefix[i]))
        if window:
            seen = seen & (p - r < window)
        seen = seen & present
        for h in range(heads):
            s = q[first:first + count, h * hd:(h + 1) * hd].astype(np.float64) @ k[:, h * pool.kvh // heads].T * scale
            if cap:
                s = cap * np.tanh(s / cap)
            if slopes is not None:
                s = s - np.float64(slopes[h]) * np.abs(p - r)
            s = np.where(seen, s, -np.inf)
            top = s.max(-1, keepdims=True)
            w = np.exp(s - np.where(np.isfinite(top), top, 0))
            total = w.sum(-1, keepdims=True)
            out[first:first + count, h] = w @ v[:, h * pool.kvh // heads] / np.where(total > 0, total, 1)
    return out.reshape(pool.n, -1)


def run(qk, t, pool, q, heads, workspace=True, scale=0.0, **terms):
    assert chunks(pool, heads, **terms)
    kv, batch = pool.dev(qk, t)
    out = t.full((pool.n, heads * pool.hd), np.nan, device="cuda")
    nb = qk.paged_attention_workspace_bytes(batch, heads, pool.kvh, pool.hd, window=terms.get("window", 0)) if workspace else 0
    ws = t.full((nb,), 0xFF, dtype=t.uint8, device="cuda") if nb else None
    dev = {k: to_dev(t, v) if isinstance(v, np.ndarray) else v for k, v in terms.items()}
    qk.paged_attention(kv, batch, to_dev(t, q), out, heads, scale=scale, workspace=ws, **dev)
    t.cuda.synchronize()
    return out.cpu().numpy()


def queries(rng, pool, heads, gain=1.0):
    return (gain * rng.standard_normal((pool.n, heads * pool.hd))).astype(np.float32)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hd", LAYOUTS)
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 30, 2 ** 30])
def test_windows_beyond_all_rows_leave_a_prefix_seen(qk, torch_gpu, kind, heads, kvh, hd, window):
    """The first row of a window far before row 0, for tokens before their prefix's end."""
    rng = np.random.default_rng(hd)
    pool = ref.Pool(rng, kind, kvh, hd, 32, SEQS)
    q = queries(rng, pool, heads)
    prefix = np.array([50, 0, 100, 170, 1111, 502, 77, 145, 2 ** 31 - 1], dtype=np.int32)
    got = run(qk, torch_gpu, pool, q, heads, window=window, prefix=prefix)
    assert rel_l2(got, attention(pool, q, heads, window=window, prefix=prefix)) < TOL


def slopes(heads):
    return np.exp2(-8 * np.arange(1, heads + 1) / heads).astype(np.float32)


PREFIX = np.array([50, 0, 100, 70, 1111, 502, -5, 145, 64], dtype=np.int32)
TERMS = {"window 1": dict(window=1), "window 40": dict(window=40), "window 75": dict(window=75), "window 300": dict(window=300),
         "window 1000": dict(window=1000), "window and prefix": dict(window=90, prefix=PREFIX), "cap": dict(cap=5.0),
         "slopes": dict(slopes=True), "all": dict(cap=8.0, window=130, slopes=True, prefix=PREFIX)}


def of(terms, heads):
    return dict(terms, slopes=slopes(heads)) if "slopes" in terms else dict(terms)


def behind(pool, window):
    """Mask [pages, page_rows] of the rows before every token's window; their whole pages
    leave the table."""
    mask = np.zeros((pool.pages, pool.page_rows), bool)
    for first, count, pos, t in pool.seqs:
        for r in range(max(pos - window + 1, 0)):
            mask[pool.table[t, r // pool.page_rows], r % pool.page_rows] = True
        pool.table[t, : max(pos - window + 1, 0) // pool.page_rows] = -1
    return mask


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hd", LAYOUTS)
@pytest.mark.parametrize("terms", TERMS)
def test_terms_of_chunks(qk, torch_gpu, kind, heads, kvh, hd, terms):
    """What lies behind every window is not finite, or its page is absent."""
    rng = np.random.default_rng(hd + len(terms))
    pool = ref.Pool(rng, kind, kvh, hd, 16 if hd == 96 else 64, SEQS)
    t = of(TERMS[terms], heads)
    mask = pool.unused()
    if "window" in t:
        mask |= behind(pool, t["window"])
    pool.poison(mask)
    q = queries(rng, pool, heads, 4.0 if "cap" in t else 1.0)
    tol = TOL * (4 if "cap" in t else 1)   # scores four times as large
    assert rel_l2(run(qk, torch_gpu, pool, q, heads, **t), attention(pool, q, heads, **t)) < tol


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hd,window", [(32, 8, 64, 300), (32, 8, 128, 1000), (24, 2, 96, 600), (32, 8, 64, 64)])
def test_splits_of_a_window(qk, torch_gpu, kind, heads, kvh, hd, window):
    """One chunk whose rows are divided: splits begin at the first token's window."""
    rng = np.random.default_rng(window)
    pool = ref.Pool(rng, kind, kvh, hd, 32, [(700, 900)])
    if window == 64:   # (more tokens, for the rule's sake)
        pool = ref.Pool(rng, kind, kvh, hd, 32, [(1100, 900)])
    pool.poison(pool.unused() | behind(pool, window))
    q = queries(rng, pool, heads)
    prefix = np.array([1000], dtype=np.int32)
    for t in (dict(window=window), dict(window=window, prefix=prefix, slopes=slopes(heads))):
        got = run(qk, torch_gpu, pool, q, heads, **t)
        assert rel_l2(got, attention(pool, q, heads, **t)) < TOL
        assert rel_l2(got, run(qk, torch_gpu, pool, q, heads, workspace=False, **t)) < TOL


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,prefix", [(30, False), (100, False), (100, True)])
def test_one_row_that_is_not_finite(qk, torch_gpu, kind, window, prefix):
    """It reaches the tokens that see it, in chunks and beside them, and no other."""
    heads, kvh = 32, 8
    rng = np.random.default_rng(window)
    pool = ref.Pool(rng, kind, kvh, 64, 16, SEQS)
    q = queries(rng, pool, heads)
    t = dict(window=window) | (dict(prefix=np.array([150, 0, 100, 170, 1200, 0, 700, 140, 1100], dtype=np.int32)) if prefix else {})
    want = attention(pool, q, heads, **t)
    mask = np.zeros((pool.pages, 16), bool)
    sees = np.zeros(pool.n, bool)
    for i, (first, count, pos, tab) in enumerate(pool.seqs):
        row = pos + count // 2 - (1 if count == 1 else 0)
        mask[pool.table[tab, row // 16], row % 16] = True
        p = pos + np.arange(count)
        sees[first:first + count] = ((row <= p) | (prefix and row < t["prefix"][i])) & (p - row < window)
    pool.poison(mask)
    got = run(qk, torch_gpu, pool, q, heads, **t)
    assert sees.any() and not sees.all() and not np.isfinite(got[sees]).any()
    assert rel_l2(got[~sees], want[~sees]) < TOL


@pytest.mark.parametrize("kind", ["i8", "e4m3", "i4"])
@pytest.mark.parametrize("terms", ["window 75", "cap", "slopes", "all"])
def test_large_keys(qk, torch_gpu, kind, terms):
    """Key scales above 2^96: tiles with units of their own.  (Some rows' are small: both
    kinds of tile in a sequence.)"""
    heads, kvh, hd = 32, 8, 64
    rng = np.random.default_rng(9)
    draw = lambda *s: (rng.standard_normal(s) * np.where(rng.random((s[0], 1, 1, 1)) < 0.3, 1e24, 1e36)).astype(np.float32)
    pool = ref.Pool(rng, kind, kvh, hd, 64, SEQS, draw=draw)
    q = queries(rng, pool, heads) * np.float32(1e-36)
    t = of(TERMS[terms], heads)
    want = attention(pool, q, heads, **t)
    assert rel_l2(run(qk, torch_gpu, pool, q, heads, **t), want) < TOL


@pytest.mark.parametrize("kind", ["i8", "e4m3", "i4"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("terms", ["window 40", "window 300", "cap", "slopes", "all"])
def test_values_far_apart(qk, torch_gpu, kind, hd, terms):
    """Value rows 2^60 apart, each token's own head by head: a product of weight and value
    is within the score's error of itself (or 2^-32 of the token's largest), and few of
    them make up a token's sum: three times the bound of scores as large."""
    heads, kvh = 32, 8
    rng = np.random.default_rng(11)
    pool = ref.Pool(rng, kind, kvh, hd, 64, SEQS)
    pool.value = list((ref.encode4 if kind == "i4" else lambda x: ref.paged_ref.encode(x, kind))(
        (rng.standard_normal((pool.pages, kvh, 64, hd)) * np.exp2(rng.uniform(-30, 30, (pool.pages, 1, 64, 1)))).astype(np.float32)))
    q = queries(rng, pool, heads)
    t = of(TERMS[terms], heads)
    got, want = run(qk, torch_gpu, pool, q, heads, **t).reshape(-1, hd), attention(pool, q, heads, **t).reshape(-1, hd)
    norm = np.linalg.norm(want, axis=1)
    assert (np.linalg.norm(got - want, axis=1) <= 3 * TOL * norm).all()
