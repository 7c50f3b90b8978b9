"""qk_paged_attention_f32 against softmax attention in 64 bits over the values
that the pages stand for."""
import numpy as np
import pytest

import paged_ref
from conftest import rel_l2, to_dev

pytestmark = pytest.mark.gpu
KINDS = ["f16", "i8", "e4m3"]
# A score is sum q k / sqrt(hd) of normal values: |q| |k| / sqrt(hd) is about
# sqrt(hd), 16 at most.  q keeps 2^-22 of its largest value, products and sums
# of hd / 32 steps in fp32 2^-24 each, so a score is within 16 * 1.45 * (2^-22 +
# 8 * 2^-24) in base 2 were all errors alike, e.g. 1.7e-5; they are not (32 and
# more independent ones): a sixth of it, 3e-6, bounds what a probability is off
# by, and the output, an average of them.
TOL = 3e-6
LAYOUTS = [(32, 8, 64), (6, 6, 64), (16, 2, 96), (5, 1, 96), (24, 8, 128), (8, 8, 128), (20, 1, 128), (8, 1, 256), (4, 2, 256)]


PAIRS = 3 << 22   # of a query row and a cache row: from there on chunks have a kernel of their own


@pytest.fixture(params=["own bound", "wide bound"], autouse=True)
def wide(request):
    """Every test twice: max_rows as the batch has it, and so large that what is
    chosen by it is what long contexts take."""
    run.wide = request.param == "wide bound"


def bound(pool, heads):
    return {"max_rows": max(pool.max_rows, -(-PAIRS // (pool.n * heads)))} if run.wide else {}


def run(qk, t, pool, q, heads, workspace=True, scale=0.0, **over):
    kv, batch = pool.dev(qk, t, **(bound(pool, heads) | over))
    out = t.full((batch.n_tokens, heads * pool.hd), np.nan, device="cuda")
    nb = qk.paged_attention_workspace_bytes(batch, heads, pool.kvh, pool.hd) if workspace is True else workspace
    ws = t.full((nb,), 0xFF, dtype=t.uint8, device="cuda") if nb else None   # stale partials are not numbers
    qk.paged_attention(kv, batch, to_dev(t, q), out, heads, scale=scale, workspace=ws)
    t.cuda.synchronize()
    return out.cpu().numpy()


def queries(rng, pool, heads):
    return rng.standard_normal((pool.n, heads * pool.hd)).astype(np.float32)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hd", LAYOUTS)
@pytest.mark.parametrize("page_rows", [16, 64])
def test_decoding_sequences(qk, torch_gpu, kind, heads, kvh, hd, page_rows):
    """One token each, lengths around the tiles and the pages, unused rows not
    finite."""
    rng = np.random.default_rng(hd)
    pool = paged_ref.Pool(rng, kind, kvh, hd, page_rows, [(1, n - 1) for n in (1, 2, 15, 16, 17, 31, 32, 33, 64, 127, 129, 400)])
    pool.poison(pool.unused())
    q = queries(rng, pool, heads)
    assert rel_l2(run(qk, torch_gpu, pool, q, heads), pool.attention(q, heads)) < TOL


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hd", LAYOUTS)
@pytest.mark.parametrize("seqs", [[(70, 0)], [(3, 90), (33, 31), (1, 64), (64, 0)]], ids=["fresh", "mixed"])
def test_chunks(qk, torch_gpu, kind, heads, kvh, hd, seqs):
    rng = np.random.default_rng(hd + len(seqs))
    pool = paged_ref.Pool(rng, kind, kvh, hd, 32, seqs)
    pool.poison(pool.unused())
    q = queries(rng, pool, heads)
    assert rel_l2(run(qk, torch_gpu, pool, q, heads), pool.attention(q, heads)) < TOL


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hd,count,pos", [(32, 8, 64, 1, 5000), (24, 8, 128, 1, 9000), (8, 1, 256, 3, 4000),
                                                    (16, 2, 96, 2, 3001), (8, 2, 128, 300, 1200), (8, 8, 64, 517, 300),
                                                    (8, 1, 256, 130, 1700), (16, 2, 96, 150, 1500)])
def test_long_rows_and_chunks(qk, torch_gpu, kind, heads, kvh, hd, count, pos):
    """Rows split over workgroups, and long chunks: a few tokens against the
    oracle, all of them against the call without a workspace (one split)."""
    rng = np.random.default_rng(pos)
    pool = paged_ref.Pool(rng, kind, kvh, hd, 128, [(count, pos)])
    pool.poison(pool.unused())
    q = queries(rng, pool, heads)
    got = run(qk, torch_gpu, pool, q, heads)
    assert rel_l2(got, run(qk, torch_gpu, pool, q, heads, workspace=0)) < TOL
    k, v, _ = pool.rows(0, pos + count)
    for i in sorted({0, count // 3, count - 1}):
        for h in (0, heads - 1):
            s = k[: pos + i + 1, h * kvh // heads] @ q[i, h * hd:(h + 1) * hd].astype(np.float64) / np.sqrt(hd)
            p = np.exp(s - s.max())
            assert rel_l2(got[i, h * hd:(h + 1) * hd], p @ v[: pos + i + 1, h * kvh // heads] / p.sum()) < 2 * TOL


@pytest.mark.parametrize("kind", KINDS)
def test_smaller_workspaces(qk, torch_gpu, kind):
    """Fewer splits where fewer fit; a few bytes are none."""
    rng = np.random.default_rng(3)
    pool = paged_ref.Pool(rng, kind, 2, 64, 64, [(1, 3000), (1, 100), (2, 1500)])
    q = queries(rng, pool, 8)
    want = pool.attention(q, 8)
    for nb in (0, 100, 3 * pool.n * 8 * 68 * 4 + 16, 5 * pool.n * 8 * 68 * 4):
        assert rel_l2(run(qk, torch_gpu, pool, q, 8, workspace=nb), want) < TOL


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,heads,kvh", [(64, 8, 2), (128, 4, 4)])
def test_absent_pages(qk, torch_gpu, kind, hd, heads, kvh):
    """Rows of absent pages take no part: in the middle, all of a sequence
    (zeros), all that the chunk's first tokens see, entries beyond the pool."""
    rng = np.random.default_rng(4)
    pool = paged_ref.Pool(rng, kind, kvh, hd, 16, [(1, 200), (1, 40), (40, 0), (5, 30), (1, 900)])
    pool.table[0, 3:7] = -1
    pool.table[1, :] = -1
    pool.table[2, 0] = pool.pages
    pool.table[3, 1] = -2 ** 31
    pool.table[4, ::2] = 2 ** 31 - 1
    pool.poison(pool.unused())
    pool.poison(np.arange(pool.pages)[:, None] * 0 + np.zeros((1, 16)) > 1)
    q = queries(rng, pool, heads)
    got, want = run(qk, torch_gpu, pool, q, heads), pool.attention(q, heads)
    assert not got[1].any() and not want[1].any() and not got[2:18].any()
    assert rel_l2(got, want) < TOL


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("count,pos", [(1, 300), (40, 60), (200, 0)])
def test_left_out_sequences(qk, torch_gpu, kind, count, pos):
    """A sequence that does not fit the batch leaves its outputs as they were,
    and so do tokens that no sequence holds."""
    rng = np.random.default_rng(4)
    pool = paged_ref.Pool(rng, kind, 2, 64, 16, [(2, 5), (count, pos), (3, 9)])
    q = queries(rng, pool, 4)
    want = pool.attention(q, 4)
    for bad in ((2, -1), (3, 3), (0, pool.n), (1, 0), (2, 2 ** 31 - 2)):
        keep = pool.seqs[1].copy()
        pool.seqs[1, bad[0]] = bad[1]
        got = run(qk, torch_gpu, pool, q, 4)
        pool.seqs[1] = keep
        rows = np.r_[0:2, 2 + count: pool.n]
        assert rel_l2(got[rows], want[rows]) < TOL and np.isnan(got[2: 2 + count]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_strides_scale_and_streams(qk, torch_gpu, kind):
    """q and out inside wider rows, a scale of the caller's, another stream."""
    t = torch_gpu
    rng = np.random.default_rng(6)
    pool = paged_ref.Pool(rng, kind, 2, 64, 32, [(1, 100), (9, 20)])
    q = queries(rng, pool, 8)
    kv, batch = pool.dev(qk, t)
    wide = t.full((pool.n, 8 * 64 + 12), 7.0, device="cuda")
    wide[:, : 8 * 64] = to_dev(t, q)
    out = t.full((pool.n, 8 * 64 + 4), 7.0, device="cuda")
    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(side):
        qk.paged_attention(kv, batch, wide[:, : 8 * 64], out[:, : 8 * 64], 8, scale=0.03)
    side.synchronize()
    assert rel_l2(out[:, : 8 * 64].cpu().numpy(), pool.attention(q, 8, 0.03)) < TOL
    assert (out[:, 8 * 64:] == 7).all() and (wide[:, 8 * 64:] == 7).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gain", [1e-30, 1e-4, 30.0])
@pytest.mark.parametrize("spread", [0.0, 4.0])
@pytest.mark.parametrize("count", [1, 130])
def test_magnitudes(qk, torch_gpu, kind, gain, spread, count):
    """Small and large queries, rows whose magnitudes differ by e^+-8 (the value
    scales' exponents with them)."""
    rng = np.random.default_rng(7)
    row_gain = lambda *s: rng.standard_normal(s).astype(np.float32) * np.exp(spread * rng.standard_normal(s[:-1] + (1,)) / 2).astype(np.float32)
    pool = paged_ref.Pool(rng, kind, 2, 64, 16, [(count, 350)], draw=row_gain)
    q = queries(rng, pool, 4) * np.float32(gain)
    got, want = run(qk, torch_gpu, pool, q, 4), pool.attention(q, 4)
    # Scores of up to |q| |k| / 8 in natural units, each within a few 2^-23 of
    # its size: gain 30 and rows of e^4 give scores of some thousands, of which
    # the largest decides; their error moves probabilities by itself.
    k = pool.rows(0, 350 + count)[0]
    size = np.linalg.norm(q.reshape(-1, 64), axis=1).max() * np.linalg.norm(k, axis=-1).max() / 8
    assert rel_l2(got, want) < max(TOL, size * 2.0 ** -23 * 2)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("count", [1, 200])
def test_scales_of_other_writers(qk, torch_gpu, kind, count):
    """Rows of zeros (scale 1 and scale 0), scales far apart."""
    rng = np.random.default_rng(8)
    pool = paged_ref.Pool(rng, kind, 1, 64, 16, [(count, 200)])
    if kind != "f16":
        for part in (pool.value, pool.key):
            part[0][:, :, 3] = 0
            part[2][:, :, 3] = 0
            part[1][:, :, 3] = 0
        f = np.float32(2.0) ** rng.integers(-60, 40, pool.value[1].shape).astype(np.float32)
        pool.value[1] = pool.value[1] * f
        pool.value[2] = pool.value[2] * f[..., None].astype(np.float64)
    q = queries(rng, pool, 2)
    assert rel_l2(run(qk, torch_gpu, pool, q, 2), pool.attention(q, 2)) < TOL


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("count,pos", [(40, 30), (300, 10)])
def test_not_finite_rows_reach_only_those_who_see_them(qk, torch_gpu, kind, count, pos):
    rng = np.random.default_rng(9)
    at = pos + count // 2
    for part in ("key", "value"):
        for bad in (np.nan, np.inf):
            pool = paged_ref.Pool(rng, kind, 2, 64, 16, [(count, pos)])
            codes, scale, _ = getattr(pool, part)
            page = pool.table[0, at // 16]
            if kind == "f16":
                codes[page, 1, at % 16, 5] = bad
            elif kind == "i8":
                scale[page, 1, at % 16] = np.nan
            else:
                codes[page, 1, at % 16, 5] = 0x7F
            clean = paged_ref.Pool(np.random.default_rng(9), kind, 2, 64, 16, [(count, pos)])
            q = queries(np.random.default_rng(1), pool, 4)
            got = run(qk, torch_gpu, pool, q, 4).reshape(count, 4, 64)
            sees = np.arange(pos, pos + count) >= at
            assert np.isfinite(got[~sees]).all() and np.isfinite(got[:, :2]).all()
            assert (~np.isfinite(got[sees][:, 2:])).any(-1).all()
            pool_ok = pool.attention(q, 4).reshape(count, 4, 64)
            assert rel_l2(got[~sees], pool_ok[~sees]) < TOL and rel_l2(got[:, :2], pool_ok[:, :2]) < TOL
            del clean


@pytest.mark.parametrize("count", [1, 200])
def test_not_finite_queries(qk, torch_gpu, count):
    rng = np.random.default_rng(10)
    pool = paged_ref.Pool(rng, "i8", 2, 64, 16, [(count, 30), (2, 9)])
    q = queries(rng, pool, 4)
    q[0, 70], q[count, 3], q[count + 1, 255] = np.nan, np.inf, -np.inf
    got, want = run(qk, torch_gpu, pool, q, 4).reshape(-1, 4, 64), None
    q2 = np.where(np.isfinite(q), q, 0)
    want = pool.attention(q2, 4).reshape(-1, 4, 64)
    bad = [(0, 1), (count, 0), (count + 1, 3)]
    for b in bad:
        assert np.isnan(got[b]).all()
        got[b] = want[b]
    assert rel_l2(got, want) < TOL


@pytest.mark.parametrize("kind", KINDS)
def test_the_same_call_twice_and_captured(qk, torch_gpu, kind):
    """Bit for bit the same again, and in a graph replayed over new inputs,
    between eager calls on another workspace."""
    t = torch_gpu
    rng = np.random.default_rng(11)
    pool = paged_ref.Pool(rng, kind, 2, 64, 32, [(1, 2000), (1, 50), (130, 20)])
    kv, batch = pool.dev(qk, t, **bound(pool, 8))
    nb = qk.paged_attention_workspace_bytes(batch, 8, 2, 64)
    ws = [t.empty(max(nb, 16), dtype=t.uint8, device="cuda") for _ in range(2)]
    q = to_dev(t, queries(rng, pool, 8))
    out, eager = t.empty_like(q), t.empty_like(q)
    call = lambda o, w: qk.paged_attention(kv, batch, q, o, 8, workspace=w)
    call(out, ws[0])
    call(eager, ws[1])
    assert t.equal(out, eager)
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g):
        call(out, ws[0])
    for i in range(4):
        q.copy_(to_dev(t, queries(rng, pool, 8)))
        out.fill_(7)
        g.replay()
        call(eager, ws[1])
        t.cuda.synchronize()
        assert t.equal(out, eager)


@pytest.mark.parametrize("workspace", [0, True, 200000])
def test_the_largest_bound(qk, torch_gpu, workspace):
    """max_rows may be as large as rows can be counted."""
    rng = np.random.default_rng(12)
    pool = paged_ref.Pool(rng, "f16", 2, 64, 1024, [(1, 1500), (150, 900), (1, 0)])
    q = queries(rng, pool, 4)
    got = run(qk, torch_gpu, pool, q, 4, workspace=workspace, max_rows=2 ** 31 - 1 - 1024)
    assert rel_l2(got, pool.attention(q, 4)) < TOL


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("count", [1, 150])
def test_shared_pages_and_a_negative_scale(qk, torch_gpu, kind, count):
    """Two sequences that begin with the same pages, and the same one twice, at
    other positions; a scale that prefers the farthest rows."""
    rng = np.random.default_rng(13)
    pool = paged_ref.Pool(rng, kind, 2, 128, 16, [(count, 100), (count, 100), (count, 64)])
    pool.table[1, :4] = pool.table[0, :4]
    pool.seqs[2, 3] = 0
    q = queries(rng, pool, 6)
    for scale in (0.0, -0.05):
        assert rel_l2(run(qk, torch_gpu, pool, q, 6, scale=scale), pool.attention(q, 6, scale or None)) < TOL   # 0: the default


@pytest.mark.parametrize("kind", KINDS)
def test_two_calls_at_once(qk, torch_gpu, kind):
    """On two streams, a workspace each, over the same cache."""
    t = torch_gpu
    rng = np.random.default_rng(14)
    pool = paged_ref.Pool(rng, kind, 2, 64, 64, [(1, 3000), (140, 900), (1, 40)])
    kv, batch = pool.dev(qk, t, **bound(pool, 8))
    nb = qk.paged_attention_workspace_bytes(batch, 8, 2, 64)
    qs = [to_dev(t, queries(rng, pool, 8)) for _ in range(2)]
    outs, ws = [t.empty_like(x) for x in qs], [t.empty(max(nb, 16), dtype=t.uint8, device="cuda") for _ in qs]
    streams = [t.cuda.Stream() for _ in qs]
    t.cuda.synchronize()
    for _ in range(20):
        for x, o, w, s in zip(qs, outs, ws, streams):
            with t.cuda.stream(s):
                qk.paged_attention(kv, batch, x, o, 8, workspace=w)
    t.cuda.synchronize()
    for x, o in zip(qs, outs):
        assert rel_l2(o.cpu().numpy(), pool.attention(x.cpu().numpy(), 8)) < TOL


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("count", [1, 150])
def test_a_query_that_is_not_finite_and_sees_no_row(qk, torch_gpu, kind, count):
    """Zeros like any that sees none."""
    rng = np.random.default_rng(15)
    pool = paged_ref.Pool(rng, kind, 1, 64, 16, [(count, 10), (1, 5)])
    pool.table[0, :] = -1
    q = queries(rng, pool, 2)
    q[0, 3], q[count - 1, 70] = np.nan, np.inf
    got = run(qk, torch_gpu, pool, q, 2)
    assert not got[:count].any()
    assert rel_l2(got[count:], pool.attention(np.nan_to_num(q, posinf=0), 2)[count:]) < TOL


def test_refusals(qk, torch_gpu):
    t = torch_gpu
    pool = paged_ref.Pool(np.random.default_rng(1), "i8", 2, 64, 16, [(1, 3)])
    kv, batch = pool.dev(qk, t)
    x = t.zeros(1, 256, device="cuda")
    with pytest.raises(qk.QKError, match="shape"):
        qk.paged_attention(kv, batch, x, x.clone(), 3)
    with pytest.raises(qk.QKError, match="multiple of kv_heads"):
        qk.paged_attention(kv, batch, x[:, :192], x.clone()[:, :192], 3)
    with pytest.raises(qk.QKError, match="float32"):
        qk.paged_attention(kv, batch, x.half(), x.clone(), 4)
    with pytest.raises(qk.QKError, match="GPU"):
        qk.paged_attention(kv, batch, x.cpu(), x.clone(), 4)


# --------------------------------------------- every token for itself --
#
# Scores of these cases are at most 8 |q| |k| / |q||k| in natural units (hd 64,
# normal values): off by 8 * 1.45 * (2^-22 + 8 * 2^-24) = 8.3e-6 in base 2 were
# all errors alike, 5.8e-6 of a weight, and so of its share; numerator and sum
# both: 1.2e-5 of a token's sum of |weight * value|.  Halves and fp32 sums add
# 2^-22 and some 2^-24.
EACH = 1.3e-5


def place(pool, part, t, rows, x):
    """Rows of sequence t anew, encoded: x [rows, kvh, hd]."""
    codes, scale, value = (getattr(pool, part) + [None])[:3]
    c, s, v = paged_ref.encode(x, pool.kind)
    for i, r in enumerate(rows):
        page, slot = pool.table[t, r // pool.page_rows], r % pool.page_rows
        codes[page, :, slot], value[page, :, slot] = c[i], v[i]
        if scale is not None:
            scale[page, :, slot] = s[i]


def each(got, pool, q, heads):
    """The largest error of any token and head, of its sum of |weight * value|."""
    worst, hd, G = 0.0, pool.hd, heads // pool.kvh
    got = got.reshape(pool.n, heads, hd)
    for first, count, pos, t in pool.seqs:
        k, v, present = pool.rows(t, pos + count)
        for i in range(count):
            seen = present & (np.arange(pos + count) <= pos + i)
            for h in range(heads):
                s = k[seen, h // G] @ q[first + i, h * hd:(h + 1) * hd].astype(np.float64) / np.sqrt(hd)
                p = np.exp(s - s.max())
                p /= p.sum()
                size = (p @ np.abs(v[seen, h // G])).max()
                worst = max(worst, np.nan_to_num(np.abs(got[first + i, h] - p @ v[seen, h // G]).max(), nan=np.inf) / size)
    return worst


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("part", ["key", "value"])
@pytest.mark.parametrize("group", [1, 2, 4])
@pytest.mark.parametrize("pos", [0, 40, 63])
def test_not_finite_rows_under_every_wave(qk, torch_gpu, kind, part, group, pos):
    """A row that is not finite just behind a chunk's first tokens: later ones see
    the whole tile that these see in part, and get no number either."""
    count, at = 300, pos + 5
    rng = np.random.default_rng(20)
    pool = paged_ref.Pool(rng, kind, 1, 64, 16, [(count, pos)])
    q = queries(rng, pool, group)
    want = pool.attention(q, group).reshape(count, -1)
    codes, scale, _ = getattr(pool, part)
    page = pool.table[0, at // 16]
    if kind == "f16":
        codes[page, 0, at % 16, 5] = np.inf
    elif kind == "i8":
        scale[page, 0, at % 16] = np.nan
    else:
        codes[page, 0, at % 16, 5] = 0x7F
    got = run(qk, torch_gpu, pool, q, group)
    sees = np.arange(pos, pos + count) >= at
    assert rel_l2(got[~sees], want[~sees]) < TOL
    assert (~np.isfinite(got[sees].reshape(-1, 64))).any(-1).all()


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("octaves", [20, 30, 40, 90])
@pytest.mark.parametrize("count", [2, 70, 200])
def test_a_large_value_row_of_later_tokens(qk, torch_gpu, kind, octaves, count):
    """It costs the tokens before it nothing."""
    rng = np.random.default_rng(21)
    pool = paged_ref.Pool(rng, kind, 1, 64, 16, [(count, 50)])
    at = 50 + count // 2
    place(pool, "value", 0, [at], rng.standard_normal((1, 1, 64)) * 2.0 ** octaves)
    q = queries(rng, pool, 2)
    assert each(run(qk, torch_gpu, pool, q, 2), pool, q, 2) < EACH


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("octaves", [24, 40])
@pytest.mark.parametrize("count", [1, 100])
@pytest.mark.parametrize("at", [0, 37, 300])
def test_a_large_value_row_of_no_weight(qk, torch_gpu, kind, octaves, count, at):
    """Every token sees it and gives it e^-80 of another's weight; what it adds,
    2^40 e^-80, is below 2^-75."""
    rng = np.random.default_rng(22)
    pool = paged_ref.Pool(rng, kind, 1, 64, 16, [(count, 400)])
    place(pool, "value", 0, [at], rng.standard_normal((1, 1, 64)) * 2.0 ** octaves)
    place(pool, "key", 0, [at], np.full((1, 1, 64), -12.0))   # score -12 * 64 / 8 for q of ones
    q = queries(rng, pool, 2) * np.float32(0.1) + 1
    assert each(run(qk, torch_gpu, pool, q, 2), pool, q, 2) < EACH


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("octaves", [-20, -40, -70])
@pytest.mark.parametrize("count", [1, 130])
def test_rows_of_zeros_among_small_values(qk, torch_gpu, kind, octaves, count):
    """A row of zeros has scale 1, far above its neighbours' scales; and one has
    every zero but its last."""
    rng = np.random.default_rng(23)
    small = lambda *s: rng.standard_normal(s) * 2.0 ** octaves
    pool = paged_ref.Pool(rng, kind, 1, 64, 16, [(count, 300)])
    total = 300 + count
    place(pool, "value", 0, range(total), small(total, 1, 64))
    zero = [0, 5, 31, 32, 100, 101, 102, 250, 300, total - 1]
    place(pool, "value", 0, zero, np.zeros((len(zero), 1, 64)))
    one = small(1, 1, 64)
    one[..., :63] = 0
    place(pool, "value", 0, [17], one)
    q = queries(rng, pool, 2)
    assert each(run(qk, torch_gpu, pool, q, 2), pool, q, 2) < EACH


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("count", [1, 200])
def test_value_scales_far_apart_token_by_token(qk, torch_gpu, kind, count):
    """Scales over 2^100, in any order and falling with the position."""
    for order in ("any", "falling", "rising"):
        rng = np.random.default_rng(24)
        pool = paged_ref.Pool(rng, kind, 1, 64, 16, [(count, 200)])
        e = rng.uniform(-60, 40, 200 + count)
        e = {"any": e, "falling": -np.sort(-e), "rising": np.sort(e)}[order]
        place(pool, "value", 0, range(200 + count), rng.standard_normal((200 + count, 1, 64)) * 2.0 ** np.floor(e)[:, None, None])
        q = queries(rng, pool, 2)
        assert each(run(qk, torch_gpu, pool, q, 2), pool, q, 2) < EACH, order


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("count", [1, 40, 300])
@pytest.mark.parametrize("bad", [np.inf, -np.inf])
def test_an_infinite_key_scale(qk, torch_gpu, kind, count, bad):
    """Its product with a query is -inf half of the time: no number all the same,
    to the tokens that see it."""
    rng = np.random.default_rng(25)
    pool = paged_ref.Pool(rng, kind, 1, 64, 16, [(count, 90)])
    q = queries(rng, pool, 4)
    want = pool.attention(q, 4)
    at = 90 + count // 3
    pool.key[1][pool.table[0, at // 16], 0, at % 16] = bad
    got = run(qk, torch_gpu, pool, q, 4)
    sees = np.arange(90, 90 + count) >= at
    assert not np.isfinite(got[sees]).any()
    if count > 1:
        assert rel_l2(got[~sees], want[~sees]) < TOL


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("count", [1, 130])
@pytest.mark.parametrize("octaves", [60, 112])
def test_large_keys_and_small_queries(qk, torch_gpu, kind, count, octaves):
    """Ordinary scores of keys some 2^112 and queries some 2^-112, next to rows of
    2^-20 of such keys."""
    rng = np.random.default_rng(26)
    pool = paged_ref.Pool(rng, kind, 1, 64, 16, [(count, 150)])
    total = 150 + count
    g = np.where(rng.random(total) < 0.3, -20.0, 0.0) + octaves
    place(pool, "key", 0, range(total), rng.standard_normal((total, 1, 64)) * 2.0 ** g[:, None, None])
    q = queries(rng, pool, 2) * np.float32(2.0 ** -octaves)
    assert each(run(qk, torch_gpu, pool, q, 2), pool, q, 2) < EACH


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("count", [1, 130])
def test_peaked_rows_element_by_element(qk, torch_gpu, kind, count):
    """One row of far the highest score: its value, to the halves' bits."""
    rng = np.random.default_rng(27)
    pool = paged_ref.Pool(rng, kind, 1, 64, 16, [(count, 350)])
    q = queries(rng, pool, 1)
    best = rng.integers(0, 350, count)
    best = best if count == 1 else np.arange(count) * 350 // count   # a row each
    place(pool, "key", 0, best, q.reshape(count, 1, 64) * 20)        # score 20 |q|^2 / 8, of others some 20 |q| at most
    k, v, _ = pool.rows(0, 350 + count)
    got = run(qk, torch_gpu, pool, q, 1)
    for i in range(count):
        s = np.sort(k[: 351 + i, 0] @ q[i].astype(np.float64) / 8)
        assert s[-1] - s[-2] > 40   # e^-40 = 2^-57
        assert np.abs(got[i] - v[best[i], 0]).max() <= 2.0 ** -21 * np.abs(v[best[i], 0]).max()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("count", [1, 150])
def test_absent_pages_read_nothing_of_the_first_page(qk, torch_gpu, kind, count):
    """Page 0, which no sequence holds, is full of what is not finite."""
    rng = np.random.default_rng(28)
    pool = paged_ref.Pool(rng, kind, 2, 64, 16, [(count, 200), (1, 40)])
    held = pool.table == 0
    free = np.setdiff1d(np.arange(pool.pages), pool.table[pool.table >= 0])[0]
    for part in (pool.key, pool.value):       # page 0 changes places with a free one
        for a in part:
            if a is not None:
                a[[0, free]] = a[[free, 0]]
    pool.table[held] = free
    pool.table[0, 3:7] = -1
    pool.table[0, 9] = pool.pages
    assert not (pool.table == 0).any()
    pool.poison(pool.unused())
    q = queries(rng, pool, 4)
    assert rel_l2(run(qk, torch_gpu, pool, q, 4), pool.attention(q, 4)) < TOL


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("heads,kvh,hd", [(4, 2, 64), (3, 1, 96), (4, 2, 128), (8, 1, 256)])
@pytest.mark.parametrize("count,pos", [(1, 1700), (130, 1500)])
@pytest.mark.parametrize("workspace", [True, 0])
def test_value_scales_apart_in_every_head_size(qk, torch_gpu, kind, heads, kvh, hd, count, pos, workspace):
    """Rows split over workgroups, whole and by one workgroup: a first row far
    below the others, zeros, rows from some tile on 2^7 and 2^30 as large, the
    largest seen by later tokens alone."""
    rng = np.random.default_rng(29)
    pool = paged_ref.Pool(rng, kind, kvh, hd, 64, [(count, pos)])
    total = pos + count
    e = np.zeros(total)
    e[0], e[500:520], e[1000], e[pos + count // 2:] = -9, 7, -40, 30
    x = rng.standard_normal((total, kvh, hd)) * 2.0 ** e[:, None, None]
    x[[3, 64, 700, 1100]] = 0
    place(pool, "value", 0, range(total), x * 2.0 ** -10)
    q = queries(rng, pool, heads)
    got = run(qk, torch_gpu, pool, q, heads, workspace=workspace)
    assert each(got, pool, q, heads) < EACH * (hd / 64) ** 0.5


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("octaves", [4, 5, 6, 7, 8, 12])
@pytest.mark.parametrize("count", [1, 150])
def test_value_scales_about_the_limit_of_alike(qk, torch_gpu, kind, octaves, count):
    """Every other row's values so many octaves below the rest, and tokens that see
    only small ones first."""
    rng = np.random.default_rng(30)
    pool = paged_ref.Pool(rng, kind, 1, 64, 16, [(count, 300)])
    total = 300 + count
    e = np.where((np.arange(total) % 2 == 0) & (np.arange(total) > 70), 0.0, -octaves)
    place(pool, "value", 0, range(total), rng.standard_normal((total, 1, 64)) * 2.0 ** e[:, None, None])
    q = queries(rng, pool, 2)
    assert each(run(qk, torch_gpu, pool, q, 2), pool, q, 2) < EACH


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("workspace", [True, 0])
def test_in_place(qk, torch_gpu, kind, workspace):
    """Outputs over their queries, bit for bit those elsewhere: both kernels, rows
    split and whole."""
    t = torch_gpu
    rng = np.random.default_rng(31)
    pool = paged_ref.Pool(rng, kind, 2, 128, 32, [(1, 2000), (170, 900), (1, 50), (3, 700)])
    q = queries(rng, pool, 8)
    want = run(qk, t, pool, q, 8, workspace=workspace)
    kv, batch = pool.dev(qk, t, **bound(pool, 8))
    nb = qk.paged_attention_workspace_bytes(batch, 8, 2, 128) if workspace else 0
    ws = t.empty(nb, dtype=t.uint8, device="cuda") if nb else None
    x = to_dev(t, q)
    qk.paged_attention(kv, batch, x, x, 8, workspace=ws)
    assert np.array_equal(x.cpu().numpy(), want)


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("count,pos", [(1, 3), (1, 3000), (1, 400), (150, 800)])
@pytest.mark.parametrize("workspace", [True, 0])
def test_values_next_to_the_largest(qk, torch_gpu, kind, count, pos, workspace):
    """Values of up to 3e38, which sums of many would pass: their mean does not."""
    rng = np.random.default_rng(32)
    pool = paged_ref.Pool(rng, kind, 1, 64, 64, [(count, pos)])
    x = rng.uniform(0.5, 1, (pos + count, 1, 64)) * 3e38
    place(pool, "value", 0, range(pos + count), x)
    q = queries(rng, pool, 2)
    got = run(qk, torch_gpu, pool, q, 2, workspace=workspace)
    assert np.isfinite(got).all() and each(got, pool, q, 2) < EACH
