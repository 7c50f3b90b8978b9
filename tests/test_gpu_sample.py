"""qk_sample_rows_f32 against the definition in numpy: the token's interval of
the kept weights' running sum holds the given random number."""
import numpy as np
import pytest

from conftest import to_dev

pytestmark = pytest.mark.gpu


def kept_weights(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Weights of the kept tokens, of the largest (0: dropped), by a sort."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    n, top = len(x), x.max()
    order = np.argsort(-x, kind="stable")
    if top == -np.inf:
        return None
    if not temperature > 0 or not top_p > 0 or not min_p <= 1 or top_k == 1:
        w = np.zeros(n)
        w[order[0]] = 1
        return w
    if top == np.inf:
        w = np.where(x == np.inf, 1.0, 0.0)
    else:
        with np.errstate(over="ignore", invalid="ignore"):
            w = np.exp((x - top) / np.float64(temperature))
        w = np.where(x == -np.inf, 0, w)
    keep = np.ones(n, dtype=bool)
    if top_k > 0:
        keep[top_k:] = False
    ws = w[order] * keep
    if top_p < 1:
        before = np.cumsum(ws) - ws
        keep &= before < np.float64(top_p) * ws.sum()
    keep &= ws >= np.float64(min_p)
    keep[0] = True
    out = np.zeros(n)
    out[order[keep]] = ws[keep]
    return out


def check(qk, t, x, u, ldv=None, **params):
    """Tokens of rows x by u; params: a list a row each."""
    rows, n = x.shape
    buf = t.full((rows, ldv or n), 9e30, device="cuda")
    buf[:, :n] = to_dev(t, x)
    dev = {k: to_dev(t, np.asarray(v, dtype=np.int32 if k == "top_k" else np.float32)) for k, v in params.items()}
    out = t.full((rows + 1,), -7, dtype=t.int32, device="cuda")
    prob = t.full((rows + 1,), -7.0, device="cuda")
    ws = t.full((max(1, qk.sample_workspace_bytes(n, rows)),), 0xFF, dtype=t.uint8, device="cuda")
    uu = to_dev(t, np.asarray(u, dtype=np.float32))
    qk.sample_rows(buf[:, :n], uu, out[:rows], prob=prob[:rows], workspace=ws, **dev)
    only = t.empty(rows, dtype=t.int32, device="cuda")
    qk.sample_rows(buf[:, :n], uu, only, workspace=ws, **dev)   # without prob, over a used workspace
    got, pr = out.cpu().numpy(), prob.cpu().numpy()
    assert got[rows] == -7 and pr[rows] == -7 and np.array_equal(only.cpu().numpy(), got[:rows])
    for r in range(rows):
        w = kept_weights(x[r], **{k: (v[r] if k == "top_k" else np.float32(v[r])) for k, v in params.items()})
        if w is None:
            assert got[r] == 0 and pr[r] == 0
            continue
        i, c, total = got[r], np.cumsum(w), w.sum()
        assert 0 <= i < n and w[i] > 0, (r, i)
        # Each of n weights is held to 2^-30 of itself, or has none below 2^-45
        # of the largest; sums in 64 bits add nothing to that.
        eps = n * 2.0 ** -45 + total * 2.0 ** -29
        uv = min(max(np.float64(np.float32(u[r])), 0), 1) if u[r] == u[r] else 0.0
        target = uv * total
        assert c[i] - w[i] <= target + eps and c[i] > target - eps, (r, i, c[i] / total, uv)
        # One rounding to fp32 of a quotient whose parts are off by 2^-30, and by
        # what the tokens without weight leave out.
        assert abs(pr[r] - w[i] / total) <= (2.0 ** -23 * w[i] + 2.0 ** -45 + n * 2.0 ** -45 * w[i]) / total
    return got[:rows]


def logits(rng, rows, n, spread=2.2):
    x = rng.standard_normal((rows, n)).astype(np.float32) * np.float32(spread)
    for r in range(rows):
        at = rng.integers(0, n, min(n, 30))
        x[r, at] = 8 + 3 * rng.standard_normal(len(at))
    return x


PARAMS = {
    "plain": dict(),
    "temperature": dict(temperature=[0.3, 1.7, 1e-6, 50.0]),
    "top_k": dict(top_k=[2, 50, 999, 5000]),
    "top_p": dict(top_p=[0.1, 0.9, 0.999, 1e-6]),
    "min_p": dict(min_p=[0.01, 0.5, 1.0, 1e-6]),
    "all": dict(temperature=[0.7, 0.0, 1.2, 0.9], top_k=[40, 0, 7, 200], top_p=[0.9, 1.0, 0.5, 0.99],
                min_p=[0.05, 0.0, 0.0, 0.001]),
    "off": dict(temperature=[1.0, 1.0, -1.0, 0.0], top_k=[0, -3, 1 << 30, 1], top_p=[1.0, 2.0, 1.0, 1.0],
                min_p=[0.0, -1.0, 0.0, 0.0]),
    "greedy": dict(top_p=[0.0, -1.0, np.nan, 0.5], min_p=[0.0, 0.0, 0.0, 1.5]),
    "not numbers": dict(temperature=[np.nan, np.inf, 1.0, 1.0], min_p=[0.0, 0.0, np.nan, 0.0]),
}


@pytest.mark.parametrize("n", [1, 2, 63, 1000, 4097, 32003, 128256])
@pytest.mark.parametrize("which", PARAMS)
def test_rows(qk, torch_gpu, n, which):
    rng = np.random.default_rng(n)
    p = PARAMS[which]
    for u in ([0.0, 0.25, 0.7, 1 - 2.0 ** -24], rng.random(4).astype(np.float32)):
        check(qk, torch_gpu, logits(rng, 4, n), u, **p)


@pytest.mark.parametrize("rows", [1, 3, 17, 64, 300])
def test_batches(qk, torch_gpu, rows):
    """Each row by its own parameters, whatever the rows beside it; the same
    row alone gives the same token."""
    rng = np.random.default_rng(rows)
    x, u = logits(rng, rows, 5003), rng.random(rows).astype(np.float32)
    p = dict(temperature=rng.uniform(0, 1.5, rows), top_k=rng.integers(-5, 300, rows), top_p=rng.uniform(0.3, 1.1, rows),
             min_p=rng.uniform(-0.1, 0.2, rows))
    got = check(qk, torch_gpu, x, u, **p)
    for r in {0, rows // 2, rows - 1}:
        alone = check(qk, torch_gpu, x[r:r + 1], u[r:r + 1], **{k: v[r:r + 1] for k, v in p.items()})
        assert alone[0] == got[r]


@pytest.mark.parametrize("spread", [0.0, 0.01, 30.0])
@pytest.mark.parametrize("n", [1000, 50001])
def test_flat_and_peaked_rows(qk, torch_gpu, spread, n):
    """Equal logits (every filter cuts among ties), nearly equal ones, and rows
    where a few tokens hold everything."""
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((6, n)) * spread).astype(np.float32)
    check(qk, torch_gpu, x, [0.0, 0.2, 0.5, 0.9, 0.99, 0.4], top_k=[0, n // 3, 77, n - 1, 2, 0],
          top_p=[0.5, 0.75, 1.0, 0.25, 0.9, 0.999], min_p=[0, 0, 0, 0, 0, 0.5])


def test_ties_go_by_index(qk, torch_gpu):
    """Quantised logits: many ties at every threshold, signed zeros among them."""
    rng = np.random.default_rng(2)
    x = np.rint(rng.standard_normal((8, 9001)) * 2).astype(np.float32)
    x[:, ::3] *= np.float32(-1)
    assert (np.signbit(x) & (x == 0)).any()
    check(qk, torch_gpu, x, rng.random(8), top_k=[5, 50, 500, 5000, 0, 0, 3000, 9000], top_p=[1, 1, 1, 1, 0.1, 0.7, 0.6, 0.9])


def test_masked_rows(qk, torch_gpu):
    """-inf, the type's lowest value, NaN, +inf, and rows that leave nothing."""
    low = np.finfo(np.float32).min
    n = 5000
    x = np.full((10, n), -np.inf, dtype=np.float32)
    x[1, 4321] = -3
    x[2] = low
    x[3] = np.nan
    x[4, [7, 4000]] = np.inf
    x[4, 8] = 5
    x[5, :100], x[5, 200] = np.nan, 1
    x[6] = low
    x[6, [10, 20]] = [low / 2, 3e38]
    x[7, 1000:1003] = [1, 2, 3]
    x[8], x[8, 17] = low, 0
    x[9, ::2] = 0
    for params in (dict(), dict(top_k=[3] * 10), dict(top_p=[0.6] * 10), dict(min_p=[0.3] * 10),
                   dict(top_k=[4000] * 10, top_p=[0.95] * 10, temperature=[0.5] * 10), dict(temperature=[1e30] * 10)):
        for u in (0.0, 0.6, 1 - 2.0 ** -24):
            check(qk, torch_gpu, x, [u] * 10, **params)


def test_random_numbers_out_of_range(qk, torch_gpu):
    rng = np.random.default_rng(3)
    x = logits(rng, 5, 700)
    check(qk, torch_gpu, x, [-1.0, 1.0, 5.0, np.nan, np.inf], top_p=[0.9] * 5)


@pytest.mark.parametrize("n,ldv", [(1000, 1001), (4097, 5000), (7, 9)])
def test_strides(qk, torch_gpu, n, ldv):
    rng = np.random.default_rng(4)
    check(qk, torch_gpu, logits(rng, 5, n), rng.random(5), ldv=ldv, top_p=[0.9] * 5, top_k=[30] * 5)


def test_frequencies(qk, torch_gpu):
    """Over 4096 evenly spaced numbers a token is drawn in proportion to its
    weight: its interval holds that many of them, to one at either end."""
    rng = np.random.default_rng(5)
    x = np.repeat(logits(rng, 1, 300), 4096, 0)
    u = (np.arange(4096) + 0.5) / 4096
    p = dict(temperature=[0.9] * 4096, top_p=[0.95] * 4096)
    got = np.bincount(check(qk, torch_gpu, x, u, **p), minlength=300)
    w = kept_weights(x[0], 0.9 * np.float32(1), 0, np.float32(0.95))
    assert np.abs(got - 4096 * w / w.sum()).max() <= 1.001


def test_captured(qk, torch_gpu):
    """Two captured graphs with workspaces of their own, replayed in turn over
    new logits."""
    t = torch_gpu
    rng = np.random.default_rng(6)
    x, u = t.empty(20, 30000, device="cuda"), t.empty(20, device="cuda")
    p = t.full((20,), 0.9, device="cuda")
    outs = [t.empty(20, dtype=t.int32, device="cuda") for _ in range(3)]
    ws = [t.empty(max(1, qk.sample_workspace_bytes(30000, 20)), dtype=t.uint8, device="cuda") for _ in range(3)]
    call = lambda i: qk.sample_rows(x, u, outs[i], top_p=p, workspace=ws[i])
    x.copy_(to_dev(t, logits(rng, 20, 30000)))
    u.uniform_()
    graphs = []
    call(2)
    for i in range(2):
        graphs.append(t.cuda.CUDAGraph())
        with t.cuda.graph(graphs[i]):
            call(i)
    for i in range(5):
        x.copy_(to_dev(t, logits(rng, 20, 30000)))
        u.uniform_()
        graphs[i % 2].replay()
        graphs[1 - i % 2].replay()
        call(2)
        t.cuda.synchronize()
        assert t.equal(outs[0], outs[2]) and t.equal(outs[1], outs[2])


@pytest.mark.parametrize("count", [1, 2, 7, 8, 127, 129, 505, 511, 512, 513, 600, 1025, 2040, 2047, 2048, 2049, 4000])
@pytest.mark.parametrize("min_p", [0.0, 0.993])
def test_as_many_tokens_at_the_cut(qk, torch_gpu, count, min_p):
    """So many tokens within a fiftieth of each other's weight, the rest far
    below; a third, two thirds and nearly all of them kept."""
    rng = np.random.default_rng(count)
    x = np.full((6, 20000), -30, np.float32)
    for r in x:
        r[rng.choice(20000, count, replace=False)] = 3 + 0.02 * rng.random(count)
    check(qk, torch_gpu, x, rng.random(6).astype(np.float32), top_p=np.float32([0.33, 0.67, 0.99] * 2),
          min_p=np.full(6, min_p, np.float32), top_k=np.int32([0, 0, 0, 1, count // 2 + 1, count]))


def test_two_calls_at_once(qk, torch_gpu):
    """On two streams, a workspace each, over the same logits."""
    t = torch_gpu
    rng = np.random.default_rng(8)
    x, n = to_dev(t, logits(rng, 24, 50000)), 50000
    us, tops = [t.rand(24, device="cuda") for _ in range(2)], [t.full((24,), p, device="cuda") for p in (0.95, 0.6)]
    outs = [[t.empty(24, dtype=t.int32, device="cuda") for _ in range(2)] for _ in range(2)]
    ws = [t.empty(qk.sample_workspace_bytes(n, 24), dtype=t.uint8, device="cuda") for _ in range(2)]
    streams = [t.cuda.Stream() for _ in range(2)]
    t.cuda.synchronize()
    for u, p, w, o in zip(us, tops, ws, outs):
        qk.sample_rows(x, u, o[0], top_p=p, workspace=w)
    t.cuda.synchronize()
    for _ in range(20):
        for u, p, w, o, s in zip(us, tops, ws, outs, streams):
            with t.cuda.stream(s):
                qk.sample_rows(x, u, o[1], top_p=p, workspace=w)
    t.cuda.synchronize()
    for o in outs:
        assert t.equal(o[0], o[1])


def test_refusals(qk, torch_gpu):
    t = torch_gpu
    x, u, o = t.zeros(2, 10, device="cuda"), t.zeros(2, device="cuda"), t.zeros(2, dtype=t.int32, device="cuda")
    with pytest.raises(qk.QKError, match="int32"):
        qk.sample_rows(x, u, o.long())
    with pytest.raises(qk.QKError, match="shape"):
        qk.sample_rows(x, u[:1], o)
    with pytest.raises(qk.QKError, match="int32"):
        qk.sample_rows(x, u, o, top_k=u)
    with pytest.raises(qk.QKError, match="float32"):
        qk.sample_rows(x.half(), u, o)
    with pytest.raises(qk.QKError, match="contiguous"):
        qk.sample_rows(x.t().contiguous().t(), u, o)


@pytest.mark.parametrize("n", [5, 1000, 3000, 20000, 40000])
@pytest.mark.parametrize("t", [np.inf, 3e38, 1e30, 2e18, 1e15])
def test_flat_temperatures_with_filters(qk, torch_gpu, n, t):
    """A temperature that leaves all logits alike, up to an infinite one: top-k and
    top-p cut by the logits' order; logits of 0 and next to it among them."""
    rng = np.random.default_rng(n)
    x = logits(rng, 8, n)
    x[:, ::5] = 0
    x[:, 1::5] = rng.choice(np.float32([-1e-20, 1e-20, -1e-30, -0.0, 1e-40, -1e-40]), x[:, 1::5].shape)
    x[7, : n // 2] = -np.inf
    half = max(n // 2, 1)
    params = dict(temperature=[t] * 8, top_k=[0, 2, half, n, 0, 77, 0, 0], top_p=[0.5, 1.0, 0.75, 0.25, 1.0, 0.9, 0.999, 0.5],
                  min_p=[0, 0, 0, 0, 1.0, 0, 0.5, 0])
    # Row 4's filter is at the weights' border: they are e^(-d / t), d the distance
    # to the largest logit, at t = 1e15 below 2^-45 t (28): within 2^-45 of 1, far
    # closer than the 2^-30 that a weight is held to (at 2e18 and more they are 1 in
    # 64 bits).  Any token may be kept there.
    edge = 4 if t == 1e15 else -1
    rows = [r for r in range(8) if r != edge]
    for u in (0.0, 0.37, 1 - 2.0 ** -24):
        check(qk, torch_gpu, x[rows], [u] * len(rows), **{k: [v[r] for r in rows] for k, v in params.items()})
    if edge >= 0:
        assert x[4].max() - x[4].min() < 2.0 ** -45 * t
        got = torch_gpu.empty(1, dtype=torch_gpu.int32, device="cuda")
        ws = torch_gpu.empty(qk.sample_workspace_bytes(n, 1), dtype=torch_gpu.uint8, device="cuda")
        one = lambda v: to_dev(torch_gpu, np.float32([v]))
        qk.sample_rows(to_dev(torch_gpu, x[4:5]), one(0.37), got, temperature=one(t), min_p=one(1.0), workspace=ws)
        assert 0 <= int(got[0]) < n


@pytest.mark.parametrize("n", [131073, 151936, 262144, 524288])
def test_rows_of_many_segments(qk, torch_gpu, n):
    """More than eight segments of 16384 logits, whose heads and histograms are
    gone through by eights; the largest logits in the first, the last or any."""
    rng = np.random.default_rng(n)
    x = logits(rng, 6, n)
    x[1, -100:] = 20 + rng.random(100)
    x[2, :100] = 20 + rng.random(100)
    x[3, 16384 * 8: 16384 * 8 + 1] = 30
    x[4, : n - 16384 - 3] = -np.inf
    for params in (dict(), dict(top_k=[40] * 6, top_p=[0.9] * 6), dict(top_p=[0.9, 0.6, 0.99, 0.999, 0.5, 0.95], temperature=[1.5, 1, 0.7, 3, 1, 2]),
                   dict(min_p=[0.05] * 6), dict(top_k=[3000] * 6, min_p=[1e-4] * 6)):
        for u in (0.1, 0.6, 1 - 2.0 ** -24):
            check(qk, torch_gpu, x, [u] * 6, **params)


@pytest.mark.parametrize("low", [-1e4, -1e9, float(np.finfo(np.float32).min), -np.inf])
def test_masked_vocabularies(qk, torch_gpu, low):
    """All but a few tokens at a finite value or -inf, over whole segments of the
    row, next to a row without a mask."""
    rng = np.random.default_rng(12)
    n = 128256
    x = logits(rng, 5, n)
    keep = rng.choice(n, 200, replace=False)
    for r in (0, 2):
        masked = np.full(n, low, np.float32)
        masked[keep] = x[r, keep]
        x[r] = masked
    x[1, 16384: 5 * 16384] = low
    x[4, :] = low
    for params in (dict(), dict(top_k=[50] * 5, top_p=[0.9] * 5), dict(top_p=[0.95] * 5, temperature=[0.7] * 5), dict(min_p=[0.1] * 5)):
        for u in (0.0, 0.5, 1 - 2.0 ** -24):
            check(qk, torch_gpu, x, [u] * 5, **params)


@pytest.mark.parametrize("n,spread,t,p", [(151936, 2.2, 2.0, 0.9), (262144, 2.2, 1.5, 0.9), (128256, 1.5, 1.5, 0.9), (128256, 2.2, 3.0, 0.9)])
def test_more_tokens_at_the_cut_than_its_list(qk, torch_gpu, n, spread, t, p):
    """Ordinary logits at high temperatures: some thousands share the cut's bin."""
    rng = np.random.default_rng(13)
    x = (rng.standard_normal((3, n)) * spread).astype(np.float32)
    check(qk, torch_gpu, x, [0.3, 0.9, 0.999], temperature=[t] * 3, top_p=[p] * 3)
