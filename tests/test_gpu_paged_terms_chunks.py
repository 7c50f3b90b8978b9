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
