"""Serving steps over a paged cache as a server runs them: prompts of two
sequences in chunks, then single tokens of both, one layer: the projections'
GEMV, rotary tables, rotation and paged write, attention, the LM head's GEMV,
and sampled tokens -- against the same layer in 64 bits over the values that
the cache holds."""
import numpy as np
import pytest

import paged_ref
from conftest import rel_l2, to_dev
from test_gpu_sample import kept_weights

pytestmark = pytest.mark.gpu
HEADS, KVH, HD, VOCAB, DIM = 8, 2, 64, 1000, 512


@pytest.mark.parametrize("kind", ["f16", "i8", "e4m3"])
@pytest.mark.parametrize("half,scaling", [(False, None), (True, dict(type="llama3", factor=8.0, low_freq_factor=1.0,
                                                                     high_freq_factor=4.0, original_context=64.0))])
@pytest.mark.parametrize("scale", [0.0, 1e-4], ids=["sharp", "even"])
def test_prompts_then_tokens(qk, torch_gpu, workloads, oracle, kind, half, scaling, scale):
    """The projections' outputs are some hundreds, so at the usual scale one row
    takes nearly all of a token's weight; at 1e-4 many share it."""
    t = torch_gpu
    rng = np.random.default_rng(1)
    wqkv, _ = workloads.gemv_case(qk.Q4_K, DIM, (HEADS + 2 * KVH) * HD, seed=5)
    whead, _ = workloads.gemv_case(qk.Q6_K, HEADS * HD, VOCAB, seed=6)
    qkv = qk.Tensor((DIM, (HEADS + 2 * KVH) * HD), qk.Q4_K, to_dev(t, wqkv))
    head = qk.Tensor((HEADS * HD, VOCAB), qk.Q6_K, to_dev(t, whead))
    deq = lambda ty, w, c, r: oracle.dequant(ty, w, c, r).astype(np.float64).reshape(r, c)
    w64, h64 = deq(qk.Q4_K, wqkv, DIM, qkv.rows()), deq(qk.Q6_K, whead, HEADS * HD, VOCAB)
    kv = qk.PagedKV.empty(getattr(qk, paged_ref.NAMES[kind]), 20, KVH, 16, HD)
    table = np.full((2, 8), -1, dtype=np.int32)
    table[0], table[1] = [3, 17, 0, 9, 5, 12, 1, 8], [2, 19, 4, 11, 7, 6, 10, 13]
    table_d = to_dev(t, table)
    cos, sin = (t.empty(128, HD // 2, device="cuda") for _ in range(2))
    qk.rope_tables(500000.0, HD, cos, sin, scaling=scaling)
    c_host, s_host = cos.cpu().numpy(), sin.cpu().numpy()
    pos = [0, 0]
    seen = [[], []]     # (key values, value values) of each sequence's rows
    for counts in [(37, 20), (30, 1), (1, 45), (1, 1), (1, 1), (0, 1)]:
        n = sum(counts)
        x = rng.standard_normal((n, DIM)).astype(np.float32)
        seqs = np.array([[0, counts[0], pos[0], 0], [counts[0], counts[1], pos[1], 1]], dtype=np.int32)
        batch = qk.PagedBatch(table_d, to_dev(t, seqs), n, max(counts), max(p + c for p, c in zip(pos, counts)))
        proj = t.empty(n, qkv.rows(), device="cuda")
        nb = qk.batch_workspace_bytes(DIM, qkv.rows(), n)
        ws = t.empty(max(nb, 256), dtype=t.uint8, device="cuda")
        qk.batch_matvec(qkv, to_dev(t, x), proj, DIM, qkv.rows(), n, ws, nb)
        q, k, v = proj[:, : HEADS * HD], proj[:, HEADS * HD: (HEADS + KVH) * HD], proj[:, (HEADS + KVH) * HD:]
        q_in, k_in, v_in = (a.cpu().numpy() for a in (q, k, v))
        qk.rope_paged_write(kv, batch, q, q, k, v, cos, sin, HEADS, half=half)
        o = t.empty(n, HEADS * HD, device="cuda")
        ab = qk.paged_attention_workspace_bytes(batch, HEADS, KVH, HD)
        qk.paged_attention(kv, batch, q, o, HEADS, scale=scale, workspace=t.empty(max(ab, 16), dtype=t.uint8, device="cuda"))
        logits = t.empty(n, VOCAB, device="cuda")
        nb = qk.batch_workspace_bytes(HEADS * HD, VOCAB, n)
        ws = t.empty(max(nb, 256), dtype=t.uint8, device="cuda")
        qk.batch_matvec(head, o, logits, HEADS * HD, VOCAB, n, ws, nb)
        u = rng.random(n).astype(np.float32)
        token, prob = t.empty(n, dtype=t.int32, device="cuda"), t.empty(n, device="cuda")
        p_d = t.full((n,), 0.9, device="cuda")
        k_d = t.full((n,), 200, dtype=t.int32, device="cuda")
        qk.sample_rows(logits, to_dev(t, u), token, top_k=k_d, top_p=p_d, prob=prob,
                       workspace=t.empty(max(1, qk.sample_workspace_bytes(VOCAB, n)), dtype=t.uint8, device="cuda"))
        # The layer in 64 bits, the cache's rounding taken from the products
        # that were written (a code is a step function of them).
        assert rel_l2(np.concatenate([q_in, k_in, v_in], 1), x.astype(np.float64) @ w64.T) < 1e-6
        want, size = np.empty((n, HEADS, HD)), 0.0
        for s, (first, count, p0, _) in enumerate(seqs):
            at = np.arange(p0, p0 + count)
            rows = lambda a: a[first:first + count].reshape(count, a.shape[1] // HD, HD)
            kr = paged_ref.encode(paged_ref.rotate(rows(k_in), c_host[at], s_host[at], HD, half), kind)[2]
            vr = paged_ref.encode(rows(v_in), kind)[2]
            qr = paged_ref.rotate(rows(q_in), c_host[at], s_host[at], HD, half).astype(np.float64)
            seen[s] += list(zip(kr, vr))
            for i in range(count):
                ks, vs = (np.array([r[j] for r in seen[s][: p0 + i + 1]]) for j in (0, 1))
                for h in range(HEADS):
                    sc = ks[:, h // (HEADS // KVH)] @ qr[i, h] * (scale or HD ** -0.5)
                    size = max(size, np.linalg.norm(qr[i, h]) * np.linalg.norm(ks[:, h // (HEADS // KVH)], axis=1).max() *
                               (scale or HD ** -0.5))
                    e = np.exp(sc - sc.max())
                    want[first + i, h] = e @ vs[:, h // (HEADS // KVH)] / e.sum()
            pos[s] += count
        got = o.cpu().numpy()
        # A score is within 2 * 2^-23 of |q| |k| * scale (q's 22 bits, the
        # product's few fp32 roundings), and moves a probability by that.
        assert rel_l2(got, want.reshape(n, -1)) < max(3e-6, size * 2.0 ** -22)
        lg = logits.cpu().numpy()
        assert rel_l2(lg, got.astype(np.float64) @ h64.T) < 1e-6
        tok = token.cpu().numpy()
        for i in range(n):
            w = kept_weights(lg[i], 1.0, 200, np.float32(0.9))
            c = np.cumsum(w) / w.sum()
            assert w[tok[i]] > 0 and c[tok[i]] > u[i] - 1e-9 and c[tok[i]] - w[tok[i]] / w.sum() <= u[i] + 1e-9


def test_a_step_captured_and_replayed(qk, torch_gpu):
    """Rotate + write, attention and sampling in one graph whose positions move
    on between replays, against the eager calls on a second cache."""
    t = torch_gpu
    rng = np.random.default_rng(2)
    seqs0 = np.array([[0, 1, 0, 0], [1, 1, 40, 1], [2, 1, 100, 2]], dtype=np.int32)
    table = to_dev(t, np.arange(24, dtype=np.int32).reshape(3, 8)[:, ::-1])
    cos, sin = (t.empty(128, HD // 2, device="cuda") for _ in range(2))
    qk.rope_tables(10000.0, HD, cos, sin)
    sides = []
    x = t.empty(3, (HEADS + 2 * KVH) * HD, device="cuda")
    u, p = t.empty(3, device="cuda"), t.full((3,), 0.8, device="cuda")
    seqs = to_dev(t, seqs0)
    batch = qk.PagedBatch(table, seqs, 3, 1, 128)
    fill = to_dev(t, rng.standard_normal((2, 3, 100, KVH * HD)).astype(np.float32))
    for _ in range(2):
        kv = qk.PagedKV.empty(qk.I8, 24, KVH, 16, HD)
        pre = qk.PagedBatch(table, to_dev(t, np.array([[100 * i, 100, 0, i] for i in range(3)], dtype=np.int32)), 300, 100, 100)
        qk.rope_paged_write(kv, pre, None, None, fill[0].reshape(300, -1), fill[1].reshape(300, -1), None, None, HEADS, rot_dim=0)
        nb = qk.paged_attention_workspace_bytes(batch, HEADS, KVH, HD)
        sides.append(dict(kv=kv, q=t.empty(3, HEADS * HD, device="cuda"), o=t.empty(3, HEADS * HD, device="cuda"),
                          ws=t.empty(max(nb, 16), dtype=t.uint8, device="cuda"),
                          sw=t.empty(max(1, qk.sample_workspace_bytes(HEADS * HD, 3)), dtype=t.uint8, device="cuda"),
                          tok=t.empty(3, dtype=t.int32, device="cuda")))

    def step(d):
        q, k, v = x[:, : HEADS * HD], x[:, HEADS * HD: (HEADS + KVH) * HD], x[:, (HEADS + KVH) * HD:]
        qk.rope_paged_write(d["kv"], batch, q, d["q"], k, v, cos, sin, HEADS)
        qk.paged_attention(d["kv"], batch, d["q"], d["o"], HEADS, workspace=d["ws"])
        qk.sample_rows(d["o"], u, d["tok"], top_p=p, workspace=d["sw"])

    new = lambda: (x.copy_(to_dev(t, rng.standard_normal(x.shape).astype(np.float32))), u.uniform_())
    new()
    step(sides[1])   # not captured: also loads the kernels
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g):
        step(sides[0])
    for i in range(6):
        new()
        seqs.copy_(to_dev(t, seqs0 + np.array([0, 0, i, 0], dtype=np.int32)))
        g.replay()
        step(sides[1])
        t.cuda.synchronize()
        assert t.equal(sides[0]["o"], sides[1]["o"]) and t.equal(sides[0]["tok"], sides[1]["tok"])
        assert t.isfinite(sides[0]["o"]).all()
