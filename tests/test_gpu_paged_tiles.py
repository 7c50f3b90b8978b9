"""qk_paged_attention_f32 by the tiles of 32 rows that a wave goes over (each takes every
fourth), and by the workgroups of a call: one tile, two, more, none; as many workgroups
as CUs, and more."""
import numpy as np
import pytest

import paged_more_ref as ref
from conftest import rel_l2, to_dev

pytestmark = pytest.mark.gpu
TOL = 3e-6   # as in the tests of attention without terms
LAYOUTS = [(4, 4, 64), (6, 2, 96), (8, 2, 128), (16, 8, 256), (8, 1, 256)]
LENGTHS = {"one tile": [1, 31, 32, 33, 96, 97, 127, 128], "two tiles": [129, 160, 200, 255, 256], "more": [257, 300, 384, 385, 512, 641]}


def run(qk, t, pool, q, heads, workspace):
    kv, batch = pool.dev(qk, t)
    out = t.full((pool.n, heads * pool.hd), np.nan, device="cuda")
    nb = qk.paged_attention_workspace_bytes(batch, heads, pool.kvh, pool.hd) if workspace else 0
    ws = t.full((nb,), 0xFF, dtype=t.uint8, device="cuda") if nb else None
    qk.paged_attention(kv, batch, to_dev(t, q), out, heads, workspace=ws)
    t.cuda.synchronize()
    return out.cpu().numpy()


@pytest.mark.parametrize("kind", ["f16", "i8", "e4m3", "i4"])
@pytest.mark.parametrize("heads,kvh,hd", LAYOUTS)
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("count", [1, 9])
@pytest.mark.parametrize("workspace", [False, True])
def test_tiles_of_a_wave(qk, torch_gpu, kind, heads, kvh, hd, lengths, count, workspace):
    rng = np.random.default_rng(hd + count)
    pool = ref.Pool(rng, kind, kvh, hd, 16, [(count, max(n - count, 0)) for n in LENGTHS[lengths]])
    pool.poison(pool.unused())
    q = rng.standard_normal((pool.n, heads * hd)).astype(np.float32)
    assert rel_l2(run(qk, torch_gpu, pool, q, heads, workspace), pool.attention(q, heads)) < TOL


@pytest.mark.parametrize("kind", ["f16", "i8", "e4m3", "i4"])
@pytest.mark.parametrize("heads,kvh,seqs", [(16, 8, [(1, 20 + 9 * i) for i in range(32)]), (16, 8, [(1, 20 + 9 * i) for i in range(33)]),
                                            (8, 1, [(128, 30), (127, 0), (100, 200), (1, 60)]), (8, 1, [(129, 30), (127, 0), (100, 200), (1, 60)])],
                         ids=["256 of tokens", "264 of tokens", "256 of prompts", "260 of prompts"])
def test_workgroups_of_heads_of_256(qk, torch_gpu, kind, heads, kvh, seqs):
    """(A workgroup: 16 query rows of a KV head.)"""
    rng = np.random.default_rng(len(seqs))
    pool = ref.Pool(rng, kind, kvh, 256, 32, seqs)
    pool.poison(pool.unused())
    q = rng.standard_normal((pool.n, heads * 256)).astype(np.float32)
    assert rel_l2(run(qk, torch_gpu, pool, q, heads, False), pool.attention(q, heads)) < TOL
