"""qk_rope_tables_f32 against the formulas in 64 bits, angle by angle."""
import math

import numpy as np
import pytest

from conftest import to_dev

pytestmark = pytest.mark.gpu


def reference(theta, rot, positions, s=None, factors=None):
    """cos, sin [positions][rot / 2] in 64 bits, from the scaling's own words."""
    amp, freq = 1.0, []
    for i in range(rot // 2):
        f = theta ** (-2.0 * i / rot)
        if factors is not None:
            f /= float(factors[i])
        if s and s["type"] == "linear":
            f /= s["factor"]
        elif s and s["type"] == "llama3":
            wave = 2 * math.pi / f
            long, short = s["original_context"] / s["low_freq_factor"], s["original_context"] / s["high_freq_factor"]
            if wave > long:
                f /= s["factor"]
            elif wave >= short:
                m = (s["original_context"] / wave - s["low_freq_factor"]) / (s["high_freq_factor"] - s["low_freq_factor"])
                f = (1 - m) * f / s["factor"] + m * f
        elif s and s["type"] == "yarn":
            at = lambda b: rot * math.log(s["original_context"] / (b * 2 * math.pi)) / (2 * math.log(theta))
            lo, hi = max(math.floor(at(s["beta_fast"])), 0), min(math.ceil(at(s["beta_slow"])), rot - 1)
            m = min(max((i - lo) / max(hi - lo, 0.001), 0), 1)
            f = f / s["factor"] * m + f * (1 - m)
            amp = s.get("attention_factor") or 0.1 * math.log(s["factor"]) + 1
        freq.append(f)
    a = np.asarray(positions, dtype=np.float64)[:, None] * np.array(freq)
    return amp * np.cos(a), amp * np.sin(a)


def close(got, want, top, amp=1.0):
    """One rounding to fp32 (half a step of a value up to amp: amp * 2^-24),
    and angles whose products differ by 2^-52 of themselves, top at most, on
    either side, plus that of a frequency's own few operations (8 of them)."""
    tol = amp * (2.0 ** -24 + top * 10 * 2.0 ** -52)
    assert np.abs(got.astype(np.float64) - want).max() <= tol


@pytest.mark.parametrize("rot", [2, 6, 64, 80, 128, 510, 512])
@pytest.mark.parametrize("positions,first", [(1, 0), (3, 131071), (257, 1000), (20000, 0)])
def test_plain_tables(qk, torch_gpu, rot, positions, first):
    t = torch_gpu
    cos, sin = (t.full((positions + 1, rot // 2), 7.0, device="cuda") for _ in range(2))
    qk.rope_tables(500000.0, rot, cos[:positions], sin[:positions], first_pos=first)
    pos = sorted({0, positions // 3, positions // 2, positions - 1})
    want = reference(500000.0, rot, [first + p for p in pos])
    for got, w in zip((cos, sin), want):
        close(got[pos].cpu().numpy(), w, first + positions)
        assert (got[positions] == 7).all()   # the row behind is left as it was


SCALINGS = [dict(type="none"), dict(type="linear", factor=4.0),
            dict(type="llama3", factor=32.0, low_freq_factor=1.0, high_freq_factor=4.0, original_context=8192.0),
            dict(type="yarn", factor=16.0, original_context=4096.0, beta_fast=32.0, beta_slow=1.0),
            dict(type="yarn", factor=0.5, original_context=100.0, beta_fast=1.0, beta_slow=1.0, attention_factor=1.25)]


@pytest.mark.parametrize("s", SCALINGS, ids=lambda s: f"{s['type']}-{s.get('factor')}")
@pytest.mark.parametrize("factors", [False, True])
@pytest.mark.parametrize("rot,theta", [(64, 500000.0), (128, 10000.0), (20, 10000.0)])
def test_scaled_tables(qk, torch_gpu, s, factors, rot, theta):
    t = torch_gpu
    n = 9000
    ff = np.random.default_rng(3).uniform(0.5, 8, rot // 2).astype(np.float32) if factors else None
    cos, sin = (t.empty(n, rot // 2, device="cuda") for _ in range(2))
    qk.rope_tables(theta, rot, cos, sin, scaling=s, freq_factors=None if ff is None else to_dev(t, ff))
    pos = list(range(0, n, 7))
    want = reference(theta, rot, pos, s, ff)
    amp = np.abs(want[0]).max()
    for got, w in zip((cos, sin), want):
        close(got[pos].cpu().numpy(), w, 2.0 * n / min(1.0, s.get("factor", 1.0)), amp)


def test_tables_are_the_drivers_formula(qk, torch_gpu):
    """What rope_kv_write_batched rotates by: cos and sin of pos * theta^(-2 i / hd)."""
    t = torch_gpu
    heads, kvh, hd, pos = 8, 2, 64, 777
    cos, sin = (t.empty(1024, hd // 2, device="cuda") for _ in range(2))
    qk.rope_tables(500000.0, hd, cos, sin)
    rng = np.random.default_rng(1)
    q, k = (rng.standard_normal((1, w * hd)).astype(np.float32) for w in (heads, kvh))
    qd, kd = to_dev(t, q), to_dev(t, k)
    cache = t.zeros(2, 1024, kvh * hd, device="cuda")
    desc = to_dev(t, np.array([[pos, 0]], dtype=np.int64))
    qk.check(qk.lib().qk_rope_kv_write_batched(qd.data_ptr(), kd.data_ptr(), kd.data_ptr(), cos.data_ptr(),
                                               sin.data_ptr(), cache[0].data_ptr(), cache[1].data_ptr(), 0, 1024,
                                               desc.data_ptr(), 1, 1024, heads, kvh, hd, None), "rope")
    a = pos * 500000.0 ** (-np.arange(0, hd, 2) / hd)
    z = q.reshape(heads, -1, 2).astype(np.float64) @ [1, 1j] * np.exp(1j * a)
    want = np.stack([z.real, z.imag], -1).reshape(1, -1)
    # Two products and a sum in fp32, of table entries rounded once: 4 half
    # steps of values below 8.
    assert np.abs(qd.cpu().numpy() - want).max() <= 8 * 4 * 2.0 ** -24


def test_refusals(qk, torch_gpu):
    t = torch_gpu
    c = t.empty(10, 32, device="cuda")
    with pytest.raises(qk.QKError, match="unknown scaling"):
        qk.rope_tables(1e4, 64, c, c, scaling=dict(type="cubic"))
    with pytest.raises(qk.QKError, match="unknown scaling"):
        qk.rope_tables(1e4, 64, c, c, scaling=dict(type="linear", factr=2.0))
    with pytest.raises(qk.QKError, match="shape"):
        qk.rope_tables(1e4, 62, c, c)
    with pytest.raises(qk.QKError, match="float32"):
        qk.rope_tables(1e4, 64, c.double(), c)
    with pytest.raises(qk.QKError, match="contiguous"):
        qk.rope_tables(1e4, 64, t.empty(10, 64, device="cuda")[:, ::2], c)
