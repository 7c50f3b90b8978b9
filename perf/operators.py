"""Operators of a serving step over a paged, quantised KV cache, as a program
that serves a Llama model calls them:

  tables  cosine and sine tables of rotary positions whose frequencies are
          scaled for long contexts
  cache   new tokens' q and k rotated, k and v quantised into cache pages, and
          the written rows read back (a copy of a sequence's rows, say)
  attn    attention of each sequence's new tokens over its pages, single tokens
          (decoding) or chunks (prefill)
  sample  the next token of each row of logits: temperature, top-k, top-p and
          min-p, from given random numbers

With `own` false, run() computes them from elementary torch operations; with
`own` true, it calls the package.  exact() is each operator's definition in 64
bits, written without either.

Cache format (both sides): a pool of pages [pages][kv_heads][page_rows]
[head_dim]; a sequence's row r is row r % page_rows of page table[r //
page_rows].  "i8": int8 codes, one fp32 scale (largest magnitude / 127) a row
and KV head.  "e4m3": float8 codes, the scale the least power of two that keeps
the row within 448.  "f16": the values themselves.
"""
import importlib.util
import math
import pathlib
import sys

import torch

own = False

PACKAGE = "inferencer_jetson_amd"
DEV = "cuda:0"
#: Sampling weights are multiples of 2^-44 of the largest one.
UNIT = 2.0 ** 44
VOCAB = 128256


def _qk():
    if PACKAGE not in sys.modules:
        folder = pathlib.Path.cwd() / "inferencer-jetson_amd"
        spec = importlib.util.spec_from_file_location(PACKAGE, folder / "__init__.py",
                                                      submodule_search_locations=[str(folder)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[PACKAGE] = mod
        spec.loader.exec_module(mod)
    return sys.modules[PACKAGE]


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # The tables of the package's own workloads: context 1024, heads of 64.
        dict(name="tables_1024", kind="tables", positions=1024, rot=64, theta=500000.0, scaling="none", factor=1.0),
        # A context of 131072 by interpolated frequencies, heads of 128.
        dict(name="tables_131072_yarn", kind="tables", positions=131072, rot=128, theta=500000.0, scaling="yarn",
             factor=16.0),
        # 32 sequences decoding: one token of each into its pages, 1B heads.
        dict(name="cache_decode_32_i8", kind="cache", type="i8", heads=32, kv_heads=8, head_dim=64, page_rows=64,
             seqs=32, count_lo=1, count_hi=1, pos_lo=64, pos_hi=2048, rot=64, half=False),
        # Prompts of odd lengths in one batch, adjacent halves, a half-rotated
        # head, the smallest pages.
        dict(name="cache_ragged_f16", kind="cache", type="f16", heads=24, kv_heads=8, head_dim=128, page_rows=16,
             seqs=5, count_lo=37, count_hi=301, pos_lo=0, pos_hi=500, rot=64, half=True),
        # A long prompt's chunk into float8 pages.
        dict(name="cache_chunk_8192_e4m3", kind="cache", type="e4m3", heads=32, kv_heads=8, head_dim=128,
             page_rows=128, seqs=1, count_lo=8192, count_hi=8192, pos_lo=8192, pos_hi=8192, rot=128, half=True),
        # One sequence decoding at the position of the package's decode workload.
        dict(name="attn_1_700_f16", kind="attn", type="f16", heads=32, kv_heads=8, head_dim=64, page_rows=64, seqs=1,
             count_lo=1, count_hi=1, pos_lo=700, pos_hi=700),
        # 64 ragged sequences decoding over long contexts.
        dict(name="attn_decode_64_i8", kind="attn", type="i8", heads=32, kv_heads=8, head_dim=128, page_rows=64,
             seqs=64, count_lo=1, count_hi=1, pos_lo=1000, pos_hi=8000),
        # An odd chunk over 600 earlier rows, 3B heads.
        dict(name="attn_chunk_517_i8", kind="attn", type="i8", heads=24, kv_heads=8, head_dim=128, page_rows=32,
             seqs=1, count_lo=517, count_hi=517, pos_lo=600, pos_hi=600),
        # A long prompt's chunk over 8192 earlier rows.
        dict(name="attn_chunk_2048_e4m3", kind="attn", type="e4m3", heads=32, kv_heads=8, head_dim=128, page_rows=128,
             seqs=1, count_lo=2048, count_hi=2048, pos_lo=8192, pos_hi=8192),
        # One sequence's next token, the usual filters.
        dict(name="sample_1", kind="sample", rows=1, vocab=VOCAB, mode="top-k top-p"),
        # A decode batch whose requests each bring their own filters.
        dict(name="sample_64_mixed", kind="sample", rows=64, vocab=VOCAB, mode="mixed"),
        # A large batch by nucleus alone.
        dict(name="sample_512_top_p", kind="sample", rows=512, vocab=VOCAB, mode="top-p"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "cache", "cache", "attn", "attn", "attn", "sample", "sample"])
    if kind == "tables":
        return dict(kind=kind, positions=_log(rng, 256, 131072), rot=2 * rng.randint(16, 64),
                    theta=rng.choice([10000.0, 500000.0]), scaling=rng.choice(["none", "linear", "llama3", "yarn"]),
                    factor=rng.choice([2.0, 8.0, 16.0]))
    if kind == "sample":
        return dict(kind=kind, rows=_log(rng, 1, 256), vocab=_log(rng, 1000, VOCAB),
                    mode=rng.choice(["top-k top-p", "top-p", "min-p", "temperature", "mixed"]))
    heads, kv_heads, hd = rng.choice([(32, 8, 64), (24, 8, 128), (16, 2, 96), (8, 8, 128), (32, 8, 128), (8, 1, 256),
                                      (5, 5, 64)])
    c = dict(kind=kind, type=rng.choice(["f16", "i8", "e4m3"]), heads=heads, kv_heads=kv_heads, head_dim=hd,
             page_rows=rng.choice([16, 32, 64, 128]))
    form = rng.random()
    if form < 0.45:      # sequences that decode
        lo = _log(rng, 1, 4000)
        c |= dict(seqs=_log(rng, 1, 64), count_lo=1, count_hi=1, pos_lo=lo, pos_hi=lo + rng.randint(0, 3000))
    elif form < 0.8:     # one chunk
        n = _log(rng, 2, 2048)
        lo = rng.choice([0, _log(rng, 1, 6000)])
        c |= dict(seqs=1, count_lo=n, count_hi=n, pos_lo=lo, pos_hi=lo)
    else:                # chunks and single tokens in one batch
        lo = _log(rng, 1, 1000)
        c |= dict(seqs=rng.randint(2, 12), count_lo=1, count_hi=_log(rng, 2, 200), pos_lo=lo,
                  pos_hi=lo + rng.randint(0, 500))
    if kind == "cache":
        c |= dict(rot=rng.choice([hd, hd // 2]), half=rng.random() < 0.5)
    return c


# ----------------------------------------------------------------- inputs --

def _gen(seed, stream):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000 + stream)
    return g


def _normal(seed, stream, *shape):
    return torch.randn(*shape, generator=_gen(seed, stream), device=DEV)


def _seq_lists(case):
    """Counts and positions of a case's sequences: spread evenly over their ranges."""
    n = case["seqs"]
    at = [0.5 if n == 1 else i * 7 % n / (n - 1) for i in range(n)]
    mid = lambda lo, hi, x: int(round(lo + (hi - lo) * x))
    counts = [mid(case["count_lo"], case["count_hi"], x) for x in at]
    pos = [mid(case["pos_lo"], case["pos_hi"], at[-1 - i]) for i in range(n)]
    return counts, pos


def _scaling(case):
    """The parameters of a case's frequency scaling, as model files give them."""
    return dict(type=case["scaling"], factor=case["factor"], low_freq_factor=1.0, high_freq_factor=4.0,
                original_context=8192.0, beta_fast=32.0, beta_slow=1.0, attention_factor=0.0)


def _encode(t, kind):
    """Rows [..., head_dim] as a filled cache holds them: (codes, scales)."""
    if kind == "f16":
        return t.half(), None
    amax = t.abs().amax(-1)
    if kind == "i8":
        scale = amax / 127
        return torch.round(t.double() / scale.double()[..., None]).to(torch.int8), scale
    mant, e = torch.frexp(amax)
    scale = torch.ldexp(torch.ones_like(amax), e - 9 + (mant > 0.875).int())
    return (t / scale[..., None]).to(torch.float8_e4m3fn), scale


def _batch(case, seed, filled):
    """A pool, the page table of a case's sequences (pages in any order) and their descriptors."""
    counts, pos = _seq_lists(case)
    rows, kvh, hd = case["page_rows"], case["kv_heads"], case["head_dim"]
    need = [-(-(c + p) // rows) for c, p in zip(counts, pos)]
    pages = sum(need) + 3
    ids = torch.randperm(pages, generator=_gen(seed, 1), device=DEV)[: sum(need)].to(torch.int32)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device=DEV)
    seqs, at, first = [], 0, 0
    for s, (c, p, k) in enumerate(zip(counts, pos, need)):
        table[s, :k] = ids[at:at + k]
        seqs.append([first, c, p, s])
        at, first = at + k, first + c
    st = dict(case=case, table=table, seqs=torch.tensor(seqs, dtype=torch.int32, device=DEV), n=first,
              max_count=max(counts), max_rows=max(c + p for c, p in zip(counts, pos)))
    for i, name in enumerate(("key", "value")):
        if filled:
            codes, scale = _encode(_normal(seed, 4 + i, pages, kvh, rows, hd), case["type"])
        else:
            dt = {"f16": torch.float16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}[case["type"]]
            codes = torch.zeros(pages, kvh, rows, hd, device=DEV).to(dt)
            scale = None if case["type"] == "f16" else torch.zeros(pages, kvh, rows, device=DEV)
        st[name], st[name + "_scale"] = codes, scale
    return st


def prepare(case, seed):
    kind = case["kind"]
    if kind == "tables":
        # Some model files bring a divisor for each frequency beside the scaling.
        ff = 1 + torch.rand(case["rot"] // 2, generator=_gen(seed, 2), device=DEV)
        out = torch.empty(2, case["positions"], case["rot"] // 2, device=DEV)
        st = dict(case=case, factors=ff, cos=out[0], sin=out[1])
    elif kind == "sample":
        n, rows = case["vocab"], case["rows"]
        g = _gen(seed, 3)
        logits = torch.randn(rows, n, generator=g, device=DEV) * 2.2
        # A few dozen tokens stand out, as a trained model's do.
        at = torch.randint(0, n, (rows, 40), generator=g, device=DEV)
        logits.scatter_(1, at, 8 + 3 * torch.randn(rows, 40, generator=g, device=DEV))
        draws = torch.rand(rows, 5, generator=g, device=DEV)
        mode = case["mode"]
        which = torch.arange(rows, device=DEV) % 5   # of a mixed batch: each kind of request in turn
        has = lambda name, k: torch.tensor(name in mode, device=DEV) | ((which == k) if mode == "mixed" else False)
        temp = 0.6 + 0.6 * draws[:, 0]
        if mode == "mixed":
            temp = torch.where(which == 4, torch.zeros_like(temp), temp)   # greedy requests
        top_k = torch.where(has("top-k", 0), (10 + 90 * draws[:, 1]).int(), 0).int()
        top_p = torch.where(has("top-p", 0) | has("top-p", 1), 0.8 + 0.19 * draws[:, 2], 1.0)
        min_p = torch.where(has("min-p", 2), 0.02 + 0.1 * draws[:, 3], 0.0)
        st = dict(case=case, logits=logits, temperature=temp, top_k=top_k, top_p=top_p, min_p=min_p,
                  uniform=draws[:, 4].contiguous(), token=torch.empty(rows, dtype=torch.int32, device=DEV),
                  prob=torch.empty(rows, device=DEV))
        if own:
            qk = _qk()
            st["workspace"] = torch.empty(max(1, qk.sample_workspace_bytes(n, rows)), dtype=torch.uint8, device=DEV)
    else:
        st = _batch(case, seed, kind == "attn")
        n, heads, kvh, hd = st["n"], case["heads"], case["kv_heads"], case["head_dim"]
        gains = torch.exp(0.4 * _normal(seed, 6, heads * hd))   # channels differ, as trained ones do
        st["q"] = _normal(seed, 7, n, heads * hd) * gains
        st["out"] = torch.empty(n, heads * hd, device=DEV)
        if kind == "cache":
            st["k"] = _normal(seed, 8, n, kvh * hd) * gains[: kvh * hd]
            st["v"] = _normal(seed, 9, n, kvh * hd) * gains[: kvh * hd]
            f = 500000.0 ** (-torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float64) / case["rot"])
            angle = torch.arange(st["max_rows"], device=DEV, dtype=torch.float64)[:, None] * f
            st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
            st["k_back"], st["v_back"] = torch.empty(n, kvh * hd, device=DEV), torch.empty(n, kvh * hd, device=DEV)
        if own:
            qk = _qk()
            st["kv"] = qk.PagedKV({"f16": qk.F16, "i8": qk.I8, "e4m3": qk.F8_E4M3}[case["type"]], st["key"], st["value"],
                                  st["key_scale"], st["value_scale"])
            st["batch"] = qk.PagedBatch(st["table"], st["seqs"], n, st["max_count"], st["max_rows"])
            if kind == "attn":
                nb = qk.paged_attention_workspace_bytes(st["batch"], heads, kvh, hd)
                st["workspace"] = torch.empty(max(1, nb), dtype=torch.uint8, device=DEV)
    return st


# -------------------------------------------------------------- plain forms --

def _frequencies(case, factors):
    rot, theta, s = case["rot"], case["theta"], _scaling(case)
    f = theta ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot) / factors.double()
    amp = 1.0
    if s["type"] == "linear":
        f = f / s["factor"]
    elif s["type"] == "llama3":
        turns = s["original_context"] * f / (2 * math.pi)   # turns over the original context
        mix = ((turns - s["low_freq_factor"]) / (s["high_freq_factor"] - s["low_freq_factor"])).clamp(0, 1)
        f = f / s["factor"] * (1 - mix) + f * mix
    elif s["type"] == "yarn":
        at = lambda beta: rot * math.log(s["original_context"] / (beta * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(at(s["beta_fast"])), 0), min(math.ceil(at(s["beta_slow"])), rot - 1)
        ramp = ((torch.arange(rot // 2, device=DEV, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f / s["factor"] * ramp + f * (1 - ramp)
        amp = 0.1 * math.log(s["factor"]) + 1
    return f, amp


def _plain_tables(st):
    f, amp = _frequencies(st["case"], st["factors"])
    angle = torch.arange(st["case"]["positions"], device=DEV, dtype=torch.float64)[:, None] * f
    return (angle.cos() * amp).float(), (angle.sin() * amp).float()


def _tokens(st):
    """Of every token: its sequence and its position."""
    first, pos = st["seqs"][:, 0].contiguous(), st["seqs"][:, 2]
    t = torch.arange(st["n"], device=DEV, dtype=torch.int32)
    s = torch.searchsorted(first, t, right=True) - 1
    return s, (pos[s] + t - first[s]).long()


def _rotate(x, cos, sin, rot, half):
    """x [tokens, heads, head_dim] by [tokens, rot / 2] tables, in 64 bits, rounded once."""
    c, s = cos.double()[:, None], sin.double()[:, None]
    r = x[..., :rot].double()
    if half:
        a, b = r[..., : rot // 2], r[..., rot // 2:]
        r = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([r.float(), x[..., rot:]], -1)


def _plain_cache(st):
    case = st["case"]
    hd, n, rows = case["head_dim"], st["n"], case["page_rows"]
    s, pos = _tokens(st)
    cos, sin = st["cos"][pos], st["sin"][pos]
    q = _rotate(st["q"].view(n, -1, hd), cos, sin, case["rot"], case["half"])
    k = _rotate(st["k"].view(n, -1, hd), cos, sin, case["rot"], case["half"])
    page, slot = st["table"][s, pos // rows].long(), pos % rows
    back = []
    for name, x in (("key", k), ("value", st["v"].view(n, -1, hd))):
        codes, scale = _encode(x, case["type"])
        pool = st[name]
        if case["type"] == "e4m3":   # indexed as bytes
            pool, codes = pool.view(torch.uint8), codes.view(torch.uint8)
        pool[page, :, slot] = codes
        got = pool[page, :, slot]
        if case["type"] == "e4m3":
            got = got.view(torch.float8_e4m3fn)
        got = got.float()
        if scale is not None:
            st[name + "_scale"][page, :, slot] = scale
            got = got * st[name + "_scale"][page, :, slot][..., None]
        back.append(got.reshape(n, -1))
    return q.reshape(n, -1), back[0], back[1]


def _gather(st, name, rows, dtype):
    """Every sequence's rows 0 .. rows - 1, [seqs, kv_heads, rows, head_dim]."""
    case = st["case"]
    r = torch.arange(rows, device=DEV)
    page = st["table"][st["seqs"][:, 3].long()][:, r // case["page_rows"]].clamp(min=0).long()
    slot = (r % case["page_rows"]).expand_as(page)
    pool = st[name]
    x = pool.view(torch.uint8)[page, :, slot].view(pool.dtype) if case["type"] == "e4m3" else pool[page, :, slot]
    x = x.to(dtype)
    if case["type"] != "f16":
        x = x * st[name + "_scale"][page, :, slot].to(dtype)[..., None]
    return x.transpose(1, 2)


def _attention(st, dtype):
    case, n = st["case"], st["n"]
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    g, count, rows = heads // kvh, st["max_count"], st["max_rows"]
    first, pos = st["seqs"][:, 0].long(), st["seqs"][:, 2].long()
    i = torch.arange(count, device=DEV)
    tok = (first[:, None] + i).clamp(max=n - 1)
    q = st["q"].view(n, kvh, g, hd)[tok].to(dtype)                                  # [seqs, count, kvh, g, hd]
    q = q.permute(0, 2, 1, 3, 4).reshape(-1, kvh, count * g, hd)
    k = _gather(st, "key", rows, dtype)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(hd))
    del k
    seen = torch.arange(rows, device=DEV) <= (pos[:, None] + i)[..., None]          # [seqs, count, rows]
    s.view(-1, kvh, count, g, rows).masked_fill_(~seen[:, None, :, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s, _gather(st, "value", rows, dtype)) / total
    o = o.view(-1, kvh, count, g, hd).transpose(1, 2)                               # [seqs, count, kvh, g, hd]
    at, p = _tokens(st)
    return o[at, p - pos[at]].reshape(n, heads * hd)


def _plain_sample(st):
    x = st["logits"]
    n = x.shape[1]
    greedy = st["temperature"] <= 0
    t = torch.where(greedy, 1.0, st["temperature"]).double()[:, None]
    top = x.amax(-1, keepdim=True).double()
    w = torch.round(torch.exp((x.double() - top) / t) * UNIT).long()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(n, device=DEV)
    k = torch.where(st["top_k"] <= 0, n, st["top_k"])
    k = torch.where(greedy, 1, k)[:, None]
    ws = torch.where(rank < k, ws, 0)
    before = torch.cumsum(ws, -1) - ws
    total = ws.sum(-1, keepdim=True)
    p = st["top_p"].double()[:, None]
    keep = (rank < k) & ((p >= 1) | (before.double() < p * total.double()))
    keep = (keep & (ws.double() >= st["min_p"].double()[:, None] * UNIT)) | (rank == 0)
    w = torch.where(torch.zeros_like(keep).scatter_(1, order, keep), w, 0)
    upto = torch.cumsum(w, -1)
    total = upto[:, -1:]
    target = torch.minimum((st["uniform"].double()[:, None] * total.double()).long(), total - 1)
    token = (upto <= target).sum(-1)
    prob = w.gather(1, token[:, None]).double() / total.double()
    return token.int(), prob[:, 0].float()


# --------------------------------------------------------------------- run --

def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        qk = _qk()
        if kind == "tables":
            qk.rope_tables(case["theta"], case["rot"], st["cos"], st["sin"], scaling=_scaling(case),
                           freq_factors=st["factors"])
            return st["cos"], st["sin"]
        if kind == "cache":
            qk.rope_paged_write(st["kv"], st["batch"], st["q"], st["out"], st["k"], st["v"], st["cos"], st["sin"],
                                case["heads"], rot_dim=case["rot"], half=case["half"])
            qk.paged_read(st["kv"], st["batch"], st["k_back"], st["v_back"])
            return st["out"], st["k_back"], st["v_back"]
        if kind == "attn":
            qk.paged_attention(st["kv"], st["batch"], st["q"], st["out"], case["heads"], workspace=st["workspace"])
            return st["out"]
        qk.sample_rows(st["logits"], st["uniform"], st["token"], temperature=st["temperature"], top_k=st["top_k"],
                       top_p=st["top_p"], min_p=st["min_p"], prob=st["prob"], workspace=st["workspace"])
        return st["token"], st["prob"]
    if kind == "tables":
        return _plain_tables(st)
    if kind == "cache":
        return _plain_cache(st)
    if kind == "attn":
        return _attention(st, torch.float32)
    return _plain_sample(st)


# -------------------------------------------------------------------- work --

def work(case):
    kind = case["kind"]
    if kind == "tables":
        pairs = case["positions"] * case["rot"] // 2
        return dict(bytes=8 * pairs + 2 * case["rot"], flops=0)
    if kind == "sample":
        return dict(bytes=case["rows"] * (4 * case["vocab"] + 28), flops=0)
    counts, pos = _seq_lists(case)
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    tokens = sum(counts)
    row = kvh * (2 * hd if case["type"] == "f16" else hd + 4)   # one cache row of keys or of values
    if kind == "cache":
        tables = 4 * case["rot"] * sum(counts)
        return dict(bytes=tokens * (4 * hd * (2 * heads + 4 * kvh) + 4 * row) + tables, flops=0)
    seen = sum(c * p + c * (c + 1) // 2 for c, p in zip(counts, pos))
    rows = sum(c + p for c, p in zip(counts, pos))
    return dict(bytes=2 * rows * row + 8 * tokens * heads * hd, flops=4 * heads * hd * seen)


# ------------------------------------------------------------------- exact --

def _exact_values(st, name):
    """A whole pool's values in 64 bits."""
    x = st[name].double()
    return x if st[name + "_scale"] is None else x * st[name + "_scale"].double()[..., None]


def _exact_attn(st):
    """Sequence by sequence, head by head, in 64 bits."""
    case = st["case"]
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    key, value = _exact_values(st, "key"), _exact_values(st, "value")
    out = torch.zeros(st["n"], heads, hd, dtype=torch.float64, device=DEV)
    q = st["q"].double().view(st["n"], heads, hd)
    for first, count, pos, s in st["seqs"].tolist():
        total = pos + count
        pages = st["table"][s, : -(-total // case["page_rows"])].long()
        hidden = torch.arange(total, device=DEV)[None] > torch.arange(pos, total, device=DEV)[:, None]
        for h in range(kvh):
            k, v = (x[pages, h].reshape(-1, hd)[:total] for x in (key, value))
            for j in range(h * heads // kvh, (h + 1) * heads // kvh):
                p = torch.softmax((q[first:first + count, j] @ k.t() / hd ** 0.5).masked_fill(hidden, -math.inf), -1)
                out[first:first + count, j] = p @ v
    return out.view(st["n"], -1)


def _exact_code(x, kind):
    """The stored value of each entry of rows x [..., head_dim] (fp32 values held in 64 bits)."""
    if kind == "f16":
        return x.half().double()
    amax = x.abs().max(-1, keepdim=True).values
    if kind == "i8":
        scale = (amax / 127).float().double()
        return torch.round(x / scale) * scale
    scale = 2.0 ** torch.ceil(torch.log2(amax / 448))
    y = x / scale
    # Three bits below the leading one, down to steps of 2^-9.
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * scale


def _exact_cache(st):
    case = st["case"]
    hd, rot, n = case["head_dim"], case["rot"], st["n"]
    seqs = st["seqs"].tolist()
    pos = torch.cat([torch.arange(p, p + c, device=DEV) for _, c, p, _ in seqs])
    turn = torch.complex(st["cos"][pos].double(), st["sin"][pos].double())[:, None]
    res = []
    for name in ("q", "k", "v"):
        x = st[name].double().view(n, -1, hd).clone()
        if name != "v":
            re = x[..., : rot // 2] if case["half"] else x[..., 0:rot:2]
            im = x[..., rot // 2: rot] if case["half"] else x[..., 1:rot:2]
            z = torch.complex(re, im) * turn
            if case["half"]:
                x[..., : rot // 2], x[..., rot // 2: rot] = z.real.clone(), z.imag.clone()
            else:
                x[..., 0:rot:2], x[..., 1:rot:2] = z.real.clone(), z.imag.clone()
        # What is quantised is the rotated value in 32 bits.
        res.append(x if name == "q" else _exact_code(x.float().double(), case["type"]))
    return tuple(x.reshape(n, -1) for x in res)


def _exact_tables(st):
    case, s = st["case"], _scaling(st["case"])
    rot, theta = case["rot"], case["theta"]
    freq, amp = [], 1.0
    for i, ff in enumerate(st["factors"].tolist()):
        f = math.exp(-2.0 * i / rot * math.log(theta)) / ff
        if s["type"] == "linear":
            f /= s["factor"]
        elif s["type"] == "llama3":
            wave = 2 * math.pi / f
            if wave > s["original_context"] / s["low_freq_factor"]:
                f /= s["factor"]
            elif wave > s["original_context"] / s["high_freq_factor"]:
                m = (s["original_context"] / wave - s["low_freq_factor"]) / (s["high_freq_factor"] - s["low_freq_factor"])
                f = (1 - m) * f / s["factor"] + m * f
        elif s["type"] == "yarn":
            dim = lambda turns: rot * math.log(s["original_context"] / (turns * 2 * math.pi)) / (2 * math.log(theta))
            lo, hi = max(math.floor(dim(s["beta_fast"])), 0), min(math.ceil(dim(s["beta_slow"])), rot - 1)
            m = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = f / s["factor"] * m + f * (1 - m)
            amp = 0.1 * math.log(s["factor"]) + 1
        freq.append(f)
    z = torch.outer(torch.arange(case["positions"], dtype=torch.float64, device=DEV),
                    torch.tensor(freq, dtype=torch.float64, device=DEV))
    z = torch.polar(torch.full_like(z, amp), z)
    return z.real.contiguous(), z.imag.contiguous()


def _exact_sample(st):
    """Row by row in 64-bit floating point: filters by the sorted row, the pick in index order."""
    tokens, probs = [], []
    cols = [st[k].tolist() for k in ("temperature", "top_k", "top_p", "min_p", "uniform")]
    for x, t, k, p, mp, u in zip(st["logits"].double(), *cols):
        if t <= 0:
            tokens.append(int(x.argmax()))
            probs.append(1.0)
            continue
        w = torch.exp((x - x.max()) / t)
        sw, at = torch.sort(w, descending=True, stable=True)
        keep = torch.ones_like(sw, dtype=torch.bool)
        if k > 0:
            keep[k:] = False
        if p < 1:
            keep &= torch.cumsum(sw * keep, 0) - sw * keep < p * (sw * keep).sum()
        keep &= sw >= mp
        keep[0] = True
        z = torch.zeros_like(w)
        z[at[keep]] = sw[keep]
        c = torch.cumsum(z, 0)
        i = int(torch.searchsorted(c, u * c[-1], right=True))
        tokens.append(i)
        probs.append(float(z[i] / c[-1]))
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(probs, dtype=torch.float64)


def exact(case, seed):
    st = prepare(case, seed)
    return {"tables": _exact_tables, "cache": _exact_cache, "attn": _exact_attn, "sample": _exact_sample}[case["kind"]](st)
