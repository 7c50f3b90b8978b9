"""Further operators of a serving step over a paged cache, as a program that
serves a Llama-like model calls them:

  cache4  new tokens' q and k rotated, k and v into pages of 4-bit codes, and
          the written rows read back
  attn    attention of each sequence's new tokens over its pages: over 4-bit
          codes, and over any cache with scores capped by a tanh, biased by
          distance, or masked by a sliding window or a prefix that is seen from
          before it too
  pages   a pool's pages given out and taken back as sequences grow, shrink and
          end, forked for several continuations of one prompt, and compacted

With `own` false, run() computes them from elementary torch operations; with
`own` true, it calls the package.  exact() is each operator's definition in 64
bits, written without either.

Cache format (both sides): a pool of pages [pages][kv_heads][page_rows]
[head_dim]; a sequence's row r is row r % page_rows of page table[r //
page_rows].  "i4": 4-bit codes of two's complement, two a byte, the earlier
value in the low half; eight bytes a row and KV head beside them, an fp32 scale
and a multiplier (one byte) for each quarter of the row; a value is code *
multiplier * scale.  The scale is the least number of 13 significant bits with
1785 scale >= the row's largest magnitude, a multiplier the least positive
integer with 7 multiplier scale >= its quarter's, a code value / (multiplier *
scale) to the nearest, ties to even.  "i8": int8 codes, one fp32 scale (largest
magnitude / 127) a row and KV head.  "e4m3": float8 codes, the scale the least
power of two that keeps the row within 448.  "f16": the values themselves.

A pool: page_table [table_rows][stride] names the page of each stretch of a
sequence (-1: none), refs [pages] counts the entries that name a page.
"""
import importlib.util
import math
import pathlib
import sys

import torch

own = False

PACKAGE = "inferencer_jetson_amd"
DEV = "cuda:0"


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

def _attn(name, type, heads, kv_heads, head_dim, page_rows, seqs, count, pos, cap=0.0, window=0, alibi=False, prefix=0):
    return dict(name=name, kind="attn", type=type, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                page_rows=page_rows, seqs=seqs, count_lo=count[0], count_hi=count[1], pos_lo=pos[0], pos_hi=pos[1],
                cap=cap, window=window, alibi=alibi, prefix=prefix)


def listed():
    return [
        # 32 sequences decoding: one token of each into its pages, 1B heads.
        dict(name="cache4_decode_32", kind="cache4", heads=32, kv_heads=8, head_dim=64, page_rows=64, seqs=32,
             count_lo=1, count_hi=1, pos_lo=64, pos_hi=2048, rot=64, half=False),
        # A long prompt's chunk into 4-bit pages.
        dict(name="cache4_chunk_8192", kind="cache4", heads=32, kv_heads=8, head_dim=128, page_rows=128, seqs=1,
             count_lo=8192, count_hi=8192, pos_lo=8192, pos_hi=8192, rot=128, half=True),
        # One sequence decoding at the position of the package's decode workload.
        _attn("attn4_1_700", "i4", 32, 8, 64, 64, 1, (1, 1), (700, 700)),
        # 64 ragged sequences decoding over long contexts: what a 4-bit cache is for.
        _attn("attn4_decode_64", "i4", 32, 8, 128, 64, 64, (1, 1), (1000, 8000)),
        # A long prompt's chunk over 8192 earlier 4-bit rows.
        _attn("attn4_chunk_2048", "i4", 32, 8, 128, 128, 1, (2048, 2048), (8192, 8192)),
        # One sequence of a model that biases by distance, no shared KV heads.
        _attn("attn_alibi_1_1500", "f16", 16, 16, 64, 32, 1, (1, 1), (1500, 1500), alibi=True),
        # Sequences decoding far into a context of which a layer sees 4096 rows.
        _attn("attn_window_decode_32", "i8", 32, 8, 128, 64, 32, (1, 1), (8000, 24000), window=4096),
        # A prompt's chunk through a layer with capped scores and a window, wide heads.
        _attn("attn_cap_window_chunk_1024", "f16", 16, 8, 256, 64, 1, (1024, 1024), (6000, 6000), cap=50.0, window=4096),
        # Prompts whose first 256 rows (an image, an instruction) see each other.
        _attn("attn_prefix_4", "e4m3", 8, 1, 256, 16, 4, (270, 400), (0, 0), prefix=256),
        # A decode batch's bookkeeping: 256 sequences, of which some end, some
        # drop what left their window, the others grow by a token.
        dict(name="pages_resize_256", kind="pages", op="resize", type="i8", layers=1, kv_heads=1, head_dim=64,
             page_rows=16, rows=256, stride=512, len_lo=100, len_hi=6000, pages=65536),
        # Sixteen prompts, three more continuations of each.
        dict(name="pages_fork_16", kind="pages", op="fork", type="i4", layers=12, kv_heads=8, head_dim=64,
             page_rows=64, rows=64, stride=64, len_lo=300, len_hi=3000, pages=1600),
        # Half the sequences have ended: the others' pages move to the pool's front.
        dict(name="pages_compact_128", kind="pages", op="compact", type="f16", layers=8, kv_heads=8, head_dim=128,
             page_rows=64, rows=128, stride=128, len_lo=500, len_hi=4000, pages=5000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache4", "cache4", "attn4", "attn4", "terms", "terms", "terms", "pages", "pages"])
    if kind == "pages":
        op = rng.choice(["resize", "fork", "compact"])
        rows, page_rows = _log(rng, 4, 256), rng.choice([16, 32, 64, 128])
        hi = _log(rng, 2 * page_rows, 60 * page_rows)
        stride = hi // page_rows + rng.randint(2, 9)
        layers = 1 if op == "resize" else rng.randint(1, 12)
        pages = rows * stride + rng.randint(0, 1000)
        # A pool of 4 GB at most.
        kvh, hd = rng.choice([(8, 64), (8, 128), (2, 96), (1, 256)]) if op != "resize" else (1, 64)
        room = int(4e9 / (4 * layers * kvh * hd * page_rows))
        return dict(kind=kind, op=op, type=rng.choice(["f16", "i8", "i4"]), layers=layers, kv_heads=kvh, head_dim=hd,
                    page_rows=page_rows, rows=rows, stride=stride, len_lo=max(1, hi // rng.randint(2, 30)), len_hi=hi,
                    pages=max(min(pages, room), 64))
    heads, kv_heads, hd = rng.choice([(32, 8, 64), (20, 4, 128), (16, 2, 96), (8, 8, 128), (32, 8, 128), (8, 1, 256),
                                      (16, 8, 256), (5, 5, 64)])
    c = dict(kind="cache4" if kind == "cache4" else "attn", heads=heads, kv_heads=kv_heads, head_dim=hd,
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
    if kind == "cache4":
        return c | dict(rot=rng.choice([hd, hd // 2]), half=rng.random() < 0.5)
    c |= dict(type="i4", cap=0.0, window=0, alibi=False, prefix=0)
    if kind == "terms":
        c |= dict(type=rng.choice(["f16", "i8", "e4m3", "i4"]))
        terms = rng.sample(["cap", "window", "alibi", "prefix"], rng.choice([1, 1, 2]))
        if "cap" in terms:
            c["cap"] = rng.choice([20.0, 30.0, 50.0])
        if "window" in terms:
            c["window"] = _log(rng, 16, 4096)
        if "alibi" in terms:
            c["alibi"] = True
        if "prefix" in terms:
            c["prefix"] = _log(rng, 8, 1000)
    return c


# ----------------------------------------------------------------- inputs --

def _gen(seed, stream):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000 + stream)
    return g


def _normal(seed, stream, *shape):
    return torch.randn(*shape, generator=_gen(seed, stream), device=DEV)


def _spread(lo, hi, n):
    """n whole numbers spread over lo .. hi, in no order of size."""
    at = [0.5 if n == 1 else i * 7 % n / (n - 1) for i in range(n)]
    return [int(round(lo + (hi - lo) * x)) for x in at]


def _seq_lists(case):
    """Counts and positions of a case's sequences."""
    n = case["seqs"]
    return _spread(case["count_lo"], case["count_hi"], n), _spread(case["pos_lo"], case["pos_hi"], n)[::-1]


def _round_up_13(t):
    """The least numbers of 13 significant bits that are no smaller than t (64 bits)."""
    mant, e = torch.frexp(t)
    return torch.ldexp(torch.ceil(mant * 8192), e - 13)


def _encode(t, kind):
    """Rows [..., head_dim] as a filled cache holds them: (codes, scales)."""
    if kind == "f16":
        return t.half(), None
    amax = t.abs().amax(-1)
    if kind == "i8":
        scale = amax / 127
        return torch.round(t.double() / scale.double()[..., None]).to(torch.int8), scale
    if kind == "i4":
        x = t.double().view(*t.shape[:-1], 4, -1)
        scale = _round_up_13(amax.double() / 1785)[..., None]
        mult = torch.ceil(x.abs().amax(-1) / (7 * scale)).clamp(min=1)
        code = (torch.round(x / (mult * scale)[..., None]).view(t.shape).int() & 15).to(torch.uint8)
        return (code[..., 0::2] | code[..., 1::2] << 4,
                torch.cat([scale.float().view(torch.uint8), mult.to(torch.uint8)], -1))
    mant, e = torch.frexp(amax)
    scale = torch.ldexp(torch.ones_like(amax), e - 9 + (mant > 0.875).int())
    return (t / scale[..., None]).to(torch.float8_e4m3fn), scale


def _empty(case, pages):
    """A layer's empty pool: codes and scales."""
    shape = (pages, case["kv_heads"], case["page_rows"])
    hd, kind = case["head_dim"], case["type"]
    if kind == "i4":
        return (torch.zeros(*shape, hd // 2, dtype=torch.uint8, device=DEV),
                torch.zeros(*shape, 8, dtype=torch.uint8, device=DEV))
    dt = {"f16": torch.float16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}[kind]
    return (torch.zeros(*shape, hd, device=DEV, dtype=torch.float32).to(dt),
            None if kind == "f16" else torch.zeros(*shape, device=DEV))


def _handle(case, st, layer=""):
    """The package's handle of a layer's pool, as a program makes it once."""
    qk = _qk()
    kind = {"f16": qk.F16, "i8": qk.I8, "e4m3": qk.F8_E4M3}.get(case["type"]) if case["type"] != "i4" else qk.I4
    return qk.PagedKV(kind, *(st[n + layer] for n in ("key", "value", "key_scale", "value_scale")))


def prepare(case, seed):
    if case["kind"] == "pages":
        return _prepare_pages(case, seed)
    counts, pos = _seq_lists(case)
    rows, kvh, hd, heads = case["page_rows"], case["kv_heads"], case["head_dim"], case["heads"]
    case = dict(case, type=case.get("type", "i4"))
    need = [-(-(c + p) // rows) for c, p in zip(counts, pos)]
    pages = sum(need) + 3
    ids = torch.randperm(pages, generator=_gen(seed, 1), device=DEV)[: sum(need)].to(torch.int32)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device=DEV)
    seqs, at, first = [], 0, 0
    for s, (c, p, k) in enumerate(zip(counts, pos, need)):
        table[s, :k] = ids[at:at + k]
        seqs.append([first, c, p, s])
        at, first = at + k, first + c
    n = first
    st = dict(case=case, table=table, seqs=torch.tensor(seqs, dtype=torch.int32, device=DEV), n=n,
              max_count=max(counts), max_rows=max(c + p for c, p in zip(counts, pos)))
    for i, name in enumerate(("key", "value")):
        if case["kind"] == "attn":
            st[name], st[name + "_scale"] = _encode(_normal(seed, 4 + i, pages, kvh, rows, hd), case["type"])
        else:
            st[name], st[name + "_scale"] = _empty(case, pages)
    gains = torch.exp(0.4 * _normal(seed, 6, heads * hd))   # channels differ, as trained ones do
    st["q"] = _normal(seed, 7, n, heads * hd) * gains
    st["out"] = torch.empty(n, heads * hd, device=DEV)
    if case["kind"] == "cache4":
        st["k"] = _normal(seed, 8, n, kvh * hd) * gains[: kvh * hd]
        st["v"] = _normal(seed, 9, n, kvh * hd) * gains[: kvh * hd]
        f = 500000.0 ** (-torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float64) / case["rot"])
        angle = torch.arange(st["max_rows"], device=DEV, dtype=torch.float64)[:, None] * f
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        st["k_back"], st["v_back"] = torch.empty(n, kvh * hd, device=DEV), torch.empty(n, kvh * hd, device=DEV)
    else:
        # Slopes that fall by octaves over the heads; a prefix for each sequence, odd ones among them.
        h = torch.arange(1, heads + 1, device=DEV, dtype=torch.float32)
        st["slopes"] = torch.exp2(-8 * h / heads) if case["alibi"] else None
        st["prefix"] = None
        if case["prefix"]:
            st["prefix"] = (case["prefix"] - torch.arange(len(need), device=DEV) % 3).clamp(min=0).to(torch.int32)
    if own:
        qk = _qk()
        st["kv"] = _handle(case, st)
        st["batch"] = qk.PagedBatch(table, st["seqs"], n, st["max_count"], st["max_rows"])
        if case["kind"] == "attn":
            nb = qk.paged_attention_workspace_bytes(st["batch"], heads, kvh, hd, window=case["window"])
            st["workspace"] = torch.empty(max(1, nb), dtype=torch.uint8, device=DEV)
    return st


def _prepare_pages(case, seed):
    rows, pages, op = case["rows"], case["pages"], case["op"]
    st = dict(case=case, table=torch.full((rows, case["stride"]), -1, dtype=torch.int32, device=DEV),
              refs=torch.zeros(pages, dtype=torch.int32, device=DEV))
    i32 = lambda t: t.to(torch.int32).contiguous()
    r = torch.arange(rows, device=DEV)
    lens = torch.randint(case["len_lo"], case["len_hi"] + 1, (rows,), generator=_gen(seed, 1), device=DEV)
    st["none"] = i32(torch.zeros_like(r))
    st["missing"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    st["moved"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    if op == "resize":
        # Of seven sequences one ends and one stays as it is; of five one drops all but its last 400 rows.
        st["come"] = i32(lens)
        st["go"] = i32(torch.where(r % 7 == 3, 0, torch.where(r % 7 == 5, -1, lens + 1)))
        st["begins"] = i32(torch.where(r % 5 == 2, (lens - 400).clamp(min=0), 0))
    elif op == "fork":
        prompts = max(1, rows // 4)   # the first rows; each later one continues one of them
        st["come"] = i32(torch.where(r < prompts, lens, 0))
        st["parents"] = i32(torch.where(r < prompts, -1, r % prompts))
        st["lengths"] = i32(lens[r % prompts])
    else:
        st["come"] = i32(lens)
        st["go"] = i32(torch.where(r % 2 == 0, 0, lens))
    if op != "resize":
        for i in range(case["layers"]):
            for j, name in enumerate(("key", "value")):
                codes, scale = _empty(case, pages)
                g = _gen(seed, 10 + 2 * i + j)
                if case["type"] == "f16":
                    codes = torch.randn(codes.shape, generator=g, device=DEV, dtype=torch.float16)
                else:
                    codes.view(torch.uint8).random_(0, 256, generator=g)
                    scale.view(torch.uint8).random_(0, 256, generator=g)
                st[f"{name}{i}"], st[f"{name}_scale{i}"] = codes, scale
    if own:
        qk = _qk()
        layers = [] if op == "resize" else [_handle(case, st, str(i)) for i in range(case["layers"])]
        st["pool"] = qk.PagePool(st["table"], st["refs"], case["page_rows"], layers)
        st["workspace"] = torch.empty(qk.pages_workspace_bytes(st["pool"]), dtype=torch.uint8, device=DEV)
    return st


# -------------------------------------------------------------- plain forms --

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


def _decode4(codes, scale, dtype):
    """The values of 4-bit rows [..., head_dim / 2] and their [..., 8] bytes of scale and multipliers."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    c = c.to(dtype) - 16 * (c > 7).to(dtype)
    unit = scale[..., :4].contiguous().view(torch.float32).to(dtype) * scale[..., 4:].to(dtype)
    return (c.view(*c.shape[:-1], 4, -1) * unit[..., None]).view(c.shape)


def _plain_cache4(st):
    case = st["case"]
    hd, n, rows = case["head_dim"], st["n"], case["page_rows"]
    s, pos = _tokens(st)
    cos, sin = st["cos"][pos], st["sin"][pos]
    q = _rotate(st["q"].view(n, -1, hd), cos, sin, case["rot"], case["half"])
    k = _rotate(st["k"].view(n, -1, hd), cos, sin, case["rot"], case["half"])
    page, slot = st["table"][s, pos // rows].long(), pos % rows

    def through(name, x):
        pool, scales = st[name], st[name + "_scale"]
        pool[page, :, slot], scales[page, :, slot] = _encode(x, "i4")
        return _decode4(pool[page, :, slot], scales[page, :, slot], torch.float32).reshape(n, -1)

    return q.reshape(n, -1), through("key", k), through("value", st["v"].view(n, -1, hd))


def _gather(st, name, rows, dtype):
    """Every sequence's rows 0 .. rows - 1, [seqs, kv_heads, rows, head_dim]."""
    case = st["case"]
    r = torch.arange(rows, device=DEV)
    page = st["table"][st["seqs"][:, 3].long()][:, r // case["page_rows"]].clamp(min=0).long()
    slot = (r % case["page_rows"]).expand_as(page)
    pool, scale = st[name], st[name + "_scale"]
    if case["type"] == "i4":
        return _decode4(pool[page, :, slot], scale[page, :, slot], dtype).transpose(1, 2)
    x = pool.view(torch.uint8)[page, :, slot].view(pool.dtype) if case["type"] == "e4m3" else pool[page, :, slot]
    x = x.to(dtype)
    if case["type"] != "f16":
        x = x * scale[page, :, slot].to(dtype)[..., None]
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
    if case["cap"]:
        s.div_(case["cap"]).tanh_().mul_(case["cap"])
    s = s.view(-1, kvh, count, g, rows)
    r = torch.arange(rows, device=DEV)
    ahead = r - (pos[:, None] + i)[..., None]                                       # [seqs, count, rows]
    if case["alibi"]:
        s.sub_(st["slopes"].to(dtype).view(1, kvh, 1, g, 1) * ahead.abs().to(dtype)[:, None, :, None])
    seen = ahead <= 0
    if case["prefix"]:
        seen = seen | ((r < st["prefix"][:, None]) & (r < (pos + st["seqs"][:, 1])[:, None]))[:, None]
    if case["window"]:
        seen = seen & (-ahead < case["window"])
    s.masked_fill_(~seen[:, None, :, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    s = s.view(-1, kvh, count * g, rows)
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s, _gather(st, "value", rows, dtype)) / total
    o = o.view(-1, kvh, count, g, hd).transpose(1, 2)                               # [seqs, count, kvh, g, hd]
    at, p = _tokens(st)
    return o[at, p - pos[at]].reshape(n, heads * hd)


def _free_by_rank(refs, count):
    """The free page of each rank 0 .. count - 1, lowest page first (-1: there are fewer)."""
    free = refs == 0
    rank = torch.where(free, torch.cumsum(free, 0) - 1, count).clamp(max=count)
    out = torch.full((count + 1,), -1, dtype=torch.int32, device=DEV)
    out[rank] = torch.arange(refs.numel(), dtype=torch.int32, device=DEV)
    out[count] = -1
    return out


def _count_pages(table, which, pages):
    """How many entries of `which` name each page."""
    c = torch.zeros(pages + 1, dtype=torch.int32, device=DEV)
    at = torch.where(which, table, pages).long()
    return c.scatter_add_(0, at.view(-1), torch.ones(at.numel(), dtype=torch.int32, device=DEV))[:pages]


def _plain_resize(st, lengths, begins):
    table, refs, rows = st["table"], st["refs"], st["case"]["page_rows"]
    e = torch.arange(table.shape[1], device=DEV)
    have = (table >= 0) & (table < refs.numel())
    change = (lengths >= 0)[:, None]
    want = e < ((lengths + rows - 1) // rows)[:, None]
    if begins is not None:
        want = want & (e >= (begins // rows)[:, None])
    drop = have & ~want & change
    refs -= _count_pages(table, drop, refs.numel())
    need = want & ~have & change
    rank = (torch.cumsum(need.view(-1), 0) - 1).view_as(table)
    given = _free_by_rank(refs, table.numel())[rank.clamp(min=0)]
    table.copy_(torch.where(drop, -1, torch.where(need, given, table)))
    refs += _count_pages(table, need & (given >= 0), refs.numel())
    st["missing"].copy_((need & (given < 0)).sum())


def _copy_pages(st, src, dst):
    """Contents of pages src to pages dst in every layer, where dst is a page."""
    ok = dst >= 0
    src, dst = src[ok].long(), dst[ok].long()
    for name in [f"{n}{i}" for i in range(st["case"]["layers"]) for n in ("key", "value", "key_scale", "value_scale")]:
        if st[name] is not None:
            st[name][dst] = st[name][src]


def _plain_fork(st):
    table, refs, rows = st["table"], st["refs"], st["case"]["page_rows"]
    parents, lengths, pages = st["parents"], st["lengths"], refs.numel()
    e = torch.arange(table.shape[1], device=DEV)
    child = (parents >= 0) & (parents != torch.arange(parents.numel(), device=DEV))
    was = table[parents.clamp(min=0).long()]
    full, part = lengths // rows, lengths % rows != 0
    shared = torch.where((e < full[:, None]) & (was >= 0), was, -1)
    source = was.gather(1, full.clamp(max=table.shape[1] - 1)[:, None].long())[:, 0]
    fresh = child & part & (source >= 0)
    rank = torch.cumsum(fresh, 0) - 1
    given = torch.where(fresh, _free_by_rank(refs, table.shape[0])[rank.clamp(min=0)], -1)
    shared = torch.where((e == full[:, None]) & fresh[:, None], given[:, None], shared)
    refs -= _count_pages(table, (table >= 0) & child[:, None], pages)
    table.copy_(torch.where(child[:, None], shared, table))
    refs += _count_pages(table, (table >= 0) & child[:, None], pages)
    st["missing"].copy_((fresh & (given < 0)).sum())
    _copy_pages(st, source, given)


def _plain_compact(st):
    table, refs = st["table"], st["refs"]
    pages = refs.numel()
    live = refs > 0
    total = live.sum()
    p = torch.arange(pages, device=DEV, dtype=torch.int32)
    moves = live & (p >= total)
    rank = torch.cumsum(moves, 0) - 1
    to = torch.where(moves, _free_by_rank(refs, pages)[rank.clamp(min=0)], p)
    ok = (table >= 0) & (table < pages)
    table.copy_(torch.where(ok, to[table.clamp(0, pages - 1).long()], table))
    counts = _count_pages(to, live, pages)   # which pages are live now
    new = torch.zeros_like(refs).scatter_add_(0, to.long(), torch.where(live, refs, 0))
    refs.copy_(torch.where(counts > 0, new, 0))
    st["moved"].copy_(moves.sum())
    _copy_pages(st, p, torch.where(moves, to, -1))


def _plain_pages(st):
    op = st["case"]["op"]
    _plain_resize(st, st["none"], None)
    _plain_resize(st, st["come"], None)
    if op == "resize":
        _plain_resize(st, st["go"], st["begins"])
    elif op == "fork":
        _plain_fork(st)
    else:
        _plain_resize(st, st["go"], None)
        _plain_compact(st)


# --------------------------------------------------------------------- run --

def _own_pages(qk, st):
    """All sequences leave and others come; then what the case stands for."""
    pool, ws, op = st["pool"], st["workspace"], st["case"]["op"]
    qk.pages_resize(pool, st["none"], missing=st["missing"], workspace=ws)
    qk.pages_resize(pool, st["come"], missing=st["missing"], workspace=ws)
    if op == "resize":
        qk.pages_resize(pool, st["go"], begins=st["begins"], missing=st["missing"], workspace=ws)
    elif op == "fork":
        qk.pages_fork(pool, st["parents"], st["lengths"], missing=st["missing"], workspace=ws)
    else:
        qk.pages_resize(pool, st["go"], missing=st["missing"], workspace=ws)
        qk.pages_compact(pool, moved=st["moved"], workspace=ws)


def run(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "pages":
        if own:
            _own_pages(_qk(), st)
        else:
            _plain_pages(st)
        # The pool as whole numbers: what its pages hold is moved, not computed.
        names = [f"{n}{i}" for i in range(case["layers"]) for n in ("key", "value", "key_scale", "value_scale")]
        held = [st[n] for n in names if st.get(n) is not None]
        return (st["table"], st["refs"], st["missing"], st["moved"],
                [t.view(torch.int16 if t.dtype == torch.float16 else torch.uint8) for t in held])
    if own:
        qk = _qk()
        if kind == "cache4":
            qk.rope_paged_write(st["kv"], st["batch"], st["q"], st["out"], st["k"], st["v"], st["cos"], st["sin"],
                                case["heads"], rot_dim=case["rot"], half=case["half"])
            qk.paged_read(st["kv"], st["batch"], st["k_back"], st["v_back"])
            return st["out"], st["k_back"], st["v_back"]
        qk.paged_attention(st["kv"], st["batch"], st["q"], st["out"], case["heads"], workspace=st["workspace"],
                           cap=case["cap"], window=case["window"], slopes=st["slopes"], prefix=st["prefix"])
        return st["out"]
    if kind == "cache4":
        return _plain_cache4(st)
    return _attention(st, torch.float32)


# -------------------------------------------------------------------- work --

def _row_bytes(case):
    """One cache row of keys or of values, of all KV heads."""
    hd = case["head_dim"]
    return case["kv_heads"] * {"f16": 2 * hd, "i8": hd + 4, "e4m3": hd + 4, "i4": hd // 2 + 8}[case.get("type", "i4")]


def work(case):
    if case["kind"] == "pages":
        # The table and the counts read and written, and each moved page.
        entries, rows = 8 * (case["rows"] * case["stride"] + case["pages"]), case["rows"]
        mean = (case["len_lo"] + case["len_hi"]) / 2 / case["page_rows"]
        moved = {"resize": 0, "fork": rows - rows // 4, "compact": rows * mean / 4}[case["op"]]
        page = 2 * case["layers"] * case["page_rows"] * _row_bytes(case)
        return dict(bytes=int(entries + 2 * moved * page), flops=0)
    counts, pos = _seq_lists(case)
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    tokens, row = sum(counts), _row_bytes(case)
    if case["kind"] == "cache4":
        tables = 4 * case["rot"] * tokens
        return dict(bytes=tokens * (4 * hd * (2 * heads + 4 * kvh) + 4 * row) + tables, flops=0)
    window = case["window"] or 1 << 40
    pairs = rows = 0
    for s, (c, p) in enumerate(zip(counts, pos)):
        pre = min(max(case["prefix"] - s % 3, 0), c + p) if case["prefix"] else 0
        pairs += sum(max(t + 1, pre) - max(0, t + 1 - window) for t in range(p, p + c))
        rows += c + p - max(0, p + 1 - window)
    return dict(bytes=2 * rows * row + 8 * tokens * heads * hd, flops=4 * heads * hd * pairs)


# ------------------------------------------------------------------- exact --

def exact(case, seed):
    if case["kind"] == "pages":   # whole numbers, all of it
        return None
    st = prepare(case, seed)
    case = st["case"]
    heads, kvh, hd, n = case["heads"], case["kv_heads"], case["head_dim"], st["n"]

    def values(name):
        """A whole pool's values in 64 bits."""
        x, s = st[name], st[name + "_scale"]
        if case["type"] != "i4":
            return x.double() if s is None else x.double() * s.double()[..., None]
        half = torch.stack([x.int() % 16, x.int() // 16], -1).view(*x.shape[:-1], hd)
        half = torch.where(half >= 8, half - 16, half).double()
        of = torch.arange(hd, device=DEV) * 4 // hd   # the quarter of each value
        return half * s[..., 4:].double()[..., of] * s[..., :4].contiguous().view(torch.float32).double()

    def stored(x):
        """The value that 4-bit rows keep of each entry of x (fp32 values held in 64 bits)."""
        t = x.abs().max(-1, keepdim=True).values / 1785
        unit = 2.0 ** (torch.floor(torch.log2(t)) - 12)
        scale = torch.ceil(t / unit) * unit
        part = x.view(*x.shape[:-1], 4, hd // 4)
        step = torch.ceil(part.abs().max(-1, keepdim=True).values / (7 * scale[..., None])).clamp(min=1) * scale[..., None]
        return (torch.round(part / step) * step).view(x.shape)

    if case["kind"] == "cache4":
        rot = case["rot"]
        pos = torch.cat([torch.arange(p, p + c, device=DEV) for _, c, p, _ in st["seqs"].tolist()])
        turn = torch.complex(st["cos"][pos].double(), st["sin"][pos].double())[:, None]
        res = []
        for name in ("q", "k", "v"):
            x = st[name].double().view(n, -1, hd).clone()
            if name != "v":
                re = x[..., : rot // 2] if case["half"] else x[..., 0:rot:2]
                im = x[..., rot // 2: rot] if case["half"] else x[..., 1:rot:2]
                z = torch.complex(re, im) * turn
                re.copy_(z.real)
                im.copy_(z.imag)
            # What is quantised is the rotated value in 32 bits.
            res.append(x if name == "q" else stored(x.float().double()))
        return tuple(x.reshape(n, -1) for x in res)

    # Sequence by sequence, head by head.
    key, value = values("key"), values("value")
    out = torch.zeros(n, heads, hd, dtype=torch.float64, device=DEV)
    q = st["q"].double().view(n, heads, hd)
    for i, (first, count, pos, s) in enumerate(st["seqs"].tolist()):
        total = pos + count
        pages = st["table"][s, : -(-total // case["page_rows"])].long()
        far = torch.arange(pos, total, device=DEV)[:, None] - torch.arange(total, device=DEV)[None]
        hidden = far < 0
        if case["prefix"]:
            hidden[:, : int(st["prefix"][i])] = False
        if case["window"]:
            hidden |= far >= case["window"]
        for h in range(kvh):
            k, v = (x[pages, h].reshape(-1, hd)[:total] for x in (key, value))
            for j in range(h * heads // kvh, (h + 1) * heads // kvh):
                x = q[first:first + count, j] @ k.t() / hd ** 0.5
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                if case["alibi"]:
                    x = x - float(st["slopes"][j]) * far.abs()
                out[first:first + count, j] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v
    return out.view(n, -1)
