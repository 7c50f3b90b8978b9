"""4-bit paged rows, attention with terms, and page pools in plain numpy, 64 bits."""
import numpy as np

import paged_ref

FMAX = float(np.finfo(np.float32).max)


def round_up_13(t):
    """The least numbers of 13 significant bits no smaller than t (64 bits, positive)."""
    m, e = np.frexp(t)
    return np.ldexp(np.ceil(m * 8192), e - 13)


def encode4(x):
    """Rows x [..., head_dim] of fp32 values: (codes [..., head_dim / 2], entries
    [..., 8] of scale and multipliers, the values they stand for in 64 bits)."""
    x = np.asarray(x, dtype=np.float32)
    amax = np.abs(x).max(-1)
    bad, none = ~np.isfinite(x).all(-1), amax < 2.0 ** -100
    safe = np.where(bad | none, 1.0, amax.astype(np.float64))
    x64 = np.where((bad | none)[..., None], 0.0, x.astype(np.float64))
    # Quotients of numbers of 24 bits by ones of 16 and fewer are no closer to a whole
    # number, or to a tie, than 2^-25 of it without being one: 64 bits decide.
    most = np.floor(FMAX / 1785 / 2.0 ** 105) * 2.0 ** 105   # 13 bits: of 2^117 steps of 2^105
    scale = np.where(none | bad, 1.0, np.minimum(round_up_13(safe / 1785), most))
    parts = x64.reshape(*x.shape[:-1], 4, -1)
    mult = np.clip(np.ceil(np.abs(parts).max(-1) / (7 * scale[..., None])), 1, 255)
    code = np.rint(parts / (mult * scale[..., None])[..., None]).reshape(x.shape).astype(np.int8)
    scale = np.where(bad, np.nan, scale).astype(np.float32)
    entries = np.concatenate([scale[..., None].view(np.uint8), mult.astype(np.uint8)], -1)
    u = (code & 15).astype(np.uint8)
    return u[..., 0::2] | u[..., 1::2] << 4, entries, decode4(u[..., 0::2] | u[..., 1::2] << 4, entries)


def decode4(codes, entries):
    """The values of 4-bit rows in 64 bits."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1).astype(np.int8)
    c = np.where(c > 7, c - 16, c).astype(np.float64)
    scale = np.ascontiguousarray(entries[..., :4]).view(np.float32)[..., 0].astype(np.float64)
    part = c.reshape(*c.shape[:-1], 4, -1) * entries[..., 4:].astype(np.float64)[..., None]
    return part.reshape(c.shape) * scale[..., None]


class Pool(paged_ref.Pool):
    """paged_ref.Pool with 4-bit rows ("i4") too, and attention with terms."""

    def __init__(self, rng, kind, *args, draw=None, **kw):
        kept = []
        draw = draw or (lambda *s: rng.standard_normal(s).astype(np.float32))

        def keep(*shape):
            kept.append(draw(*shape))
            return kept[-1]

        super().__init__(rng, "i8" if kind == "i4" else kind, *args, draw=keep, **kw)
        if kind == "i4":
            self.kind = kind
            self.key, self.value = (list(encode4(x)) for x in kept)

    def poison(self, mask):
        if self.kind != "i4":
            return super().poison(mask)
        for codes, entries, _ in (self.key, self.value):
            codes.transpose(0, 2, 1, 3)[mask] = 0x88
            entries.transpose(0, 2, 1, 3)[mask] = 0xFF   # scales that are not numbers

    def attention(self, q, heads, scale=None, cap=0.0, window=0, slopes=None, prefix=None):
        """[n, heads * hd]; left-out tokens NaN."""
        hd, G = self.hd, heads // self.kvh
        scale = 1 / np.sqrt(hd) if scale is None else scale
        out = np.full((self.n, heads, hd), np.nan)
        for i, (first, count, pos, t) in enumerate(self.seqs):
            total = pos + count
            k, v, present = self.rows(t, total)
            r = np.arange(total)
            for j in range(count):
                p = pos + j
                seen = r <= p
                if prefix is not None:
                    seen = seen | (r < prefix[i])
                if window:
                    seen = seen & (p - r < window)
                seen = seen & present
                if not seen.any():
                    out[first + j] = 0
                    continue
                for h in range(heads):
                    s = k[seen, h // G] @ q[first + j, h * hd:(h + 1) * hd].astype(np.float64) * scale
                    if cap:
                        s = cap * np.tanh(s / cap)
                    if slopes is not None:
                        s = s - np.float64(slopes[h]) * np.abs(p - r[seen])
                    w = np.exp(s - s.max())
                    out[first + j, h] = w @ v[seen, h // G] / w.sum()
        return out.reshape(self.n, -1)

    def dev(self, qk, torch, max_count=None, max_rows=None, n_tokens=None):
        if self.kind != "i4":
            return super().dev(qk, torch, max_count, max_rows, n_tokens)
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        kv = qk.PagedKV(qk.I4, up(self.key[0]), up(self.value[0]), up(self.key[1]), up(self.value[1]))
        return kv, qk.PagedBatch(up(self.table), up(self.seqs), self.n if n_tokens is None else n_tokens,
                                 max_count or self.max_count, max_rows or self.max_rows)


class Pages:
    """A pool's table, counts and contents (any integer arrays [pages][...]), entry by entry."""

    def __init__(self, rows, stride, pages, page_rows, contents=()):
        self.table = np.full((rows, stride), -1, dtype=np.int32)
        self.refs = np.zeros(pages, dtype=np.int32)
        self.page_rows, self.contents = page_rows, [c.copy() for c in contents]

    def held(self, p):
        return 0 <= p < len(self.refs)

    def take(self, taken):
        """The lowest page that was free in `taken`, which loses it; -1."""
        for p in range(taken["next"], len(self.refs)):
            if taken["refs"][p] == 0:
                taken["next"] = p + 1
                return p
        taken["next"] = len(self.refs)
        return -1

    def resize(self, lengths, begins=None):
        rows, stride = self.table.shape
        want = [None] * rows
        for r in range(rows):
            if lengths[r] < 0:
                continue
            first = max(int(begins[r]), 0) // self.page_rows if begins is not None else 0
            want[r] = (first, -(-int(lengths[r]) // self.page_rows))
            for e in range(stride):
                if self.held(self.table[r, e]) and not first <= e < want[r][1]:
                    self.refs[self.table[r, e]] -= 1
                    self.table[r, e] = -1
        missing, free = 0, dict(refs=self.refs.copy(), next=0)
        for r in range(rows):
            for e in range(*(want[r] or (0, 0))):
                if e >= stride:
                    missing += 1
                elif not self.held(self.table[r, e]):
                    p = self.take(free)
                    self.table[r, e] = p
                    if p < 0:
                        missing += 1
                    else:
                        self.refs[p] = 1
        return missing

    def fork(self, parents, lengths):
        rows, stride = self.table.shape
        old, free = self.table.copy(), dict(refs=self.refs.copy(), next=0)
        missing, copies = 0, []
        for c in range(rows):
            p = parents[c]
            if not 0 <= p < rows or p == c:
                continue
            full, part = divmod(max(int(lengths[c]), 0), self.page_rows)
            new = np.full(stride, -1, dtype=np.int32)
            for e in range(stride):
                if e < full and self.held(old[p, e]):
                    new[e] = old[p, e]
                elif e == full and part and self.held(old[p, e]):
                    new[e] = self.take(free)
                    if new[e] < 0:
                        missing += 1
                    else:
                        copies.append((old[p, e], new[e]))
            for e in range(stride):
                if self.held(old[c, e]):
                    self.refs[old[c, e]] -= 1
                if new[e] >= 0:
                    self.refs[new[e]] += 1
            self.table[c] = new
        for src, dst in copies:
            for a in self.contents:
                a[dst] = a[src]
        return missing

    def compact(self):
        live = [p for p in range(len(self.refs)) if self.refs[p] > 0]
        holes = [p for p in range(len(live)) if self.refs[p] == 0]
        moves = dict(zip([p for p in live if p >= len(live)], holes))
        for src, dst in moves.items():
            for a in self.contents:
                a[dst] = a[src]
            self.refs[dst], self.refs[src] = self.refs[src], 0
        for i, p in np.ndenumerate(self.table):
            self.table[i] = moves.get(int(p), p)
        return len(moves)
