"""The paged cache in plain numpy, 64 bits: its row formats, a pool with pages
in any order, and attention over it."""
import numpy as np

NAMES = {"f16": "F16", "i8": "I8", "e4m3": "F8_E4M3"}


def e4m3_values():
    """The 256 float8 values (4-bit exponent of bias 7, 3-bit mantissa, no
    infinities, 0x7F and 0xFF not a number)."""
    out = np.empty(256)
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        v = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out[b] = np.nan if b & 127 == 127 else (-v if b & 128 else v)
    return out


E4M3 = e4m3_values()


def encode(x, kind):
    """Rows x [..., head_dim] of fp32 values: (stored codes, scales or None,
    the values they stand for in 64 bits)."""
    x = np.asarray(x, dtype=np.float32)
    if kind == "f16":
        h = x.astype(np.float16)
        return h, None, h.astype(np.float64)
    amax = np.abs(x).max(-1)
    bad = ~np.isfinite(x).all(-1)
    none = amax < 2.0 ** -100
    safe = np.where(bad | none, np.float32(1), amax)
    x64 = np.where((bad | none)[..., None], 0.0, x.astype(np.float64))
    if kind == "i8":
        scale = (safe / np.float32(127)).astype(np.float32)
        scale = np.where(none, np.float32(1), scale)
        # The quotient of two fp32 values is no closer to a tie than an ulp of
        # 64 bits without being one: rint of it is the exact rounding.
        codes = np.rint(x64 / scale.astype(np.float64)[..., None]).astype(np.int8)
        value = codes.astype(np.float64)
    else:
        mant, e = np.frexp(safe.astype(np.float64))
        scale = np.where(none, 1.0, 2.0 ** (e - 9 + (mant > 0.875))).astype(np.float32)
        y = x64 / scale.astype(np.float64)[..., None]
        step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
        value = np.rint(y / step) * step
        order = np.argsort(E4M3[:127])
        codes = order[np.searchsorted(E4M3[:127][order], np.abs(value))].astype(np.uint8) | \
            (np.signbit(y).astype(np.uint8) << 7)
    scale = np.where(bad, np.float32(np.nan), scale).astype(np.float32)
    return codes, scale, value * scale.astype(np.float64)[..., None]


def rotate(x, cos, sin, rot, half):
    """x [tokens, heads, head_dim] by table rows [tokens, rot / 2], one rounding."""
    out = np.array(x, dtype=np.float32)
    a, b = (x[..., : rot // 2], x[..., rot // 2: rot]) if half else (x[..., 0:rot:2], x[..., 1:rot:2])
    a, b, c, s = (v.astype(np.float64) for v in (a, b, cos[:, None], sin[:, None]))
    re, im = (a * c - b * s).astype(np.float32), (b * c + a * s).astype(np.float32)
    if half:
        out[..., : rot // 2], out[..., rot // 2: rot] = re, im
    else:
        out[..., 0:rot:2], out[..., 1:rot:2] = re, im
    return out


class Pool:
    """A pool of pages filled with rows of a given kind, and the page table of
    sequences (count, pos), in numpy; dev() puts it on the GPU."""

    def __init__(self, rng, kind, kvh, hd, page_rows, seqs, spare=2, draw=None, table_extra=1):
        self.kind, self.kvh, self.hd, self.page_rows = kind, kvh, hd, page_rows
        need = [-(-(c + p) // page_rows) for c, p in seqs]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(seqs), max(need + [1]) + table_extra), -1, dtype=np.int32)
        self.seqs = np.zeros((len(seqs), 4), dtype=np.int32)
        at = first = 0
        for i, ((c, p), k) in enumerate(zip(seqs, need)):
            self.table[i, :k] = order[at:at + k]
            self.seqs[i] = (first, c, p, i)
            at, first = at + k, first + c
        self.n = first
        self.max_count = max(c for c, _ in seqs)
        self.max_rows = max(c + p for c, p in seqs)
        draw = draw or (lambda *s: rng.standard_normal(s).astype(np.float32))
        shape = (self.pages, kvh, page_rows, hd)
        self.key = list(encode(draw(*shape), kind))
        self.value = list(encode(draw(*shape), kind))

    def unused(self):
        """Mask [pages, page_rows] of the rows no sequence holds."""
        free = np.ones((self.pages, self.page_rows), dtype=bool)
        for _, c, p, t in self.seqs:
            for r in range(c + p):
                page = self.table[t, r // self.page_rows]
                if 0 <= page < self.pages:
                    free[page, r % self.page_rows] = False
        return free

    def poison(self, mask):
        """Rows of a mask [pages, page_rows] filled with what is not finite."""
        for part in (self.key, self.value):
            codes = part[0].transpose(0, 2, 1, 3)
            codes[mask] = {"f16": np.float16(np.nan), "i8": np.int8(-128), "e4m3": np.uint8(0x7F)}[self.kind]
            if part[1] is not None:
                part[1].transpose(0, 2, 1)[mask] = np.nan

    def rows(self, t, n):
        """Values of rows 0 .. n - 1 of table row t, [n, kvh, hd], and which are present."""
        k, v = np.zeros((n, self.kvh, self.hd)), np.zeros((n, self.kvh, self.hd))
        present = np.zeros(n, dtype=bool)
        for r in range(n):
            page = self.table[t, r // self.page_rows]
            if 0 <= page < self.pages:
                present[r] = True
                k[r], v[r] = self.key[2][page, :, r % self.page_rows], self.value[2][page, :, r % self.page_rows]
        return k, v, present

    def attention(self, q, heads, scale=None):
        """Softmax attention of every token, [n, heads * hd]; left-out tokens NaN."""
        hd, G = self.hd, heads // self.kvh
        scale = 1 / np.sqrt(hd) if scale is None else scale
        out = np.full((self.n, heads, hd), np.nan)
        for first, count, pos, t in self.seqs:
            k, v, present = self.rows(t, pos + count)
            for i in range(count):
                seen = present & (np.arange(pos + count) <= pos + i)
                for h in range(heads):
                    if not seen.any():
                        out[first + i, h] = 0
                        continue
                    s = k[seen, h // G] @ q[first + i, h * hd:(h + 1) * hd].astype(np.float64) * scale
                    p = np.exp(s - s.max())
                    out[first + i, h] = p @ v[seen, h // G] / p.sum()
        return out.reshape(self.n, -1)

    def dev(self, qk, torch, max_count=None, max_rows=None, n_tokens=None):
        """(PagedKV, PagedBatch) on the GPU."""
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        codes = [up(p[0]) for p in (self.key, self.value)]
        if self.kind == "e4m3":
            codes = [c.view(torch.float8_e4m3fn) for c in codes]
        scales = [None if p[1] is None else up(p[1]) for p in (self.key, self.value)]
        kv = qk.PagedKV(getattr(qk, NAMES[self.kind]), *codes, *scales)
        return kv, qk.PagedBatch(up(self.table), up(self.seqs), self.n if n_tokens is None else n_tokens,
                                 max_count or self.max_count, max_rows or self.max_rows)
