// qk_paged_attention.hip - attention of new tokens over a paged cache.
//
// The rows of a (sequence, KV head) tile are query rows: row i * G + g is query
// head g (of G) of new token i.  Both products run on the fp16 matrix
// instructions: a cache code (int8, float8 or fp16) is exact in fp16, and a
// query value or a probability is the sum of two fp16 halves, 22 bits of it.
// The products are taken transposed, scores S^T = K Q^T and outputs O^T = V^T
// P^T: a lane then holds the scores of one query row, the softmax needs two
// cross-lane steps, and the probabilities are the second product's operand as
// they stand.
//
//   score(row) = (K code . q 2^e) * 2^-e log2(e) scale * key_scale(row), e the
//                exponent that brings a query row's largest value to 2^13;
//   weight     = exp2(score - m), m the running maximum; its sum l in fp32;
//   operand    = weight * value_scale(row) * 2^(14 - ev), ev the exponent of the
//                largest value scale so far, so the halves neither overflow
//                nor lose the bits of a small weight.
#include "qk_paged.h"

#include <algorithm>
#include <cmath>

namespace qk {
namespace {

hipStream_t S(qk_stream s) { return static_cast<hipStream_t>(s); }

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

struct PagedAttn {
    qk_paged_kv kv;
    qk_paged_batch b;
    const float *q;
    float *out, *parts;
    int64_t ldq, ldout;
    int heads, page_shift, splits, split_rows;
    float scale;   // log2(e) * the softmax scale
};

constexpr int kTile = 32;      // cache rows of a tile
constexpr int kRowTile = 16;   // query rows of a workgroup

// A split's partial of one (token, head): the running maximum and the sum (in
// base-2 units), padded to 4, then head_dim sums.
constexpr int part_floats(int hd) { return 4 + hd; }

constexpr int code_bytes(int type) { return type == QK_TYPE_F16 ? 2 : 1; }

// ------------------------------------------------ codes to fp16 operands --

// Two unsigned bytes u (code + 128) as fp16: 0x6400 | u is 1024 + u.
__device__ __forceinline__ half2v biased_pair(uint32_t bytes, uint32_t sel) {
    const uint32_t w = __builtin_amdgcn_perm(0x64646464u, bytes, sel);
    const half2v off = {static_cast<_Float16>(1152.f), static_cast<_Float16>(1152.f)};
    return __builtin_bit_cast(half2v, w) - off;
}
// Four codes of one dword, in order.
template <int TYPE>
__device__ __forceinline__ void codes4(uint32_t w, half2v &a, half2v &b) {
    if constexpr (TYPE == QK_TYPE_I8) {
        w ^= 0x80808080u;
        a = biased_pair(w, 0x04010400u);
        b = biased_pair(w, 0x04030402u);
    } else {
        a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true);
    }
}

__device__ __forceinline__ half8 join(half2v a, half2v b, half2v c, half2v d) {
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <int BYTES>
struct Bytes {
    uint32_t w[(BYTES + 3) / 4];
};
template <int BYTES>
__device__ __forceinline__ Bytes<BYTES> load_bytes(const char *p) {
    Bytes<BYTES> r{};
    __builtin_memcpy(r.w, p, BYTES);
    return r;
}

// --------------------------------------------------------------- layouts --
//
// Key operand of step s (32 dimensions): lane (row l % 16, g = l / 16) holds
// 8 dimensions.  Which ones is free as long as the query operand agrees: with
// 8-bit codes a lane loads 16 bytes that serve two steps.
template <int HD, int TYPE>
__device__ __forceinline__ constexpr int key_dim(int s, int g) {
    if (TYPE == QK_TYPE_F16 || (HD % 64 && s == HD / 32 - 1)) return 32 * s + 8 * g;
    return s / 2 * 64 + g * 16 + (s & 1) * 8;
}
// Value operand c (16 dimensions, 32 rows): lane i = l % 16 holds dimension
// value_dim(i, c), so a lane loads HD / 16 neighbours of a row at once (96
// 8-bit codes: four of the first 64 and two of the rest).
template <int HD, int TYPE>
__device__ __forceinline__ constexpr int value_dim(int i, int c) {
    if (HD == 96 && TYPE != QK_TYPE_F16) return c < 4 ? i * 4 + c : 64 + i * 2 + c - 4;
    return i * (HD / 16) + c;
}

template <int HD, int TYPE>
struct KeyTile {   // 32 rows: two halves of 16
    static constexpr int kB = HD / 4 * code_bytes(TYPE);   // bytes a lane holds of a row
    uint4v w[2][(kB + 15) / 16];
    __device__ __forceinline__ void load(int h, const char *row, int g) {
        #pragma unroll
        for (int j = 0; j < kB / 16; ++j) __builtin_memcpy(&w[h][j], row + j * 64 + g * 16, 16);
        if constexpr (kB % 16 != 0) __builtin_memcpy(&w[h][kB / 16], row + kB / 16 * 64 + g * 8, 8);
    }
    __device__ __forceinline__ half8 operand(int h, int s) const {
        if constexpr (TYPE == QK_TYPE_F16) {
            return __builtin_bit_cast(half8, w[h][s]);
        } else {
            const bool tail = HD % 64 != 0 && s == HD / 32 - 1;
            const uint4v &v = w[h][s / 2];
            const uint32_t lo = tail || !(s & 1) ? v[0] : v[2], hi = tail || !(s & 1) ? v[1] : v[3];
            half2v a, b, c, d;
            codes4<TYPE>(lo, a, b);
            codes4<TYPE>(hi, c, d);
            return join(a, b, c, d);
        }
    }
};

template <int HD, int TYPE>
struct ValueTile {   // 8 rows a lane: slot j < 4 row 4 g + j, else 16 + 4 g + j - 4
    static constexpr int kB = HD / 16 * code_bytes(TYPE);
    static constexpr bool kSplit = HD == 96 && TYPE != QK_TYPE_F16;   // 4 + 2 bytes
    uint32_t w[8][(kB + 3) / 4];
    __device__ __forceinline__ void load(int j, const char *row, int i) {
        if constexpr (kSplit) {
            uint16_t tail;
            __builtin_memcpy(&w[j][0], row + i * 4, 4);
            __builtin_memcpy(&tail, row + 64 + i * 2, 2);
            w[j][1] = tail;
        } else {
            __builtin_memcpy(w[j], row + i * kB, kB);
        }
    }
    // Operand of dimension c: its codes of the 8 rows, slot order.
    __device__ __forceinline__ half8 operand(int c) const {
        half2v p[4];
        if constexpr (TYPE == QK_TYPE_F16) {
            const uint32_t sel = c & 1 ? 0x07060302u : 0x05040100u;
            #pragma unroll
            for (int k = 0; k < 4; ++k)
                p[k] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(w[2 * k + 1][c / 2], w[2 * k][c / 2], sel));
            return join(p[0], p[1], p[2], p[3]);
        } else {
            // Byte c % 4 of four rows into one dword, then as key codes.
            const int b = c & 3, d = c / 4;
            const uint32_t pair = static_cast<uint32_t>(b | (4 + b) << 8) | 0x0c0c0000u;
            uint32_t q[2];
            #pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t lo = __builtin_amdgcn_perm(w[4 * k + 1][d], w[4 * k][d], pair);
                const uint32_t hi = __builtin_amdgcn_perm(w[4 * k + 3][d], w[4 * k + 2][d], pair);
                q[k] = lo | hi << 16;
            }
            codes4<TYPE>(q[0], p[0], p[1]);
            codes4<TYPE>(q[1], p[2], p[3]);
            return join(p[0], p[1], p[2], p[3]);
        }
    }
};

// Zeroes the values of an operand that are not finite; whether there are any,
// by slot.
__device__ __forceinline__ void clear_not_finite(half8 &v, uint32_t &bad) {
    uint4v w = __builtin_bit_cast(uint4v, v);
    #pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t all = j & 1 ? 0x7C000000u : 0x7C00u;
        if ((w[j / 2] & all) == all) {
            bad |= 1u << j;
            w[j / 2] &= j & 1 ? 0xFFFFu : 0xFFFF0000u;
        }
    }
    v = __builtin_bit_cast(half8, w);
}

__device__ __forceinline__ void split_half(float x, _Float16 &hi, _Float16 &lo) {
    hi = static_cast<_Float16>(x);
    lo = static_cast<_Float16>(x - static_cast<float>(hi));
}

// A workgroup: 16 query rows of one (sequence, KV head) over a split's rows,
// its four waves every fourth tile of 32 rows each; the waves' states meet in
// LDS.
template <int HD, int TYPE>
__global__ __launch_bounds__(256) void paged_attention_kernel(PagedAttn a) {
    constexpr int NS = HD / 32, NC = HD / 16, kCode = code_bytes(TYPE);
    constexpr bool kScaled = TYPE != QK_TYPE_F16;
    __shared__ float meet[3][HD * 16 + 64];
    const qk_paged_seq s = a.b.seqs[blockIdx.y];
    if (!paged_seq_ok(s, a.b, a.page_shift)) return;
    const int kvh = a.kv.kv_heads, G = a.heads / kvh;
    const int split = blockIdx.x % a.splits, unit = blockIdx.x / a.splits;
    const int h = unit % kvh, row0 = unit / kvh * kRowTile;
    const int rows = s.count * G;
    if (row0 >= rows) return;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // This lane's query row, the last row it sees, and the rows the tile sees.
    const int row = row0 + n, tok = row / G;
    const bool have = row < rows;
    const int mine = have ? s.pos + tok : -1;
    const int last = s.pos + min(row0 + kRowTile - 1, rows - 1) / G;   // of the tile's last token
    const int seen = s.pos + row0 / G;                                // of its first
    const int64_t begin64 = static_cast<int64_t>(split) * a.split_rows;
    if (begin64 > last) return;   // the merge takes the splits that reach a token
    const int begin = static_cast<int>(begin64), end = static_cast<int>(min(begin64 + a.split_rows, int64_t(last) + 1));

    half8 qh[NS], ql[NS];
    float qscale;
    {
        const float *qrow = a.q + (s.first + tok) * a.ldq + static_cast<int64_t>(h * G + row % G) * HD;
        float v[NS][8], top = 0.f;
        bool finite = true;
        #pragma unroll
        for (int st = 0; st < NS; ++st)
            #pragma unroll
            for (int e = 0; e < 8; e += 4) {
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                if (have) x = *reinterpret_cast<const float4 *>(qrow + key_dim<HD, TYPE>(st, g) + e);
                const float y[4] = {x.x, x.y, x.z, x.w};
                #pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[st][e + k] = y[k];
                    top = fmaxf(top, fabsf(y[k]));
                    finite = finite && isfinite(y[k]);
                }
            }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        int fin = finite;
        fin &= __shfl_xor(fin, 16);
        fin &= __shfl_xor(fin, 32);
        const int e = fin && top > 0.f ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
        qscale = fin ? ldexpf(a.scale, -e) : __builtin_nanf("");
        #pragma unroll
        for (int st = 0; st < NS; ++st)
            #pragma unroll
            for (int k = 0; k < 8; ++k) {
                _Float16 hi, lo;
                split_half(fin ? ldexpf(v[st][k], e) : 0.f, hi, lo);
                qh[st][k] = hi;
                ql[st][k] = lo;
            }
    }

    float4v o[NC];
    #pragma unroll
    for (int c = 0; c < NC; ++c) o[c] = float4v{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    int ev = -126;

    const int32_t *table = a.b.page_table + static_cast<int64_t>(s.table) * a.b.table_stride;
    const int64_t page_stride = static_cast<int64_t>(kvh) * a.kv.page_rows, head_row = static_cast<int64_t>(h) * a.kv.page_rows;
    for (int t0 = begin + wave * kTile; t0 < end; t0 += 4 * kTile) {
        // Each half of a tile lies in one page; rows past the sequence's last
        // are read from the first page (in bounds, masked).
        KeyTile<HD, TYPE> kt;
        ValueTile<HD, TYPE> vt;
        float4v ks[2], vs[2];
        bool present[2];
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const int r = t0 + 16 * hf;
            const int64_t page = r <= last ? paged_page(table, r >> a.page_shift, a.kv.pages) : -1;
            present[hf] = page >= 0;
            const int64_t base = max(page, int64_t(0)) * page_stride + head_row + (r & (a.kv.page_rows - 1));
            kt.load(hf, static_cast<const char *>(a.kv.key) + (base + n) * (HD * kCode), g);
            #pragma unroll
            for (int j = 0; j < 4; ++j)
                vt.load(4 * hf + j, static_cast<const char *>(a.kv.value) + (base + 4 * g + j) * (HD * kCode), n);
            if constexpr (kScaled) {
                ks[hf] = *reinterpret_cast<const float4v *>(a.kv.key_scale + base + 4 * g);
                vs[hf] = *reinterpret_cast<const float4v *>(a.kv.value_scale + base + 4 * g);
            }
        }
        float4v st[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        #pragma unroll
        for (int x = 0; x < NS; ++x)
            #pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const half8 k = kt.operand(hf, x);
                st[hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[x], st[hf], 0, 0, 0);
                st[hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[x], st[hf], 0, 0, 0);
            }
        // Register r of half hf: row t0 + 16 hf + 4 g + r.
        float mx = -INFINITY, vtop = 0.f;
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf)
            #pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int at = t0 + 16 * hf + 4 * g + r;
                float x = st[hf][r] * qscale;
                if constexpr (kScaled)
                    x *= ks[hf][r];
                else
                    x = fmaf(x, 0.f, x);   // an infinite key's score: not a number, whatever its sign
                st[hf][r] = present[hf] && at <= mine ? x : -INFINITY;
                mx = fmaxf(mx, st[hf][r]);
                if constexpr (kScaled) {
                    vs[hf][r] = present[hf] && at <= last ? vs[hf][r] : 0.f;
                    vtop = fmaxf(vtop, vs[hf][r]);
                }
            }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        float f = 1.f;
        const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
        int en = ev;
        if constexpr (kScaled) {
            vtop = fmaxf(vtop, __shfl_xor(vtop, 16));
            vtop = fmaxf(vtop, __shfl_xor(vtop, 32));
            en = max(ev, vtop > 0.f ? __builtin_amdgcn_frexp_expf(vtop) : -126);
            en = __builtin_amdgcn_readfirstlane(en);
        }
        f = __builtin_amdgcn_exp2f(m - ref);
        m = mn;
        l *= f;
        const float fo = kScaled ? ldexpf(f, ev - en) : f;
        ev = en;
        #pragma unroll
        for (int c = 0; c < NC; ++c)
            #pragma unroll
            for (int r = 0; r < 4; ++r) o[c][r] *= fo;
        half8 ph, pl;
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf)
            #pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float w = __builtin_amdgcn_exp2f(st[hf][r] - ref);
                l += w;
                float x = w * (kScaled ? ldexpf(vs[hf][r], 14 - ev) : 0x1p14f);
                if constexpr (kScaled) x = st[hf][r] == -INFINITY ? 0.f : x;   // a masked row's scale may be NaN
                _Float16 hi, lo;
                split_half(x, hi, lo);
                ph[4 * hf + r] = hi;
                pl[4 * hf + r] = lo;
            }
        // A row that some token does not see meets it as 0 * value.
        const bool edge = TYPE != QK_TYPE_I8 && (t0 + kTile - 1 > seen || !present[0] || !present[1]);
        uint32_t bad = 0;
        #pragma unroll
        for (int c = 0; c < NC; ++c) {
            half8 v = vt.operand(c);
            if (edge) clear_not_finite(v, bad);
            o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, o[c], 0, 0, 0);
            o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, o[c], 0, 0, 0);
        }
        if (edge && __builtin_amdgcn_ballot_w64(bad != 0)) {
            // The tokens that see such a row: not finite.
            #pragma unroll
            for (int off = 1; off < 16; off <<= 1) bad |= static_cast<uint32_t>(__shfl_xor(static_cast<int>(bad), off));
            #pragma unroll
            for (int hf = 0; hf < 2; ++hf)
                #pragma unroll
                for (int r = 0; r < 4; ++r)
                    if ((bad >> (4 * hf + r) & 1) && present[hf] && t0 + 16 * hf + 4 * g + r <= mine)
                        l = __builtin_nanf("");
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    // The waves' states to a common exponent, then into wave 0, in wave order.
    const float back = kScaled ? ldexpf(1.f, ev - 14) : 0x1p-14f;
    #pragma unroll
    for (int c = 0; c < NC; ++c)
        #pragma unroll
        for (int r = 0; r < 4; ++r) o[c][r] *= back;
    if (wave > 0) {
        float *mineat = meet[wave - 1];
        #pragma unroll
        for (int c = 0; c < NC; ++c) *reinterpret_cast<float4v *>(mineat + (c * 64 + lane) * 4) = o[c];
        if (g == 0) {
            mineat[HD * 16 + 2 * n] = m;
            mineat[HD * 16 + 2 * n + 1] = l;
        }
    }
    __syncthreads();
    if (wave > 0) return;
    #pragma unroll 1
    for (int w = 0; w < 3; ++w) {
        const float *other = meet[w];
        const float mo = other[HD * 16 + 2 * n], lo = other[HD * 16 + 2 * n + 1];
        const float mn = fmaxf(m, mo), ref = mn == -INFINITY ? 0.f : mn;
        const float f = __builtin_amdgcn_exp2f(m - ref), fo = __builtin_amdgcn_exp2f(mo - ref);
        m = mn;
        l = l * f + lo * fo;
        #pragma unroll
        for (int c = 0; c < NC; ++c) {
            const float4v po = *reinterpret_cast<const float4v *>(other + (c * 64 + lane) * 4);
            #pragma unroll
            for (int r = 0; r < 4; ++r) o[c][r] = fmaf(po[r], fo, o[c][r] * f);
        }
    }
    if (!have) return;
    const int head = h * G + row % G;
    float *dst;
    float norm = 1.f;
    if (a.splits > 1) {
        dst = a.parts + ((static_cast<int64_t>(s.first + tok) * a.heads + head) * a.splits + split) * part_floats(HD);
        if (g == 0) *reinterpret_cast<float4 *>(dst) = make_float4(m, l, 0.f, 0.f);
        dst += 4;
    } else {
        dst = a.out + (s.first + tok) * a.ldout + static_cast<int64_t>(head) * HD;
        norm = m == -INFINITY && l == 0.f ? 0.f : 1.f / l;   // no row seen: zeros
    }
    #pragma unroll
    for (int r = 0; r < 4; ++r)
        #pragma unroll
        for (int c = 0; c < NC; ++c) dst[value_dim<HD, TYPE>(4 * g + r, c)] = o[c][r] * norm;
}

// The splits that reach a token, in order; one wave a (token, head).
template <int HD>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttn a) {
    const qk_paged_seq s = a.b.seqs[blockIdx.y];
    if (!paged_seq_ok(s, a.b, a.page_shift)) return;
    const int lane = threadIdx.x & 63;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (at >= static_cast<int64_t>(s.count) * a.heads) return;
    const int tok = static_cast<int>(at / a.heads), head = static_cast<int>(at % a.heads);
    // As the kernel's: a tile's splits go to its last token's last row, and
    // those beyond this token's own hold nothing of it.
    const int live = min(a.splits, (s.pos + tok) / a.split_rows + 1);
    const float *p = a.parts + (static_cast<int64_t>(s.first + tok) * a.heads + head) * a.splits * part_floats(HD);
    constexpr int kD = HD > 64 ? (HD + 63) / 64 : 1;
    float m = -INFINITY, l = 0.f, o[kD] = {};
    for (int i = 0; i < live; ++i) {
        const float mo = p[i * part_floats(HD)], lo = p[i * part_floats(HD) + 1];
        const float mn = fmaxf(m, mo), ref = mn == -INFINITY ? 0.f : mn;
        const float f = __builtin_amdgcn_exp2f(m - ref), fo = __builtin_amdgcn_exp2f(mo - ref);
        m = mn;
        l = l * f + lo * fo;
        #pragma unroll
        for (int d = 0; d < kD; ++d)
            if (d * 64 + lane < HD) o[d] = fmaf(p[i * part_floats(HD) + 4 + d * 64 + lane], fo, o[d] * f);
    }
    const float norm = m == -INFINITY && l == 0.f ? 0.f : 1.f / l;
    float *out = a.out + (s.first + tok) * a.ldout + static_cast<int64_t>(head) * HD;
    #pragma unroll
    for (int d = 0; d < kD; ++d)
        if (d * 64 + lane < HD) out[d * 64 + lane] = o[d] * norm;
}

// Splits of a call's rows: enough workgroups for the chip, at least two tiles
// a wave.
int wanted_splits(const qk_paged_batch &b, int heads, int kv_heads) {
    const int64_t tiles = (static_cast<int64_t>(b.max_count) * (heads / kv_heads) + kRowTile - 1) / kRowTile;
    const int64_t units = std::max<int64_t>(1, tiles * kv_heads * b.n_seqs);
    const int64_t most = (b.max_rows + 8 * kTile - 1) / (8 * kTile);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({1024 / units, most, 64})));
}

size_t split_bytes(const qk_paged_batch &b, int heads, int hd) {
    return static_cast<size_t>(b.n_tokens) * heads * part_floats(hd) * sizeof(float);
}

template <int HD, int TYPE>
int launch(const PagedAttn &a, hipStream_t stream) {
    const int64_t G = a.heads / a.kv.kv_heads;
    const int64_t tiles = (a.b.max_count * G + kRowTile - 1) / kRowTile;
    hipLaunchKernelGGL((paged_attention_kernel<HD, TYPE>),
                       dim3(static_cast<unsigned>(tiles * a.kv.kv_heads * a.splits), a.b.n_seqs), dim3(256), 0,
                       stream, a);
    if (a.splits > 1)
        hipLaunchKernelGGL((paged_merge_kernel<HD>),
                           dim3(static_cast<unsigned>((static_cast<int64_t>(a.b.max_count) * a.heads + 3) / 4),
                                a.b.n_seqs),
                           dim3(256), 0, stream, a);
    return launch_status("qk_paged_attention_f32 launch");
}

template <int HD>
int launch_type(const PagedAttn &a, hipStream_t stream) {
    if (a.kv.type == QK_TYPE_F16) return launch<HD, QK_TYPE_F16>(a, stream);
    if (a.kv.type == QK_TYPE_I8) return launch<HD, QK_TYPE_I8>(a, stream);
    return launch<HD, QK_TYPE_F8_E4M3>(a, stream);
}

}  // namespace
}  // namespace qk

extern "C" {

size_t qk_paged_attention_workspace_bytes(const qk_paged_batch *batch, int heads, int kv_heads, int head_dim) {
    if (qk::check_paged_batch("qk_paged_attention_workspace_bytes", batch) || heads < 1 || kv_heads < 1 ||
        heads % kv_heads || head_dim < 1 || head_dim > 256 || batch->n_seqs == 0 || batch->n_tokens == 0)
        return 0;
    const int splits = qk::wanted_splits(*batch, heads, kv_heads);
    return splits > 1 ? splits * qk::split_bytes(*batch, heads, head_dim) : 0;
}

int qk_paged_attention_f32(const qk_paged_kv *kv, const qk_paged_batch *batch, const float *q, int ldq, float *out,
                           int ldout, int heads, float scale, void *workspace, size_t workspace_bytes,
                           qk_stream stream) {
    const char *where = "qk_paged_attention_f32";
    if (int s = qk::check_paged_kv(where, kv)) return s;
    if (int s = qk::check_paged_batch(where, batch)) return s;
    if (heads < 1 || heads > 65536 || heads % kv->kv_heads)
        return qk::fail(QK_ERR_INVALID_ARG, "qk_paged_attention_f32: heads must be a multiple of kv_heads");
    if (!std::isfinite(scale)) return qk::fail(QK_ERR_INVALID_ARG, "qk_paged_attention_f32: scale is not finite");
    if (batch->n_seqs == 0 || batch->n_tokens == 0) return qk::ok();
    if (!q || !out) return qk::fail(QK_ERR_INVALID_ARG, "qk_paged_attention_f32: null pointer");
    const int64_t dim = static_cast<int64_t>(heads) * kv->head_dim;
    if (ldq < dim || ldout < dim)
        return qk::fail(QK_ERR_INVALID_ARG, "qk_paged_attention_f32: leading dimension smaller than the row");
    if (!qk::aligned(q, 16) || !qk::aligned(out, 16) || !qk::aligned(workspace, 16) || ldq % 4 || ldout % 4)
        return qk::fail(QK_ERR_ALIGN, "qk_paged_attention_f32: q and out need 16-byte rows, workspace 16 bytes");
    const int64_t tiles = (static_cast<int64_t>(batch->max_count) * (heads / kv->kv_heads) + qk::kRowTile - 1) / qk::kRowTile;
    if (tiles * kv->kv_heads > 0x7FFFFFFF / 64)
        return qk::fail(QK_ERR_LIMIT, "qk_paged_attention_f32: too many query rows in one launch");
    qk::PagedAttn a{};
    a.kv = *kv;
    a.b = *batch;
    a.q = q;
    a.out = out;
    a.parts = static_cast<float *>(workspace);
    a.ldq = ldq;
    a.ldout = ldout;
    a.heads = heads;
    a.page_shift = __builtin_ctz(kv->page_rows);
    a.scale = 1.4426950408889634f * (scale != 0.f ? scale : 1.f / std::sqrt(static_cast<float>(kv->head_dim)));
    const size_t per = qk::split_bytes(*batch, heads, kv->head_dim);
    const int64_t fit = workspace ? static_cast<int64_t>(workspace_bytes / per) : 0;
    a.splits = static_cast<int>(std::min<int64_t>(qk::wanted_splits(*batch, heads, kv->kv_heads), fit < 2 ? 1 : fit));
    // Splits of whole rounds of the four waves' tiles.
    a.split_rows = ((batch->max_rows + a.splits - 1) / a.splits + 4 * qk::kTile - 1) / (4 * qk::kTile) * (4 * qk::kTile);
    a.splits = (batch->max_rows + a.split_rows - 1) / a.split_rows;
    switch (kv->head_dim) {
        case 64: return qk::launch_type<64>(a, qk::S(stream));
        case 96: return qk::launch_type<96>(a, qk::S(stream));
        case 128: return qk::launch_type<128>(a, qk::S(stream));
        default: return qk::launch_type<256>(a, qk::S(stream));
    }
}

}  // extern "C"
