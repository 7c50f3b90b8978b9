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
//   operand    = weight * value_scale(row) * 2^(15 - e), e by the largest of these
//                products of the query row so far (fp16 rows: 2^15): the halves do
//                not overflow, and keep 22 bits of a product above 2^-10 of the
//                largest and 2^-32 of that of any other.
#include "qk_paged.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

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
    int heads, group, page_shift;   // group: query heads a KV head
    // Splits of the rows of a sequence of few query rows a KV head and of one of
    // many (more than few_rows, which the chunk kernel takes).
    int splits[2], split_rows[2], part_splits;
    int few_rows;
    float scale;   // log2(e) * the softmax scale
};

constexpr int kTile = 32;      // cache rows of a tile
constexpr int kRowTile = 16;   // query rows of a workgroup

// A split's partial of one (token, head): the largest score and the sum of weights
// (in base-2 units), padded to 4, then head_dim means.
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

// The bits of four 8-bit codes that make them other than 0 (float8 has a -0).
template <int TYPE>
constexpr uint32_t code_bits = TYPE == QK_TYPE_I8 ? 0xFFFFFFFFu : 0x7F7F7F7Fu;

// The bits of all lanes of each 16.
__device__ __forceinline__ uint32_t or16(uint32_t bits) {
    auto turned = [](uint32_t v, auto by) {
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x120 + decltype(by)::value, 0xF, 0xF, false));
    };
    bits |= turned(bits, std::integral_constant<int, 8>{});   // row_ror
    bits |= turned(bits, std::integral_constant<int, 4>{});
    bits |= turned(bits, std::integral_constant<int, 2>{});
    return bits | turned(bits, std::integral_constant<int, 1>{});
}

__device__ __forceinline__ half8 join(half2v a, half2v b, half2v c, half2v d) {
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
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
    // Slots whose row is not all zeros (8-bit codes); by all lanes of 16 that hold it.
    __device__ __forceinline__ uint32_t live() const {
        uint32_t bits = 0;
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t any = 0;
            #pragma unroll
            for (int d = 0; d < (kB + 3) / 4; ++d) any |= w[j][d];
            if (any & code_bits<TYPE>) bits |= 1u << j;
        }
        return or16(bits);
    }
    // Operands of four dimensions (two of the rest of 96) from one dword of each
    // row: rows are interleaved in pairs, and a pair's bytes are as they stand
    // what a conversion takes.
    __device__ __forceinline__ void operands(int d, half8 (&v)[4]) const {
        if constexpr (TYPE == QK_TYPE_F16) {
            #pragma unroll
            for (int c = 0; c < 4 && 4 * d + c < HD / 16; ++c) {
                const uint32_t sel = c & 1 ? 0x07060302u : 0x05040100u;
                half2v p[4];
                #pragma unroll
                for (int k = 0; k < 4; ++k)
                    p[k] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(w[2 * k + 1][2 * d + c / 2], w[2 * k][2 * d + c / 2], sel));
                v[c] = join(p[0], p[1], p[2], p[3]);
            }
        } else {
            half2v p[4][4];
            #pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t x = w[2 * k][d], y = w[2 * k + 1][d];
                codes4<TYPE>(__builtin_amdgcn_perm(y, x, 0x05010400u), p[0][k], p[1][k]);
                codes4<TYPE>(__builtin_amdgcn_perm(y, x, 0x07030602u), p[2][k], p[3][k]);
            }
            #pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = join(p[c][0], p[c][1], p[c][2], p[c][3]);
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

// Two values as halves each: hi cut off, lo what is left (one mixed fma a value).
// The values are pinned: a product that ends here would otherwise be rounded to
// fp16 at once where hi is used and by way of fp32 where lo is made of it, and the
// two differ by a step now and then.
__device__ __forceinline__ void split_pair(float x, float y, half2v &hi, half2v &lo) {
    float minus = -1.f;   // a constant here would make two conversions and a difference of the fma
    asm("" : "+v"(x), "+v"(y), "+s"(minus));
    hi = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(x, y));
    lo = half2v{static_cast<_Float16>(fmaf(static_cast<float>(hi[0]), minus, x)),
                static_cast<_Float16>(fmaf(static_cast<float>(hi[1]), minus, y))};
}

// The largest of three, without the steps that make a signalling NaN quiet first
// (results of arithmetic are quiet already); NaN only of three.  The compiler does
// not see that a vector instruction wrote the result: one that it does see has to
// come between this and a lane exchange, which needs wait states behind it.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}

// Both halves' maximum, of a lane and the one 32 from it.
__device__ __forceinline__ float max_halves(float v) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, v);
    const auto both = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    const uint32_t low = both[0], high = both[1];
    return fmaxf(__builtin_bit_cast(float, low), __builtin_bit_cast(float, high));
}

// A wave's values joined by op, `none` for a lane without one; in every lane.
template <typename Op>
__device__ __forceinline__ float wave_join(float v, float none, Op op) {
    const int fill = __builtin_bit_cast(int, none);
    auto moved = [&](int bits) { return __builtin_bit_cast(float, bits); };
    v = op(v, moved(__builtin_amdgcn_update_dpp(fill, __builtin_bit_cast(int, v), 0x111, 0xF, 0xF, false)));   // row_shr 1, 2, 4, 8
    v = op(v, moved(__builtin_amdgcn_update_dpp(fill, __builtin_bit_cast(int, v), 0x112, 0xF, 0xF, false)));
    v = op(v, moved(__builtin_amdgcn_update_dpp(fill, __builtin_bit_cast(int, v), 0x114, 0xF, 0xF, false)));
    v = op(v, moved(__builtin_amdgcn_update_dpp(fill, __builtin_bit_cast(int, v), 0x118, 0xF, 0xF, false)));
    v = op(v, moved(__builtin_amdgcn_update_dpp(fill, __builtin_bit_cast(int, v), 0x142, 0xA, 0xF, false)));   // row_bcast 15 into rows 1 and 3
    v = op(v, moved(__builtin_amdgcn_update_dpp(fill, __builtin_bit_cast(int, v), 0x143, 0xC, 0xF, false)));   // row_bcast 31 into rows 2 and 3
    return moved(__builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ float wave_max(float v) {
    return wave_join(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}
// The largest and the least exponent of a wave's values that are not 0 (none:
// below and above all others), each 2^(e - 1) to 2^e, in one go.
__device__ __forceinline__ void wave_exponents(float v, int &top, int &low) {
    typedef uint16_t two __attribute__((ext_vector_type(2)));
    const int e = __builtin_amdgcn_frexp_expf(v) + 512;
    two b = v != 0.f ? two{static_cast<uint16_t>(e), static_cast<uint16_t>(1024 - e)} : two{0, 0};
    auto join = [&](auto ctrl, auto rows) {
        const int moved = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, b), decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
        b = __builtin_elementwise_max(b, __builtin_bit_cast(two, moved));
    };
    join(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xF>{});   // row_shr 1, 2, 4, 8
    join(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xF>{});
    join(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xF>{});
    join(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xF>{});
    join(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});   // row_bcast 15 into rows 1 and 3
    join(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});   // row_bcast 31 into rows 2 and 3
    const uint32_t all = __builtin_amdgcn_readlane(__builtin_bit_cast(int, b), 63);
    top = static_cast<int>(all & 0xFFFF) - 512;
    low = 512 - static_cast<int>(all >> 16);
}
__device__ __forceinline__ float wave_sum(float v) {
    return wave_join(v, 0.f, [](float a, float b) { return a + b; });
}

// |v| as an integer, ordered as the values are, infinity and NaN above them.
__device__ __forceinline__ int magnitude(float v) { return __builtin_bit_cast(int, v) & 0x7FFFFFFF; }

// What a query row of largest magnitude top is multiplied by (a power of two that
// brings that below 2^14) and what its scores are.  All scores of a row that is
// not finite are not numbers.
__device__ __forceinline__ void query_units(int top, float scale, float &factor, float &qscale) {
    const int e = top > 0 ? min(14 - __builtin_amdgcn_frexp_expf(__builtin_bit_cast(float, top)), 126) : 0;
    const bool fin = top < 0x7F800000;
    factor = fin ? ldexpf(1.f, e) : __builtin_nanf("");
    qscale = fin ? ldexpf(scale, -e) : 1.f;
}

// The units of one query row's products of weights and value scales, 2^(15 - e).
// e follows the largest product, not the largest scale: a row that this query row
// does not see, or gives no weight, may have a scale 2^40 times the others'.
// Products are looked at where the maximum grows, and where the tile's largest
// scale alone does not say that none overflows.  Nor do rows of zeros count, whose
// scale says nothing: codes are looked at where a scale is 1, which the writer gives
// such rows, or a product is 64 times what was known.
constexpr int kLeastExponent = -112;   // the halves' least step is below fp32's then
struct ValueUnits {
    float known = 0.f;                // the largest product, by the present weights
    float factor = 0x1p127f;          // 2^(15 - e)
    __device__ __forceinline__ int exponent() const { return 16 - __builtin_amdgcn_frexp_expf(factor); }
    __device__ __forceinline__ bool holds(float product) const { return product * factor <= 65504.f; }
    __device__ __forceinline__ bool strange(float product) const { return product > 64.f * known; }
    // New units by the largest product of a tile and its largest scale, for which
    // they leave room (2^2); earlier weights (and known) times f: what the sums are
    // multiplied by.  (Those that are not finite stay so in any units.)
    __device__ __forceinline__ float renew(float product, float scale, float f) {
        known = fmaxf(known, product);
        const int old = exponent();
        int e = kLeastExponent;
        if (known > 0.f) {
            const int ek = __builtin_amdgcn_frexp_expf(known);
            e = known < INFINITY ? max(max(ek, min(ek + 2, __builtin_amdgcn_frexp_expf(scale))), kLeastExponent) : old;
        }
        factor = ldexpf(1.f, 15 - e);
        return ldexpf(f, old - e);
    }
};

// A workgroup: 16 query rows of one (sequence, KV head) over a split's rows,
// its four waves every fourth tile of 32 rows each; the waves' states meet in
// LDS.  Few query rows leave the cache as the bound, so nothing is staged: a lane
// loads its own share of both operands, the next tile's while this one is
// multiplied.  64 sequences over 1000 to 8000 rows, 8 KV heads of 128 int8 values:
// 611 MB in 136 us, 4.5 TB/s (a copy reaches 4.7, a plain reading 6.15); one over
// 700 rows of 64 fp16 values: 5.9 us, the latency of its loads, and 3.1 of the
// merge.  Two workgroups a CU up to 128 dimensions: left to itself the compiler
// takes registers beyond that (fp16 rows of 128, 4 sequences of 8000: 33 us, with
// the bound 28).
template <int HD, int TYPE>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void paged_attention_kernel(PagedAttn a) {
    constexpr int NS = HD / 32, NC = HD / 16, kCode = code_bytes(TYPE);
    constexpr bool kScaled = TYPE != QK_TYPE_F16;
    __shared__ float meet[3][HD * 16 + 64];
    const qk_paged_seq s = a.b.seqs[blockIdx.y];
    if (!paged_seq_ok(s, a.b, a.page_shift)) return;
    const int kvh = a.kv.kv_heads, G = a.group;
    // A chip's XCDs take workgroups in turn: the splits rotate, or the first ones
    // (which every sequence has) would all fall to the same XCDs.
    const int splits = a.splits[0], unit = blockIdx.x / splits, split = (blockIdx.x + unit + blockIdx.y) % splits;
    const int h = unit % kvh, row0 = unit / kvh * kRowTile;
    const int rows = s.count * G;
    if (row0 >= rows || rows > a.few_rows) return;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // This lane's query row, the last row it sees, and the rows the tile sees.
    // (Past the last row: that one again, masked and not written.)
    const int row = row0 + n, tok = min(row, rows - 1) / G, own = min(row, rows - 1) - tok * G;
    const bool have = row < rows;
    const int mine = have ? s.pos + tok : -1;
    const int last = s.pos + __builtin_amdgcn_readlane(tok, 15);   // of the tile's last token
    const int seen = s.pos + __builtin_amdgcn_readlane(tok, 0);    // of its first
    const int64_t begin64 = static_cast<int64_t>(split) * a.split_rows[0];
    if (begin64 > last) return;   // the merge takes the splits that reach a token
    const int begin = static_cast<int>(begin64), end = static_cast<int>(min(begin64 + a.split_rows[0], int64_t(last) + 1));

    half8 qh[NS], ql[NS];
    float qscale;
    {
        const float *qrow = a.q + (s.first + tok) * a.ldq + static_cast<int64_t>(h * G + own) * HD;
        float v[NS][8];
        #pragma unroll
        for (int st = 0; st < NS; ++st)
            #pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 x = *reinterpret_cast<const float4 *>(qrow + key_dim<HD, TYPE>(st, g) + e);
                v[st][e] = x.x, v[st][e + 1] = x.y, v[st][e + 2] = x.z, v[st][e + 3] = x.w;
            }
        int top = 0;
        #pragma unroll
        for (int st = 0; st < NS; ++st)
            #pragma unroll
            for (int k = 0; k < 8; ++k) top = max(top, magnitude(v[st][k]));
        top = max(top, __shfl_xor(top, 16));
        top = max(top, __shfl_xor(top, 32));
        float factor;
        query_units(top, a.scale, factor, qscale);
        #pragma unroll
        for (int st = 0; st < NS; ++st) {
            half2v u[4], w[4];
            #pragma unroll
            for (int k = 0; k < 4; ++k)
                split_pair(factor * v[st][2 * k], factor * v[st][2 * k + 1], u[k], w[k]);
            qh[st] = join(u[0], u[1], u[2], u[3]);
            ql[st] = join(w[0], w[1], w[2], w[3]);
        }
    }

    float4v o[NC];
    #pragma unroll
    for (int c = 0; c < NC; ++c) o[c] = float4v{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    ValueUnits units;

    const int32_t *table = a.b.page_table + static_cast<int64_t>(s.table) * a.b.table_stride;
    const int64_t page_stride = static_cast<int64_t>(kvh) * a.kv.page_rows, head_row = static_cast<int64_t>(h) * a.kv.page_rows;
    // Each half of a tile lies in one page; rows past the sequence's last are
    // read from the first page (in bounds, masked).  A tile's pages are looked up
    // two tiles ahead, its rows loaded one ahead.
    struct Pages {
        int64_t id[2];
    };
    struct Tile {
        KeyTile<HD, TYPE> k;
        ValueTile<HD, TYPE> v;
        float4v ks[2], vs[2];
        bool present[2];
    };
    auto pages_of = [&](int t0) {
        Pages p;
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const int r = min(t0 + 16 * hf, last);
            const int64_t page = paged_page(table, r >> a.page_shift, a.kv.pages);
            p.id[hf] = t0 + 16 * hf <= last ? page : -1;
        }
        return p;
    };
    auto load = [&](Tile &t, int t0, const Pages &p) {
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            t.present[hf] = p.id[hf] >= 0;
            const int64_t base = max(p.id[hf], int64_t(0)) * page_stride + head_row + ((t0 + 16 * hf) & (a.kv.page_rows - 1));
            t.k.load(hf, static_cast<const char *>(a.kv.key) + (base + n) * (HD * kCode), g);
            #pragma unroll
            for (int j = 0; j < 4; ++j)
                t.v.load(4 * hf + j, static_cast<const char *>(a.kv.value) + (base + 4 * g + j) * (HD * kCode), n);
            if constexpr (kScaled) {
                t.ks[hf] = *reinterpret_cast<const float4v *>(a.kv.key_scale + base + 4 * g);
                t.vs[hf] = *reinterpret_cast<const float4v *>(a.kv.value_scale + base + 4 * g);
            }
        }
    };
    auto take = [&](Tile &t, int t0) {
        float4v st[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        #pragma unroll
        for (int x = 0; x < NS; ++x)
            #pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const half8 k = t.k.operand(hf, x);
                st[hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[x], st[hf], 0, 0, 0);
                st[hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[x], st[hf], 0, 0, 0);
            }
        // Register r of half hf: row t0 + 16 hf + 4 g + r.
        float mx = -INFINITY, vtop = 0.f;
        bool one = false;
        const bool edge = t0 + kTile - 1 > seen || !t.present[0] || !t.present[1];
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf)
            #pragma unroll
            for (int r = 0; r < 4; ++r) {
                float x = st[hf][r] * qscale;
                // An infinite key's score: not a number, whatever its sign.
                if constexpr (kScaled)
                    x *= fmaf(t.ks[hf][r], 0.f, t.ks[hf][r]);
                else
                    x = fmaf(x, 0.f, x);
                st[hf][r] = x;
            }
        if (edge) {
            #pragma unroll
            for (int hf = 0; hf < 2; ++hf)
                #pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at = t0 + 16 * hf + 4 * g + r;
                    st[hf][r] = t.present[hf] && at <= mine ? st[hf][r] : -INFINITY;
                }
        }
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf)
            #pragma unroll
            for (int r = 0; r < 4; ++r) {
                mx = fmaxf(mx, st[hf][r]);
                if constexpr (kScaled) {
                    vtop = fmaxf(vtop, fabsf(t.vs[hf][r]));
                    one = one || t.vs[hf][r] == 1.f;
                }
            }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        if constexpr (kScaled) {
            vtop = fmaxf(vtop, __shfl_xor(vtop, 16));
            vtop = fmaxf(vtop, __shfl_xor(vtop, 32));
        }
        const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
        // The sums follow a larger maximum, of which there are few.
        const bool more = __builtin_amdgcn_ballot_w64(mn > m);
        float f = 1.f;
        if (more) {
            f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            l *= f;
            m = mn;
        }
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf)
            #pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float w = __builtin_amdgcn_exp2f(st[hf][r] - ref);
                l += w;
                if constexpr (kScaled)   // a masked row's scale may be anything
                    st[hf][r] = st[hf][r] == -INFINITY ? 0.f : w * t.vs[hf][r];
                else
                    st[hf][r] = w;
            }
        if (more || (kScaled && __builtin_amdgcn_ballot_w64(m != -INFINITY && !units.holds(vtop)))) {
            float fo = f;
            if constexpr (kScaled) {
                auto largest = [&] {
                    float y = 0.f;
                    #pragma unroll
                    for (int j = 0; j < 8; ++j) y = fmaxf(y, fabsf(st[j / 4][j % 4]));
                    y = fmaxf(y, __shfl_xor(y, 16));
                    return fmaxf(y, __shfl_xor(y, 32));
                };
                float y = largest();
                units.known *= f;
                if (__builtin_amdgcn_ballot_w64(one || units.strange(y))) {
                    const uint32_t live = t.v.live();
                    #pragma unroll
                    for (int j = 0; j < 8; ++j)   // (a scale that is not finite stays)
                        if (!(live >> j & 1) && fabsf(st[j / 4][j % 4]) < INFINITY) st[j / 4][j % 4] = 0.f;
                    y = largest();
                }
                fo = units.renew(y, vtop, f);
            }
            #pragma unroll
            for (int c = 0; c < NC; ++c)
                #pragma unroll
                for (int r = 0; r < 4; ++r) o[c][r] *= fo;
        }
        half2v pu[4], pw[4];
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const float k = kScaled ? units.factor : 0x1p15f;
            split_pair(st[hf][0] * k, st[hf][1] * k, pu[2 * hf], pw[2 * hf]);
            split_pair(st[hf][2] * k, st[hf][3] * k, pu[2 * hf + 1], pw[2 * hf + 1]);
        }
        const half8 ph = join(pu[0], pu[1], pu[2], pu[3]), pl = join(pw[0], pw[1], pw[2], pw[3]);
        // A row that some token does not see meets it as 0 * value.
        uint32_t bad = 0;
        #pragma unroll
        for (int d = 0; d < (NC + 3) / 4; ++d) {
            half8 v[4];
            t.v.operands(d, v);
            #pragma unroll
            for (int k = 0; k < 4 && 4 * d + k < NC; ++k) {
                if (TYPE != QK_TYPE_I8 && edge) clear_not_finite(v[k], bad);
                float4v &c = o[4 * d + k];
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[k], pl, c, 0, 0, 0);
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[k], ph, c, 0, 0, 0);
            }
        }
        if (TYPE != QK_TYPE_I8 && edge && __builtin_amdgcn_ballot_w64(bad != 0)) {
            // The tokens that see such a row: not finite.
            #pragma unroll
            for (int off = 1; off < 16; off <<= 1) bad |= static_cast<uint32_t>(__shfl_xor(static_cast<int>(bad), off));
            #pragma unroll
            for (int hf = 0; hf < 2; ++hf)
                #pragma unroll
                for (int r = 0; r < 4; ++r)
                    if ((bad >> (4 * hf + r) & 1) && t.present[hf] && t0 + 16 * hf + 4 * g + r <= mine)
                        l = __builtin_nanf("");
        }
    };
    constexpr int kStep = 4 * kTile;
    int t0 = begin + wave * kTile;
    if (t0 < end) {
        Tile cur;
        load(cur, t0, pages_of(t0));
        Pages ahead = pages_of(t0 + kStep);
        for (; t0 < end; t0 += kStep) {
            Tile next;
            if (t0 + kStep < end) load(next, t0 + kStep, ahead);
            ahead = pages_of(t0 + 2 * kStep);
            take(cur, t0);
            cur = next;
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    // The waves' means (sums could pass fp32's range), then into wave 0, in wave order.
    auto share_of = [](float l) { return l == 0.f ? 0.f : 1.f / l; };   // no row seen: zeros
    const int back = (kScaled ? units.exponent() : 0) - 15;
    const float inverse = share_of(l);
    #pragma unroll
    for (int c = 0; c < NC; ++c)
        #pragma unroll
        for (int r = 0; r < 4; ++r) o[c][r] = ldexpf(o[c][r] * inverse, back);
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
    float mw[4] = {m}, lw[4] = {l};
    #pragma unroll
    for (int w = 0; w < 3; ++w) {
        mw[w + 1] = meet[w][HD * 16 + 2 * n];
        lw[w + 1] = meet[w][HD * 16 + 2 * n + 1];
    }
    m = fmaxf(fmaxf(mw[0], mw[1]), fmaxf(mw[2], mw[3]));
    l = 0.f;
    #pragma unroll
    for (int w = 0; w < 4; ++w) {
        lw[w] *= __builtin_amdgcn_exp2f(mw[w] - (m == -INFINITY ? 0.f : m));
        l += lw[w];
    }
    const float whole = share_of(l);
    #pragma unroll
    for (int c = 0; c < NC; ++c)
        #pragma unroll
        for (int r = 0; r < 4; ++r) o[c][r] *= lw[0] * whole;
    #pragma unroll
    for (int w = 0; w < 3; ++w) {
        const float f = lw[w + 1] * whole;
        #pragma unroll
        for (int c = 0; c < NC; ++c) {
            const float4v po = *reinterpret_cast<const float4v *>(meet[w] + (c * 64 + lane) * 4);
            #pragma unroll
            for (int r = 0; r < 4; ++r) o[c][r] = fmaf(po[r], f, o[c][r]);
        }
    }
    if (!have) return;
    const int head = h * G + own;
    float *dst = a.out + (s.first + tok) * a.ldout + static_cast<int64_t>(head) * HD;
    if (splits > 1) {
        dst = a.parts + ((static_cast<int64_t>(s.first + tok) * a.heads + head) * a.part_splits + split) * part_floats(HD);
        if (g == 0) *reinterpret_cast<float4 *>(dst) = make_float4(m, l, 0.f, 0.f);
        dst += 4;
    }
    #pragma unroll
    for (int r = 0; r < 4; ++r)
        #pragma unroll
        for (int c = 0; c < NC; ++c) dst[value_dim<HD, TYPE>(4 * g + r, c)] = o[c][r];
}

// -------------------------------------------------------------- chunks --
//
// Sequences of many query rows: a workgroup takes 128 of them (32 a wave) over
// tiles of 64 cache rows, which all four waves read from LDS as fp16, converted
// once.  Keys lie there as they are, values transposed, [dimension][row], so both
// are operands of v_mfma_f32_32x32x16_f16 as 16-byte reads.  The rows of a tile
// are permuted as the scores' registers hold them: lane half hi has, of each 16
// rows, 4 hi .. + 3 and 8 + 4 hi .. + 3.  While a tile is multiplied the next one
// is in registers on its way from memory; two LDS buffers, a barrier a tile.
//
// The bound is the matrix instructions, twice the products of one fp16 pass: 2048
// tokens over 8192 earlier rows, 32 heads of 128 float8 values, are 620 GFLOP of
// them, in 616 to 645 us 1.0 PFLOP/s, where a library product of two fp16 matrices
// of 8192 reaches 1.15 (both below the instructions' peak, at a clock of 1.9 GHz).
// The 16-row kernel took 1150 us.  Short chunks are bound by the latency of a
// workgroup's steps: 517 tokens over 600, 24 heads, 31 us and 7.5 of the merge,
// where the matrix instructions are 10.
constexpr int kChunkTile = 64, kChunkRows = 128;

// The units of products of weights and value scales are 2^(15 - ev), ev the exponent
// of the largest scale so far, as long as no two scales of the split differ by more
// than kAlike octaves (a query row's largest product, of its largest weight, is 2^8
// of them then): nothing is to be done for a query row.  From the first tile on
// where they do, a query row's weights are taken 2^lift as large, by an addend of
// the exponential's argument: its own products count, where it sees and weighs the
// rows and these are not all zeros, and are looked at when the largest known has
// sunk below 2^8 by larger scores and scales, or when the tile may hold one of more
// than 2^16.  (With a first row of 2^-8 of the others' values 517 tokens of int8 take
// 44 us instead of 39, 2048 of float8 759 instead of 629.)
constexpr int kAlike = 6;
constexpr float kCoarse = 0x1p8f, kMostLift = 96.f;

template <int HD, int TYPE>
struct Chunk {
    static constexpr int kCode = code_bytes(TYPE), kWidth = HD == 96 ? 128 : HD;
    // A thread's share of a tile: 16 bytes of kKeys key rows, kValCols values of
    // four rows (of 96 dimensions as of 128, a quarter of the threads idle, so that
    // a wave's rows lie within 16 of one page).
    static constexpr int kKeyCols = 16 / kCode, kKeyLine = kWidth / kKeyCols, kKeys = kChunkTile * kKeyLine / 256;
    static constexpr int kValCols = kWidth / 16, kValBytes = kValCols * kCode;
    static_assert(kValCols % 4 == 0, "values go by four");
    // Keys: 16 bytes between rows put the 8 rows of a read into different
    // banks.  Values: 128 bytes a dimension, 16-byte pieces exchanged by it.
    static constexpr int kKeyStride = 2 * HD + 16;
    static constexpr int kKeyBytes = kChunkTile * kKeyStride, kValueBytes = HD * 2 * kChunkTile;

    struct Head {
        float ks[kChunkTile], vs[kChunkTile];   // vs times 2^(15 - ev)
        uint32_t bad[2];                        // rows that are not finite
        int ev;                                 // the exponent of the largest value scale so far
        int room;                               // 0, or, once scales are apart, 1 + octaves from the tile's largest to 2^ev
        int big;                                // ks are times 2^-24: there is one above 2^96
        int pad[3];
    };
    static_assert(sizeof(Head) % 16 == 0, "the second buffer's 16-byte reads");
    static constexpr int kBuffer = kKeyBytes + kValueBytes + sizeof(Head);

    // Of col + d, col a multiple of kValCols and d below it: that of col xor that of d.
    static __device__ __forceinline__ int exchange(int d) { return (d ^ (d >> 3)) & 7; }
};

typedef float float16v __attribute__((ext_vector_type(16)));

template <int HD, int TYPE>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void paged_chunk_kernel(PagedAttn a) {
    using C = Chunk<HD, TYPE>;
    constexpr int NS = HD / 16, ND = HD / 32, kCode = C::kCode;
    constexpr bool kScaled = TYPE != QK_TYPE_F16;
    extern __shared__ __align__(16) char lds[];
    const qk_paged_seq s = a.b.seqs[blockIdx.y];
    if (!paged_seq_ok(s, a.b, a.page_shift)) return;
    const int kvh = a.kv.kv_heads, G = a.group;
    const int splits = a.splits[1], unit = blockIdx.x / splits, split = (blockIdx.x + unit + blockIdx.y) % splits;
    const int rows = s.count * G, tiles = (rows + kChunkRows - 1) / kChunkRows;
    if (unit / kvh >= tiles || rows <= a.few_rows) return;
    // The last tiles first: they see the most rows.
    const int h = unit % kvh, row0 = (tiles - 1 - unit / kvh) * kChunkRows;
    const int lane = threadIdx.x & 63, n = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int last = s.pos + min(row0 + kChunkRows - 1, rows - 1) / G, seen = s.pos + row0 / G;
    const int64_t begin64 = static_cast<int64_t>(split) * a.split_rows[1];
    if (begin64 > last) return;
    const int begin = static_cast<int>(begin64), end = static_cast<int>(min(begin64 + a.split_rows[1], int64_t(last) + 1));

    // Of a row past the last one: that one again, masked and not written.
    const int wrow = row0 + 32 * wave, row = wrow + n, tok = min(row, rows - 1) / G, own = min(row, rows - 1) - tok * G;
    const bool have = row < rows;
    const int mine = have ? s.pos + tok : -1;
    const int wave_seen = s.pos + __builtin_amdgcn_readlane(tok, 0);
    const int wave_last = wrow < rows ? s.pos + __builtin_amdgcn_readlane(tok, 31) : -1;

    // ------------------------------------------------------ staging ------
    const int32_t *table = a.b.page_table + static_cast<int64_t>(s.table) * a.b.table_stride;
    const int64_t page_stride = static_cast<int64_t>(kvh) * a.kv.page_rows, head_row = static_cast<int64_t>(h) * a.kv.page_rows;
    const int mask = a.kv.page_rows - 1;
    // Renewed every tile: what follows from it is then computed anew, instead of
    // kept in registers through the loop (30 of them, which spilled).
    int tid = threadIdx.x;
    // The page of each lane's row of a tile, 16 rows of one page (past the last
    // row: of the last): it is read a tile ahead, and as uniform values the four
    // would be waited for, with all loads before them, as soon as asked for.
    auto pages_of = [&](int t0) { return table[min(t0 + (lane & 48), last) >> a.page_shift]; };
    struct Stage {
        uint4v key[C::kKeys];
        uint32_t value[4][C::kValBytes / 4];
        float scale;
        uint32_t absent;   // of the 16 rows that there are, those whose page is not
    };
    auto load = [&](Stage &g, int t0, int32_t pages) {
        const bool there = pages >= 0 && pages < a.kv.pages;
        const int group = t0 + (lane & 48);
        const uint64_t gone = __builtin_amdgcn_ballot_w64(!there && group <= last);
        g.absent = (gone & 1) | (gone >> 15 & 2) | (gone >> 30 & 4) | (gone >> 45 & 8);
        const int page = there ? pages : 0;
        // First row of 16 rows i, a uniform number.
        auto row_of = [&](int i) {
            return __builtin_amdgcn_readlane(page, 16 * i) * page_stride + head_row + ((t0 + 16 * i) & mask);
        };
        #pragma unroll
        for (int i = 0; i < C::kKeys; ++i) {
            const int row = tid / C::kKeyLine + i * (256 / C::kKeyLine), col = min(tid % C::kKeyLine * C::kKeyCols, HD - C::kKeyCols);
            const char *base = static_cast<const char *>(a.kv.key) +
                               row_of((64 * wave / C::kKeyLine + i * (256 / C::kKeyLine)) / 16) * (HD * kCode);
            g.key[i] = *reinterpret_cast<const uint4v *>(base + ((row & 15) * HD + col) * kCode);
        }
        const int quad = tid / 16, col = min(tid % 16 * C::kValCols, HD - C::kValCols);
        const char *base = static_cast<const char *>(a.kv.value) + row_of(wave) * (HD * kCode);
        #pragma unroll
        for (int r = 0; r < 4; ++r)
            __builtin_memcpy(g.value[r], base + ((4 * (quad & 3) + r) * HD + col) * kCode, C::kValBytes);
        if constexpr (kScaled)
            if (wave < 2)
                g.scale = (wave == 0 ? a.kv.value_scale : a.kv.key_scale)[page * page_stride + head_row + (group & mask) + (tid & 15)];
    };
    int top_ev = kLeastExponent, low_ev = INT32_MAX;   // wave 0's: exponents of the value scales so far
    auto store = [&](const Stage &g, int t0, char *buf) {
        auto &head = *reinterpret_cast<typename C::Head *>(buf + C::kKeyBytes + C::kValueBytes);
        const bool edge = t0 + kChunkTile - 1 > seen;
        if constexpr (kScaled) {
            if (wave == 0) {
                // A row that some token does not see meets it as 0 * value: what
                // is not finite counts as 0 there, and is flagged.
                const bool there = t0 + lane <= last && !(g.absent >> (lane >> 4) & 1);
                const bool bad = there && edge && !isfinite(g.scale);
                const uint64_t all_bad = __builtin_amdgcn_ballot_w64(bad);
                if (lane < 2 && all_bad) atomicOr(&head.bad[lane], static_cast<uint32_t>(all_bad >> (32 * lane)));
                const float v = there && !bad ? g.scale : 0.f;
                int top, low;
                wave_exponents(v, top, low);
                top_ev = max(top_ev, top);
                low_ev = min(low_ev, low);
                head.vs[lane] = ldexpf(v, 15 - top_ev);
                if (lane == 0) head.ev = top_ev, head.room = low_ev < top_ev - kAlike ? 1 + top_ev - max(top, kLeastExponent) : 0;
            } else if (wave == 1) {
                // Products without it are 2^31 at most (2^14 by 448 by 256 dimensions),
                // with it 2^14 by 2^128 by 256: 2^126 in the units of such tiles.
                const bool big = __builtin_amdgcn_ballot_w64(fabsf(g.scale) > 0x1p96f);
                const float v = big ? g.scale * 0x1p-24f : g.scale;
                head.ks[lane] = fmaf(v, 0.f, v);   // infinite: all its scores are not numbers
                if (lane == 0) head.big = big;
            }
        }
        #pragma unroll
        for (int i = 0; i < C::kKeys; ++i) {
            const int row = tid / C::kKeyLine + i * (256 / C::kKeyLine), col = tid % C::kKeyLine * C::kKeyCols;
            if (HD != C::kWidth && col >= HD) continue;
            char *at = buf + row * C::kKeyStride + col * 2;
            if constexpr (TYPE == QK_TYPE_F16) {
                *reinterpret_cast<uint4v *>(at) = g.key[i];
            } else {
                half2v c[8];
                #pragma unroll
                for (int w = 0; w < 4; ++w) codes4<TYPE>(g.key[i][w], c[2 * w], c[2 * w + 1]);
                *reinterpret_cast<half8 *>(at) = join(c[0], c[1], c[2], c[3]);
                *reinterpret_cast<half8 *>(at + 16) = join(c[4], c[5], c[6], c[7]);
            }
        }
        const int quad = tid / 16, col = tid % 16 * C::kValCols;
        if (HD != C::kWidth && col >= HD) return;
        const int piece = quad / 4 * 2 + (quad & 1), half = quad >> 1 & 1;
        const int exchanged = (piece ^ C::exchange(col)) << 4;
        char *const at = buf + C::kKeyBytes + col * 2 * kChunkTile + 8 * half;
        uint2 w[C::kValCols];   // of a dimension: rows 0 and 1, rows 2 and 3
        #pragma unroll
        for (int d4 = 0; d4 < C::kValCols / 4; ++d4) {
            half2v p[4][2];
            if constexpr (TYPE == QK_TYPE_F16) {
                #pragma unroll
                for (int c = 0; c < 4; ++c)
                    #pragma unroll
                    for (int k = 0; k < 2; ++k)
                        p[c][k] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(g.value[2 * k + 1][2 * d4 + c / 2],
                                                                                   g.value[2 * k][2 * d4 + c / 2],
                                                                                   c & 1 ? 0x07060302u : 0x05040100u));
            } else {
                #pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t x = g.value[2 * k][d4], y = g.value[2 * k + 1][d4];
                    codes4<TYPE>(__builtin_amdgcn_perm(y, x, 0x05010400u), p[0][k], p[1][k]);
                    codes4<TYPE>(__builtin_amdgcn_perm(y, x, 0x07030602u), p[2][k], p[3][k]);
                }
            }
            #pragma unroll
            for (int c = 0; c < 4; ++c)
                w[4 * d4 + c] = make_uint2(__builtin_bit_cast(uint32_t, p[c][0]), __builtin_bit_cast(uint32_t, p[c][1]));
        }
        const bool gone = g.absent >> wave & 1;
        if (TYPE != QK_TYPE_I8 && (edge || gone)) {
            uint32_t bad = 0;
            #pragma unroll
            for (int d = 0; d < C::kValCols; ++d) {
                if ((w[d].x & 0x7C00u) == 0x7C00u) w[d].x &= 0xFFFF0000u, bad |= 1u;
                if ((w[d].x & 0x7C000000u) == 0x7C000000u) w[d].x &= 0xFFFFu, bad |= 2u;
                if ((w[d].y & 0x7C00u) == 0x7C00u) w[d].y &= 0xFFFF0000u, bad |= 4u;
                if ((w[d].y & 0x7C000000u) == 0x7C000000u) w[d].y &= 0xFFFFu, bad |= 8u;
            }
            if (bad && !gone) atomicOr(&head.bad[quad / 8], bad << (4 * quad % 32));
        }
        #pragma unroll
        for (int d = 0; d < C::kValCols; ++d)
            *reinterpret_cast<uint2 *>(at + (exchanged ^ (C::exchange(d) << 4)) + d * 2 * kChunkTile) = w[d];
    };

    // ------------------------------------------------------- queries -----
    half8 qh[NS], ql[NS];
    float qscale;
    {
        const float *qrow = a.q + (s.first + tok) * a.ldq + static_cast<int64_t>(h * G + own) * HD + 8 * hi;
        float4 v[NS][2];
        #pragma unroll
        for (int x = 0; x < NS; ++x)
            #pragma unroll
            for (int k = 0; k < 2; ++k) v[x][k] = *reinterpret_cast<const float4 *>(qrow + 16 * x + 4 * k);
        int top = 0;
        #pragma unroll
        for (int x = 0; x < NS; ++x)
            #pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float4 y = v[x][k];
                top = max(max(top, max(magnitude(y.x), magnitude(y.y))), max(magnitude(y.z), magnitude(y.w)));
            }
        top = max(top, __shfl_xor(top, 32));
        // The running maximum is one of the products, whose order a negative scale
        // would turn: its sign goes to the queries.
        float factor;
        query_units(top, fabsf(a.scale), factor, qscale);
        qscale = fmaxf(qscale, 0x1p-149f);   // one that underflows is as good as that
        factor = a.scale < 0.f ? -factor : factor;
        #pragma unroll
        for (int x = 0; x < NS; ++x) {
            half2v u[4], w[4];
            #pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float4 y = v[x][k];
                split_pair(factor * y.x, factor * y.y, u[2 * k], w[2 * k]);
                split_pair(factor * y.z, factor * y.w, u[2 * k + 1], w[2 * k + 1]);
            }
            qh[x] = join(u[0], u[1], u[2], u[3]);
            ql[x] = join(w[0], w[1], w[2], w[3]);
        }
    }

    float16v o[ND];
    #pragma unroll
    for (int d = 0; d < ND; ++d)
        #pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    // The largest score so far, in base 2 (-c) and in the products' units (after large
    // key scales: that or less).
    float m = -INFINITY, c = INFINITY, l = 0.f;
    int ev = kLeastExponent;
    float lift = 0.f, known = 0.f;   // once scales are apart: l is 2^lift as large; the row's largest product
    bool apart = false;

    auto take = [&](char *buf, int t0, uint32_t absent) {
        auto &head = *reinterpret_cast<typename C::Head *>(buf + C::kKeyBytes + C::kValueBytes);
        const int en = kScaled ? __builtin_amdgcn_readfirstlane(head.ev) : ev;
        const int room = kScaled ? __builtin_amdgcn_readfirstlane(head.room) : 0;
        const bool big = kScaled && __builtin_amdgcn_readfirstlane(head.big);
        const float unit = big ? fminf(qscale * 0x1p24f, 0x1.fffffep127f) : qscale;   // a score's, of the products
        const bool edge = t0 + kChunkTile - 1 > wave_seen || absent;   // some token does not see it whole
        auto scores = [&](int hf, float16v &st) {
            #pragma unroll
            for (int r = 0; r < 16; ++r) st[r] = 0.f;
            const char *keys = buf + (32 * hf + n) * C::kKeyStride + 16 * hi;
            #pragma unroll
            for (int x = 0; x < NS; ++x) {
                const half8 k = *reinterpret_cast<const half8 *>(keys + 32 * x);
                st = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[x], st, 0, 0, 0);
                st = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[x], st, 0, 0, 0);
            }
        };
        // Half a tile at a time, the second half's scores begun before the first
        // one's weights, which run beside them: 2 % of a long chunk's time (all 32
        // scores a lane at once left too few registers).
        float16v st, ahead;
        scores(0, st);
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            // Register r: row t0 + 32 hf + 8 (r / 4) + 4 hi + r % 4.
            #pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                if constexpr (kScaled) {
                    const float4v ks = *reinterpret_cast<const float4v *>(head.ks + 32 * hf + 8 * r4 + 4 * hi);
                    #pragma unroll
                    for (int r = 0; r < 4; ++r) st[4 * r4 + r] *= ks[r];
                } else {
                    #pragma unroll
                    for (int r = 0; r < 4; ++r)   // an infinite key's score: not a number, whatever its sign
                        st[4 * r4 + r] = fmaf(st[4 * r4 + r], 0.f, st[4 * r4 + r]);
                }
            }
            if (edge) {
                const uint32_t two = absent >> (2 * hf), hide = ((two & 1 ? 0xFFFFu : 0) | (two & 2 ? 0xFFFF0000u : 0)) >> (4 * hi);
                const int left = mine - t0 - 32 * hf - 4 * hi;
                #pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int at = 8 * (r / 4) + r % 4;
                    st[r] = at <= left && !(hide >> at & 1) ? st[r] : -INFINITY;
                }
            }
            float mn = big ? -INFINITY : m;
            #pragma unroll
            for (int r = 0; r < 14; r += 2) mn = max3(mn, st[r], st[r + 1]);
            mn = max_halves(fmaxf(fmaxf(mn, st[14]), st[15]));
            const char *values = buf + C::kKeyBytes;
            auto operand = [&](int b, int d) {   // 16 rows of 32 dimensions
                return *reinterpret_cast<const half8 *>(
                    values + (32 * d + n) * 2 * kChunkTile + (((4 * hf + 2 * b + hi) ^ C::exchange(32 * d + n)) << 4));
            };
            if (room && !apart) {
                apart = true;
                known = c == INFINITY ? 0.f : kCoarse;   // of alike scales, at least
            }
            // Besides: scales are apart, and the tile may hold a product beyond a row's units.
            if (en != ev || big || __builtin_amdgcn_ballot_w64(mn > m || (room && c != INFINITY && lift > static_cast<float>(room)))) {
                // c is what the weights so far were taken with, rounding and all.
                const float cn = kScaled ? fminf(c, -mn * unit) : mn == -INFINITY ? INFINITY : -mn * qscale;
                const float f = cn == INFINITY ? 1.f : __builtin_amdgcn_exp2f(cn - c);
                l *= f;
                float fo = kScaled ? ldexpf(f, ev - en) : f;
                m = big ? -INFINITY : mn;
                c = cn;
                ev = en;
                known *= fo;
                if (__builtin_expect(room != 0, 0) &&
                    __builtin_amdgcn_ballot_w64(c != INFINITY && (lift > static_cast<float>(room) || known < kCoarse))) {
                    uint32_t live = 0;   // rows that are not all zeros, in the scores' order
                    #pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        uint4v any = {0, 0, 0, 0};
                        #pragma unroll
                        for (int d = 0; d < ND; ++d) any |= __builtin_bit_cast(uint4v, operand(b, d));
                        #pragma unroll
                        for (int j = 0; j < 8; ++j) live |= any[j / 2] & (j & 1 ? 0x7FFF0000u : 0x7FFFu) ? 1u << (8 * b + j) : 0;
                    }
                    live = or16(live);
                    live |= static_cast<uint32_t>(__shfl_xor(static_cast<int>(live), 16));
                    #pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        float &at = head.vs[32 * hf + 8 * (r / 4) + 4 * hi + r % 4];
                        const float vs = at;
                        // The scale of a row of zeros (a finite one) goes: no sum has
                        // anything of it, whichever of the two another wave reads.
                        const bool zeros = !(live >> r & 1) && fabsf(vs) < INFINITY;
                        if (zeros && n == 0) at = 0.f;
                        known = fmaxf(known, zeros ? 0.f : fabsf(__builtin_amdgcn_exp2f(fmaf(st[r], unit, (c == INFINITY ? 0.f : c) + lift)) * vs));
                    }
                    known = max_halves(known);
                    const float to = known > 0.f ? fminf(fmaxf(lift + static_cast<float>(12 - __builtin_amdgcn_frexp_expf(known)), 0.f), kMostLift) : kMostLift;
                    const float up = known < INFINITY ? __builtin_amdgcn_exp2f(to - lift) : 1.f;
                    lift = known < INFINITY ? to : lift;
                    known *= up;
                    l *= up;
                    fo *= up;
                }
                #pragma unroll
                for (int d = 0; d < ND; ++d)
                    #pragma unroll
                    for (int r = 0; r < 16; ++r) o[d][r] *= fo;
            }
            const float ref = (c == INFINITY ? 0.f : c) + lift;   // nothing seen: weights of exp2(-inf)
            if (t0 + kChunkTile - 1 > seen) {   // flagged for all waves, those that see the whole tile too
                const uint32_t bad = head.bad[hf] >> (4 * hi);
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(bad != 0) != 0, 0)) {
                    #pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if ((bad >> (8 * (r / 4) + r % 4) & 1) && st[r] != -INFINITY) l = __builtin_nanf("");
                }
            }
            if (hf == 0) scores(1, ahead);
            #pragma unroll
            for (int b = 0; b < 2; ++b) {   // 16 rows
                half2v pu[4], pw[4];
                #pragma unroll
                for (int r4 = 0; r4 < 2; ++r4) {
                    float4v vs;
                    if constexpr (kScaled)
                        vs = *reinterpret_cast<const float4v *>(head.vs + 32 * hf + 16 * b + 8 * r4 + 4 * hi);
                    float y[4];
                    #pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float x = st[8 * b + 4 * r4 + r];
                        const float w = __builtin_amdgcn_exp2f(fmaf(x, unit, ref));
                        l += w;
                        y[r] = w * (kScaled ? vs[r] : 0x1p15f);
                    }
                    split_pair(y[0], y[1], pu[2 * r4], pw[2 * r4]);
                    split_pair(y[2], y[3], pu[2 * r4 + 1], pw[2 * r4 + 1]);
                }
                const half8 ph = join(pu[0], pu[1], pu[2], pu[3]), pl = join(pw[0], pw[1], pw[2], pw[3]);
                half8 v[ND];
                #pragma unroll
                for (int d = 0; d < ND; ++d) {
                    v[d] = operand(b, d);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], pl, o[d], 0, 0, 0);
                }
                #pragma unroll
                for (int d = 0; d < ND; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], ph, o[d], 0, 0, 0);
            }
            st = ahead;
        }
    };

    Stage g;
    load(g, begin, pages_of(begin));
    int32_t ahead = pages_of(begin + kChunkTile);
    int b = 0;
    for (int t0 = begin; t0 < end; t0 += kChunkTile, b ^= 1) {
        char *buf = lds + b * C::kBuffer;
        asm volatile("" : "+v"(tid));
        if (t0 + kChunkTile - 1 > seen) {   // flags that all waves may set
            auto &head = *reinterpret_cast<typename C::Head *>(buf + C::kKeyBytes + C::kValueBytes);
            if (tid == 0) head.bad[0] = head.bad[1] = 0;
            __syncthreads();
        }
        store(g, t0, buf);
        const uint32_t absent = g.absent;
        __syncthreads();   // the tile is in; every wave is done with the one before
        if (t0 + kChunkTile < end) {
            load(g, t0 + kChunkTile, ahead);
            ahead = pages_of(t0 + 2 * kChunkTile);
        }
        if (t0 <= wave_last) take(buf, t0, absent);
    }
    l += __shfl_xor(l, 32);
    if (!have) return;
    const int head = h * G + own;
    const int back = kScaled ? ev - 15 : -15;
    const float inverse = l == 0.f ? 0.f : 1.f / l;   // no row seen: zeros
    float *dst = a.out + (s.first + tok) * a.ldout + static_cast<int64_t>(head) * HD;
    if (splits > 1) {
        dst = a.parts + ((static_cast<int64_t>(s.first + tok) * a.heads + head) * a.part_splits + split) * part_floats(HD);
        if (hi == 0) *reinterpret_cast<float4 *>(dst) = make_float4(-c, kScaled ? l * __builtin_amdgcn_exp2f(-lift) : l, 0.f, 0.f);
        dst += 4;
    }
    #pragma unroll
    for (int d = 0; d < ND; ++d)
        #pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            float v[4];
            #pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = ldexpf(o[d][4 * r4 + r] * inverse, back);
            *reinterpret_cast<float4 *>(dst + 32 * d + 8 * r4 + 4 * hi) = make_float4(v[0], v[1], v[2], v[3]);
        }
}

// The splits that reach a token, 64 at most; one wave a (token, head): a lane has a
// split's maximum and sum, then all lanes the dimensions, eight splits at a time
// (read one after the other, 64 splits took 10 us longer).
template <int HD>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttn a) {
    const qk_paged_seq s = a.b.seqs[blockIdx.y];
    if (!paged_seq_ok(s, a.b, a.page_shift)) return;
    const int lane = threadIdx.x & 63;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (at >= static_cast<int64_t>(s.count) * a.heads) return;
    const int tok = static_cast<int>(at / a.heads), head = static_cast<int>(at % a.heads);
    // As the kernel's: a tile's splits go to its last token's last row, and
    // those beyond this token's own hold nothing of it.
    const int many = static_cast<int64_t>(s.count) * a.group > a.few_rows;
    if (a.splits[many] == 1) return;
    const int live = min(a.splits[many], (s.pos + tok) / a.split_rows[many] + 1);
    const float *p = a.parts + (static_cast<int64_t>(s.first + tok) * a.heads + head) * a.part_splits * part_floats(HD);
    constexpr int kD = (HD + 63) / 64, kBatch = 8;
    float ms = -INFINITY, ls = 0.f;
    if (lane < live) {
        const float2 state = *reinterpret_cast<const float2 *>(p + lane * part_floats(HD));
        ms = state.x;
        ls = state.y;
    }
    const float *col[kD];
    #pragma unroll
    for (int d = 0; d < kD; ++d) col[d] = p + 4 + min(d * 64 + lane, HD - 1);
    const float m = wave_max(ms);
    float fs = ls * __builtin_amdgcn_exp2f(ms - (m == -INFINITY ? 0.f : m));
    const float l = wave_sum(fs);
    fs *= l == 0.f ? 0.f : 1.f / l;   // no row seen: zeros
    float o[kD] = {};
    for (int i0 = 0; i0 < live; i0 += kBatch) {
        float v[kBatch][kD];
        #pragma unroll
        for (int i = 0; i < kBatch; ++i)
            #pragma unroll
            for (int d = 0; d < kD; ++d) v[i][d] = col[d][min(i0 + i, live - 1) * part_floats(HD)];
        #pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, fs), min(i0 + i, 63)));
            if (i0 + i < live)
                #pragma unroll
                for (int d = 0; d < kD; ++d) o[d] = fmaf(v[i][d], f, o[d]);
        }
    }
    float *out = a.out + (s.first + tok) * a.ldout + static_cast<int64_t>(head) * HD;
    #pragma unroll
    for (int d = 0; d < kD; ++d)
        if (d * 64 + lane < HD) out[d * 64 + lane] = o[d];
}

// A sequence of more query rows a KV head than kFewRows takes the chunk kernel,
// if the call's chunks are kManyUnits workgroups of it unsplit, or have kManyPairs
// pairs of a query row and a cache row.  Four query heads for each of eight KV
// heads of 128 int8 values, the chunk kernel against the first, in us: one
// sequence, 68 query rows a KV head over 4000 cache rows (2.2 million pairs) 23
// and 19, 256 over 4000 (8.3 million) 30 and 30, 1600 over 500 (12 million) 36 and
// 38, 512 over 4000 (17 million) 40 and 56, 2000 over none (8 million, 128
// workgroups) 32 and 23; eight sequences, 256 over 500 (9.2 million, 128
// workgroups) 33 and 33, 68 over 4000 (17 million) 48 and 76, 512 over none (256
// workgroups) 16 and 28; 64 sequences, 68 over none (512 workgroups) 15 and 30.
// Eight query heads of 256 for one KV head, one sequence of 2048 tokens over 4000:
// int8 344 and 413, fp16 355 and 405; eight of 64 over 4000: 88 and 87, 95 and 85,
// where the first kernel would be the faster one: the rule sees neither head size
// nor type.
constexpr int kFewRows = 64, kManyUnits = 256;
constexpr int64_t kManyPairs = 3 << 22;
// Query rows a KV head up to which a sequence of this call takes the first
// kernel; a call of one sequence launches one of the two.
int few_rows(const qk_paged_batch &b, int heads, int kv_heads) {
    const int64_t rows = static_cast<int64_t>(b.max_count) * (heads / kv_heads);
    if (rows <= kFewRows) return INT32_MAX;
    const int64_t units = (rows + kChunkRows - 1) / kChunkRows * kv_heads * b.n_seqs;
    const double pairs = static_cast<double>(b.n_tokens) * heads * b.max_rows;
    if (units < kManyUnits && pairs < kManyPairs) return INT32_MAX;
    return b.n_seqs == 1 ? 0 : kFewRows;
}

// Splits of a call's rows, 64 at most.  Few query rows: the workgroups that the
// chip holds at once, two a CU (one of 256 dimensions), of at least 128 rows, or
// 256 in more than 32 splits, and none for 256 rows or less.  (One sequence, 8 KV
// heads of 128 int8 values: 250 rows whole 8.2 us, in two splits 10.2; 2000 rows
// in 16 splits 9.7, in eight 11.0; 8000 rows in 32 splits 12.5, in 63 14.0.  16
// sequences of 8000 rows: in one round of workgroups 51 us, in two 55.)  Sequences
// that fill the chip as they are even out in four splits, if those are long: 64
// sequences of 1000 to 8000 rows 136 us, 146 whole (of equal lengths the other way
// round, 217 and 197); of 125 to 1000 rows whole 24, in four splits 31.
// Chunks: a round of workgroups likewise, of at least four tiles; those that lie
// behind all that a chunk's first tokens see end at once and do not count.
struct Splits {
    int few, many;
};
Splits wanted_splits(const qk_paged_batch &b, int heads, int kv_heads, int head_dim) {
    const int64_t few = few_rows(b, heads, kv_heads), rows = static_cast<int64_t>(b.max_count) * (heads / kv_heads);
    const int64_t per_tile = static_cast<int64_t>(kv_heads) * b.n_seqs;
    const int64_t round = head_dim > 128 ? 256 : 512;
    Splits splits{1, 1};
    if (few > 0) {
        const int64_t units = std::max<int64_t>((std::min(rows, few) + kRowTile - 1) / kRowTile * per_tile, 1);
        int64_t n = round / units;
        if (b.max_rows >= 4096) n = std::max(n, std::min<int64_t>(4, 4 * round / units));
        const int64_t most = std::max<int64_t>(std::min<int64_t>(32, (int64_t(b.max_rows) + 127) / 128), b.max_rows / 256);
        splits.few = b.max_rows <= 256 ? 1 : static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({n, most, 64})));
    }
    if (rows > few) {
        const int64_t units = (rows + kChunkRows - 1) / kChunkRows * per_tile;
        const double mean = b.max_rows - 0.5 * std::min(b.max_count, b.max_rows);
        auto live = [&](int n) { return units * std::min<double>(n, mean * n / b.max_rows + 0.5); };
        while (splits.many < 64 && live(splits.many + 1) <= round && b.max_rows > splits.many * 4 * kChunkTile) ++splits.many;
    }
    return splits;
}

size_t split_bytes(const qk_paged_batch &b, int heads, int hd) {
    return static_cast<size_t>(b.n_tokens) * heads * part_floats(hd) * sizeof(float);
}

template <int HD, int TYPE>
int launch(const PagedAttn &a, hipStream_t stream) {
    const int64_t rows = static_cast<int64_t>(a.b.max_count) * (a.heads / a.kv.kv_heads);
    auto grid = [&](int64_t n, int tile, int splits) {
        return dim3(static_cast<unsigned>((n + tile - 1) / tile * a.kv.kv_heads * splits), a.b.n_seqs);
    };
    if (a.few_rows > 0)
        hipLaunchKernelGGL((paged_attention_kernel<HD, TYPE>),
                           grid(std::min<int64_t>(rows, a.few_rows), kRowTile, a.splits[0]), dim3(256), 0, stream, a);
    constexpr size_t kLds = 2 * Chunk<HD, TYPE>::kBuffer;
    if (rows > a.few_rows)
        hipLaunchKernelGGL((paged_chunk_kernel<HD, TYPE>), grid(rows, kChunkRows, a.splits[1]), dim3(256), kLds, stream,
                           a);
    if (a.part_splits > 1)
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
    const qk::Splits splits = qk::wanted_splits(*batch, heads, kv_heads, head_dim);
    const int most = std::max(splits.few, splits.many);
    return most > 1 ? most * qk::split_bytes(*batch, heads, head_dim) : 0;
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
    qk::PagedAttn a{};
    a.kv = *kv;
    a.b = *batch;
    a.q = q;
    a.out = out;
    a.parts = static_cast<float *>(workspace);
    a.ldq = ldq;
    a.ldout = ldout;
    a.heads = heads;
    a.group = heads / kv->kv_heads;
    a.page_shift = __builtin_ctz(kv->page_rows);
    a.scale = 1.4426950408889634f * (scale != 0.f ? scale : 1.f / std::sqrt(static_cast<float>(kv->head_dim)));
    const size_t per = qk::split_bytes(*batch, heads, kv->head_dim);
    const int64_t fit = workspace ? static_cast<int64_t>(workspace_bytes / per) : 0;
    const qk::Splits wanted = qk::wanted_splits(*batch, heads, kv->kv_heads, kv->head_dim);
    // Splits of whole rounds of a workgroup's tiles.
    auto plan = [&](int kind, int splits, int round) {
        const int64_t n = std::min<int64_t>(splits, fit < 2 ? 1 : fit), rows = batch->max_rows;
        const int64_t each = ((rows + n - 1) / n + round - 1) / round * round;
        a.split_rows[kind] = static_cast<int>(each);
        a.splits[kind] = static_cast<int>((rows + each - 1) / each);
    };
    a.few_rows = qk::few_rows(*batch, heads, kv->kv_heads);
    plan(0, wanted.few, 4 * qk::kTile);
    plan(1, wanted.many, qk::kChunkTile);
    a.part_splits = std::max(a.splits[0], a.splits[1]);
    // A launch has fewer than 2^32 threads a dimension, of 256 a workgroup.
    const int64_t tiles = (static_cast<int64_t>(batch->max_count) * a.group + qk::kRowTile - 1) / qk::kRowTile;
    if (tiles * kv->kv_heads * std::max(a.part_splits, 4) >= 1 << 24)   // (the merge: four tokens' heads)
        return qk::fail(QK_ERR_LIMIT, "qk_paged_attention_f32: too many query rows in one launch");
    // (In place it may be: a workgroup reads its query rows before it writes them.)
    if ((q != out || ldq != ldout) && qk::rows_meet(q, ldq, dim, out, ldout, dim, batch->n_tokens))
        return qk::fail(QK_ERR_INVALID_ARG, "qk_paged_attention_f32: out overlaps a part of q");
    switch (kv->head_dim) {
        case 64: return qk::launch_type<64>(a, qk::S(stream));
        case 96: return qk::launch_type<96>(a, qk::S(stream));
        case 128: return qk::launch_type<128>(a, qk::S(stream));
        default: return qk::launch_type<256>(a, qk::S(stream));
    }
}

}  // extern "C"
