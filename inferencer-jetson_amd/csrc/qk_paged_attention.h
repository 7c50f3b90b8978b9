// qk_paged_attention.h - attention of new tokens over a paged cache: the kernels,
// compiled a cache type at a time (csrc/qk_paged_attention_*.hip).
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
// With terms (a cap, a bias by distance, a window, a prefix) a score is brought to
// base-2 units of its own as soon as it is a product, and takes them there.
#pragma once

#include "qk_paged.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace qk {

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
    // Terms: scores capped (in base-2 units; 0: not), biased by slopes[head] times the
    // distance, of rows within a window (0: none) and of a prefix of each sequence.
    float cap;
    int window;
    const float *slopes;
    const int32_t *prefix;
};

// The attention launches of each cache type, with terms or without.
int attend_f16(const PagedAttn &a, bool terms, hipStream_t stream);
int attend_i8(const PagedAttn &a, bool terms, hipStream_t stream);
int attend_e4m3(const PagedAttn &a, bool terms, hipStream_t stream);
int attend_i4(const PagedAttn &a, bool terms, hipStream_t stream);

// Rows of a sequence's prefix that there are (a negative one is none).
__device__ __forceinline__ int prefix_rows(const PagedAttn &a, const qk_paged_seq &s) {
    return a.prefix ? max(min(a.prefix[blockIdx.y], s.pos + s.count), 0) : 0;
}
// Where the rows that a windowed sequence's splits divide begin: a multiple of 64
// (a tile's rows lie in whole groups of 16 of a page), no row that a token sees
// before it.
__device__ __forceinline__ int first_row(const PagedAttn &a, const qk_paged_seq &s) {
    return a.window ? max(s.pos - a.window + 1, 0) & ~63 : 0;
}

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;      // cache rows of a tile
constexpr int kRowTile = 16;   // query rows of a workgroup

// A split's partial of one (token, head): the largest score and the sum of weights
// (in base-2 units), padded to 4, then head_dim means.
constexpr int part_floats(int hd) { return 4 + hd; }

// Bytes of n codes, and of the scale that a row has beside them.
constexpr int code_bytes(int type, int n) { return type == QK_TYPE_F16 ? 2 * n : type == QK_TYPE_I4 ? n / 2 : n; }
// Codes that are whole numbers are finite.
constexpr bool whole_codes(int type) { return type == QK_TYPE_I8 || type == QK_TYPE_I4; }

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

// 4-bit codes become code * multiplier in fp16, a whole number of at most 2040: with
// u = code + 8, a nibble of two's complement but for its upper bit, in bits 6 to 9 of
// 0x4C00 it is 16 + u, and (16 + u) m - 24 m is one packed fma, exact (24 m is 8 times
// a number of ten bits).
struct Mult {
    half2v m, off;
    // Of each half, the byte of its dword that sel names.
    __device__ __forceinline__ void set(uint32_t lo, uint32_t hi, uint32_t sel) {
        const half2v bias = {static_cast<_Float16>(1024.f), static_cast<_Float16>(1024.f)};
        const half2v by = {static_cast<_Float16>(-24.f), static_cast<_Float16>(-24.f)};
        m = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(hi, lo, sel) | 0x64006400u) - bias;
        off = m * by;
    }
};
// The selector of byte k of both dwords.
__device__ __forceinline__ uint32_t mult_sel(int k) { return 0x0C040C00u + 0x10001u * k; }
// The constants in registers: a nibble's bits are then cut out and joined with them in
// one instruction, which takes no literals (one in a scalar and one in a vector
// register; they are made anew where the compiler likes).
struct Nibbles {
    uint32_t mask = 0x03C003C0u, base = 0x4E004E00u;
    __device__ __forceinline__ Nibbles() { asm("" : "+s"(mask), "+v"(base)); }
    __device__ __forceinline__ half2v code(uint32_t at6, const Mult &m) const {   // in bits 6 to 9 of each half
        return __builtin_elementwise_fma(__builtin_bit_cast(half2v, (at6 & mask) ^ base), m.m, m.off);
    }
    // Eight codes of one dword: pair k holds values k and k + 4.
    __device__ __forceinline__ half8 eight(uint32_t w, const Mult &m) const {
        const half2v a = code(w << 6, m), b = code(w << 2, m), c = code(w >> 2, m), d = code(w >> 6, m);
        return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
    // Four of two rows each, x and y: pair k their values k.
    __device__ __forceinline__ void four(uint32_t x, uint32_t y, uint32_t sel, const Mult &m, half2v (&p)[4]) const {
        const uint32_t w = __builtin_amdgcn_perm(y, x, sel);
        p[0] = code(w << 6, m), p[1] = code(w << 2, m), p[2] = code(w >> 2, m), p[3] = code(w >> 6, m);
    }
};
// The selector of the lower or upper two bytes of two rows, for four().
__device__ __forceinline__ constexpr uint32_t four_sel(int half) { return half ? 0x07060302u : 0x05040100u; }
// Query values of one step in the order in which its key codes stand.
template <int TYPE>
__device__ __forceinline__ half8 key_order(half2v a, half2v b, half2v c, half2v d) {
    if constexpr (TYPE == QK_TYPE_I4) return half8{a[0], c[0], a[1], c[1], b[0], d[0], b[1], d[1]};
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The bits of four 8-bit codes that make them other than 0 (float8 has a -0).
template <int TYPE>
constexpr uint32_t code_bits = whole_codes(TYPE) ? 0xFFFFFFFFu : 0x7F7F7F7Fu;

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
// 8-bit codes a lane loads 16 bytes that serve two steps, with 4-bit ones a quarter
// of the row, which has one multiplier.
template <int HD, int TYPE>
__device__ __forceinline__ constexpr int key_dim(int s, int g) {
    if (TYPE == QK_TYPE_I4) return g * (HD / 4) + 8 * s;
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
    static constexpr int kB = code_bytes(TYPE, HD / 4);   // bytes a lane holds of a row
    uint4v w[2][(kB + 15) / 16];
    uint32_t mults[2];   // the rows' multipliers (4-bit codes)
    __device__ __forceinline__ void load(int h, const char *row, int g) {
        if constexpr (TYPE == QK_TYPE_I4) {
            #pragma unroll
            for (int j = 0; j < (kB + 15) / 16; ++j)
                __builtin_memcpy(&w[h][j], row + g * kB + j * 16, kB - 16 * j < 16 ? kB - 16 * j : 16);
            return;
        }
        #pragma unroll
        for (int j = 0; j < kB / 16; ++j) __builtin_memcpy(&w[h][j], row + j * 64 + g * 16, 16);
        if constexpr (kB % 16 != 0) __builtin_memcpy(&w[h][kB / 16], row + kB / 16 * 64 + g * 8, 8);
    }
    __device__ __forceinline__ half8 operand(int h, int s, const Mult &m, const Nibbles &codes) const {
        if constexpr (TYPE == QK_TYPE_I4) {
            return codes.eight(w[h][s / 4][s % 4], m);
        } else if constexpr (TYPE == QK_TYPE_F16) {
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
    static constexpr int kB = code_bytes(TYPE, HD / 16);
    static constexpr bool kSplit = HD == 96 && TYPE != QK_TYPE_F16;   // 4 + 2 values
    uint32_t w[8][(kB + 3) / 4];
    __device__ __forceinline__ void load(int j, const char *row, int i) {
        if constexpr (TYPE == QK_TYPE_I4 && kSplit) {
            uint16_t most;
            __builtin_memcpy(&most, row + i * 2, 2);
            w[j][0] = most | static_cast<uint32_t>(static_cast<uint8_t>(row[32 + i])) << 16;
        } else if constexpr (TYPE == QK_TYPE_I4 && kB == 2) {
            uint16_t all;
            __builtin_memcpy(&all, row + i * 2, 2);
            w[j][0] = all;
        } else if constexpr (kSplit) {
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
    // (4-bit codes: from two bytes of each row, times the multipliers of the rows'
    // pairs, of the quarter that holds these dimensions.)
    __device__ __forceinline__ void operands(int d, half8 (&v)[4], const Mult (&m)[4], const Nibbles &codes) const {
        if constexpr (TYPE == QK_TYPE_I4) {
            half2v p[4][4];   // [pair of rows][dimension]
            #pragma unroll
            for (int k = 0; k < 4; ++k) codes.four(w[2 * k][d / 2], w[2 * k + 1][d / 2], four_sel(d & 1), m[k], p[k]);
            #pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = join(p[0][c], p[1][c], p[2][c], p[3][c]);
        } else if constexpr (TYPE == QK_TYPE_F16) {
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

// cap tanh(x / cap) of N scores, inverse 1 / cap.  Where all of a wave are below
// 0.55 of the cap, which is where trained scores lie, by y + y^3 P(y^2), P the
// minimax polynomial of (tanh(y) / y - 1) / y^2 there (its error is below fp32's
// rounding): eight operations instead of two quarter-rate ones and eight.  Why 0.55: the
// quotient (1 - e) / (1 + e) passes the rounding of e on 1 / sinh(2 y) times, less than
// once from y = 0.44 on (five times at 0.1), and the polynomial, fitted to a little more
// than that, has there an error of 4.9e-9 of tanh(y) / y, a twelfth of a rounding.
// (Four at a time: all of a tile's side by side would take the registers of the sums.)
template <int N, typename V>
__device__ __forceinline__ void cap_scores(V &x, float cap, float inverse) {
    constexpr int kBy = N < 4 ? N : 4;
    float top = 0.f;
    #pragma unroll
    for (int r = 0; r < N; ++r) top = fmaxf(top, fabsf(x[r]));
    auto cubic = [](float z) {
        float p = fmaf(-0.00661022774875164f, z, 0.021309388801455498f);
        p = fmaf(p, z, -0.05390942841768265f);
        p = fmaf(p, z, 0.13333113491535187f);
        return fmaf(p, z, -0.3333333134651184f);
    };
    if (__builtin_amdgcn_ballot_w64(top * inverse > 0.55f)) {
        #pragma unroll
        for (int r0 = 0; r0 < N; r0 += kBy) {
            __builtin_amdgcn_sched_barrier(0);
            #pragma unroll
            for (int r = r0; r < r0 + kBy; ++r) {
                const float y = x[r] * inverse, e = __builtin_amdgcn_exp2f(-2.8853900817779268f * fabsf(y));
                const float t = (1.f - e) * __builtin_amdgcn_rcpf(1.f + e), z = y * y;
                x[r] = cap * (fabsf(y) > 0.55f ? copysignf(t, y) : fmaf(cubic(z), z * y, y));
            }
        }
    } else {
        #pragma unroll
        for (int r0 = 0; r0 < N; r0 += kBy) {
            __builtin_amdgcn_sched_barrier(0);
            #pragma unroll
            for (int r = r0; r < r0 + kBy; ++r) {
                const float y = x[r] * inverse, z = y * y;
                x[r] = fmaf(cap * cubic(z), z * y, x[r]);
            }
        }
    }
    __builtin_amdgcn_sched_barrier(0);
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

// A query row as the operands of the scores' product, lane group g's dimensions of
// it: two halves each, times what qscale undoes.
template <int HD, int TYPE, int NS>
__device__ __forceinline__ void load_query(const float *qrow, int g, float scale, half8 (&qh)[NS], half8 (&ql)[NS],
                                           float &qscale) {
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
    query_units(top, scale, factor, qscale);
    #pragma unroll
    for (int st = 0; st < NS; ++st) {
        half2v u[4], w[4];
        #pragma unroll
        for (int k = 0; k < 4; ++k)
            split_pair(factor * v[st][2 * k], factor * v[st][2 * k + 1], u[k], w[k]);
        qh[st] = key_order<TYPE>(u[0], u[1], u[2], u[3]);
        ql[st] = key_order<TYPE>(w[0], w[1], w[2], w[3]);
    }
}

// A workgroup: 16 query rows of one (sequence, KV head) over a split's rows,
// its four waves every fourth tile of 32 rows each; the waves' states meet in
// LDS.  Few query rows leave the cache as the bound, so nothing is staged: a lane
// loads its own share of both operands, the next tile's while this one is
// multiplied.  64 sequences over 1000 to 8000 rows, 8 KV heads of 128 int8 values:
// 611 MB in 126 us, 4.8 TB/s (a copy reaches 4.95, a plain reading 6.15); one over
// 700 rows of 64 fp16 values: 5.5 us, the latency of its loads, and 3.4 of the
// merge.  Two workgroups a CU: left to itself the compiler takes registers beyond
// that (fp16 rows of 128, 4 sequences of 8000: 33 us, with the bound 28).  Heads of 256
// need all of a CU's registers for two tiles and the query; SHARED has the query in LDS,
// read for each tile, and one tile in registers, whose loads a second workgroup hides
// (attend_launch says when).
template <int HD, int TYPE, bool TERMS, bool SHARED>
__global__ __launch_bounds__(256, HD <= 128 || SHARED ? 2 : 1) void paged_attention_kernel(PagedAttn a) {
    constexpr int NS = HD / 32, NC = HD / 16, kRow = code_bytes(TYPE, HD);
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
    const int lane = threadIdx.x & 63;
    int n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // This lane's query row, the last row it sees, and the rows the tile sees.
    // (Past the last row: that one again, masked and not written.)
    const int row = row0 + n, tok = min(row, rows - 1) / G, own = min(row, rows - 1) - tok * G;
    const bool have = row < rows;
    const int mine = have ? s.pos + tok : -1;
    int last = s.pos + __builtin_amdgcn_readlane(tok, 15);   // of the tile's last token
    int seen = s.pos + __builtin_amdgcn_readlane(tok, 0);    // of its first
    // With terms: this query row sees rows low .. up, all of the tile rows hidden .. seen.
    int up = mine, low = 0, hidden = 0;
    int64_t begin64 = static_cast<int64_t>(split) * a.split_rows[0];
    if constexpr (TERMS) {
        const int prefix = prefix_rows(a, s);
        up = have ? max(mine, prefix - 1) : -1;
        low = a.window ? mine - a.window + 1 : 0;
        hidden = a.window ? last - a.window + 1 : 0;
        begin64 += first_row(a, s);
        last = max(last, prefix - 1);
    }
    if (begin64 > last) return;   // the merge takes the splits that reach a token
    int begin = static_cast<int>(begin64);
    const int end = static_cast<int>(min(begin64 + a.split_rows[0], int64_t(last) + 1));
    if constexpr (TERMS) {
        // No tile before the first token's window.
        if (a.window) begin = max(begin, (seen - a.window + 1) & ~(kTile - 1));
        seen = max(seen, prefix_rows(a, s) - 1);
    }

    half8 qh[NS], ql[NS];
    float qscale;
    load_query<HD, TYPE, NS>(a.q + (s.first + tok) * a.ldq + static_cast<int64_t>(h * G + own) * HD, g, a.scale, qh, ql, qscale);
    __shared__ half8 queries[SHARED ? 2 : 1][SHARED ? NS : 1][64];
    if constexpr (SHARED) {
        if (wave == 0)
            #pragma unroll
            for (int x = 0; x < NS; ++x) queries[0][x][lane] = qh[x], queries[1][x][lane] = ql[x];
        __syncthreads();
    }

    float4v o[NC];
    #pragma unroll
    for (int c = 0; c < NC; ++c) o[c] = float4v{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    ValueUnits units;
    const Nibbles codes;
    const float slope = TERMS && a.slopes ? 1.4426950408889634f * a.slopes[h * G + own] : 0.f;
    const float inverse_cap = TERMS && a.cap > 0.f ? 1.f / a.cap : 0.f;

    // (Of the constant address space: looked up by scalar loads, which no wait for a
    // tile's loads includes.)
    typedef const __attribute__((address_space(4))) int32_t *Table;
    const Table table = (Table)(a.b.page_table + static_cast<int64_t>(s.table) * a.b.table_stride);
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
        uint32_t vm[8];   // 4-bit codes: the value rows' multipliers
        bool present[2];
    };
    // Scales (and multipliers) of rows base + 4 g .. + 3.
    auto scales4 = [&](const float *at, int64_t base, int g, float4v &scale, uint32_t *mults) {
        if constexpr (TYPE == QK_TYPE_I4) {
            // (No part of a load unused: its register would be given to something else,
            // which then waits for the load.)
            if (mults) {
                const uint4v *e = reinterpret_cast<const uint4v *>(at + 2 * (base + 4 * g));
                const uint4v lo = e[0], hi = e[1];
                const uint32_t s[4] = {lo[0], lo[2], hi[0], hi[2]};   // (a cast of an element of a vector is one of its first)
                scale = __builtin_bit_cast(float4v, s);
                mults[0] = lo[1], mults[1] = lo[3], mults[2] = hi[1], mults[3] = hi[3];
            } else {
                #pragma unroll
                for (int r = 0; r < 4; ++r) scale[r] = at[2 * (base + 4 * g + r)];
            }
        } else {
            scale = *reinterpret_cast<const float4v *>(at + base + 4 * g);
        }
    };
    auto pages_of = [&](int t0) {
        Pages p;
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const int r = min(t0 + 16 * hf, last);
            const int64_t page = table[r >> a.page_shift];
            p.id[hf] = t0 + 16 * hf <= last && page >= 0 && page < a.kv.pages ? page : -1;
        }
        return p;
    };
    auto load = [&](Tile &t, int t0, const Pages &p, int n, int g) {
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            t.present[hf] = p.id[hf] >= 0;
            const int64_t base = max(p.id[hf], int64_t(0)) * page_stride + head_row + ((t0 + 16 * hf) & (a.kv.page_rows - 1));
            t.k.load(hf, static_cast<const char *>(a.kv.key) + (base + n) * kRow, g);
            #pragma unroll
            for (int j = 0; j < 4; ++j)
                t.v.load(4 * hf + j, static_cast<const char *>(a.kv.value) + (base + 4 * g + j) * kRow, n);
            if constexpr (kScaled) {
                scales4(a.kv.key_scale, base, g, t.ks[hf], nullptr);
                scales4(a.kv.value_scale, base, g, t.vs[hf], t.vm + 4 * hf);
            }
            if constexpr (TYPE == QK_TYPE_I4)
                t.k.mults[hf] = __builtin_bit_cast(uint32_t, a.kv.key_scale[2 * (base + n) + 1]);
        }
    };
    auto take = [&](Tile &t, int t0) {
        float4v st[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        Mult km[2];
        if constexpr (TYPE == QK_TYPE_I4)
            #pragma unroll
            for (int hf = 0; hf < 2; ++hf) km[hf].set(t.k.mults[hf], t.k.mults[hf], mult_sel(g));
        #pragma unroll
        for (int x = 0; x < NS; ++x) {
            const half8 upper = SHARED ? queries[0][SHARED ? x : 0][lane] : qh[x], lower = SHARED ? queries[SHARED ? 1 : 0][SHARED ? x : 0][lane] : ql[x];
            #pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const half8 k = t.k.operand(hf, x, km[hf], codes);
                st[hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, lower, st[hf], 0, 0, 0);
                st[hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, upper, st[hf], 0, 0, 0);
            }
        }
        // Register r of half hf: row t0 + 16 hf + 4 g + r.
        float mx = -INFINITY, vtop = 0.f;
        bool one = false;
        const bool edge = t0 + kTile - 1 > seen || !t.present[0] || !t.present[1] || (TERMS && t0 < hidden);
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
        if constexpr (TERMS) {
            if (a.cap > 0.f) {
                cap_scores<4>(st[0], a.cap, inverse_cap);
                cap_scores<4>(st[1], a.cap, inverse_cap);
            }
            if (a.slopes) {
                const float far = static_cast<float>(mine - t0 - 4 * g);
                #pragma unroll
                for (int hf = 0; hf < 2; ++hf)
                    #pragma unroll
                    for (int r = 0; r < 4; ++r)
                        st[hf][r] = fmaf(-slope, fabsf(far - static_cast<float>(16 * hf + r)), st[hf][r]);
            }
        }
        if (edge) {
            #pragma unroll
            for (int hf = 0; hf < 2; ++hf)
                #pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at = t0 + 16 * hf + 4 * g + r;
                    st[hf][r] = t.present[hf] && at <= up && (!TERMS || at >= low) ? st[hf][r] : -INFINITY;
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
        Mult vm[4];
        #pragma unroll
        for (int d = 0; d < (NC + 3) / 4; ++d) {
            half8 v[4];
            if constexpr (TYPE == QK_TYPE_I4)
                if (d == 0 || HD == 96)   // (of 96 values a lane's first four and last two lie apart)
                    #pragma unroll
                    for (int k = 0; k < 4; ++k)
                        vm[k].set(t.vm[2 * k], t.vm[2 * k + 1], mult_sel(value_dim<HD, TYPE>(n, 4 * d) / (HD / 4)));
            t.v.operands(d, v, vm, codes);
            #pragma unroll
            for (int k = 0; k < 4 && 4 * d + k < NC; ++k) {
                if (!whole_codes(TYPE) && edge) clear_not_finite(v[k], bad);
                float4v &c = o[4 * d + k];
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[k], pl, c, 0, 0, 0);
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[k], ph, c, 0, 0, 0);
            }
        }
        if (!whole_codes(TYPE) && edge && __builtin_amdgcn_ballot_w64(bad != 0)) {
            // The tokens that see such a row: not finite.
            #pragma unroll
            for (int off = 1; off < 16; off <<= 1) bad |= static_cast<uint32_t>(__shfl_xor(static_cast<int>(bad), off));
            #pragma unroll
            for (int hf = 0; hf < 2; ++hf)
                #pragma unroll
                for (int r = 0; r < 4; ++r)
                    if ((bad >> (4 * hf + r) & 1) && t.present[hf] && t0 + 16 * hf + 4 * g + r <= up &&
                        (!TERMS || t0 + 16 * hf + 4 * g + r >= low))
                        l = __builtin_nanf("");
        }
    };
    // Two tiles in registers by turns, one multiplied while the other loads; a tile's
    // pages are looked up before its turn to load comes.  Past the wave's last tile
    // a line of it again, by all lanes: loads that may be left out would have every wait
    // for a tile wait for all that is under way.
    constexpr int kStep = 4 * kTile;
    int t0 = begin + wave * kTile;
    if (t0 < end) {
        const int final = t0 + (end - 1 - t0) / kStep * kStep;
        if constexpr (SHARED) {
            Pages ahead = pages_of(t0);
            for (; t0 < end; t0 += kStep) {
                Tile tile;
                load(tile, t0, ahead, n, g);
                ahead = pages_of(min(t0 + kStep, final));
                take(tile, t0);
            }
        } else if (t0 == final) {
            // One tile, as of short splits: nothing is loaded beside it (8 sequences of 700
            // rows, 8 KV heads of 128 fp16 values, 11.0 us, with a second tile's loads 12.8).
            // What follows from the lane's numbers is computed for it alone: shared with the
            // loop's it spills (64 sequences of 3000 rows 154 us, 138 without).
            asm volatile("" : "+v"(n), "+v"(g));
            Tile tile;
            load(tile, t0, pages_of(t0), n, g);
            take(tile, t0);
        } else {
            Tile tiles[2];
            load(tiles[0], t0, pages_of(t0), n, g);
            Pages ahead = pages_of(min(t0 + kStep, final));
            for (bool more = true; more;) {
                #pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int keep = t0 == final ? 0 : 63;
                    load(tiles[i ^ 1], min(t0 + kStep, final), ahead, n & keep, g & keep);
                    asm volatile("" ::: "memory");   // or they would sink to where the tile is known to be needed
                    ahead = pages_of(min(t0 + 2 * kStep, final));
                    take(tiles[i], t0);
                    if ((t0 += kStep) >= end) {
                        more = false;
                        break;
                    }
                }
            }
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

// ---------------------------------------------------------- few rows --
//
// Sequences of at most 16 / DUP query rows a KV head (single tokens, mostly): each
// query row stands in DUP neighbouring columns of the scores' product, so a lane of
// them need take no more than 4 / DUP of each four scores through the softmax, and
// the lanes share what the 16-row kernel does DUP times over.  Of the second
// product's columns the first of a query row's holds the weights' upper halves, the
// second the lower ones, added at the end: one matrix instruction for two.  Rows
// pair as 4 g + k of a tile's two halves, so that a lane's weights are whole pairs.
// 64 sequences over 1000 to 8000 4-bit rows, 8 KV heads of 128: 332 MB in 90 us, the
// vector instructions 55 % of the issue slots (404 a tile; the 16-row kernel's 640
// take 114 us); its loads alone take 75.
// Lanes of four: the value of lane `from` of each.
template <int A, int B, int C, int D>
__device__ __forceinline__ uint32_t quad(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), A | B << 2 | C << 4 | D << 6, 0xF, 0xF, true));
}
template <int A, int B, int C, int D>
__device__ __forceinline__ float quad(float v) {
    return __builtin_bit_cast(float, quad<A, B, C, D>(__builtin_bit_cast(uint32_t, v)));
}
// Joined over the DUP lanes of a query row and the four groups of 16 lanes.
template <int DUP, typename Op>
__device__ __forceinline__ float join_row(float v, Op op) {
    v = op(v, quad<1, 0, 3, 2>(v));
    if constexpr (DUP == 4) v = op(v, quad<2, 3, 0, 1>(v));
    uint32_t bits = __builtin_bit_cast(uint32_t, v);
    const auto rows = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
    const uint32_t even = rows[0], odd = rows[1];
    v = op(__builtin_bit_cast(float, even), __builtin_bit_cast(float, odd));
    bits = __builtin_bit_cast(uint32_t, v);
    const auto halves = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    const uint32_t low = halves[0], high = halves[1];
    return op(__builtin_bit_cast(float, low), __builtin_bit_cast(float, high));
}

template <int HD, int TYPE, bool TERMS, int DUP>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void paged_decode_kernel(PagedAttn a) {
    constexpr int NS = HD / 32, NC = HD / 16, kRow = code_bytes(TYPE, HD), kRows = 16 / DUP, kOwn = 4 / DUP;
    static_assert(TYPE != QK_TYPE_F16, "rows have scales");
    __shared__ float meet[3][kRows * (HD + 4)];
    __shared__ half8 queries[2][NS][64];
    const qk_paged_seq s = a.b.seqs[blockIdx.y];
    if (!paged_seq_ok(s, a.b, a.page_shift)) return;
    const int kvh = a.kv.kv_heads, G = a.group;
    // A chip's XCDs take workgroups in turn: the splits rotate, or the first ones
    // (which every sequence has) would all fall to the same XCDs.
    const int splits = a.splits[0], h = blockIdx.x / splits, split = (blockIdx.x + h + blockIdx.y) % splits;
    const int rows = s.count * G;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, part = n % DUP;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // This lane's query row (past the last: that one again, masked and not written),
    // the cache rows low .. up that it sees, those that all of them do, hidden .. seen.
    const int row = n / DUP, tok = min(row, rows - 1) / G, own = min(row, rows - 1) - tok * G;
    const bool have = row < rows;
    const int mine = have ? s.pos + tok : -1;
    int last = s.pos + s.count - 1, seen = s.pos, up = mine, low = 0, hidden = 0;
    int64_t begin64 = static_cast<int64_t>(split) * a.split_rows[0];
    if constexpr (TERMS) {
        const int prefix = prefix_rows(a, s);
        up = have ? max(mine, prefix - 1) : -1;
        low = a.window ? mine - a.window + 1 : 0;
        hidden = a.window ? last - a.window + 1 : 0;
        begin64 += first_row(a, s);
        last = max(last, prefix - 1);
        seen = max(seen, prefix - 1);
    }
    if (begin64 > last) return;   // the merge takes the splits that reach a token
    int begin = static_cast<int>(begin64);
    const int end = static_cast<int>(min(begin64 + a.split_rows[0], int64_t(last) + 1));
    if constexpr (TERMS)
        if (a.window) begin = max(begin, (s.pos - a.window + 1) & ~(kTile - 1));   // no tile before the first token's window

    // The queries in LDS, read for each tile (the same for all four waves): 8 NS
    // registers fewer.
    float qscale;
    {
        half8 qh[NS], ql[NS];
        load_query<HD, TYPE, NS>(a.q + (s.first + tok) * a.ldq + static_cast<int64_t>(h * G + own) * HD, g, a.scale, qh, ql, qscale);
        if (wave == 0)
            #pragma unroll
            for (int x = 0; x < NS; ++x) queries[0][x][lane] = qh[x], queries[1][x][lane] = ql[x];
        __syncthreads();
    }

    float4v o[NC];
    #pragma unroll
    for (int c = 0; c < NC; ++c) o[c] = float4v{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    ValueUnits units;
    const Nibbles codes;
    const float slope = TERMS && a.slopes ? 1.4426950408889634f * a.slopes[h * G + own] : 0.f;
    const float inverse_cap = TERMS && a.cap > 0.f ? 1.f / a.cap : 0.f;

    // (Of the constant address space: looked up by scalar loads, which no wait for a
    // tile's loads includes.)
    typedef const __attribute__((address_space(4))) int32_t *Table;
    const Table table = (Table)(a.b.page_table + static_cast<int64_t>(s.table) * a.b.table_stride);
    const int64_t page_stride = static_cast<int64_t>(kvh) * a.kv.page_rows, head_row = static_cast<int64_t>(h) * a.kv.page_rows;
    struct Pages {
        int64_t id[2];
    };
    struct Tile {
        KeyTile<HD, TYPE> k;
        ValueTile<HD, TYPE> v;   // slot 2 k + hf: row 4 g + k of half hf
        float ks[2][kOwn], vs[2][kOwn];   // of rows 4 g + part * kOwn ..
        uint4v entry[2][2];               // 4-bit codes: scales and multipliers of value rows 4 g .. + 3
        bool present[2];
    };
    auto pages_of = [&](int t0) {
        Pages p;
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const int r = min(t0 + 16 * hf, last);
            const int64_t page = table[r >> a.page_shift];
            p.id[hf] = t0 + 16 * hf <= last && page >= 0 && page < a.kv.pages ? page : -1;
        }
        return p;
    };
    auto load = [&](Tile &t, int t0, const Pages &p) {
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            t.present[hf] = p.id[hf] >= 0;
            const int64_t base = max(p.id[hf], int64_t(0)) * page_stride + head_row + ((t0 + 16 * hf) & (a.kv.page_rows - 1));
            t.k.load(hf, static_cast<const char *>(a.kv.key) + base * kRow + n * kRow, g);
            #pragma unroll
            for (int k = 0; k < 4; ++k)
                t.v.load(2 * k + hf, static_cast<const char *>(a.kv.value) + base * kRow + (4 * g + k) * kRow, n);
            constexpr int kEntry = TYPE == QK_TYPE_I4 ? 2 : 1;
            #pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                t.ks[hf][i] = (a.kv.key_scale + base * kEntry)[(4 * g + part * kOwn + i) * kEntry];
                if constexpr (TYPE != QK_TYPE_I4) t.vs[hf][i] = (a.kv.value_scale + base)[4 * g + part * kOwn + i];
            }
            if constexpr (TYPE == QK_TYPE_I4) {
                t.k.mults[hf] = __builtin_bit_cast(uint32_t, (a.kv.key_scale + base * 2)[2 * n + 1]);
                // (Whole entries, and all of them used: a register of a load that is not
                // would be given to something else, which then waits for the load.)
                const uint4v *e = reinterpret_cast<const uint4v *>(a.kv.value_scale + base * 2) + 2 * g;
                t.entry[hf][0] = e[0];
                t.entry[hf][1] = e[1];
            }
        }
    };
    // Of four values of rows 4 g + 0 .. 3 this lane's.
    auto pick = [&](float r0, float r1, float r2, float r3, float *x) {
        if constexpr (DUP == 4) {
            const float even = part & 2 ? r2 : r0, odd = part & 2 ? r3 : r1;
            x[0] = part & 1 ? odd : even;
        } else {
            x[0] = part ? r2 : r0;
            x[1] = part ? r3 : r1;
        }
    };
    auto take = [&](Tile &t, int t0) {
        if constexpr (TYPE == QK_TYPE_I4)
            #pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const uint32_t s[4] = {t.entry[hf][0][0], t.entry[hf][0][2], t.entry[hf][1][0], t.entry[hf][1][2]};
                const float4v scale = __builtin_bit_cast(float4v, s);
                pick(scale[0], scale[1], scale[2], scale[3], t.vs[hf]);
            }
        float4v st[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        Mult km[2];
        if constexpr (TYPE == QK_TYPE_I4)
            #pragma unroll
            for (int hf = 0; hf < 2; ++hf) km[hf].set(t.k.mults[hf], t.k.mults[hf], mult_sel(g));
        #pragma unroll
        for (int x = 0; x < NS; ++x) {
            const half8 qh = queries[0][x][lane], ql = queries[1][x][lane];
            #pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const half8 k = t.k.operand(hf, x, km[hf], codes);
                st[hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql, st[hf], 0, 0, 0);
                st[hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh, st[hf], 0, 0, 0);
            }
        }
        // Of rows t0 + 16 hf + 4 g + 0 .. 3 this lane's: x[kOwn hf + i] of row part * kOwn + i.
        float x[2 * kOwn];
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf) pick(st[hf][0], st[hf][1], st[hf][2], st[hf][3], x + hf * kOwn);
        const bool edge = t0 + kTile - 1 > seen || !t.present[0] || !t.present[1] || (TERMS && t0 < hidden);
        #pragma unroll
        for (int i = 0; i < 2 * kOwn; ++i) {
            // An infinite key's score: not a number, whatever its sign.
            x[i] *= qscale;
            x[i] *= fmaf(t.ks[i / kOwn][i % kOwn], 0.f, t.ks[i / kOwn][i % kOwn]);
        }
        const int first = t0 + 4 * g + part * kOwn;   // the row of x[0]
        if constexpr (TERMS) {
            if (a.cap > 0.f) cap_scores<2 * kOwn>(x, a.cap, inverse_cap);
            if (a.slopes) {
                const float far = static_cast<float>(mine - first);
                #pragma unroll
                for (int i = 0; i < 2 * kOwn; ++i)
                    x[i] = fmaf(-slope, fabsf(far - static_cast<float>(i / kOwn * 16 + i % kOwn)), x[i]);
            }
        }
        if (edge) {
            #pragma unroll
            for (int i = 0; i < 2 * kOwn; ++i) {
                const int at = first + i / kOwn * 16 + i % kOwn;
                x[i] = t.present[i / kOwn] && at <= up && (!TERMS || at >= low) ? x[i] : -INFINITY;
            }
        }
        // A larger maximum, or a product beyond the units, is met in few tiles: lanes look
        // at their own rows, and join what they have only then.
        auto larger = [](float a, float b) { return fmaxf(a, b); };
        float mx = x[0], vtop = 0.f, f = 1.f;
        #pragma unroll
        for (int i = 1; i < 2 * kOwn; ++i) mx = fmaxf(mx, x[i]);
        const bool more = __builtin_amdgcn_ballot_w64(mx > m);
        if (more) {
            const float mn = fmaxf(m, join_row<DUP>(mx, larger));
            f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            l *= f;
            m = mn;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        #pragma unroll
        for (int i = 0; i < 2 * kOwn; ++i) {
            const float w = __builtin_amdgcn_exp2f(x[i] - ref);
            l += w;
            x[i] = x[i] == -INFINITY ? 0.f : w * t.vs[i / kOwn][i % kOwn];   // a masked row's scale may be anything
            vtop = fmaxf(vtop, fabsf(t.vs[i / kOwn][i % kOwn]));
        }
        if (more || __builtin_amdgcn_ballot_w64(m != -INFINITY && !units.holds(vtop))) {
            bool one = false;
            #pragma unroll
            for (int i = 0; i < 2 * kOwn; ++i) one = one || t.vs[i / kOwn][i % kOwn] == 1.f;
            auto largest = [&] {
                float y = 0.f;
                #pragma unroll
                for (int i = 0; i < 2 * kOwn; ++i) y = fmaxf(y, fabsf(x[i]));
                return join_row<DUP>(y, larger);
            };
            float y = largest();
            units.known *= f;
            if (__builtin_amdgcn_ballot_w64(one || units.strange(y))) {
                const uint32_t live = t.v.live();
                #pragma unroll
                for (int i = 0; i < 2 * kOwn; ++i)   // (a scale that is not finite stays)
                    if (!(live >> (2 * (part * kOwn + i % kOwn) + i / kOwn) & 1) && fabsf(x[i]) < INFINITY) x[i] = 0.f;
                y = largest();
            }
            const float fo = units.renew(y, join_row<DUP>(vtop, larger), f);
            #pragma unroll
            for (int c = 0; c < NC; ++c)
                #pragma unroll
                for (int r = 0; r < 4; ++r) o[c][r] *= fo;
        }
        // Pairs of this lane, then of all four rows: upper halves in a query row's
        // first column, lower ones in its others.
        uint4v p;
        {
            const float k = units.factor;
            uint32_t hi[kOwn], lo[kOwn];
            #pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                half2v ph, pl;
                split_pair(x[i] * k, x[kOwn + i] * k, ph, pl);
                hi[i] = __builtin_bit_cast(uint32_t, ph);
                lo[i] = __builtin_bit_cast(uint32_t, pl);
            }
            // (Both sides of a choice are taken before it: lanes have to be active to be read.)
            auto choose = [&](uint32_t up, uint32_t down) { return part == 0 ? up : down; };
            if constexpr (DUP == 4) {
                p[0] = choose(quad<0, 0, 0, 0>(hi[0]), quad<0, 0, 0, 0>(lo[0]));
                p[1] = choose(quad<1, 1, 1, 1>(hi[0]), quad<1, 1, 1, 1>(lo[0]));
                p[2] = choose(quad<2, 2, 2, 2>(hi[0]), quad<2, 2, 2, 2>(lo[0]));
                p[3] = choose(quad<3, 3, 3, 3>(hi[0]), quad<3, 3, 3, 3>(lo[0]));
            } else {
                p[0] = choose(quad<0, 0, 2, 2>(hi[0]), quad<0, 0, 2, 2>(lo[0]));
                p[1] = choose(quad<0, 0, 2, 2>(hi[1]), quad<0, 0, 2, 2>(lo[1]));
                p[2] = choose(quad<1, 1, 3, 3>(hi[0]), quad<1, 1, 3, 3>(lo[0]));
                p[3] = choose(quad<1, 1, 3, 3>(hi[1]), quad<1, 1, 3, 3>(lo[1]));
            }
        }
        const half8 weights = __builtin_bit_cast(half8, p);
        // A row that some token does not see meets it as 0 * value.
        uint32_t bad = 0;
        Mult vm[4];
        #pragma unroll
        for (int d = 0; d < (NC + 3) / 4; ++d) {
            half8 v[4];
            if constexpr (TYPE == QK_TYPE_I4)
                if (d == 0 || HD == 96)   // (of 96 values a lane's first four and last two lie apart)
                    #pragma unroll
                    for (int k = 0; k < 4; ++k)
                        vm[k].set(t.entry[0][k / 2][k % 2 * 2 + 1], t.entry[1][k / 2][k % 2 * 2 + 1],
                                  mult_sel(value_dim<HD, TYPE>(n, 4 * d) / (HD / 4)));
            t.v.operands(d, v, vm, codes);
            #pragma unroll
            for (int k = 0; k < 4 && 4 * d + k < NC; ++k) {
                if (!whole_codes(TYPE) && edge) clear_not_finite(v[k], bad);
                o[4 * d + k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[k], weights, o[4 * d + k], 0, 0, 0);
            }
        }
        if (!whole_codes(TYPE) && edge && __builtin_amdgcn_ballot_w64(bad != 0)) {
            // The tokens that see such a row: not finite.
            #pragma unroll
            for (int off = 1; off < 16; off <<= 1) bad |= static_cast<uint32_t>(__shfl_xor(static_cast<int>(bad), off));
            #pragma unroll
            for (int hf = 0; hf < 2; ++hf)
                #pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at = t0 + 16 * hf + 4 * g + r;
                    if ((bad >> (2 * r + hf) & 1) && t.present[hf] && at <= up && (!TERMS || at >= low)) l = __builtin_nanf("");
                }
        }
    };
    // Tiles in registers by turns, one multiplied while the others load; a tile's
    // pages are looked up before its turn to load comes.  Past the wave's last tile
    // that one again: loads that may be left out would have every wait for a tile wait
    // for all that is under way.
    constexpr int kStep = 4 * kTile;
    int t0 = begin + wave * kTile;
    if (t0 < end) {
        const int final = t0 + (end - 1 - t0) / kStep * kStep;
        Tile tiles[2];
        load(tiles[0], t0, pages_of(t0));
        Pages ahead = pages_of(min(t0 + kStep, final));
        for (bool more = true; more;) {
            #pragma unroll
            for (int i = 0; i < 2; ++i) {
                load(tiles[i ^ 1], min(t0 + kStep, final), ahead);
                asm volatile("" ::: "memory");   // or they would sink to where the tile is known to be needed
                ahead = pages_of(min(t0 + 2 * kStep, final));
                take(tiles[i], t0);
                if ((t0 += kStep) >= end) {
                    more = false;
                    break;
                }
            }
        }
    }
    l = join_row<DUP>(l, [](float a, float b) { return a + b; });
    // The waves' means (sums could pass fp32's range), then into wave 0, in wave order.
    auto share_of = [](float l) { return l == 0.f ? 0.f : 1.f / l; };   // no row seen: zeros
    const int back = units.exponent() - 15;
    const float inverse = share_of(l);
    #pragma unroll
    for (int c = 0; c < NC; ++c)
        #pragma unroll
        for (int r = 0; r < 4; ++r) o[c][r] = ldexpf((o[c][r] + quad<1, 0, 3, 2>(o[c][r])) * inverse, back);
    // Of a query row's lanes the first has all of its dimensions 4 g + r of 16.
    if (wave > 0 && part == 0) {
        float *mineat = meet[wave - 1] + row * (HD + 4);
        #pragma unroll
        for (int c = 0; c < NC; ++c) *reinterpret_cast<float4v *>(mineat + (c * 4 + g) * 4) = o[c];
        if (g == 0) {
            mineat[HD] = m;
            mineat[HD + 1] = l;
        }
    }
    __syncthreads();
    if (wave > 0 || part != 0 || !have) return;
    float mw[4] = {m}, lw[4] = {l};
    #pragma unroll
    for (int w = 0; w < 3; ++w) {
        mw[w + 1] = meet[w][row * (HD + 4) + HD];
        lw[w + 1] = meet[w][row * (HD + 4) + HD + 1];
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
            const float4v po = *reinterpret_cast<const float4v *>(meet[w] + row * (HD + 4) + (c * 4 + g) * 4);
            #pragma unroll
            for (int r = 0; r < 4; ++r) o[c][r] = fmaf(po[r], f, o[c][r]);
        }
    }
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
// The 16-row kernel took 1150 us.  Of 4-bit rows 659 us, three instructions a pair of
// codes where float8 takes one.  Short chunks are bound by the latency of a
// workgroup's steps: 517 tokens over 600, 24 heads, 31 us and 7.5 of the merge,
// where the matrix instructions are 10.  Two workgroups a CU; of 64 fp16 values three,
// for which the compiler has to be asked (8 sequences of 300 tokens over 1000, 32 heads:
// 89 us, of two 102).
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
    static constexpr int kWidth = HD == 96 ? 128 : HD;

    // A thread's share of a tile: 16 bytes of kKeys key rows, kValCols values of
    // four rows (of 96 dimensions as of 128, a quarter of the threads idle, so that
    // a wave's rows lie within 16 of one page).
    // (4-bit codes: a quarter of a key row, of one multiplier.)
    static constexpr int kKeyCols = TYPE == QK_TYPE_F16 ? 8 : TYPE == QK_TYPE_I4 ? HD / 4 : 16;
    static constexpr int kKeyLine = TYPE == QK_TYPE_I4 ? 4 : kWidth / kKeyCols, kKeys = kChunkTile * kKeyLine / 256;
    static constexpr int kKeyRegs = TYPE == QK_TYPE_I4 ? (code_bytes(TYPE, kKeyCols) + 15) / 16 : kKeys;
    static constexpr int kValCols = kWidth / 16, kValBytes = code_bytes(TYPE, kValCols);
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
        int big;                                // ks are times 2^-24: there is one above 2^96 (4-bit codes: 2^94)
        int pad[3];
    };
    static_assert(sizeof(Head) % 16 == 0, "the second buffer's 16-byte reads");
    static constexpr int kBuffer = kKeyBytes + kValueBytes + sizeof(Head);

    // Of col + d, col a multiple of kValCols and d below it: that of col xor that of d.
    static __device__ __forceinline__ int exchange(int d) { return (d ^ (d >> 3)) & 7; }
};

typedef float float16v __attribute__((ext_vector_type(16)));

template <int HD, int TYPE, bool TERMS>
__global__ __launch_bounds__(256, HD > 128 ? 1 : HD == 64 && TYPE == QK_TYPE_F16 && !TERMS ? 3 : 2) void paged_chunk_kernel(PagedAttn a) {
    using C = Chunk<HD, TYPE>;
    constexpr int NS = HD / 16, ND = HD / 32, kRow = code_bytes(TYPE, HD);
    constexpr bool kScaled = TYPE != QK_TYPE_F16;
    // Scores in base-2 units of rows without scales: the maximum that weights are taken
    // from follows only when it has grown by 2^kSlack, so the sums are seldom rescaled
    // (of 32 query rows some one's maximum grows in most tiles); weights are below
    // 2^kSlack then and their halves in units of 2^(kSlack - 15).
    constexpr float kSlack = TERMS && !kScaled ? 8.f : 0.f, kUnit = TERMS && !kScaled ? 0x1p7f : 0x1p15f;
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
    int last = s.pos + min(row0 + kChunkRows - 1, rows - 1) / G, seen = s.pos + row0 / G;
    int64_t begin64 = static_cast<int64_t>(split) * a.split_rows[1];
    const int prefix = TERMS ? prefix_rows(a, s) : 0;
    int hidden = 0;   // with a window: the first row that all query rows see, of those before seen
    if constexpr (TERMS) {
        begin64 += first_row(a, s);
        hidden = a.window ? last - a.window + 1 : 0;
        last = max(last, prefix - 1);
    }
    if (begin64 > last) return;
    int begin = static_cast<int>(begin64);
    const int end = static_cast<int>(min(begin64 + a.split_rows[1], int64_t(last) + 1));
    if constexpr (TERMS) {
        // No tile before the first token's window.
        if (a.window) begin = max(begin, (seen - a.window + 1) & ~(kChunkTile - 1));
        seen = max(seen, prefix - 1);
    }
    // Whether some token does not see all of a tile that there is.
    auto cut = [&](int t0) { return t0 + kChunkTile - 1 > seen || (TERMS && t0 < hidden); };

    // Of a row past the last one: that one again, masked and not written.
    const int wrow = row0 + 32 * wave, row = wrow + n, tok = min(row, rows - 1) / G, own = min(row, rows - 1) - tok * G;
    const bool have = row < rows;
    const int mine = have ? s.pos + tok : -1;
    int wave_seen = s.pos + __builtin_amdgcn_readlane(tok, 0);
    int wave_last = wrow < rows ? s.pos + __builtin_amdgcn_readlane(tok, 31) : -1;
    // With terms: this query row sees rows low .. up, all of the wave's rows wave_hidden
    // .. wave_seen, none of them any before wave_first.
    int up = mine, low = 0, wave_hidden = 0, wave_first = 0;
    if constexpr (TERMS) {
        up = have ? max(mine, prefix - 1) : -1;
        low = a.window ? max(mine - a.window + 1, 0) : 0;   // (a tile's row is taken off it below)
        wave_hidden = a.window ? wave_last - a.window + 1 : 0;
        wave_first = a.window ? wave_seen - a.window + 1 : 0;
        wave_seen = max(wave_seen, prefix - 1);
        wave_last = wrow < rows ? max(wave_last, prefix - 1) : -1;
    }
    const float slope = TERMS && a.slopes ? 1.4426950408889634f * a.slopes[h * G + own] : 0.f;
    const float inverse_cap = TERMS && a.cap > 0.f ? 1.f / a.cap : 0.f;

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
        uint4v key[C::kKeyRegs];
        uint32_t value[4][(C::kValBytes + 3) / 4];
        uint32_t key_mults, value_mults[4];   // 4-bit codes
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
        const int quad = tid / 16, col = min(tid % 16 * C::kValCols, HD - C::kValCols);
        if constexpr (TYPE == QK_TYPE_I4) {
            constexpr int kB = code_bytes(TYPE, C::kKeyCols);
            const int64_t first = row_of(wave);
            const char *keys = static_cast<const char *>(a.kv.key) + first * kRow + (tid / 4 & 15) * kRow + tid % 4 * kB;
            #pragma unroll
            for (int i = 0; i < C::kKeyRegs; ++i)
                __builtin_memcpy(&g.key[i], keys + 16 * i, kB - 16 * i < 16 ? kB - 16 * i : 16);
            g.key_mults = __builtin_bit_cast(uint32_t, a.kv.key_scale[2 * (first + (tid / 4 & 15)) + 1]);
            const float *entries = a.kv.value_scale + 2 * (first + 4 * (quad & 3));
            #pragma unroll
            for (int r = 0; r < 4; ++r) g.value_mults[r] = __builtin_bit_cast(uint32_t, entries[2 * r + 1]);
        } else {
            #pragma unroll
            for (int i = 0; i < C::kKeys; ++i) {
                const int row = tid / C::kKeyLine + i * (256 / C::kKeyLine), col = min(tid % C::kKeyLine * C::kKeyCols, HD - C::kKeyCols);
                const char *base = static_cast<const char *>(a.kv.key) +
                                   row_of((64 * wave / C::kKeyLine + i * (256 / C::kKeyLine)) / 16) * kRow;
                g.key[i] = *reinterpret_cast<const uint4v *>(base + (row & 15) * kRow + code_bytes(TYPE, col));
            }
        }
        const char *base = static_cast<const char *>(a.kv.value) + row_of(wave) * kRow;
        #pragma unroll
        for (int r = 0; r < 4; ++r) {
            const char *at = base + (4 * (quad & 3) + r) * kRow + code_bytes(TYPE, col);
            if constexpr (C::kValBytes == 2) {
                uint16_t all;
                __builtin_memcpy(&all, at, 2);
                g.value[r][0] = all;
            } else {
                __builtin_memcpy(g.value[r], at, C::kValBytes);
            }
        }
        if constexpr (kScaled)
            if (wave < 2)
                g.scale = (wave == 0 ? a.kv.value_scale : a.kv.key_scale)
                    [(page * page_stride + head_row + (group & mask) + (tid & 15)) * (TYPE == QK_TYPE_I4 ? 2 : 1)];
    };
    int top_ev = kLeastExponent, low_ev = INT32_MAX;   // wave 0's: exponents of the value scales so far
    const Nibbles codes;
    auto store = [&](const Stage &g, int t0, char *buf) {
        auto &head = *reinterpret_cast<typename C::Head *>(buf + C::kKeyBytes + C::kValueBytes);
        const bool edge = cut(t0);
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
                // Products without it are 2^31 at most (2^14 by 448 by 256 dimensions; of
                // 4-bit codes 2^33), with it 2^14 by 2^128 by 256: 2^126 in the units of
                // such tiles.
                const bool big = __builtin_amdgcn_ballot_w64(fabsf(g.scale) > (TYPE == QK_TYPE_I4 ? 0x1p94f : 0x1p96f));
                const float v = big ? g.scale * 0x1p-24f : g.scale;
                head.ks[lane] = fmaf(v, 0.f, v);   // infinite: all its scores are not numbers
                if (lane == 0) head.big = big;
            }
        }
        if constexpr (TYPE == QK_TYPE_I4) {
            char *at = buf + tid / 4 * C::kKeyStride + tid % 4 * C::kKeyCols * 2;
            Mult m;
            m.set(g.key_mults, g.key_mults, mult_sel(tid % 4));
            #pragma unroll
            for (int w = 0; w < C::kKeyCols / 8; ++w)
                *reinterpret_cast<half8 *>(at + 16 * w) = codes.eight(g.key[w / 4][w % 4], m);
        }
        #pragma unroll
        for (int i = 0; i < (TYPE == QK_TYPE_I4 ? 0 : C::kKeys); ++i) {
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
        Mult vm[2];
        if constexpr (TYPE == QK_TYPE_I4)   // (a thread's dimensions are of one quarter)
            #pragma unroll
            for (int k = 0; k < 2; ++k) vm[k].set(g.value_mults[2 * k], g.value_mults[2 * k + 1], mult_sel(col / (HD / 4)));
        #pragma unroll
        for (int d4 = 0; d4 < C::kValCols / 4; ++d4) {
            half2v p[4][2];
            if constexpr (TYPE == QK_TYPE_I4) {
                #pragma unroll
                for (int k = 0; k < 2; ++k) {
                    half2v four[4];
                    codes.four(g.value[2 * k][d4 / 2], g.value[2 * k + 1][d4 / 2], four_sel(d4 & 1), vm[k], four);
                    #pragma unroll
                    for (int c = 0; c < 4; ++c) p[c][k] = four[c];
                }
            } else if constexpr (TYPE == QK_TYPE_F16) {
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
        if (!whole_codes(TYPE) && (edge || gone)) {
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
            qh[x] = key_order<TYPE>(u[0], u[1], u[2], u[3]);
            ql[x] = key_order<TYPE>(w[0], w[1], w[2], w[3]);
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
        // Of the scores as they are then: with terms they come to base-2 units at once.
        const float by = TERMS ? 1.f : unit;
        const bool renew = big && !TERMS;
        const bool edge = t0 + kChunkTile - 1 > wave_seen || absent || (TERMS && t0 < wave_hidden);   // some token does not see it whole
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
        // (With terms there are too few registers for that.)
        float16v st, ahead;
        scores(0, st);
        #pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            if (TERMS && hf == 1) scores(1, st);
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
            if constexpr (TERMS) {
                #pragma unroll
                for (int r = 0; r < 16; ++r) st[r] *= unit;
                if (a.cap > 0.f) cap_scores<16>(st, a.cap, inverse_cap);
                if (a.slopes) {
                    const float far = static_cast<float>(mine - t0 - 32 * hf - 4 * hi);
                    #pragma unroll
                    for (int r = 0; r < 16; ++r)
                        st[r] = fmaf(-slope, fabsf(far - static_cast<float>(8 * (r / 4) + r % 4)), st[r]);
                }
            }
            if (edge) {
                const uint32_t two = absent >> (2 * hf), hide = ((two & 1 ? 0xFFFFu : 0) | (two & 2 ? 0xFFFF0000u : 0)) >> (4 * hi);
                const int left = up - t0 - 32 * hf - 4 * hi, from = low - t0 - 32 * hf - 4 * hi;
                #pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int at = 8 * (r / 4) + r % 4;
                    st[r] = at <= left && (!TERMS || at >= from) && !(hide >> at & 1) ? st[r] : -INFINITY;
                }
            }
            float mn = renew ? -INFINITY : m;
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
            if (en != ev || renew || __builtin_amdgcn_ballot_w64(mn > (kSlack > 0.f ? m + kSlack : m) || (room && c != INFINITY && lift > static_cast<float>(room)))) {
                // c is what the weights so far were taken with, rounding and all.
                const float cn = kScaled ? fminf(c, -mn * by) : mn == -INFINITY ? INFINITY : -mn * (TERMS ? 1.f : qscale);
                const float f = cn == INFINITY ? 1.f : __builtin_amdgcn_exp2f(cn - c);
                l *= f;
                float fo = kScaled ? ldexpf(f, ev - en) : f;
                m = renew ? -INFINITY : mn;
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
                        known = fmaxf(known, zeros ? 0.f : fabsf(__builtin_amdgcn_exp2f(fmaf(st[r], by, (c == INFINITY ? 0.f : c) + lift)) * vs));
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
            if (cut(t0)) {   // flagged for all waves, those that see the whole tile too
                const uint32_t bad = head.bad[hf] >> (4 * hi);
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(bad != 0) != 0, 0)) {
                    #pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if ((bad >> (8 * (r / 4) + r % 4) & 1) && st[r] != -INFINITY) l = __builtin_nanf("");
                }
            }
            if (!TERMS && hf == 0) scores(1, ahead);
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
                        const float w = __builtin_amdgcn_exp2f(fmaf(x, by, ref));
                        l += w;
                        y[r] = w * (kScaled ? vs[r] : kUnit);
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
            if constexpr (!TERMS) st = ahead;
        }
    };

    Stage g;
    load(g, begin, pages_of(begin));
    int32_t ahead = pages_of(begin + kChunkTile);
    int b = 0;
    for (int t0 = begin; t0 < end; t0 += kChunkTile, b ^= 1) {
        char *buf = lds + b * C::kBuffer;
        asm volatile("" : "+v"(tid));
        if (cut(t0)) {   // flags that all waves may set
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
        if (t0 <= wave_last && (!TERMS || t0 + kChunkTile > wave_first)) take(buf, t0, absent);
    }
    l += __shfl_xor(l, 32);
    if (!have) return;
    const int head = h * G + own;
    const int back = kScaled ? ev - 15 : TERMS ? -7 : -15;
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

template <int HD, int TYPE, bool TERMS>
int attend_launch(const PagedAttn &a, hipStream_t stream) {
    const int64_t rows = static_cast<int64_t>(a.b.max_count) * (a.heads / a.kv.kv_heads);
    auto grid = [&](int64_t n, int tile, int splits) {
        return dim3(static_cast<unsigned>((n + tile - 1) / tile * a.kv.kv_heads * splits), a.b.n_seqs);
    };
    // Few rows: 64 sequences over 1000 to 8000 4-bit rows, eight KV heads of 128, in us,
    // against the 16-row kernel: 4 query rows 95 and 114, 8 105 and 111; 16 sequences over
    // 4000 of 256, 2 query rows 42 and 49.  With terms, 32 sequences of int8 over windows
    // of 4096: 53 and 57; of 1000: 22.9 and 23.5; float8, 8 query rows over 3000: 42.7 and
    // 43.1.  Of fp16 rows the loads alone take the time (32 sequences over 3000 86 and 80).
    if constexpr (TYPE == QK_TYPE_I4 || (TERMS && TYPE != QK_TYPE_F16)) {
        if (rows <= 8) {
            auto kernel = rows <= 4 ? paged_decode_kernel<HD, TYPE, TERMS, 4> : paged_decode_kernel<HD, TYPE, TERMS, 2>;
            hipLaunchKernelGGL(kernel, grid(1, 1, a.splits[0]), dim3(256), 0, stream, a);
            return launch_status("qk_paged_attention_f32 launch");
        }
    }
    if (a.few_rows > 0) {
        const int64_t few = std::min<int64_t>(rows, a.few_rows);
        const dim3 blocks = grid(few, kRowTile, a.splits[0]);
        // Heads of 256 without terms: SHARED where there are more workgroups than CUs, of fp16
        // rows only if they share the cache rows of a sequence.  In us, SHARED second: 16
        // single tokens over 2000, 16 heads on 8, int8 32.4 and 35.5, fp16 49.9 and 50.5; 64
        // over 1000, int8 54.8 and 49.2, float8 56.0 and 51.4; 64 over 4500, int8 233 and 228,
        // fp16 402 and 417; four prompts of 300 over 100, 8 heads on 1, int8 41.6 and 31.3, fp16
        // 45.6 and 38.7.
        auto kernel = paged_attention_kernel<HD, TYPE, TERMS, (HD > 128)>;
        if constexpr (HD > 128 && !TERMS && TYPE != QK_TYPE_I4)
            if (static_cast<int64_t>(blocks.x) * blocks.y <= 256 || (TYPE == QK_TYPE_F16 && few <= kRowTile))
                kernel = paged_attention_kernel<HD, TYPE, TERMS, false>;
        hipLaunchKernelGGL(kernel, blocks, dim3(256), 0, stream, a);
    }
    if constexpr (HD <= 128 || !(TERMS || TYPE == QK_TYPE_I4)) {   // (the others have no chunks)
        constexpr size_t kLds = 2 * Chunk<HD, TYPE>::kBuffer;
        if (rows > a.few_rows)
            hipLaunchKernelGGL((paged_chunk_kernel<HD, TYPE, TERMS>), grid(rows, kChunkRows, a.splits[1]), dim3(256), kLds,
                               stream, a);
    }
    return launch_status("qk_paged_attention_f32 launch");
}

template <int TYPE, bool TERMS>
int attend_heads(const PagedAttn &a, hipStream_t stream) {
    switch (a.kv.head_dim) {
        case 64: return attend_launch<64, TYPE, TERMS>(a, stream);
        case 96: return attend_launch<96, TYPE, TERMS>(a, stream);
        case 128: return attend_launch<128, TYPE, TERMS>(a, stream);
        default: return attend_launch<256, TYPE, TERMS>(a, stream);
    }
}

template <int TYPE>
int attend_type(const PagedAttn &a, bool terms, hipStream_t stream) {
    return terms ? attend_heads<TYPE, true>(a, stream) : attend_heads<TYPE, false>(a, stream);
}

}  // namespace
}  // namespace qk
