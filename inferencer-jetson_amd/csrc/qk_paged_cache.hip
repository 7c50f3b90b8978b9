// qk_paged_cache.hip - rotary tables, and rows into and out of a paged cache.
#include "qk_paged.h"

#include <cmath>

namespace qk {
namespace {

hipStream_t S(qk_stream s) { return static_cast<hipStream_t>(s); }

// ------------------------------------------------------------- tables --
//
// f_i by the thread that holds pair i, once for all its positions; the angle
// is taken in turns, so its whole turns drop out exactly: t = p * f / 2 pi, r =
// t - rint(t) (an error of 2^-53 t, 2e-12 turns at position 131072), then the
// nearest quarter turn off, and the Taylor polynomials of sine and cosine on
// +-pi/4, whose first dropped terms are y^15/15! < 3e-14 and y^16/16! < 2e-15.
// All in 64 bits, at half the rate of 32: 131072 positions of 64 pairs, 67 MB,
// take 18 us, 3.7 TB/s (14 were the stores alone); 1024 positions 3 us, the
// latency of one launch and of the frequencies' exp().
struct TableArgs {
    double log_theta, factor, low, high, context, amplitude;
    double ramp_lo, ramp_span;
    const float *freq_factors;
    float *cosine, *sine;
    int type, half, rot, first, positions, sweep, per_block;
};

constexpr double kTurn = 6.283185307179586476925;

__device__ __forceinline__ void sincos_turns(double t, double &s, double &c) {
    const double r = t - rint(t);
    const double j = rint(4. * r);
    const double y = fma(j, -0.25, r) * kTurn, y2 = y * y;
    double ps = 1. / 6227020800.;
    ps = fma(ps, y2, -1. / 39916800.);
    ps = fma(ps, y2, 1. / 362880.);
    ps = fma(ps, y2, -1. / 5040.);
    ps = fma(ps, y2, 1. / 120.);
    ps = fma(ps, y2, -1. / 6.);
    ps = fma(ps * y2, y, y);
    double pc = -1. / 87178291200.;
    pc = fma(pc, y2, 1. / 479001600.);
    pc = fma(pc, y2, -1. / 3628800.);
    pc = fma(pc, y2, 1. / 40320.);
    pc = fma(pc, y2, -1. / 720.);
    pc = fma(pc, y2, 1. / 24.);
    pc = fma(pc, y2, -0.5);
    pc = fma(pc, y2, 1.);
    const int q = static_cast<int>(j) & 3;
    const double a = q & 1 ? pc : ps, b = q & 1 ? ps : pc;
    s = q & 2 ? -a : a;
    c = (q + 1) & 2 ? -b : b;
}

__global__ __launch_bounds__(256) void rope_tables_kernel(TableArgs a) {
    const int i = threadIdx.x % a.half, sub = threadIdx.x / a.half;
    if (sub >= a.sweep) return;
    double f = exp(-2. * i / a.rot * a.log_theta);
    if (a.freq_factors) f /= static_cast<double>(a.freq_factors[i]);
    if (a.type == QK_ROPE_LINEAR) {
        f /= a.factor;
    } else if (a.type == QK_ROPE_LLAMA3) {
        const double turns = a.context * f / kTurn;
        const double m = fmin(fmax((turns - a.low) / (a.high - a.low), 0.), 1.);
        f = f / a.factor * (1. - m) + f * m;
    } else if (a.type == QK_ROPE_YARN) {
        const double m = fmin(fmax((i - a.ramp_lo) / a.ramp_span, 0.), 1.);
        f = f / a.factor * m + f * (1. - m);
    }
    f /= kTurn;
    const int p1 = min(a.positions, (static_cast<int>(blockIdx.x) + 1) * a.per_block);
    for (int p = blockIdx.x * a.per_block + sub; p < p1; p += a.sweep) {
        double s, c;
        sincos_turns((static_cast<double>(a.first) + p) * f, s, c);
        const int64_t at = static_cast<int64_t>(p) * a.half + i;
        a.cosine[at] = static_cast<float>(c * a.amplitude);
        a.sine[at] = static_cast<float>(s * a.amplitude);
    }
}

// -------------------------------------------------------------- write --

struct WriteArgs {
    qk_paged_kv kv;
    qk_paged_batch b;
    const float *q, *k, *v, *cosine, *sine;
    float *q_out;
    int64_t ldq, ldq_out, ldk, ldv;
    int heads, positions, rot, half, page_shift;
};

// Lanes that share a row, 4 values each (96: 24 of 32).
constexpr int row_lanes(int hd) { return hd == 64 ? 16 : hd == 256 ? 64 : 32; }

__device__ __forceinline__ float4 load4(const float *p) {
    float4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// Values c .. c + 3 of a head at x, rotated.  Products of fp32 values are exact
// in 64 bits, so a * c - b * s is rounded once there and once to fp32 whatever
// the compiler fuses.
__device__ __forceinline__ float4 rotate4(const float *x, int c, const float *cosine, const float *sine, int rot,
                                          int half) {
    float v[4];
    __builtin_memcpy(v, x + c, 16);
    if (c >= rot) return make_float4(v[0], v[1], v[2], v[3]);
    float o[4], cs[4], sn[4];
    if (half) {
        const int h = rot / 2;
        if (h % 4 == 0) {
            const bool upper = c >= h;
            __builtin_memcpy(o, x + (upper ? c - h : c + h), 16);
            __builtin_memcpy(cs, cosine + (upper ? c - h : c), 16);
            __builtin_memcpy(sn, sine + (upper ? c - h : c), 16);
            #pragma unroll
            for (int e = 0; e < 4; ++e) sn[e] = upper ? sn[e] : -sn[e];
        } else {
            #pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = c + e;
                const bool upper = d >= h, in = d < rot;
                o[e] = in ? x[upper ? d - h : d + h] : 0.f;
                cs[e] = in ? cosine[upper ? d - h : d] : 1.f;
                sn[e] = in ? (upper ? sine[d - h] : -sine[d]) : 0.f;
            }
        }
    } else {
        #pragma unroll
        for (int e = 0; e < 4; e += 2) {
            const bool in = c + e < rot;
            const float cp = in ? cosine[(c + e) / 2] : 1.f, sp = in ? sine[(c + e) / 2] : 0.f;
            cs[e] = cs[e + 1] = cp;
            sn[e] = -sp;
            sn[e + 1] = sp;
            o[e] = v[e + 1];
            o[e + 1] = v[e];
        }
    }
    float r[4];
    #pragma unroll
    for (int e = 0; e < 4; ++e)
        r[e] = c + e < rot ? static_cast<float>(static_cast<double>(v[e]) * cs[e] + static_cast<double>(o[e]) * sn[e])
                           : v[e];
    return make_float4(r[0], r[1], r[2], r[3]);
}

// x / scale to the nearest integer, ties to even, exactly: of n = rint(x *
// inv), off by one at most, the remainder x - n * scale is a multiple of half
// an ulp of scale below 0.51 scale, so it is exact and decides.
__device__ __forceinline__ int round_quotient(float x, float scale, float inv) {
    const float n = rintf(x * inv);
    const float e = fmaf(-n, scale, x), h = 0.5f * scale;
    const bool odd = (static_cast<int>(n) & 1) != 0;
    if (e > h || (e == h && odd)) return static_cast<int>(n) + 1;
    if (e < -h || (e == -h && odd)) return static_cast<int>(n) - 1;
    return static_cast<int>(n);
}

constexpr uint32_t kTinyBits = (127u - 100u) << 23;   // 2^-100

// Bytes of n codes, and floats of a row's scale entry.
constexpr int code_bytes(int type, int n) { return type == QK_TYPE_F16 ? 2 * n : type == QK_TYPE_I4 ? n / 2 : n; }
constexpr int scale_floats(int type) { return type == QK_TYPE_I4 ? 2 : 1; }

// The scale of a 4-bit row of largest magnitude top: the least number of 13
// significant bits s with 1785 s >= top (a product of 24 bits: exact), found by two
// comparisons from a quotient that is off by less than a step of 13 bits.
__device__ __forceinline__ float scale_of_13(float top) {
    uint32_t b = (__builtin_bit_cast(uint32_t, top * (1.f / 1785.f)) + 0x7FFu) & ~0x7FFu;
    auto value = [](uint32_t bits) { return __builtin_bit_cast(float, bits); };
    if (1785.f * value(b) < top) b += 0x800u;
    if (1785.f * value(b - 0x800u) >= top) b -= 0x800u;
    // (Next to fp32's largest: the one below, whose values are finite.)
    return 1785.f * value(b) < INFINITY ? value(b) : value(b - 0x800u);
}
// The least positive integer m with m step >= top, step of 16 significant bits, at
// most 255.
__device__ __forceinline__ float multiplier(float top, float step) {
    float m = ceilf(top * (1.f / step));
    if ((m - 1.f) * step >= top) m -= 1.f;
    if (m * step < top) m += 1.f;
    return fminf(fmaxf(m, 1.f), 255.f);
}

// The largest of the lanes of a row's quarter (HD / 16 of them).
template <int HD>
__device__ __forceinline__ uint32_t quarter_max(uint32_t v) {
    constexpr int kLanes = HD / 16;
    if constexpr (kLanes & (kLanes - 1)) {   // 6 of 96 values
        const int row = threadIdx.x & 32, first = row + (threadIdx.x & 31) / kLanes * kLanes;
        uint32_t top = 0;   // (lanes past the row's 24 hold zeros, and read within the wave)
        #pragma unroll
        for (int i = 0; i < kLanes; ++i) top = max(top, static_cast<uint32_t>(__shfl(static_cast<int>(v), first + i)));
        return top;
    }
    #pragma unroll
    for (int off = 1; off < kLanes; off <<= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), off)));
    return v;
}

// One row's four values of a lane (zeros past head_dim) into its page; all
// row_lanes lanes call it.  (4-bit rows: the quarters' maxima on the way to the row's,
// a multiplier a quarter, gathered in the first lane; 8192 tokens of 8 KV heads of 128
// in 89 us where float8 rows take 85, memory bound as those.)
template <int HD, int TYPE, int LANES>
__device__ __forceinline__ void store_codes(const float4 &x, bool active, char *row, float *scale_at, int c) {
    if constexpr (TYPE == QK_TYPE_F16) {
        if (!active) return;
        const _Float16 h[4] = {static_cast<_Float16>(x.x), static_cast<_Float16>(x.y), static_cast<_Float16>(x.z),
                               static_cast<_Float16>(x.w)};
        __builtin_memcpy(row + 2 * c, h, 8);
        return;
    }
    // Magnitudes as integers: those that are not finite are the largest.
    const float v[4] = {x.x, x.y, x.z, x.w};
    uint32_t amax = 0;
    #pragma unroll
    for (int e = 0; e < 4; ++e) amax = max(amax, __builtin_bit_cast(uint32_t, v[e]) & 0x7FFFFFFFu);
    uint32_t part = 0;
    if constexpr (TYPE == QK_TYPE_I4) part = quarter_max<HD>(amax);
    #pragma unroll
    for (int off = 1; off < LANES; off <<= 1) amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), off)));
    const float top = __builtin_bit_cast(float, amax);
    const bool bad = amax >= 0x7F800000u, none = amax < kTinyBits;
    float scale;
    uint32_t codes = 0;
    if constexpr (TYPE == QK_TYPE_I8) {
        scale = none ? 1.f : top / 127.f;
        const float inv = 1.f / scale;
        #pragma unroll
        for (int e = 0; e < 4; ++e)
            codes |= (static_cast<uint32_t>(round_quotient(v[e], scale, inv)) & 0xFFu) << (8 * e);
    } else if constexpr (TYPE == QK_TYPE_I4) {
        scale = none ? 1.f : scale_of_13(top);
        const float m = bad || none ? 1.f : multiplier(__builtin_bit_cast(float, part), 7.f * scale);
        const float step = m * scale, inv = 1.f / step;   // a product of 21 bits; its code's is of 24
        #pragma unroll
        for (int e = 0; e < 4; ++e)
            codes |= (static_cast<uint32_t>(round_quotient(v[e], step, inv)) & 0xFu) << (4 * e);
        // The multipliers of all quarters in the row's first lane.
        const int first = threadIdx.x & (64 - LANES);
        uint32_t mults = 0;
        #pragma unroll
        for (int q = 0; q < 4; ++q)
            mults |= static_cast<uint32_t>(__shfl(static_cast<int>(m), first + q * (HD / 16))) << (8 * q);
        if (bad) scale = __builtin_nanf("");
        if (bad || none) codes = 0;
        if (!active) return;
        const uint16_t two = static_cast<uint16_t>(codes);
        __builtin_memcpy(row + c / 2, &two, 2);
        if (c == 0) *reinterpret_cast<float2 *>(scale_at) = make_float2(scale, __builtin_bit_cast(float, mults));
        return;
    } else {
        // 448 = 0.875 * 2^9: the least power of two with top / scale <= 448.
        const int s = __builtin_amdgcn_frexp_expf(top) - (__builtin_amdgcn_frexp_mantf(top) > 0.875f ? 8 : 9);
        scale = none ? 1.f : ldexpf(1.f, s);
        float y[4];
        #pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = ldexpf(v[e], none ? 0 : -s);
        codes = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        codes = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], codes, true);
    }
    if (bad) scale = __builtin_nanf("");
    if (bad || none) codes = 0;
    if (!active) return;
    __builtin_memcpy(row + c, &codes, 4);
    if (c == 0) *scale_at = scale;
}

// Rows of a group of row_lanes lanes, one after the other.  Two: 32 decoding
// sequences' rows (8 KV heads of 64 int8 values) written 4.2 us, with four 5.2;
// 8192 tokens' (32 heads, 8 KV heads of 128, float8) written 85 us and read 20,
// with one 88 and 21, with four 84 and 22, with eight 88 and 25.
constexpr int kGroupRows = 2;

// Rows (token, head) of q, then k, then v, one a group of row_lanes lanes.  Bound
// by memory: of those 8192 tokens 352 MB in and out, 4.2 TB/s (a copy reaches
// 4.7).
template <int HD, int TYPE>
__global__ __launch_bounds__(256) void paged_write_kernel(WriteArgs a) {
    constexpr int L = row_lanes(HD), kRows = 256 / L, U = kGroupRows;
    const qk_paged_seq s = a.b.seqs[blockIdx.y];
    if (!paged_seq_ok(s, a.b, a.page_shift) || (a.rot > 0 && s.pos + s.count > a.positions)) return;
    const int c = (threadIdx.x % L) * 4, kvh = a.kv.kv_heads, heads = a.q ? a.heads : 0, R = heads + 2 * kvh;
    const int64_t total = static_cast<int64_t>(s.count) * R, block0 = static_cast<int64_t>(blockIdx.x) * kRows * U;
    const bool active = c < HD;
    #pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t at = block0 + u * kRows + threadIdx.x / L;
        if (at >= total) return;   // whole groups leave, so a row's lanes stay together
        const int i = static_cast<int>(at / R), r = static_cast<int>(at - static_cast<int64_t>(i) * R);
        const int pos = s.pos + i;
        const int64_t tok = s.first + i;
        const float *cosine = a.cosine + static_cast<int64_t>(pos) * (a.rot / 2);
        const float *sine = a.sine + static_cast<int64_t>(pos) * (a.rot / 2);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < heads) {
            if (active) {
                // In place too: a row's lanes are of one wave, so all have loaded their
                // pairs before any of them stores.
                x = rotate4(a.q + tok * a.ldq + r * HD, c, cosine, sine, a.rot, a.half);
                *reinterpret_cast<float4 *>(a.q_out + tok * a.ldq_out + r * HD + c) = x;
            }
            continue;
        }
        const bool key = r < heads + kvh;
        const int h = r - heads - (key ? 0 : kvh);
        if (active)
            x = key ? rotate4(a.k + tok * a.ldk + h * HD, c, cosine, sine, a.rot, a.half)
                    : load4(a.v + tok * a.ldv + h * HD + c);
        const int64_t page = paged_page(a.b.page_table + static_cast<int64_t>(s.table) * a.b.table_stride,
                                        pos >> a.page_shift, a.kv.pages);
        const int64_t row = (max(page, int64_t(0)) * kvh + h) * a.kv.page_rows + (pos & (a.kv.page_rows - 1));
        char *base = static_cast<char *>(key ? a.kv.key : a.kv.value) + row * code_bytes(TYPE, HD);
        float *scale_at = TYPE == QK_TYPE_F16 ? nullptr : (key ? a.kv.key_scale : a.kv.value_scale) + row * scale_floats(TYPE);
        store_codes<HD, TYPE, L>(x, active && page >= 0, base, scale_at, c);
    }
}

// --------------------------------------------------------------- read --

struct ReadArgs {
    qk_paged_kv kv;
    qk_paged_batch b;
    float *key_out, *value_out;
    int64_t ldk, ldv;
    int page_shift;
};

// (4-bit codes: mult the multiplier of their quarter; code * mult is exact.)
template <int TYPE>
__device__ __forceinline__ float4 decode4(const char *p, float scale, float mult) {
    if constexpr (TYPE == QK_TYPE_I4) {
        uint16_t two;
        __builtin_memcpy(&two, p, 2);
        const uint32_t w = two ^ 0x8888u;
        auto at = [&](int e) { return (static_cast<float>(w >> (4 * e) & 15) - 8.f) * mult * scale; };
        return make_float4(at(0), at(1), at(2), at(3));
    } else if constexpr (TYPE == QK_TYPE_F16) {
        _Float16 h[4];
        __builtin_memcpy(h, p, 8);
        return make_float4(h[0], h[1], h[2], h[3]);
    } else if constexpr (TYPE == QK_TYPE_I8) {
        int8_t b[4];
        __builtin_memcpy(b, p, 4);
        return make_float4(b[0] * scale, b[1] * scale, b[2] * scale, b[3] * scale);
    } else {
        uint32_t w;
        __builtin_memcpy(&w, p, 4);
        return make_float4(__builtin_amdgcn_cvt_f32_fp8(w, 0) * scale, __builtin_amdgcn_cvt_f32_fp8(w, 1) * scale,
                           __builtin_amdgcn_cvt_f32_fp8(w, 2) * scale, __builtin_amdgcn_cvt_f32_fp8(w, 3) * scale);
    }
}

// Rows (token, head) of the keys, then of the values, as above: the 8192 tokens' 17
// MB of codes and 67 MB of fp32 in 20 us, 4.2 TB/s.
template <int HD, int TYPE>
__global__ __launch_bounds__(256) void paged_read_kernel(ReadArgs a) {
    constexpr int L = row_lanes(HD), kRows = 256 / L, U = kGroupRows;
    const qk_paged_seq s = a.b.seqs[blockIdx.y];
    if (!paged_seq_ok(s, a.b, a.page_shift)) return;
    const int c = (threadIdx.x % L) * 4, kvh = a.kv.kv_heads;
    const int first_kind = a.key_out ? 0 : 1, kinds = (a.key_out ? 1 : 0) + (a.value_out ? 1 : 0), R = kinds * kvh;
    const int64_t total = static_cast<int64_t>(s.count) * R, block0 = static_cast<int64_t>(blockIdx.x) * kRows * U;
    if (c >= HD) return;
    #pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t at = block0 + u * kRows + threadIdx.x / L;
        if (at >= total) return;
        const int i = static_cast<int>(at / R), r = static_cast<int>(at - static_cast<int64_t>(i) * R);
        const bool key = first_kind + r / kvh == 0;
        const int h = r % kvh, pos = s.pos + i;
        const int64_t page = paged_page(a.b.page_table + static_cast<int64_t>(s.table) * a.b.table_stride,
                                        pos >> a.page_shift, a.kv.pages);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (page >= 0) {
            const int64_t row = (page * kvh + h) * a.kv.page_rows + (pos & (a.kv.page_rows - 1));
            const char *base = static_cast<const char *>(key ? a.kv.key : a.kv.value);
            const float *scales = key ? a.kv.key_scale : a.kv.value_scale;
            const float scale = TYPE == QK_TYPE_F16 ? 1.f : scales[row * scale_floats(TYPE)];
            float mult = 1.f;
            if constexpr (TYPE == QK_TYPE_I4)
                mult = static_cast<float>(__builtin_bit_cast(uint32_t, scales[row * 2 + 1]) >> (8 * (c / (HD / 4))) & 0xFFu);
            x = decode4<TYPE>(base + row * code_bytes(TYPE, HD) + code_bytes(TYPE, c), scale, mult);
        }
        float *out = key ? a.key_out + (s.first + i) * a.ldk : a.value_out + (s.first + i) * a.ldv;
        *reinterpret_cast<float4 *>(out + h * HD + c) = x;
    }
}

template <template <int, int> class Launch, class... A>
int by_shape(int hd, int type, A &&...args) {
    auto of = [&](auto HD) {
        constexpr int kHd = decltype(HD)::value;
        if (type == QK_TYPE_F16) return Launch<kHd, QK_TYPE_F16>::run(args...);
        if (type == QK_TYPE_I8) return Launch<kHd, QK_TYPE_I8>::run(args...);
        if (type == QK_TYPE_I4) return Launch<kHd, QK_TYPE_I4>::run(args...);
        return Launch<kHd, QK_TYPE_F8_E4M3>::run(args...);
    };
    switch (hd) {
        case 64: return of(std::integral_constant<int, 64>{});
        case 96: return of(std::integral_constant<int, 96>{});
        case 128: return of(std::integral_constant<int, 128>{});
        default: return of(std::integral_constant<int, 256>{});
    }
}

template <int HD, int TYPE>
struct Write {
    static int run(const WriteArgs &a, dim3 grid, hipStream_t stream) {
        hipLaunchKernelGGL((paged_write_kernel<HD, TYPE>), grid, dim3(256), 0, stream, a);
        return launch_status("qk_rope_paged_write launch");
    }
};

template <int HD, int TYPE>
struct Read {
    static int run(const ReadArgs &a, dim3 grid, hipStream_t stream) {
        hipLaunchKernelGGL((paged_read_kernel<HD, TYPE>), grid, dim3(256), 0, stream, a);
        return launch_status("qk_paged_read_f32 launch");
    }
};

// Workgroups for max_count * R rows of a sequence; 0: more than a launch holds
// (fewer than 2^32 threads a dimension, of 256 a workgroup).
unsigned row_blocks(int64_t max_count, int64_t R, int hd) {
    const int64_t per = 256 / row_lanes(hd) * kGroupRows, n = (max_count * R + per - 1) / per;
    return n >= 1 << 24 ? 0 : static_cast<unsigned>(n);
}

}  // namespace

bool rows_meet(const float *a, int64_t lda, int64_t wa, const float *b, int64_t ldb, int64_t wb, int64_t n) {
    if (!a || !b || n < 1) return false;
    const int64_t d = (reinterpret_cast<intptr_t>(b) - reinterpret_cast<intptr_t>(a)) / static_cast<int64_t>(sizeof(float));
    if (d >= (n - 1) * lda + wa || -d >= (n - 1) * ldb + wb) return false;
    for (int64_t i = d < wa ? 0 : (d - wa) / lda; i < n; ++i) {
        // The first row of b that ends behind the start of row i of a.
        const int64_t from = i * lda - d - wb + 1, j = from <= 0 ? 0 : (from + ldb - 1) / ldb;
        if (j < n && d + j * ldb < i * lda + wa) return true;
        if (lda == ldb && j > 0 && j < n - 1) return false;   // the rows behind meet alike
    }
    return false;
}

int check_paged_kv(const char *where, const qk_paged_kv *kv) {
    const std::string w(where);
    if (!kv || !kv->key || !kv->value) return fail(QK_ERR_INVALID_ARG, w + ": null cache pointer");
    if (kv->type != QK_TYPE_F16 && kv->type != QK_TYPE_I8 && kv->type != QK_TYPE_F8_E4M3 && kv->type != QK_TYPE_I4)
        return fail(QK_ERR_TYPE, w + ": cache type " + std::to_string(kv->type) + " is not F16, I8, I4 or F8_E4M3");
    if (kv->type != QK_TYPE_F16 && (!kv->key_scale || !kv->value_scale))
        return fail(QK_ERR_INVALID_ARG, w + ": null scale pointer");
    if (kv->head_dim != 64 && kv->head_dim != 96 && kv->head_dim != 128 && kv->head_dim != 256)
        return fail(QK_ERR_LIMIT, w + ": head_dim must be 64, 96, 128 or 256");
    if (kv->page_rows < 16 || kv->page_rows > 1024 || (kv->page_rows & (kv->page_rows - 1)))
        return fail(QK_ERR_LIMIT, w + ": page_rows must be a power of two from 16 to 1024");
    if (kv->kv_heads < 1 || kv->kv_heads > 4096 || kv->pages < 1 || kv->pages > 0x7FFFFFFF)
        return fail(QK_ERR_INVALID_ARG, w + ": bad KV head or page count");
    if (!aligned(kv->key, 16) || !aligned(kv->value, 16) || !aligned(kv->key_scale, 16) ||
        !aligned(kv->value_scale, 16))
        return fail(QK_ERR_ALIGN, w + ": cache buffers must be 16-byte aligned");
    return QK_OK;
}

int check_paged_batch(const char *where, const qk_paged_batch *b) {
    const std::string w(where);
    if (!b || b->n_seqs < 0 || b->n_tokens < 0) return fail(QK_ERR_INVALID_ARG, w + ": null batch or negative count");
    if (b->n_seqs == 0 || b->n_tokens == 0) return QK_OK;
    if (!b->page_table || !b->seqs || b->table_rows < 1 || b->table_stride < 1)
        return fail(QK_ERR_INVALID_ARG, w + ": null or empty page table or sequences");
    if (b->max_count < 1 || b->max_rows < b->max_count || b->max_rows > 0x7FFFFFFF - 1024)
        return fail(QK_ERR_INVALID_ARG, w + ": max_count must be positive and max_rows at least max_count");
    if (b->n_seqs > 65535) return fail(QK_ERR_LIMIT, w + ": too many sequences in one launch");
    if (!aligned(b->seqs, 16) || !aligned(b->page_table, 4))
        return fail(QK_ERR_ALIGN, w + ": seqs must be 16-byte and page_table 4-byte aligned");
    return QK_OK;
}

}  // namespace qk

extern "C" {

int qk_rope_tables_f32(float theta, int rot_dim, const qk_rope_scaling *scaling, const float *freq_factors,
                       int first_pos, int positions, float *cosine, float *sine, qk_stream stream) {
    if (positions < 0 || first_pos < 0 || (positions > 0 && (!cosine || !sine)))
        return qk::fail(QK_ERR_INVALID_ARG, "qk_rope_tables_f32: null pointer or negative position");
    if (rot_dim < 2 || rot_dim % 2 || rot_dim > 512)
        return qk::fail(QK_ERR_LIMIT, "qk_rope_tables_f32: rot_dim must be even, 2 to 512");
    if (positions > 1 << 30 || positions > 0x7FFFFFFF - first_pos)
        return qk::fail(QK_ERR_LIMIT, "qk_rope_tables_f32: more than 2^30 positions, or beyond 2^31");
    if (!(theta > 0.f) || !std::isfinite(theta))
        return qk::fail(QK_ERR_INVALID_ARG, "qk_rope_tables_f32: theta must be positive");
    qk::TableArgs a{};
    const int type = scaling ? scaling->type : QK_ROPE_NONE;
    a.log_theta = std::log(static_cast<double>(theta));
    a.amplitude = a.factor = 1.;
    if (type != QK_ROPE_NONE) {
        const qk_rope_scaling &s = *scaling;
        if (type != QK_ROPE_LINEAR && type != QK_ROPE_LLAMA3 && type != QK_ROPE_YARN)
            return qk::fail(QK_ERR_TYPE, "qk_rope_tables_f32: unknown scaling " + std::to_string(type));
        if (!(s.factor > 0.f) || !std::isfinite(s.factor))
            return qk::fail(QK_ERR_INVALID_ARG, "qk_rope_tables_f32: factor must be positive");
        a.factor = s.factor;
        if (type != QK_ROPE_LINEAR && (!(s.original_context > 0.f) || !std::isfinite(s.original_context)))
            return qk::fail(QK_ERR_INVALID_ARG, "qk_rope_tables_f32: original_context must be positive");
        a.context = s.original_context;
        if (type == QK_ROPE_LLAMA3) {
            if (!(s.high_freq_factor > s.low_freq_factor) || !std::isfinite(s.high_freq_factor) ||
                !std::isfinite(s.low_freq_factor))
                return qk::fail(QK_ERR_INVALID_ARG,
                                "qk_rope_tables_f32: high_freq_factor must be larger than low_freq_factor");
            a.low = s.low_freq_factor;
            a.high = s.high_freq_factor;
        }
        if (type == QK_ROPE_YARN) {
            if (!(s.beta_slow > 0.f) || !(s.beta_fast >= s.beta_slow) || !std::isfinite(s.beta_fast) || theta == 1.f ||
                !std::isfinite(s.attention_factor))
                return qk::fail(QK_ERR_INVALID_ARG,
                                "qk_rope_tables_f32: beta_fast must be at least beta_slow, both positive, theta not 1");
            auto pair = [&](double turns) {
                return rot_dim * std::log(a.context / (turns * qk::kTurn)) / (2. * a.log_theta);
            };
            a.ramp_lo = std::max(std::floor(pair(s.beta_fast)), 0.);
            const double hi = std::min(std::ceil(pair(s.beta_slow)), rot_dim - 1.);
            a.ramp_span = std::max(hi - a.ramp_lo, 0.001);
            a.amplitude = s.attention_factor != 0.f ? s.attention_factor : 0.1 * std::log(a.factor) + 1.;
        }
    }
    if (positions == 0) return qk::ok();
    const int64_t values = static_cast<int64_t>(positions) * (rot_dim / 2);
    if (qk::rows_meet(cosine, values, values, sine, values, values, 1))
        return qk::fail(QK_ERR_INVALID_ARG, "qk_rope_tables_f32: cosine overlaps sine");
    a.type = type;
    a.rot = rot_dim;
    a.half = rot_dim / 2;
    a.first = first_pos;
    a.positions = positions;
    a.freq_factors = freq_factors;
    a.cosine = cosine;
    a.sine = sine;
    a.sweep = 256 / a.half;
    const int sweeps = std::max(1, std::min(16, positions / (a.sweep * 1024)));
    a.per_block = a.sweep * sweeps;
    hipLaunchKernelGGL(qk::rope_tables_kernel, dim3((positions + a.per_block - 1) / a.per_block), dim3(256), 0,
                       qk::S(stream), a);
    return qk::launch_status("qk_rope_tables_f32 launch");
}

int qk_rope_paged_write(const qk_paged_kv *kv, const qk_paged_batch *batch, const float *q, int ldq, float *q_out,
                        int ldq_out, const float *k, int ldk, const float *v, int ldv, int heads, const float *cosine,
                        const float *sine, int positions, int rot_dim, int half, qk_stream stream) {
    const char *where = "qk_rope_paged_write";
    if (int s = qk::check_paged_kv(where, kv)) return s;
    if (int s = qk::check_paged_batch(where, batch)) return s;
    if (rot_dim < 0 || rot_dim % 2 || rot_dim > kv->head_dim || positions < 0 || (half != 0 && half != 1))
        return qk::fail(QK_ERR_INVALID_ARG, "qk_rope_paged_write: rot_dim must be even, 0 to head_dim, half 0 or 1");
    if (batch->n_seqs == 0 || batch->n_tokens == 0) return qk::ok();
    if (!k || !v || !q != !q_out || (rot_dim > 0 && (!cosine || !sine)))
        return qk::fail(QK_ERR_INVALID_ARG, "qk_rope_paged_write: null pointer");
    const int64_t kv_dim = static_cast<int64_t>(kv->kv_heads) * kv->head_dim;
    if (q && (heads < 1 || heads > 65536 || heads % kv->kv_heads))
        return qk::fail(QK_ERR_INVALID_ARG, "qk_rope_paged_write: heads must be a multiple of kv_heads");
    const int64_t q_dim = q ? static_cast<int64_t>(heads) * kv->head_dim : 0;
    if (ldk < kv_dim || ldv < kv_dim || (q && (ldq < q_dim || ldq_out < q_dim)))
        return qk::fail(QK_ERR_INVALID_ARG, "qk_rope_paged_write: leading dimension smaller than the row");
    if (q == q_out && q && ldq != ldq_out)
        return qk::fail(QK_ERR_INVALID_ARG, "qk_rope_paged_write: in place, ldq and ldq_out must be equal");
    if (!qk::aligned(q, 16) || !qk::aligned(q_out, 16) || !qk::aligned(k, 16) || !qk::aligned(v, 16) || ldk % 4 ||
        ldv % 4 || (q && (ldq % 4 || ldq_out % 4)))
        return qk::fail(QK_ERR_ALIGN, "qk_rope_paged_write: q, q_out, k and v need 16-byte rows");
    const int R = (q ? heads : 0) + 2 * kv->kv_heads;
    const unsigned blocks = qk::row_blocks(batch->max_count, R, kv->head_dim);
    if (!blocks) return qk::fail(QK_ERR_LIMIT, "qk_rope_paged_write: too many rows in one launch");
    if (q && ((q != q_out && qk::rows_meet(q_out, ldq_out, q_dim, q, ldq, q_dim, batch->n_tokens)) ||
              qk::rows_meet(q_out, ldq_out, q_dim, k, ldk, kv_dim, batch->n_tokens) ||
              qk::rows_meet(q_out, ldq_out, q_dim, v, ldv, kv_dim, batch->n_tokens)))
        return qk::fail(QK_ERR_INVALID_ARG, "qk_rope_paged_write: q_out overlaps k, v or a part of q");
    const qk::WriteArgs a{*kv, *batch, q,   k,     v,         cosine,  sine, q_out, ldq,
                          ldq_out, ldk, ldv, heads, positions, rot_dim, half, __builtin_ctz(kv->page_rows)};
    return qk::by_shape<qk::Write>(kv->head_dim, kv->type, a, dim3(blocks, batch->n_seqs), qk::S(stream));
}

int qk_paged_read_f32(const qk_paged_kv *kv, const qk_paged_batch *batch, float *key_out, int ldk, float *value_out,
                      int ldv, qk_stream stream) {
    const char *where = "qk_paged_read_f32";
    if (int s = qk::check_paged_kv(where, kv)) return s;
    if (int s = qk::check_paged_batch(where, batch)) return s;
    if (batch->n_seqs == 0 || batch->n_tokens == 0) return qk::ok();
    if (!key_out && !value_out) return qk::fail(QK_ERR_INVALID_ARG, "qk_paged_read_f32: null pointer");
    const int64_t kv_dim = static_cast<int64_t>(kv->kv_heads) * kv->head_dim;
    if ((key_out && ldk < kv_dim) || (value_out && ldv < kv_dim))
        return qk::fail(QK_ERR_INVALID_ARG, "qk_paged_read_f32: leading dimension smaller than the row");
    if (!qk::aligned(key_out, 16) || !qk::aligned(value_out, 16) || (key_out && ldk % 4) || (value_out && ldv % 4))
        return qk::fail(QK_ERR_ALIGN, "qk_paged_read_f32: key_out and value_out need 16-byte rows");
    const int R = ((key_out ? 1 : 0) + (value_out ? 1 : 0)) * kv->kv_heads;
    const unsigned blocks = qk::row_blocks(batch->max_count, R, kv->head_dim);
    if (!blocks) return qk::fail(QK_ERR_LIMIT, "qk_paged_read_f32: too many rows in one launch");
    if (qk::rows_meet(key_out, ldk, kv_dim, value_out, ldv, kv_dim, batch->n_tokens))
        return qk::fail(QK_ERR_INVALID_ARG, "qk_paged_read_f32: key_out overlaps value_out");
    const qk::ReadArgs a{*kv, *batch, key_out, value_out, ldk, ldv, __builtin_ctz(kv->page_rows)};
    return qk::by_shape<qk::Read>(kv->head_dim, kv->type, a, dim3(blocks, batch->n_seqs), qk::S(stream));
}

}  // extern "C"
