// qk_sample.hip - the next token of rows of logits: temperature, top-k, top-p,
// min-p and the pick by a given random number.
//
// The filters keep a prefix of the row in descending order (equal logits by
// index), so what they leave is the tokens down to one of them: the cut.  Four
// launches:
//   sample_scan_kernel, a workgroup per 16384 logits (a segment): its largest,
//     and a histogram over 16 bins an octave of the weights 2^(x log2(e) / T)
//     below the segment's own power of two, as integers, so the order of adding
//     does not matter;
//   sample_plan_kernel, a workgroup per row: adds up the segments' histograms
//     and finds the bin in which the cut lies;
//   sample_collect_kernel, per segment again: lists that bin's tokens (some
//     hundreds at most; with top-k, where they fit, all that it leaves);
//   sample_pick_kernel, a workgroup per row: sorts the list and finds the cut,
//     then from the histograms the segment that holds the random number's token,
//     and the token by looking that segment over.
// A row is thus read once from memory and once from the cache, and its
// exponentials are taken once.  They are held to 2^-30 of themselves: with the 24
// bits of a float the borders between 10^5 tokens of like weight would move by
// some 10^-5 of a token's width, and with them one token in some ten thousand
// rows; in 64 bits (half the rate, its conversions a quarter) the scan of 512
// rows of 128256 took 100 us.
//
// Rows that this does not serve go through sample_plain, which finds the cut digit
// by digit from histograms of the floats' order, one workgroup in six to ten
// readings of the row:
//   an infinite logit; a temperature of 2^60 and more;
//   a segment whose largest logit has |x log2(e) / T| of 4096 and more: a finite
//     mask (-1e9, say) over a whole segment of a row that is not masked elsewhere, a
//     logit of 30 at T = 0.01;
//   more tokens in the cut's bin than its list holds: thousands of equal logits, but
//     also ordinary ones at high temperatures or of large vocabularies (of normal
//     logits of deviation 2.2 with top-p 0.9: 128256 at T = 3, 262144 at 1.5).
// One such row of 128256 logits takes 570 to 770 us, of 262144 1.5 ms; 64 of them
// take 0.8 to 0.9 and 2.1 ms.
#include "qk_internal.h"

namespace qk {
namespace {

hipStream_t S(qk_stream s) { return static_cast<hipStream_t>(s); }

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kSegment = 32 * kThreads;
constexpr int kMaxSegments = (1 << 19) / kSegment;
constexpr int kOctave = 16, kBins = 48 * kOctave;
constexpr int kFine = 128;   // steps of an octave in the weights' table
constexpr int kList = 2048;
constexpr int kRank = 8;     // of kList, whose end a step of them does not pass
static_assert(kList % kRank == 0, "");
constexpr int kGather = 8;   // segments whose bins a thread loads at once
constexpr double kUnit = 17592186044416.;   // 2^44: sample_plain's weights, of which 2^19 stay below 2^64

// A segment's largest logit, its lowest index (of greedy rows), and the power of
// two that its weights are below (kNone: no logit above -inf, kFar: out of range).
struct SegmentHead {
    float best;
    int at, e, pad;
};
constexpr int kNone = -0x40000000, kFar = 0x40000000;

// A row as its segments leave it.
struct RowPlan {
    double least;    // the weight that min-p asks for, in units of 2^(e - 31)
    float best;
    int e;           // the row's power of two
    int way;         // kDone: the token is out; kPlain: for sample_plain; kBinned
    int counted;     // top-k leaves tokens out
    int bin_k;       // the bin of top-k's last token, kBins without
    int bin_m, m_hi; // the bins around `least` (two where it is near a border), kBins without
    int lo, hi;      // the bins to list first (lo > hi: none)
};
constexpr int kDone = 0, kPlain = 1, kBinned = 2;

struct SampleArgs {
    const float *logits;
    int64_t ldv;
    int n;
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t *top_k;
    int32_t *out;
    float *prob;
    SegmentHead *heads;   // [rows][segments]
    RowPlan *plans;       // [rows]
    uint64_t *mass;       // [rows][segments][kBins]: of bin i in units of 2^(segment's e - 31 - i / 16)
    double *cum;          // [rows][kBins]: sums of the row's bins up to each, in units of 2^(e - 31)
    uint64_t *list;       // [rows][kList] tokens of the bins asked for
    uint32_t *count;      // [rows][segments][kBins] tokens, of rows with top-k
    uint32_t *counts;     // [rows][kBins]: sums up to each
    int *listed;          // [rows]
    int segments, wide;   // wide: rows are 16-byte aligned
};

// NaN as -inf; -0 as 0 in the order-preserving key.
__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// A row's parameters; greedy: only the first token is left.
struct RowParams {
    float t, p, mp;
    int k;
    bool greedy;
};
__device__ __forceinline__ RowParams row_params(const SampleArgs &a, int row) {
    RowParams r{a.temperature ? a.temperature[row] : 1.f, a.top_p ? a.top_p[row] : 1.f, a.min_p ? a.min_p[row] : 0.f,
                a.top_k ? a.top_k[row] : 0, false};
    r.greedy = !(r.t > 0.f) || !(r.p > 0.f) || !(r.mp <= 1.f) || r.k == 1;
    return r;
}

// Inclusive sums over a wave's lanes of a 64-bit type: the rows of 16 by DPP
// shifts, then the rows before (a lane without a source adds 0).
template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T dpp_part(T v) {
    static_assert(sizeof(T) == 8, "two dwords");
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, ROWS, 0xF, false);
    return __builtin_bit_cast(T, static_cast<uint64_t>(hi) << 32 | lo);
}
template <class T>
__device__ __forceinline__ T wave_scan(T v) {
    v += dpp_part<0x111, 0xF>(v);   // row_shr 1, 2, 4, 8
    v += dpp_part<0x112, 0xF>(v);
    v += dpp_part<0x114, 0xF>(v);
    v += dpp_part<0x118, 0xF>(v);
    v += dpp_part<0x142, 0xA>(v);   // row_bcast 15 into rows 1 and 3
    v += dpp_part<0x143, 0xC>(v);   // row_bcast 31 into rows 2 and 3
    return v;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false)));
}
// The largest of a wave's values, in every lane.
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    v = dpp_max<0x118, 0xF>(dpp_max<0x114, 0xF>(dpp_max<0x112, 0xF>(dpp_max<0x111, 0xF>(v))));
    v = dpp_max<0x143, 0xC>(dpp_max<0x142, 0xA>(v));
    return __builtin_amdgcn_readlane(static_cast<int>(v), 63);
}
// The last lane's value of a 64-bit type.
template <class T>
__device__ __forceinline__ T wave_last(T v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(b), 63);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), 63);
    return __builtin_bit_cast(T, static_cast<uint64_t>(hi) << 32 | lo);
}

// -------------------------------------------------- rows digit by digit --

struct RowScale {
    float top;
    double t;
};
__device__ __forceinline__ uint64_t weight(float x, const RowScale &r) {
    if (x == -INFINITY) return 0;
    if (r.top == INFINITY) return x == INFINITY ? static_cast<uint64_t>(kUnit) : 0;
    return static_cast<uint64_t>(rint(exp((static_cast<double>(x) - r.top) / r.t) * kUnit));
}

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
    return wave_last(wave_scan(v));
}
// Sum over the workgroup, to every thread.
__device__ __forceinline__ uint64_t block_sum_u64(uint64_t v, uint64_t *scratch) {
    v = wave_sum_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t s = 0;
    #pragma unroll
    for (int w = 0; w < kWaves; ++w) s += scratch[w];
    return s;
}

// The largest bin b of 256 at which the sum of bins 255 .. b reaches target
// (above: the sum of the bins over it); bin 0 if none does.
__device__ __forceinline__ void find_bin(const uint64_t *hist, double target, int &bin, uint64_t &above) {
    uint64_t sum = 0;
    int b = 255;
    for (; b > 0; --b) {
        if (static_cast<double>(sum + hist[b]) >= target) break;
        sum += hist[b];
    }
    bin = b;
    above = sum;
}

struct PlainShared {
    uint64_t hist[256];
    uint64_t scratch[kWaves];
    uint64_t found_above;
    int found_bin, found_index;
};

// A row whose largest logit is best, by all threads of the workgroup.
__device__ __forceinline__ void sample_plain(const SampleArgs &a, const RowParams &r, int row, float best,
                                             PlainShared &sh) {
    uint64_t *const hist = sh.hist, *const scratch = sh.scratch;
    uint64_t &found_above = sh.found_above;
    int &found_bin = sh.found_bin, &found_index = sh.found_index;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float *x = a.logits + static_cast<int64_t>(row) * a.ldv;
    const float p = r.p, mp = r.mp;
    const int k = r.k;
    const RowScale rs{best, r.t};

    uint32_t limit = 0;             // keys above it are kept, and at it the first `ties`
    uint64_t ties = ~0ull;
    if (k > 0 && k < a.n) {
        uint32_t prefix = 0;
        uint64_t need = k;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < a.n; i += kThreads) {
                const uint32_t key = key_of(clean(x[i]));
                if (shift == 24 || key >> (shift + 8) == prefix) atomicAdd(reinterpret_cast<unsigned long long *>(&hist[key >> shift & 255]), 1ull);
            }
            __syncthreads();
            if (tid == 0) {
                int b;
                uint64_t above;
                find_bin(hist, static_cast<double>(need), b, above);
                found_bin = b;
                found_above = above;
            }
            __syncthreads();
            need -= found_above;
            prefix = prefix << 8 | static_cast<uint32_t>(found_bin);
        }
        limit = prefix;
        ties = need;
    }
    if (p < 1.f) {
        // Weights at the limit count `ties` times.
        uint64_t mine = 0;
        for (int i = tid; i < a.n; i += kThreads) {
            const float v = clean(x[i]);
            if (key_of(v) > limit || ties == ~0ull) mine += weight(v, rs);
        }
        uint64_t total = block_sum_u64(mine, scratch);
        const uint64_t at_limit = ties == ~0ull ? 0 : ties * weight(value_of(limit), rs);
        total += at_limit;
        const double target = static_cast<double>(p) * static_cast<double>(total);
        uint32_t prefix = 0;
        uint64_t before = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < a.n; i += kThreads) {
                const float v = clean(x[i]);
                const uint32_t key = key_of(v);
                if ((key > limit || ties == ~0ull) && (shift == 24 || key >> (shift + 8) == prefix))
                    atomicAdd(reinterpret_cast<unsigned long long *>(&hist[key >> shift & 255]), static_cast<unsigned long long>(weight(v, rs)));
            }
            __syncthreads();
            if (tid == 0) {
                if (at_limit && (shift == 24 || limit >> (shift + 8) == prefix)) hist[limit >> shift & 255] += at_limit;
                // Sums from the top of the row, before and within this digit.
                uint64_t sum = before;
                int b = 255;
                for (; b > 0; --b) {
                    if (hist[b] && static_cast<double>(sum + hist[b]) >= target) break;
                    sum += hist[b];
                }
                found_bin = b;
                found_above = sum;
            }
            __syncthreads();
            before = found_above;
            prefix = prefix << 8 | static_cast<uint32_t>(found_bin);
        }
        // Of equal weights w after a sum `before`: kept while the sum is below
        // the target.
        const uint64_t w = weight(value_of(prefix), rs);
        uint64_t count = 0;
        if (w > 0 && static_cast<double>(before) < target) {
            const double n = ceil((target - static_cast<double>(before)) / static_cast<double>(w));
            count = static_cast<uint64_t>(n);
            while (count > 0 && static_cast<double>(before + (count - 1) * w) >= target) --count;
            while (static_cast<double>(before + count * w) < target) ++count;
        }
        ties = prefix == limit && ties != ~0ull ? min(ties, count) : count;
        limit = prefix;
    }
    // The index of the last kept tie.
    int cut = 0x7FFFFFFF;
    if (ties != ~0ull) {
        uint64_t seen = 0;
        cut = -1;
        for (int i0 = 0; i0 < a.n && seen < ties; i0 += kThreads) {
            const int i = i0 + tid;
            const bool tie = i < a.n && key_of(clean(x[i])) == limit;
            const uint64_t mask = __builtin_amdgcn_ballot_w64(tie);
            __syncthreads();
            if (lane == 0) scratch[wave] = __builtin_popcountll(mask);
            if (tid == 0) found_index = -1;
            __syncthreads();
            uint64_t base = seen, all = 0;
            for (int w = 0; w < kWaves; ++w) {
                if (w < wave) base += scratch[w];
                all += scratch[w];
            }
            const uint64_t rank = base + __builtin_popcountll(mask & ((1ull << lane) - 1));
            if (tie && rank < ties) atomicMax(&found_index, i);
            __syncthreads();
            cut = max(cut, found_index);
            seen += all;
        }
    }
    const double least = static_cast<double>(mp) * kUnit;
    auto kept = [&](int i) -> uint64_t {
        const float v = clean(x[i]);
        const uint32_t key = key_of(v);
        if (ties != ~0ull && !(key > limit || (key == limit && i <= cut))) return 0;
        const uint64_t w = weight(v, rs);
        return static_cast<double>(w) >= least ? w : 0;
    };
    uint64_t mine = 0;
    for (int i = tid; i < a.n; i += kThreads) mine += kept(i);
    const uint64_t total = block_sum_u64(mine, scratch);
    const double u = a.uniform[row], ut = u * static_cast<double>(total);
    uint64_t target = ut > 0. ? (ut < static_cast<double>(total) ? static_cast<uint64_t>(ut) : total - 1) : 0;
    target = min(target, total - 1);
    uint64_t sum = 0;
    for (int i0 = 0; i0 < a.n; i0 += kThreads) {
        const int i = i0 + tid;
        const uint64_t w = i < a.n ? kept(i) : 0;
        uint64_t upto = wave_scan(w);
        __syncthreads();
        if (lane == 63) scratch[wave] = upto;
        __syncthreads();
        uint64_t all = 0;
        for (int v = 0; v < kWaves; ++v) {
            if (v < wave) upto += scratch[v];
            all += scratch[v];
        }
        upto += sum;
        sum += all;
        if (w > 0 && upto > target && upto - w <= target) {
            a.out[row] = i;
            if (a.prob) a.prob[row] = static_cast<float>(static_cast<double>(w) / static_cast<double>(total));
        }
        if (sum > target) break;
    }
}

// ------------------------------------------------------------ weights --

constexpr double kLog2E = 1.4426950408889634074;

// log2(e) / T as two floats.
struct Slope {
    float hi, lo;
};
__device__ __forceinline__ Slope slope_of(float t) {
    const double c = kLog2E / static_cast<double>(t);
    const float hi = static_cast<float>(c);
    return {hi, static_cast<float>(c - static_cast<double>(hi))};
}

// The power of two above a segment's weights by its largest logit: t = x c is
// below it for every x, since p is monotone.  Slopes below 2^-60 (temperatures of
// 2^60 and more) are out of range too: x c ends in 0 for an x that the bins'
// intervals still tell from 0, and an infinite temperature leaves these without
// numbers.
__device__ __forceinline__ int exponent_of(float best, const Slope &c) {
    const float p = best * c.hi;
    return best == -INFINITY ? kNone : !(fabsf(p) < 4096.f) || c.hi < 0x1p-60f ? kFar : static_cast<int>(floorf(p)) + 1;
}

// t = x c = p + lo to some 48 bits, p = (g + 1/2) / 128 + y with y exact, f = 128
// e - 1 - g >= 0 the fine step below 2^e, or -1 from 47 octaves on (and for
// -inf).  y with lo stays within 1/256 + 2^-12.
struct Depth {
    float y;
    int f;
    __device__ __forceinline__ int bin() const { return f >> 3; }
};
static_assert(kFine == 8 * kOctave, "Depth::bin");
__device__ __forceinline__ Depth depth_of(float x, const Slope &c, int e) {
    const float p = x * c.hi, lo = fmaf(x, c.lo, fmaf(x, c.hi, -p));
    const float g = floorf(p * kFine);
    const float y = fmaf(g, -1.f / kFine, p) + (lo - 0.5f / kFine);
    const int top = kFine * e;
    const bool in = g >= static_cast<float>(top - 47 * kFine);
    return {y, in ? top - 1 - static_cast<int>(g) : -1};
}

// The weight of a step f in units of 2^(e - 31 - f / 128): 2^-((f % 128) + 1/2)/128
// from the table (as an integer and as a float), times 1 + z with z = e^(y ln 2) -
// 1 by its Taylor polynomial (the next term is 2^-38), which is so small that 24
// bits of it are 32 of the weight.
__device__ __forceinline__ uint32_t unit_weight(const Depth &d, const uint2 *table) {
    const uint2 t = table[d.f & (kFine - 1)];
    float z = fmaf(d.y, 5.5504108664821580e-2f, 2.4022650695910072e-1f);
    z = fmaf(d.y, z, 6.9314718055994531e-1f) * d.y;
    return t.x + static_cast<uint32_t>(static_cast<int>(z * __builtin_bit_cast(float, t.y)));
}

__device__ __forceinline__ void fill_table(uint2 *table) {
    if (threadIdx.x < kFine) {
        const double w = exp2(31. - (static_cast<double>(threadIdx.x) + 0.5) / kFine);
        table[threadIdx.x] = make_uint2(static_cast<uint32_t>(rint(w)), __builtin_bit_cast(uint32_t, static_cast<float>(w)));
    }
}

__device__ __forceinline__ void load_quad(const float *x, int i, int n, int wide, float (&v)[4]) {
    if (wide && i + 3 < n) {
        const float4 q = *reinterpret_cast<const float4 *>(x + i);
        v[0] = clean(q.x), v[1] = clean(q.y), v[2] = clean(q.z), v[3] = clean(q.w);
    } else {
        #pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i + e < n ? clean(x[i + e]) : -INFINITY;
    }
}

constexpr int kQuads = kSegment / (4 * kThreads);
__device__ __forceinline__ int quad_at(int seg, int j) {
    return seg * kSegment + (j * kThreads + static_cast<int>(threadIdx.x)) * 4;
}

// --------------------------------------------------------------- scan --
//
// Bound by its arithmetic (an exponential to 31 bits and an LDS atomic a logit):
// 512 rows of 128256 in 70 us, 3.7 TB/s of them, where reading them alone is 55; of
// one row 8 workgroups, 8.5 us.  Two or four copies of the histogram, for fewer
// conflicts, took as long.

__global__ __launch_bounds__(kThreads) void sample_scan_kernel(SampleArgs a) {
    __shared__ unsigned long long mass[kBins];
    __shared__ uint32_t count[kBins];
    __shared__ uint2 table[kFine];
    __shared__ float best_of[kWaves];
    __shared__ int lowest;
    const int row = blockIdx.y, seg = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float *x = a.logits + static_cast<int64_t>(row) * a.ldv;
    float v[kQuads][4];
    #pragma unroll
    for (int j = 0; j < kQuads; ++j) load_quad(x, quad_at(seg, j), a.n, a.wide, v[j]);
    const RowParams r = row_params(a, row);
    fill_table(table);
    for (int i = tid; i < kBins; i += kThreads) {
        mass[i] = 0;
        count[i] = 0;
    }
    if (tid == 0) {
        lowest = 0x7FFFFFFF;
        if (seg == 0) a.listed[row] = 0;
    }
    float best = -INFINITY;
    #pragma unroll
    for (int j = 0; j < kQuads; ++j)
        #pragma unroll
        for (int k = 0; k < 4; ++k) best = fmaxf(best, v[j][k]);
    #pragma unroll
    for (int off = 32; off > 0; off >>= 1) best = fmaxf(best, __shfl_xor(best, off));
    if (lane == 0) best_of[wave] = best;
    __syncthreads();
    #pragma unroll
    for (int w = 0; w < kWaves; ++w) best = fmaxf(best, best_of[w]);
    const Slope c = slope_of(r.t);
    const int e = exponent_of(best, c);
    const int64_t me = static_cast<int64_t>(row) * a.segments + seg;
    if (r.greedy) {
        int at = 0x7FFFFFFF;
        #pragma unroll
        for (int j = kQuads - 1; j >= 0; --j)
            #pragma unroll
            for (int k = 3; k >= 0; --k) at = v[j][k] == best ? quad_at(seg, j) + k : at;
        if (at < a.n) atomicMin(&lowest, at);
        __syncthreads();
        if (tid == 0) a.heads[me] = SegmentHead{best, lowest, kNone, 0};
        return;
    }
    if (tid == 0) a.heads[me] = SegmentHead{best, 0, e, 0};
    if (e == kNone || e == kFar) return;
    const bool counted = r.k > 0 && r.k < a.n;
    #pragma unroll
    for (int j = 0; j < kQuads; ++j)
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
            const Depth d = depth_of(v[j][k], c, e);
            if (d.f >= 0) {
                atomicAdd(&mass[d.bin()], static_cast<unsigned long long>(unit_weight(d, table)));
                if (counted) atomicAdd(&count[d.bin()], 1u);
            }
        }
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads) {
        a.mass[me * kBins + i] = mass[i];
        if (counted) a.count[me * kBins + i] = count[i];
    }
}

// --------------------------------------------------------------- plan --
//
// Bound by the latency of the histograms' loads and of a scan of 768 sums in 64
// bits: 7 us for a row, 9 for 512.

// Octaves and bins from a segment's power of two down to the row's (64: no bin
// of it is left).
__device__ __forceinline__ int octaves_down(int e, int segment_e) {
    return segment_e == kNone ? 64 : min(e - segment_e, 64);
}

// The first of kBins sums to reach target (rounding may leave two such steps:
// the lower), kBins if none does; by kBins threads or fewer, several bins each.
template <int THREADS, class T>
__device__ __forceinline__ int first_reaching(const T *cum, double target, int *found) {
    __syncthreads();
    if (threadIdx.x == 0) *found = kBins;
    __syncthreads();
    #pragma unroll
    for (int i = threadIdx.x; i < kBins; i += THREADS)
        if (static_cast<double>(cum[i]) >= target && (i == 0 || static_cast<double>(cum[i - 1]) < target))
            atomicMin(found, i);
    __syncthreads();
    return *found;
}

__global__ __launch_bounds__(kBins) void sample_plan_kernel(SampleArgs a) {
    __shared__ SegmentHead head[kMaxSegments];
    __shared__ double cum[kBins];
    __shared__ uint32_t counts[kBins];
    __shared__ uint2 table[kFine];
    __shared__ double sums[kBins / 64];
    __shared__ uint64_t tokens[kBins / 64];
    __shared__ int found;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const RowParams r = row_params(a, row);
    const int64_t first = static_cast<int64_t>(row) * a.segments;
    if (tid < a.segments) head[tid] = a.heads[first + tid];
    fill_table(table);
    __syncthreads();
    RowPlan st{0., -INFINITY, kNone, kBinned, r.k > 0 && r.k < a.n, kBins, kBins, kBins, 0, -1};
    int at = 0x7FFFFFFF;
    bool far = false;
    for (int g = 0; g < a.segments; ++g) {
        const SegmentHead h = head[g];
        arg_better(st.best, at, h.best, h.at);
        far = far || h.e == kFar;
        if (h.e != kFar) st.e = max(st.e, h.e);
    }
    if (st.best == -INFINITY || r.greedy) {
        if (tid == 0) {
            a.out[row] = st.best == -INFINITY ? 0 : at;
            if (a.prob) a.prob[row] = st.best == -INFINITY ? 0.f : 1.f;
        }
        st.way = kDone;
    } else if (far) {
        st.way = kPlain;
    } else {
        // Bin tid of the row: of a segment m octaves lower, its bin tid - 16 m.
        // The integers of one bin have one unit, so they add up exactly.
        uint64_t sum = 0, n = 0;
        for (int g0 = 0; g0 < a.segments; g0 += kGather) {
            uint64_t w[kGather];
            uint32_t m[kGather];
            #pragma unroll
            for (int k = 0; k < kGather; ++k) {   // all loads first
                const int g = min(g0 + k, a.segments - 1), from = tid - kOctave * octaves_down(st.e, head[g].e);
                const bool in = g0 + k < a.segments && from >= 0;
                const int64_t i = (first + g) * kBins + max(from, 0);
                w[k] = in ? a.mass[i] : 0;
                m[k] = in && st.counted ? a.count[i] : 0;
            }
            #pragma unroll
            for (int k = 0; k < kGather; ++k) {
                sum += w[k];
                n += m[k];
            }
        }
        const double mine = wave_scan(ldexp(static_cast<double>(sum), -(tid / kOctave)));
        const uint64_t upto = wave_scan(n);
        if (lane == 63) {
            sums[wave] = mine;
            tokens[wave] = upto;
        }
        __syncthreads();
        double before = 0.;
        uint64_t earlier = 0;
        for (int w = 0; w < wave; ++w) {
            before += sums[w];
            earlier += tokens[w];
        }
        cum[tid] = before + mine;
        counts[tid] = static_cast<uint32_t>(earlier + upto);
        a.cum[static_cast<int64_t>(row) * kBins + tid] = cum[tid];
        if (st.counted) {
            a.counts[static_cast<int64_t>(row) * kBins + tid] = counts[tid];
            st.bin_k = first_reaching<kBins>(counts, static_cast<double>(r.k), &found);
        }
        if (r.mp > 0.f) {
            const Depth d = depth_of(st.best, slope_of(r.t), st.e);
            st.least = ldexp(static_cast<double>(r.mp) * unit_weight(d, table), -(d.f / kFine));
            const double below = (d.f + 0.5) / kFine - d.y - log2(static_cast<double>(r.mp));
            // A token's bin goes by p alone, which is off by 2^-12 octaves at most.
            auto bin_at = [](double d) { return static_cast<int>(fmin(fmax(d, 0.), 48.) * kOctave); };
            st.bin_m = bin_at(below - 0x1p-11);
            st.m_hi = bin_at(below + 0x1p-11);
        }
        if (st.bin_k < kBins) {
            st.lo = counts[st.bin_k] <= kList ? 0 : st.bin_k;   // all that top-k leaves, where it fits the list
            st.hi = st.bin_k;
        } else {
            __syncthreads();
            const double target = static_cast<double>(r.p) * cum[kBins - 1];
            const int bin = min(st.bin_m, r.p < 1.f ? first_reaching<kBins>(cum, target, &found) : kBins);
            if (bin < kBins) {
                st.lo = bin;
                st.hi = bin == st.bin_m ? st.m_hi : bin;
            }
        }
    }
    if (tid == 0) a.plans[row] = st;
}

// ------------------------------------------------------------ collect --
//
// 512 rows of 128256 in 40 us, from the caches in part (6.6 TB/s); one row 5 to 6.

__device__ __forceinline__ uint64_t packed(float x, int i) {
    return static_cast<uint64_t>(key_of(x)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}

// Logits that may lie in a segment's bins lo .. hi: their interval, widened by
// more than the roundings of the bins' arithmetic, so few get the exact test.
struct Range {
    Slope c;
    int e, lo, hi;
    float low, high;
};
__device__ __forceinline__ Range range_of(int lo, int hi, float t, int e) {
    const double c = kLog2E / static_cast<double>(t);
    const double high = (e - lo * (1. / kOctave)) / c, low = (e - (hi + 1) * (1. / kOctave)) / c;
    return {slope_of(t), e, lo, hi, static_cast<float>(low - 1e-6 * (fabs(low) + 1e-20)),
            static_cast<float>(high + 1e-6 * (fabs(high) + 1e-20))};
}

// The tokens of a quad within a range, into a list of the workgroup.
__device__ __forceinline__ void list_quad(const float (&v)[4], int i, const Range &in, uint64_t *list, int *listed) {
    #pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (!(v[k] >= in.low && v[k] <= in.high)) continue;
        const Depth d = depth_of(v[k], in.c, in.e);
        if (d.f >= 0 && d.bin() >= in.lo && d.bin() <= in.hi) {
            const int slot = atomicAdd(listed, 1);
            if (slot < kList) list[slot] = packed(v[k], i + k);
        }
    }
}

__global__ __launch_bounds__(kThreads) void sample_collect_kernel(SampleArgs a) {
    __shared__ uint64_t list[kList];
    __shared__ int listed, base;
    const int row = blockIdx.y, seg = blockIdx.x, tid = threadIdx.x;
    const float *x = a.logits + static_cast<int64_t>(row) * a.ldv;
    const RowPlan &st = a.plans[row];
    const SegmentHead &head = a.heads[static_cast<int64_t>(row) * a.segments + seg];
    if (st.way != kBinned || st.lo > st.hi || head.e == kNone) return;
    const int shift = kOctave * octaves_down(st.e, head.e);
    if (st.hi < shift) return;
    float v[kQuads][4];
    #pragma unroll
    for (int j = 0; j < kQuads; ++j) load_quad(x, quad_at(seg, j), a.n, a.wide, v[j]);
    const Range in = range_of(st.lo - shift, st.hi - shift, a.temperature ? a.temperature[row] : 1.f, head.e);
    if (tid == 0) listed = 0;
    __syncthreads();
    #pragma unroll
    for (int j = 0; j < kQuads; ++j) list_quad(v[j], quad_at(seg, j), in, list, &listed);
    __syncthreads();
    const int n = listed;
    if (n == 0) return;
    if (tid == 0) base = atomicAdd(&a.listed[row], n);
    __syncthreads();
    for (int i = tid; i < min(n, kList); i += kThreads)
        if (base + i < kList) a.list[static_cast<int64_t>(row) * kList + base + i] = list[i];
}

// --------------------------------------------------------------- pick --
//
// A row's steps one after the other: what top-k leaves picked from the list alone
// 5 to 6 us (one row), a list's cut and the segment looked over 12 to 20; 512 rows
// by nucleus, two workgroups a CU, 32 to 38.

struct PickShared {
    uint64_t list[kList];         // tokens: the key's bits, then the index's complement
    uint64_t some[kList];         // those of them that are ordered
    uint64_t ordered[kList];
    double cum[kBins];
    uint64_t part_mass[kThreads]; // of the list in kThreads parts of its logits' range
    uint32_t part_count[kThreads];
    uint2 table[kFine];
    SegmentHead head[kMaxSegments];
    unsigned long long kept[kMaxSegments];   // listed kept weight of each segment
    double kept_all[kMaxSegments];           // kept weight of each segment
    uint64_t wave_mass[kWaves], wave_count[kWaves];
    uint64_t quads[kQuads * kWaves];
    uint64_t base_mass, base_count;
    uint32_t key_high, key_low;
    int listed, found, picked;
};

// Sums over the workgroup's threads up to each (inclusive) of a pair.
__device__ __forceinline__ void block_scan(uint64_t &mass, uint64_t &count, PickShared &s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    mass = wave_scan(mass);
    count = wave_scan(count);
    __syncthreads();
    if (lane == 63) {
        s.wave_mass[wave] = mass;
        s.wave_count[wave] = count;
    }
    __syncthreads();
    #pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        mass += w < wave ? s.wave_mass[w] : 0;
        count += w < wave ? s.wave_count[w] : 0;
    }
}

// The largest number i of the threads that say so (i grows with the thread), into
// *found: one atomic a wave, since a word's follow each other.
__device__ __forceinline__ void last_of(bool yes, int i, int *found) {
    const uint64_t all = __builtin_amdgcn_ballot_w64(yes);
    if (yes && !(all >> (threadIdx.x & 63) >> 1)) atomicMax(found, i);
}

// A row by its segments' histograms and its list, by all threads of the
// workgroup; false: it is one for sample_plain.
__device__ __forceinline__ bool sample_binned(const SampleArgs &a, const RowParams &r, const RowPlan &st, int row,
                                              PickShared &s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float *x = a.logits + static_cast<int64_t>(row) * a.ldv;
    const int64_t first = static_cast<int64_t>(row) * a.segments;
    const int e = st.e, listed = st.lo <= st.hi ? a.listed[row] : 0;
    if (listed > kList) return false;
    fill_table(s.table);
    if (tid < a.segments) s.head[tid] = a.heads[first + tid];
    if (tid < kMaxSegments) s.kept[tid] = 0;
    if (tid == 0) s.listed = listed;
    for (int i = tid; i < listed; i += kThreads) s.list[i] = a.list[static_cast<int64_t>(row) * kList + i];
    for (int i = tid; i < kBins; i += kThreads) s.cum[i] = a.cum[static_cast<int64_t>(row) * kBins + i];
    const Slope c = slope_of(r.t);
    __syncthreads();

    // Tokens of other bins, by reading the row; false: more than the list holds.
    auto collect = [&](int lo, int hi) {
        __syncthreads();
        if (tid == 0) s.listed = 0;
        __syncthreads();
        for (int g = 0; g < a.segments; ++g) {
            const int down = octaves_down(e, s.head[g].e) * kOctave;
            if (s.head[g].e == kNone || hi < down) continue;
            const Range in = range_of(lo - down, hi - down, r.t, s.head[g].e);
            #pragma unroll 1
            for (int j = 0; j < kQuads; ++j) {
                float v[4];
                load_quad(x, quad_at(g, j), a.n, a.wide, v);
                list_quad(v, quad_at(g, j), in, s.list, &s.listed);
            }
        }
        __syncthreads();
        return s.listed <= kList;
    };
    // A listed token's segment, and its weight in the row's units of 2^(e - 31)
    // (exact, for min-p) and as an integer of 2^(e - 47).
    auto segment_of = [&](uint64_t t) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(t)) / kSegment; };
    auto weight_of = [&](uint64_t t, uint64_t &whole) {
        const int eg = s.head[segment_of(t)].e;
        const Depth d = depth_of(value_of(static_cast<uint32_t>(t >> 32)), c, eg);
        const uint32_t m = unit_weight(d, s.table);
        const int below = e - eg + d.f / kFine;
        whole = below < 48 ? static_cast<uint64_t>(m) << 16 >> below : 0;
        return ldexp(static_cast<double>(m), -below);
    };
    constexpr double kWhole = 0x1p-16;   // 2^(e - 47) in units of 2^(e - 31)
    // The first m tokens of a list, the largest first, into s.ordered: a token a
    // thread, counting the larger ones, eight at a read's wait.
    auto order = [&](uint64_t *from, int m) {
        if (tid < kRank && m + tid < kList) from[m + tid] = 0;
        __syncthreads();
        for (int i = tid; i < m; i += kThreads) {
            const uint64_t t = from[i];
            int rank = 0;
            for (int k = 0; k < m; k += kRank)
                #pragma unroll
                for (int j = 0; j < kRank; ++j) rank += from[k + j] > t;
            s.ordered[rank] = t;
        }
        __syncthreads();
    };
    // The last listed token that is kept, in the tokens' order: as many as
    // `left`, while the sum before is below the target and the weight is not
    // below the least; ~0 if none is.  A list of more tokens than threads is cut
    // into kThreads parts of its range first, of which one then holds the cut.
    auto cut_of = [&](double above, double target, int left, double least) -> uint64_t {
        const int n = s.listed;
        auto stays = [&](uint64_t t, uint64_t &w) { return weight_of(t, w) >= least; };
        float high = 0.f, scale = 0.f;
        auto part_of = [&](uint64_t t) {
            return min(static_cast<int>((high - value_of(static_cast<uint32_t>(t >> 32))) * scale), kThreads - 1);
        };
        const bool parts = n > kThreads;
        uint64_t base_mass = 0, base_count = 0;
        int part = 0;
        if (parts) {
            __syncthreads();
            s.part_mass[tid] = 0;
            s.part_count[tid] = 0;
            if (tid == 0) {
                s.key_high = 0;
                s.key_low = ~0u;
                s.found = -1;
            }
            __syncthreads();
            uint32_t top = 0, low = ~0u;
            for (int i = tid; i < n; i += kThreads) {
                const uint32_t k = static_cast<uint32_t>(s.list[i] >> 32);
                top = max(top, k);
                low = min(low, k);
            }
            top = wave_max_u32(top);
            low = ~wave_max_u32(~low);
            if (lane == 0) {   // a wave at a time: 64 lanes' atomics on one word follow each other
                atomicMax(&s.key_high, top);
                atomicMin(&s.key_low, low);
            }
            __syncthreads();
            high = value_of(s.key_high);
            scale = fminf((kThreads - 1) / (high - value_of(s.key_low)), 1e30f);   // 1e30: all alike, one part
            for (int i = tid; i < n; i += kThreads) {
                uint64_t w;
                if (!stays(s.list[i], w)) continue;
                atomicAdd(reinterpret_cast<unsigned long long *>(&s.part_mass[part_of(s.list[i])]), static_cast<unsigned long long>(w));
                atomicAdd(&s.part_count[part_of(s.list[i])], 1u);
            }
            __syncthreads();
            uint64_t mass = s.part_mass[tid], count = s.part_count[tid];
            const uint64_t own_mass = mass, own_count = count;
            block_scan(mass, count, s);
            const uint64_t mass0 = mass - own_mass, count0 = count - own_count;
            last_of(own_count > 0 && count0 < static_cast<uint64_t>(left) &&
                        above + static_cast<double>(mass0) * kWhole < target,
                    tid, &s.found);
            __syncthreads();
            part = s.found;
            if (part < 0) return ~0ull;
            if (tid == part) {
                s.base_mass = mass0;
                s.base_count = count0;
            }
        }
        __syncthreads();
        if (parts) {
            base_mass = s.base_mass;
            base_count = s.base_count;
        }
        const bool all = !parts && least <= 0.;
        uint64_t *const some = all ? s.list : s.some;
        if (!all) {
            if (tid == 0) s.picked = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) {
                uint64_t w;
                if (stays(s.list[i], w) && (!parts || part_of(s.list[i]) == part)) some[atomicAdd(&s.picked, 1)] = s.list[i];
            }
            __syncthreads();
        }
        const int m = all ? n : s.picked;
        order(some, m);
        if (tid == 0) s.found = -1;
        for (int i0 = 0; i0 < m; i0 += kThreads) {
            const int i = i0 + tid;
            uint64_t own = 0, count = i < m;
            if (i < m) weight_of(s.ordered[i], own);
            uint64_t mass = own;
            block_scan(mass, count, s);
            mass += base_mass;
            last_of(i < m && base_count + i < static_cast<uint64_t>(left) &&
                        above + static_cast<double>(mass - own) * kWhole < target,
                    i, &s.found);
            base_mass = s.wave_mass[kWaves - 1] + base_mass;   // of full rounds only: the last has no next
            #pragma unroll
            for (int w = 0; w < kWaves - 1; ++w) base_mass += s.wave_mass[w];
        }
        __syncthreads();
        return s.found < 0 ? ~0ull : s.ordered[s.found];
    };
    // All that top-k leaves is listed, a token a thread: both cuts from one order,
    // and the token from the kept ones themselves.
    if (st.bin_k < kBins && st.lo == 0 && listed <= kThreads) {
        order(s.list, listed);
        const uint64_t mine = tid < listed ? s.ordered[tid] : 0;
        uint64_t own = 0, upto = 0, none = 0;
        bool stays = false;
        if (tid < listed) stays = weight_of(mine, own) >= st.least && tid < r.k;
        if (tid >= r.k) own = 0;
        upto = own;
        block_scan(upto, none, s);
        uint64_t total = 0;
        #pragma unroll
        for (int w = 0; w < kWaves; ++w) total += s.wave_mass[w];
        if (r.p < 1.f) stays = stays && static_cast<double>(upto - own) < static_cast<double>(r.p) * static_cast<double>(total);
        s.some[tid] = stays ? own : 0;
        if (tid == 0) s.picked = 0;
        __syncthreads();
        last_of(stays, tid + 1, &s.picked);
        __syncthreads();
        const int keep = s.picked;
        uint64_t z = 0, before = 0;
        for (int k = 0; k < keep; ++k) {   // in index order: those with a larger complement
            const uint64_t w = s.some[k];
            z += w;
            before += static_cast<uint32_t>(s.ordered[k]) > static_cast<uint32_t>(mine) ? w : 0;
        }
        const double goal = a.uniform[row] * static_cast<double>(z);
        const uint64_t want = goal > 0. ? min(goal < static_cast<double>(z) ? static_cast<uint64_t>(goal) : z, z - 1) : 0;
        if (stays && before <= want && want < before + own) {
            a.out[row] = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(mine));
            if (a.prob) a.prob[row] = static_cast<float>(static_cast<double>(own) / static_cast<double>(z));
        }
        return true;
    }
    auto left_of = [&](int lo) {
        if (st.bin_k == kBins) return s.listed;
        return min(s.listed, r.k - (lo > 0 ? static_cast<int>(a.counts[static_cast<int64_t>(row) * kBins + lo - 1]) : 0));
    };
    auto above_of = [&](int lo) { return lo > 0 ? s.cum[lo - 1] : 0.; };

    double target = INFINITY;
    int lo = st.lo <= st.hi ? st.lo : kBins;   // the list's first bin
    if (r.p < 1.f) {
        double total = s.cum[kBins - 1];
        if (st.bin_k < kBins) {   // of what top-k leaves
            const uint64_t last = cut_of(above_of(lo), INFINITY, left_of(lo), 0.);
            uint64_t mass = 0, none = 0;
            for (int i = tid; i < s.listed; i += kThreads) {
                uint64_t w;
                weight_of(s.list[i], w);
                mass += s.list[i] >= last ? w : 0;
            }
            block_scan(mass, none, s);
            mass = 0;
            #pragma unroll
            for (int w = 0; w < kWaves; ++w) mass += s.wave_mass[w];
            total = above_of(lo) + static_cast<double>(mass) * kWhole;
        }
        target = static_cast<double>(r.p) * total;
    }
    int bin = min(st.bin_k, st.bin_m);
    if (r.p < 1.f) bin = min(bin, first_reaching<kThreads>(s.cum, target, &s.found));
    int whole = kBins;      // kept: bins below `whole`, and the list's tokens down to `cut`
    uint64_t cut = ~0ull;
    if (bin < kBins) {
        if (bin < lo) {   // a smaller nucleus within a top-k beyond the list
            if (!collect(bin, bin == st.bin_m ? st.m_hi : bin)) return false;
            lo = bin;
        }
        whole = lo;
        cut = cut_of(above_of(lo), target, left_of(lo), st.least);
        for (int i = tid; i < s.listed; i += kThreads)
            if (s.list[i] >= cut) {
                uint64_t w;
                weight_of(s.list[i], w);
                atomicAdd(&s.kept[segment_of(s.list[i])], static_cast<unsigned long long>(w));
            }
    }
    __syncthreads();

    // Kept weight of each segment: its whole bins and its listed tokens.
    for (int g = wave; g < a.segments; g += kWaves) {
        const int down = octaves_down(e, s.head[g].e), n = whole - kOctave * down;
        double sum = 0.;
        if (n > 0) {
            #pragma unroll
            for (int i = 0; i < kBins; i += 64) {
                const uint64_t w = a.mass[(first + g) * kBins + i + lane];
                sum += i + lane < n ? ldexp(static_cast<double>(w), -down - (i + lane) / kOctave) : 0.;
            }
            sum = wave_last(wave_scan(sum));
        }
        if (lane == 0) s.kept_all[g] = sum + static_cast<double>(s.kept[g]) * kWhole;
    }
    __syncthreads();
    // The segment of the random number's token, and the share of its weight that
    // lies before that token.
    const double mine = lane < a.segments ? s.kept_all[lane] : 0., upto = wave_scan(mine), z = wave_last(upto);
    if (!(z > 0.)) return false;
    const double u = a.uniform[row], goal = u > 0. ? fmin(u, 1.) * z : 0.;
    const uint64_t some = __builtin_amdgcn_ballot_w64(mine > 0.), over = __builtin_amdgcn_ballot_w64(mine > 0. && goal < upto);
    const int seg = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
    const double share = (goal - (__shfl(upto, seg) - __shfl(mine, seg))) / __shfl(mine, seg);
    // The segment again, weights as integers: wave sums by quads, then the token.
    const int eg = s.head[seg].e, down = kOctave * octaves_down(e, eg);
    const bool any = cut != ~0ull;
    const float cut_x = any ? value_of(static_cast<uint32_t>(cut >> 32)) : INFINITY;
    const int cut_i = any ? static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(cut)) : -1;
    // With a cut the kept tokens are those down to it, by the logits alone: a wave
    // without any takes no exponentials.
    auto weights = [&](const float (&v)[4], int i, uint64_t (&w)[4]) {
        uint64_t sum = 0;
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
            w[k] = 0;
            if (any && !(v[k] > cut_x || (v[k] == cut_x && i + k <= cut_i))) continue;
            const Depth d = depth_of(v[k], c, eg);
            const bool kept = d.f >= 0 && (any || d.bin() + down < whole);
            w[k] = kept ? static_cast<uint64_t>(unit_weight(d, s.table)) << 16 >> (d.f / kFine) : 0;
            sum += w[k];
        }
        return sum;
    };
    float v[kQuads][4];
    #pragma unroll
    for (int j = 0; j < kQuads; ++j) load_quad(x, quad_at(seg, j), a.n, a.wide, v[j]);
    #pragma unroll
    for (int j = 0; j < kQuads; ++j) {
        uint64_t w[4];
        const uint64_t own = weights(v[j], quad_at(seg, j), w);
        const uint64_t t = __builtin_amdgcn_ballot_w64(own > 0) ? wave_scan(own) : 0;
        if (lane == 63) s.quads[j * kWaves + wave] = t;
    }
    __syncthreads();
    static_assert(kQuads * kWaves == 64, "a lane for each sum");
    const uint64_t sum = s.quads[lane], sums = wave_scan(sum), all = wave_last(sums);
    if (all == 0) return false;
    const double inside = fmax(share, 0.) * static_cast<double>(all);
    const uint64_t want = inside < static_cast<double>(all) ? min(static_cast<uint64_t>(inside), all - 1) : all - 1;
    const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sums > want));
    if (wave != at % kWaves) return true;
    uint64_t w[4];
    float q[4];
    const int i = quad_at(seg, at / kWaves);
    load_quad(x, i, a.n, a.wide, q);
    const uint64_t own = weights(q, i, w);
    uint64_t b = __shfl(sums - sum, at) + wave_scan(own) - own;
    if (b <= want && want < b + own)
        for (int k = 0; k < 4; ++k) {
            if (w[k] && b <= want && want < b + w[k]) {
                a.out[row] = i + k;
                const Depth d = depth_of(q[k], c, eg);
                if (a.prob)
                    a.prob[row] = static_cast<float>(
                        ldexp(static_cast<double>(unit_weight(d, s.table)), eg - e - d.f / kFine) / z);
            }
            b += w[k];
        }
    return true;
}

__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleArgs a) {
    __shared__ union {
        PickShared pick;
        PlainShared plain;
    } s;
    const int row = blockIdx.x;
    const RowPlan st = a.plans[row];
    if (st.way == kDone) return;
    const RowParams r = row_params(a, row);
    if (st.way == kPlain || !sample_binned(a, r, st, row, s.pick)) sample_plain(a, r, row, st.best, s.plain);
}

size_t round256(size_t b) { return (b + 255) / 256 * 256; }

// A call's arrays in its workspace; returns their bytes.
size_t lay_out(SampleArgs &a, int rows, char *ws) {
    const size_t segments = static_cast<size_t>(rows) * a.segments;
    size_t at = 0;
    auto take = [&](auto *&p, size_t n) {
        p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(ws + at);
        at += round256(n * sizeof(*p));
    };
    take(a.heads, segments);
    take(a.plans, rows);
    take(a.mass, segments * kBins);
    take(a.cum, static_cast<size_t>(rows) * kBins);
    take(a.list, static_cast<size_t>(rows) * kList);
    take(a.count, segments * kBins);
    take(a.counts, static_cast<size_t>(rows) * kBins);
    take(a.listed, rows);
    return at;
}

}  // namespace
}  // namespace qk

extern "C" {

size_t qk_sample_rows_workspace_bytes(int n, int rows) {
    if (n < 1 || n > 1 << 19 || rows < 1) return 0;
    qk::SampleArgs a{};
    a.segments = (n + qk::kSegment - 1) / qk::kSegment;
    return qk::lay_out(a, rows, nullptr);
}

int qk_sample_rows_f32(const float *logits, int n, int64_t ldv, int rows, const float *temperature,
                       const int32_t *top_k, const float *top_p, const float *min_p, const float *uniform,
                       int32_t *out, float *prob, void *workspace, size_t workspace_bytes, qk_stream stream) {
    if (n < 1 || rows < 0 || ldv < n || (rows > 0 && (!logits || !uniform || !out)))
        return qk::fail(QK_ERR_INVALID_ARG, "qk_sample_rows_f32: null pointer, empty row or bad stride");
    if (n > 1 << 19) return qk::fail(QK_ERR_LIMIT, "qk_sample_rows_f32: at most 2^19 logits a row");
    if (rows > 65535) return qk::fail(QK_ERR_LIMIT, "qk_sample_rows_f32: too many rows in one launch");
    const size_t need = qk_sample_rows_workspace_bytes(n, rows);
    if (need && (!workspace || workspace_bytes < need))
        return qk::fail(QK_ERR_INVALID_ARG, "qk_sample_rows_f32: workspace smaller than qk_sample_rows_workspace_bytes");
    if (!qk::aligned(workspace, 256)) return qk::fail(QK_ERR_ALIGN, "qk_sample_rows_f32: workspace must be 256-byte aligned");
    if (rows == 0) return qk::ok();
    qk::SampleArgs a{logits, ldv, n, temperature, top_p, min_p, uniform, top_k, out, prob};
    a.segments = (n + qk::kSegment - 1) / qk::kSegment;
    a.wide = qk::aligned(logits, 16) && ldv % 4 == 0;
    qk::lay_out(a, rows, static_cast<char *>(workspace));
    const dim3 grid(a.segments, rows), block(qk::kThreads);
    hipLaunchKernelGGL(qk::sample_scan_kernel, grid, block, 0, qk::S(stream), a);
    hipLaunchKernelGGL(qk::sample_plan_kernel, dim3(rows), dim3(qk::kBins), 0, qk::S(stream), a);
    hipLaunchKernelGGL(qk::sample_collect_kernel, grid, block, 0, qk::S(stream), a);
    hipLaunchKernelGGL(qk::sample_pick_kernel, dim3(rows), block, 0, qk::S(stream), a);
    return qk::launch_status("qk_sample_rows_f32 launch");
}

}  // extern "C"
