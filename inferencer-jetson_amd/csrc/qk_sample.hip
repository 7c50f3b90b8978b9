// qk_sample.hip - the next token of rows of logits: temperature, top-k, top-p,
// min-p and the pick by a given random number.
//
// The filters keep a prefix of the row in descending order (equal logits by
// index), so what they leave is the tokens from one of them on: the cut.  Two
// launches:
//   sample_scan_kernel, a workgroup per 16384 logits (a segment): its largest,
//     and a histogram over 16 bins an octave of the weights 2^(x log2(e) / T)
//     below the segment's own power of two 2^E, as integers in units of
//     2^(E - 46), so the order of adding does not matter;
//   sample_pick_kernel, a workgroup per row: adds up the segments' histograms,
//     finds the bin in which the cut lies, reads the row again for that bin's
//     tokens (some hundreds at most, or with top-k all that it leaves), sorts
//     them and finds the cut; then the segment that holds the random number's
//     token from the histograms, and the token by looking that segment over.
// A row is thus read once from memory and once from the cache, and each
// weight's exponential (in 64 bits: 32 would move the borders between tokens by
// 1e-8 of the sum, and with them one token in some thousands of rows) is taken
// once.  Rows that this does not serve -- an infinite logit, more tokens in the
// cut's bin than its list holds (thousands of equal logits, or a temperature
// that leaves all of them alike), |x log2(e) / T| of 2^20 and more -- go through
// sample_plain, which finds the cut digit by digit from histograms of the
// floats' order.
#include "qk_internal.h"

namespace qk {
namespace {

hipStream_t S(qk_stream s) { return static_cast<hipStream_t>(s); }

struct SampleArgs {
    const float *logits;
    int64_t ldv;
    int n;
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t *top_k;
    int32_t *out;
    float *prob;
    struct SegmentHead *heads;   // [rows][segments]
    uint64_t *mass;              // [rows][segments][kBins]
    uint32_t *count;             // the same, of rows with top-k
    int segments, wide;          // wide: rows are 16-byte aligned
};

// A segment's largest logit, its lowest index, and the power of two that its
// weights are below (kNone: no logit above -inf, kFar: out of range).
struct SegmentHead {
    float best;
    int at, e, pad;
};
constexpr int kNone = -0x40000000, kFar = 0x40000000;

constexpr int kThreads = 512, kWaves = kThreads / 64;   // of sample_pick_kernel
constexpr int kScanThreads = 1024, kSegment = 16 * kScanThreads;
constexpr int kMaxSegments = (1 << 19) / kSegment;
constexpr int kBins = 768, kOctave = 16;   // 48 octaves; a weight has 46 bits
constexpr int kList = 2048;
constexpr double kUnit = 17592186044416.;   // 2^44: sample_plain's weights, of which 2^19 stay below 2^64

// Order-preserving key; NaN as -inf, -0 as 0.
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.f; }
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
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
    #pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
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
        uint64_t upto = w;
        #pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint64_t o = __shfl_up(upto, off);
            if (lane >= off) upto += o;
        }
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

// 2^-d in units of 2^-46, d = i / 16 + r below 47 and bin i: 2^-(i % 16 + 1/2)/16
// from the table, e^(-y ln 2) of |y| <= 1/32 by its Taylor polynomial to y^6
// (the next term is 4e-16), the power of two into the exponent, rounded by
// adding 2^52.
__device__ __forceinline__ uint64_t unit_weight(double d, int i, const double *table) {
    const double y = fma(static_cast<double>(i), -1. / kOctave, d) - 0.5 / kOctave;
    double p = 1.5403530393381609954e-4;
    p = fma(p, y, -1.3333558146428443423e-3);
    p = fma(p, y, 9.6181291076284771619e-3);
    p = fma(p, y, -5.5504108664821579953e-2);
    p = fma(p, y, 2.4022650695910071233e-1);
    p = fma(p, y, -6.9314718055994530942e-1);
    p = fma(p, y, 1.);
    const double v = p * table[i & (kOctave - 1)];
    const uint64_t scaled = __builtin_bit_cast(uint64_t, v) + (static_cast<uint64_t>(46 - i / kOctave) << 52);
    return __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, scaled) + 4503599627370496.) - 0x4330000000000000ull;
}

// How far a logit's weight lies below 2^e, in octaves (inf for none).
__device__ __forceinline__ double octaves_below(float x, double c, int e) {
    return fma(-static_cast<double>(x), c, static_cast<double>(e));
}
constexpr double kDepth = 47.;   // from here on a weight rounds to 0
__device__ __forceinline__ int bin_of(double d) { return static_cast<int>(fmax(d, 0.) * kOctave); }

__device__ __forceinline__ void load_quad(const float *x, int i, int n, int wide, float (&v)[4]) {
    if (wide && i + 3 < n) {
        const float4 q = *reinterpret_cast<const float4 *>(x + i);
        v[0] = clean(q.x), v[1] = clean(q.y), v[2] = clean(q.z), v[3] = clean(q.w);
    } else {
        #pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i + e < n ? clean(x[i + e]) : -INFINITY;
    }
}

__device__ __forceinline__ void fill_table(double *table) {
    if (threadIdx.x < kOctave) table[threadIdx.x] = exp2(-(static_cast<double>(threadIdx.x) + 0.5) / kOctave);
}

// --------------------------------------------------------------- scan --

__global__ __launch_bounds__(kScanThreads) void sample_scan_kernel(SampleArgs a) {
    __shared__ unsigned long long mass[kBins];
    __shared__ uint32_t count[kBins];
    __shared__ double table[kOctave];
    __shared__ uint64_t best_of[kScanThreads / 64];
    const int row = blockIdx.y, seg = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float *x = a.logits + static_cast<int64_t>(row) * a.ldv;
    float v[4][4];
    #pragma unroll
    for (int j = 0; j < 4; ++j) load_quad(x, seg * kSegment + (j * kScanThreads + tid) * 4, a.n, a.wide, v[j]);
    const RowParams r = row_params(a, row);
    fill_table(table);
    for (int i = tid; i < kBins; i += kScanThreads) mass[i] = 0, count[i] = 0;
    float best = -INFINITY;
    int at = 0x7FFFFFFF;
    #pragma unroll
    for (int j = 0; j < 4; ++j)
        #pragma unroll
        for (int e = 0; e < 4; ++e) arg_better(best, at, v[j][e], seg * kSegment + (j * kScanThreads + tid) * 4 + e);
    #pragma unroll
    for (int off = 32; off > 0; off >>= 1) arg_better(best, at, __shfl_xor(best, off), __shfl_xor(at, off));
    if (lane == 0) best_of[wave] = static_cast<uint64_t>(key_of(best)) << 32 | static_cast<uint32_t>(at);
    __syncthreads();
    for (int w = 0; w < kScanThreads / 64; ++w)
        arg_better(best, at, value_of(static_cast<uint32_t>(best_of[w] >> 32)),
                   static_cast<int>(best_of[w] & 0xFFFFFFFFu));
    const double c = kLog2E / static_cast<double>(r.t), top = static_cast<double>(best) * c;
    const int e = best == -INFINITY ? kNone : !(fabs(top) < 1048576.) ? kFar : static_cast<int>(ceil(top));
    const int64_t me = static_cast<int64_t>(row) * a.segments + seg;
    if (tid == 0) a.heads[me] = SegmentHead{best, at, e, 0};
    if (r.greedy || e == kNone || e == kFar) return;
    const bool counted = r.k > 0 && r.k < a.n;
    #pragma unroll
    for (int j = 0; j < 4; ++j)
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
            const double d = octaves_below(v[j][k], c, e);
            if (d < kDepth) {
                const int bin = bin_of(d);
                atomicAdd(&mass[bin], static_cast<unsigned long long>(unit_weight(d, bin, table)));
                if (counted) atomicAdd(&count[bin], 1u);
            }
        }
    __syncthreads();
    for (int i = tid; i < kBins; i += kScanThreads) {
        a.mass[me * kBins + i] = mass[i];
        if (counted) a.count[me * kBins + i] = count[i];
    }
}

// --------------------------------------------------------------- pick --

struct PickShared {
    double cum[kBins];            // sums of the row's bins up to each, in units of 2^(e - 46)
    uint64_t list[kList];         // tokens: the key's bits, then the index's complement
    double sorted[kList];         // sums of the list's weights up to each
    double table[kOctave];
    SegmentHead head[kMaxSegments];
    uint64_t kept[kMaxSegments];  // kept weight of each segment, in its own units
    uint64_t part[8][kWaves];
    double wave_sum[kWaves];
    uint32_t wave_count[kWaves];
    uint32_t counts[kBins];       // tokens of the row's bins up to each
    int listed, bin_k, bin_p, cut, found;
};

// Inclusive sums over kBins values, two a thread, in a fixed order.
template <class T>
__device__ __forceinline__ void scan_bins(T *v, T *waves) {
    static_assert(kBins <= 2 * kThreads, "two bins a thread");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = 2 * tid;
    T a = i < kBins ? v[i] : T(0), b = i + 1 < kBins ? v[i + 1] : T(0);
    T sum = a + b;
    #pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const T o = __shfl_up(sum, off);
        if (lane >= off) sum += o;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = sum;
    __syncthreads();
    T base = T(0);
    for (int w = 0; w < wave; ++w) base += waves[w];
    const T before = base + (sum - (a + b));
    if (i < kBins) v[i] = before + a;
    if (i + 1 < kBins) v[i + 1] = base + sum;
    __syncthreads();
}

// The first of kBins non-decreasing sums to reach target, kBins if none does.
template <class T>
__device__ __forceinline__ int first_reaching(const T *cum, double target, int *found) {
    if (threadIdx.x == 0) *found = kBins;
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads)
        if (static_cast<double>(cum[i]) >= target && (i == 0 || static_cast<double>(cum[i - 1]) < target))
            atomicMin(found, i);   // rounding may leave two such steps
    __syncthreads();
    const int r = *found;
    __syncthreads();
    return r;
}

__device__ __forceinline__ uint64_t packed(float x, int i) {
    return static_cast<uint64_t>(key_of(x)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}

// Descending bitonic sort of list[0 .. size), size a power of two.
__device__ __forceinline__ void sort_list(uint64_t *list, int size) {
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int t = threadIdx.x; t < size / 2; t += kThreads) {
                const int i = 2 * t - (t & (j - 1)), o = i + j;
                const uint64_t p = list[i], q = list[o];
                if ((p < q) == ((i & k) == 0)) list[i] = q, list[o] = p;
            }
        }
    __syncthreads();
}

// A row by its segments' histograms, by all threads of the workgroup; false:
// it is one for sample_plain, with its largest logit in best.
__device__ __forceinline__ bool sample_binned(const SampleArgs &a, const RowParams &r, int row, float &best,
                                              PickShared &s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float *x = a.logits + static_cast<int64_t>(row) * a.ldv;
    const int64_t first = static_cast<int64_t>(row) * a.segments;
    best = -INFINITY;
    int at = 0x7FFFFFFF, e = kNone;
    bool far = false;
    for (int g = 0; g < a.segments; ++g) {
        const SegmentHead h = a.heads[first + g];
        arg_better(best, at, h.best, h.at);
        far = far || h.e == kFar;
        if (h.e != kFar) e = max(e, h.e);
        if (tid == 0) s.head[g] = h;
    }
    if (best == -INFINITY || r.greedy) {
        if (tid == 0) {
            a.out[row] = best == -INFINITY ? 0 : at;
            if (a.prob) a.prob[row] = best == -INFINITY ? 0.f : 1.f;
        }
        return true;
    }
    if (far) return false;

    // The row's bins: of a segment whose power of two lies m octaves lower,
    // bin i - 16 m.
    const bool counted = r.k > 0 && r.k < a.n;
    fill_table(s.table);
    for (int i = tid; i < kBins; i += kThreads) {
        double sum = 0.;
        uint32_t n = 0;
        for (int g = 0; g < a.segments; ++g) {
            const int eg = a.heads[first + g].e;
            const int lower = min(e - eg, 64), from = i - kOctave * lower;
            if (eg == kNone || from < 0) continue;
            sum += ldexp(static_cast<double>(a.mass[(first + g) * kBins + from]), -lower);
            if (counted) n += a.count[(first + g) * kBins + from];
        }
        s.cum[i] = sum;
        s.counts[i] = n;
    }
    __syncthreads();
    scan_bins(s.cum, s.wave_sum);
    if (counted) scan_bins(s.counts, s.wave_count);
    const double c = kLog2E / static_cast<double>(r.t);

    // Tokens of bins lo .. hi into the list; false: more than it holds.
    auto collect = [&](int lo, int hi) {
        __syncthreads();
        if (tid == 0) s.listed = 0;
        __syncthreads();
        for (int g = 0; g < a.segments; ++g) {
            const int eg = s.head[g].e, lower = min(e - eg, 64) * kOctave;
            if (eg == kNone) continue;
            const int end = min(a.n, (g + 1) * kSegment);
            #pragma unroll 2
            for (int i = g * kSegment + tid * 4; i < end; i += kThreads * 4) {
                float v[4];
                load_quad(x, i, a.n, a.wide, v);
                #pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const double d = octaves_below(v[k], c, eg);
                    if (!(d < kDepth)) continue;
                    const int bin = bin_of(d) + lower;
                    if (bin >= lo && bin <= hi) {
                        const int slot = atomicAdd(&s.listed, 1);
                        if (slot < kList) s.list[slot] = packed(v[k], i + k);
                    }
                }
            }
        }
        __syncthreads();
        if (s.listed > kList) return false;
        int size = 2;
        while (size < s.listed) size <<= 1;
        for (int i = s.listed + tid; i < size; i += kThreads) s.list[i] = 0;
        sort_list(s.list, size);
        return true;
    };
    // A listed token's weight in its segment's units, and in the row's.
    auto listed_weight = [&](int i, int &g) -> uint64_t {
        const uint64_t t = s.list[i];
        g = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(t)) / kSegment;
        const double d = octaves_below(value_of(static_cast<uint32_t>(t >> 32)), c, s.head[g].e);
        return unit_weight(d, bin_of(d), s.table);
    };
    auto row_weight = [&](int i) {
        int g;
        const uint64_t w = listed_weight(i, g);
        return ldexp(static_cast<double>(w), s.head[g].e - e);
    };
    // Sums of the list's weights up to each, four a thread.
    auto sum_list = [&]() {
        static_assert(kList == 4 * kThreads, "four tokens a thread");
        double w[4], sum = 0.;
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = tid * 4 + k;
            w[k] = i < s.listed ? row_weight(i) : 0.;
            sum += w[k];
        }
        double upto = sum;
        #pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const double o = __shfl_up(upto, off);
            if (lane >= off) upto += o;
        }
        if (lane == 63) s.wave_sum[wave] = upto;
        __syncthreads();
        double base = 0.;
        for (int v = 0; v < wave; ++v) base += s.wave_sum[v];
        base += upto - sum;
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
            base += w[k];
            s.sorted[tid * 4 + k] = base;
        }
        __syncthreads();
    };

    const int last = kBins - 1;
    int bin_k = kBins, lo = 0, left = 0;   // top-k: the bin of its last token, and how many of the list are left
    bool listed = false;
    if (counted) bin_k = first_reaching(s.counts, static_cast<double>(r.k), &s.found);
    double total = s.cum[last];
    if (bin_k < kBins) {
        const bool all = s.counts[bin_k] <= kList;   // the whole of what top-k leaves fits the list
        lo = all ? 0 : bin_k;
        if (!collect(lo, bin_k)) return false;
        sum_list();
        listed = true;
        left = r.k - (lo > 0 ? static_cast<int>(s.counts[lo - 1]) : 0);
        total = (lo > 0 ? s.cum[lo - 1] : 0.) + s.sorted[left - 1];
    }
    const double target = r.p < 1.f ? static_cast<double>(r.p) * total : INFINITY;
    // The largest token's weight, and the least one that min-p keeps.
    const double dbest = octaves_below(best, c, e);
    const double least = r.mp > 0.f ? static_cast<double>(r.mp) * static_cast<double>(unit_weight(dbest, bin_of(dbest), s.table)) : 0.;
    int bin = bin_k;
    if (r.p < 1.f) bin = min(bin, first_reaching(s.cum, target, &s.found));
    if (r.mp > 0.f) bin = min(bin, bin_of(fmin(dbest - log2(static_cast<double>(r.mp)), 48.)));
    int whole = kBins, keep = 0;   // kept: bins below `whole`, and the list's first `keep` tokens
    uint64_t cut = ~0ull;          // the last of these
    if (bin < kBins) {
        if (!listed || bin < lo) {
            if (!collect(bin, bin)) return false;
            sum_list();
            lo = bin;
            left = s.listed;
        }
        whole = lo;
        const double above = lo > 0 ? s.cum[lo - 1] : 0.;
        if (tid == 0) s.cut = 0;
        __syncthreads();
        // Kept: as many as top-k leaves, while the sum before is below the
        // target and the weight not below the least.
        int mine = 0;
        for (int i = tid; i < left; i += kThreads) {
            const double before = above + (i > 0 ? s.sorted[i - 1] : 0.);
            if (before < target && (least == 0. || row_weight(i) >= least)) mine = i + 1;
        }
        if (mine) atomicMax(&s.cut, mine);
        __syncthreads();
        keep = s.cut;
        if (keep > 0) cut = s.list[keep - 1];
    }

    // Kept weight of each segment, in its own units.
    for (int g = wave; g < a.segments; g += kWaves) {
        const int eg = s.head[g].e;
        uint64_t sum = 0;
        if (eg != kNone)
            for (int i = lane; i < min(whole, kBins) - kOctave * min(e - eg, 64); i += 64) sum += a.mass[(first + g) * kBins + i];
        sum = wave_sum_u64(sum);
        if (lane == 0) s.kept[g] = sum;
    }
    __syncthreads();
    for (int i = tid; i < keep; i += kThreads) {
        int g;
        const uint64_t w = listed_weight(i, g);
        atomicAdd(reinterpret_cast<unsigned long long *>(&s.kept[g]), static_cast<unsigned long long>(w));
    }
    __syncthreads();
    double z = 0.;
    for (int g = 0; g < a.segments; ++g)
        if (s.head[g].e != kNone) z += ldexp(static_cast<double>(s.kept[g]), max(s.head[g].e - e, -64));
    // The segment of the random number's token, and how much of its weight
    // lies before that token.
    const double u = a.uniform[row], goal = u > 0. ? fmin(u, 1.) * z : 0.;
    double sum = 0.;
    int seg = -1;
    uint64_t want = 0;
    for (int g = 0; g < a.segments; ++g) {
        const uint64_t w = s.head[g].e == kNone ? 0 : s.kept[g];
        if (!w) continue;
        const int lower = max(s.head[g].e - e, -64);
        const double part = ldexp(static_cast<double>(w), lower);
        seg = g;
        const double inside = ldexp(fmax(goal - sum, 0.), -lower);
        want = inside < static_cast<double>(w) ? min(static_cast<uint64_t>(inside), w - 1) : w - 1;
        if (goal < sum + part) break;
        sum += part;
    }
    // The segment again: thread sums by tiles of 4 * kThreads tokens, then the
    // wave and the token.
    constexpr int kTiles = kSegment / (4 * kThreads);
    static_assert(kTiles == 8, "s.part");
    const int eg = s.head[seg].e;
    auto weights = [&](int i, uint64_t (&w)[4]) {
        float v[4];
        load_quad(x, i, a.n, a.wide, v);
        uint64_t sum = 0;
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
            const double d = octaves_below(v[k], c, eg);
            const bool kept = d < kDepth && (bin_of(d) + kOctave * (e - eg) < whole || packed(v[k], i + k) >= cut);
            w[k] = kept ? unit_weight(d, bin_of(d), s.table) : 0;
            sum += w[k];
        }
        return sum;
    };
    uint64_t tile_sum[kTiles];
    #pragma unroll
    for (int j = 0; j < kTiles; ++j) {
        uint64_t w[4];
        const int i = seg * kSegment + (j * kThreads + tid) * 4;
        tile_sum[j] = i < a.n ? weights(i, w) : 0;
    }
    #pragma unroll
    for (int j = 0; j < kTiles; ++j) {
        const uint64_t t = wave_sum_u64(tile_sum[j]);
        if (lane == 0) s.part[j][wave] = t;
    }
    __syncthreads();
    int tile = 0, mine = 0;
    uint64_t before = 0;
    bool done = false;
    for (int j = 0; j < kTiles && !done; ++j)
        for (int w = 0; w < kWaves; ++w) {
            if (before + s.part[j][w] > want) {
                tile = j;
                mine = w;
                done = true;
                break;
            }
            before += s.part[j][w];
        }
    if (wave != mine || !done) return true;
    uint64_t w[4];
    const int i = seg * kSegment + (tile * kThreads + tid) * 4;
    uint64_t own = i < a.n ? weights(i, w) : 0, upto = own;
    #pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint64_t o = __shfl_up(upto, off);
        if (lane >= off) upto += o;
    }
    uint64_t b = before + upto - own;
    if (own && b <= want && want < b + own)
        for (int k = 0; k < 4; ++k) {
            if (w[k] && b <= want && want < b + w[k]) {
                a.out[row] = i + k;
                if (a.prob) a.prob[row] = static_cast<float>(ldexp(static_cast<double>(w[k]), max(eg - e, -64)) / z);
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
    const RowParams r = row_params(a, blockIdx.x);
    float best;
    if (!sample_binned(a, r, blockIdx.x, best, s.pick)) sample_plain(a, r, blockIdx.x, best, s.plain);
}

size_t round256(size_t b) { return (b + 255) / 256 * 256; }

}  // namespace
}  // namespace qk

extern "C" {

size_t qk_sample_rows_workspace_bytes(int n, int rows) {
    if (n < 1 || n > 1 << 19 || rows < 1) return 0;
    const size_t segments = static_cast<size_t>(rows) * ((n + qk::kSegment - 1) / qk::kSegment);
    return qk::round256(segments * sizeof(qk::SegmentHead)) + segments * qk::kBins * (sizeof(uint64_t) + sizeof(uint32_t));
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
    const size_t segments = static_cast<size_t>(rows) * a.segments;
    char *ws = static_cast<char *>(workspace);
    a.heads = reinterpret_cast<qk::SegmentHead *>(ws);
    a.mass = reinterpret_cast<uint64_t *>(ws + qk::round256(segments * sizeof(qk::SegmentHead)));
    a.count = reinterpret_cast<uint32_t *>(a.mass + segments * qk::kBins);
    hipLaunchKernelGGL(qk::sample_scan_kernel, dim3(a.segments, rows), dim3(qk::kScanThreads), 0, qk::S(stream), a);
    hipLaunchKernelGGL(qk::sample_pick_kernel, dim3(rows), dim3(qk::kThreads), 0, qk::S(stream), a);
    return qk::launch_status("qk_sample_rows_f32 launch");
}

}  // extern "C"
