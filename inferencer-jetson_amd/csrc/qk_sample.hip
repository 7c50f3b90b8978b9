// qk_sample.hip - the next token of rows of logits: temperature, top-k, top-p,
// min-p and the pick by a given random number.
//
// Weights are integers, w = rint(exp((x - max) / T) * 2^44), so every sum is
// exact and neither the filters nor the pick depend on an order of adding.
// The filters keep the tokens whose key (the float's order as an unsigned
// integer) is above a threshold, and of those at the threshold the first `ties`
// by index; the threshold is found digit by digit from histograms of counts
// (top-k) or of weights (top-p).
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
};

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr double kUnit = 17592186044416.;   // 2^44

// Order-preserving key; NaN as -inf, -0 as 0.
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.f; }
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
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

__global__ __launch_bounds__(kThreads) void sample_rows_kernel(SampleArgs a) {
    __shared__ uint64_t hist[256];
    __shared__ uint64_t scratch[kWaves];
    __shared__ uint64_t found_above;
    __shared__ int found_bin, found_index;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float *x = a.logits + static_cast<int64_t>(row) * a.ldv;
    const float t = a.temperature ? a.temperature[row] : 1.f;
    const float p = a.top_p ? a.top_p[row] : 1.f, mp = a.min_p ? a.min_p[row] : 0.f;
    const int k = a.top_k ? a.top_k[row] : 0;

    // The largest key and its lowest index.
    float best = -INFINITY;
    int at = 0x7FFFFFFF;
    for (int i = tid; i < a.n; i += kThreads) arg_better(best, at, clean(x[i]), i);
    #pragma unroll
    for (int off = 32; off > 0; off >>= 1) arg_better(best, at, __shfl_xor(best, off), __shfl_xor(at, off));
    if (lane == 0) scratch[wave] = static_cast<uint64_t>(key_of(best)) << 32 | static_cast<uint32_t>(at);
    __syncthreads();
    for (int w = 0; w < kWaves; ++w)
        arg_better(best, at, value_of(static_cast<uint32_t>(scratch[w] >> 32)), static_cast<int>(scratch[w] & 0xFFFFFFFFu));
    if (best == -INFINITY) {
        if (tid == 0) {
            a.out[row] = 0;
            if (a.prob) a.prob[row] = 0.f;
        }
        return;
    }
    if (!(t > 0.f) || !(p > 0.f) || !(mp <= 1.f) || k == 1) {
        if (tid == 0) {
            a.out[row] = at;
            if (a.prob) a.prob[row] = 1.f;
        }
        return;
    }
    const RowScale rs{best, t};

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

}  // namespace
}  // namespace qk

extern "C" {

size_t qk_sample_rows_workspace_bytes(int n, int rows) {
    (void)n;
    (void)rows;
    return 0;
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
    const qk::SampleArgs a{logits, ldv, n, temperature, top_p, min_p, uniform, top_k, out, prob};
    hipLaunchKernelGGL(qk::sample_rows_kernel, dim3(rows), dim3(qk::kThreads), 0, qk::S(stream), a);
    return qk::launch_status("qk_sample_rows_f32 launch");
}

}  // extern "C"
