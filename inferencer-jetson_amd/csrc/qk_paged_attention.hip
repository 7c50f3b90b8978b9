// qk_paged_attention.hip - attention of new tokens over a paged cache: which kernel
// a call takes, its splits, and the merge of their partials.
#include "qk_paged_attention.h"

#include <cmath>

namespace qk {
namespace {

hipStream_t S(qk_stream s) { return static_cast<hipStream_t>(s); }

// The splits that reach a token, 64 at most; one wave a (token, head): a lane has a
// split's maximum and sum, then all lanes the dimensions, eight splits at a time
// (read one after the other, 64 splits took 10 us longer).
// (MASKED: with a window or a prefix.  Asked for by every wave, of calls without them
// too, the two took 2 us of 10: four chunks of 512 tokens, 32 heads.)
template <int HD, bool MASKED>
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
    const int upto = MASKED ? max(s.pos + tok, prefix_rows(a, s) - 1) - first_row(a, s) : s.pos + tok;
    const int live = min(a.splits[many], upto / a.split_rows[many] + 1);
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
// sequence, 68 query rows a KV head over 4000 cache rows (2.2 million pairs) 24
// and 19, 256 over 4000 (8.3 million) 31 and 29, 1600 over 500 (12 million) 36 and
// 36, 512 over 4000 (17 million) 42 and 53, 2000 over none (8 million, 128
// workgroups) 32 and 23; eight sequences, 256 over 500 (9.2 million, 128
// workgroups) 36 and 31, 68 over 4000 (17 million) 52 and 68, 512 over none (256
// workgroups) 19 and 28; 64 sequences, 68 over none (512 workgroups) 20 and 30.
// Eight query heads of 256 for one KV head, one sequence of 2048 tokens over 4000:
// int8 344 and 280, fp16 348 and 380; eight of 64 over 4000: 91 and 83, 97 and 83,
// where the first kernel would be the faster one three times of four: the rule sees
// neither head size nor type.
constexpr int kFewRows = 64, kManyUnits = 256;
constexpr int64_t kManyPairs = 3 << 22;
// Heads of 256 dimensions of 4-bit rows, or with terms, all take the first (all_few),
// whose workgroups are two a CU, not one.  In us, and by the chunk kernel: 4-bit rows, 16
// heads on 8, 2048 tokens over 4000 530 and 583, 8 sequences of 300 over 1000 192 and 264;
// 8 heads on one, 2048 over 4000 with capped scores, float8 rows 306 and 375, fp16 381 and
// 384; fp16, 16 heads on 8, capped, over none 208 and 251, 1024 over 6000 and a window of
// 4096 310 and 353.  The other way round for longer fp16 chunks of 16 heads on 8, which
// the rule does not see: 2048 over 4000 capped 740 and 712, over 6000 through a window
// of 4096 602 and 506, of 1024 189 and 163.
// Query rows a KV head up to which a sequence of this call takes the first
// kernel; a call of one sequence launches one of the two.
int few_rows(const qk_paged_batch &b, int heads, int kv_heads, bool all_few) {
    const int64_t rows = static_cast<int64_t>(b.max_count) * (heads / kv_heads);
    if (rows <= kFewRows || all_few) return INT32_MAX;
    const int64_t units = (rows + kChunkRows - 1) / kChunkRows * kv_heads * b.n_seqs;
    const double pairs = static_cast<double>(b.n_tokens) * heads * b.max_rows;
    if (units < kManyUnits && pairs < kManyPairs) return INT32_MAX;
    return b.n_seqs == 1 ? 0 : kFewRows;
}

// Splits of a call's rows, 64 at most.  Few query rows: the workgroups that the
// chip holds at once, two a CU (one of 256 dimensions: 512 of those that are two a CU
// were no faster), of at least 128 rows, or 256 in more than 32 splits, and none for 256
// rows or less.  (One sequence, 8 KV heads of 128 int8 values: 250 rows whole 8.0 us, in
// two splits 9.8; 2000 rows in 16 splits 10.5, in eight 11.6; 8000 rows in 32 splits
// 13.4, in 63 15.0.  16 sequences of 8000 rows: in one round of workgroups 50 us, in two
// 52.)  Sequences that fill the chip as they are even out in four splits, if those are
// long.  64 sequences of 1000 to 8000 rows: 4-bit 91 us and whole 103, int8 130 and 132,
// fp16 222 and 223; of equal lengths the other way round, of 4500 91 and 78, 126 and 110,
// 212 and 202, which no call can tell from the others on the host; of 125 to 1000 int8
// rows whole 22, in four splits 31.
// Chunks: a round of workgroups likewise, of at least four tiles; those that lie
// behind all that a chunk's first tokens see end at once and do not count.
struct Splits {
    int few, many;
};
Splits wanted_splits(const qk_paged_batch &b, int heads, int kv_heads, int head_dim, bool all_few) {
    const int64_t few = few_rows(b, heads, kv_heads, all_few), rows = static_cast<int64_t>(b.max_count) * (heads / kv_heads);
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

template <int HD>
int merge(const PagedAttn &a, hipStream_t stream) {
    auto kernel = a.window || a.prefix ? paged_merge_kernel<HD, true> : paged_merge_kernel<HD, false>;
    hipLaunchKernelGGL(kernel,
                       dim3(static_cast<unsigned>((static_cast<int64_t>(a.b.max_count) * a.heads + 3) / 4), a.b.n_seqs),
                       dim3(256), 0, stream, a);
    return launch_status("qk_paged_attention_f32 launch");
}

int launch(const PagedAttn &a, bool terms, hipStream_t stream) {
    int status;
    switch (a.kv.type) {
        case QK_TYPE_F16: status = attend_f16(a, terms, stream); break;
        case QK_TYPE_I8: status = attend_i8(a, terms, stream); break;
        case QK_TYPE_I4: status = attend_i4(a, terms, stream); break;
        default: status = attend_e4m3(a, terms, stream);
    }
    if (status != QK_OK || a.part_splits == 1) return status;
    switch (a.kv.head_dim) {
        case 64: return merge<64>(a, stream);
        case 96: return merge<96>(a, stream);
        case 128: return merge<128>(a, stream);
        default: return merge<256>(a, stream);
    }
}

// A batch as its splits are planned: of the rows that a window leaves of a sequence.
qk_paged_batch planned(const qk_paged_batch &b, int window) {
    qk_paged_batch p = b;
    if (window > 0) p.max_rows = static_cast<int>(std::min<int64_t>(b.max_rows, int64_t(window) + b.max_count + 62));
    return p;
}

// Whether all query rows of a call take the first kernel.
bool all_few(int type, bool terms, int head_dim) { return head_dim > 128 && (terms || type == QK_TYPE_I4); }

// (Of any cache type, with any terms of this window.)
size_t workspace_bytes(const qk_paged_batch &batch, int heads, int kv_heads, int head_dim, int window) {
    int most = 1;
    for (const bool few : {false, all_few(QK_TYPE_I4, true, head_dim)}) {
        const Splits splits = wanted_splits(planned(batch, window), heads, kv_heads, head_dim, few);
        most = std::max({most, splits.few, splits.many});
    }
    return most > 1 ? most * split_bytes(batch, heads, head_dim) : 0;
}

}  // namespace
}  // namespace qk

extern "C" {

size_t qk_paged_attention_workspace_bytes(const qk_paged_batch *batch, int heads, int kv_heads, int head_dim) {
    return qk_paged_attention_terms_workspace_bytes(batch, heads, kv_heads, head_dim, 0);
}

size_t qk_paged_attention_terms_workspace_bytes(const qk_paged_batch *batch, int heads, int kv_heads, int head_dim,
                                                int window) {
    if (qk::check_paged_batch("qk_paged_attention_workspace_bytes", batch) || heads < 1 || kv_heads < 1 ||
        heads % kv_heads || head_dim < 1 || head_dim > 256 || window < 0 || batch->n_seqs == 0 || batch->n_tokens == 0)
        return 0;
    return qk::workspace_bytes(*batch, heads, kv_heads, head_dim, window);
}

int qk_paged_attention_f32(const qk_paged_kv *kv, const qk_paged_batch *batch, const float *q, int ldq, float *out,
                           int ldout, int heads, float scale, void *workspace, size_t workspace_bytes,
                           qk_stream stream) {
    return qk_paged_attention_terms_f32(kv, batch, q, ldq, out, ldout, heads, scale, nullptr, workspace, workspace_bytes,
                                        stream);
}

int qk_paged_attention_terms_f32(const qk_paged_kv *kv, const qk_paged_batch *batch, const float *q, int ldq, float *out,
                                 int ldout, int heads, float scale, const qk_attention_terms *terms, void *workspace,
                                 size_t workspace_bytes, qk_stream stream) {
    const char *where = "qk_paged_attention_f32";
    if (int s = qk::check_paged_kv(where, kv)) return s;
    if (int s = qk::check_paged_batch(where, batch)) return s;
    if (heads < 1 || heads > 65536 || heads % kv->kv_heads)
        return qk::fail(QK_ERR_INVALID_ARG, "qk_paged_attention_f32: heads must be a multiple of kv_heads");
    if (!std::isfinite(scale)) return qk::fail(QK_ERR_INVALID_ARG, "qk_paged_attention_f32: scale is not finite");
    const qk_attention_terms none{}, &t = terms ? *terms : none;
    if (!(t.cap == 0.f || (t.cap >= 0x1p-64f && t.cap <= 0x1p64f)))
        return qk::fail(QK_ERR_INVALID_ARG, "qk_paged_attention_f32: cap must be 0, or from 2^-64 to 2^64");
    if (t.window < 0) return qk::fail(QK_ERR_INVALID_ARG, "qk_paged_attention_f32: negative window");
    if (batch->n_seqs == 0 || batch->n_tokens == 0) return qk::ok();
    if (!q || !out) return qk::fail(QK_ERR_INVALID_ARG, "qk_paged_attention_f32: null pointer");
    const int64_t dim = static_cast<int64_t>(heads) * kv->head_dim;
    if (ldq < dim || ldout < dim)
        return qk::fail(QK_ERR_INVALID_ARG, "qk_paged_attention_f32: leading dimension smaller than the row");
    if (!qk::aligned(q, 16) || !qk::aligned(out, 16) || !qk::aligned(workspace, 16) || ldq % 4 || ldout % 4 ||
        !qk::aligned(t.slopes, 4) || !qk::aligned(t.prefix, 4))
        return qk::fail(QK_ERR_ALIGN, "qk_paged_attention_f32: q and out need 16-byte rows, workspace 16 bytes, slopes and prefix 4");
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
    a.cap = 1.4426950408889634f * t.cap;
    a.window = t.window;
    a.slopes = t.slopes;
    a.prefix = t.prefix;
    const qk_paged_batch plan_batch = qk::planned(*batch, t.window);
    const size_t per = qk::split_bytes(*batch, heads, kv->head_dim);
    const int64_t fit = workspace ? static_cast<int64_t>(workspace_bytes / per) : 0;
    const bool with_terms = t.cap > 0.f || t.window > 0 || t.slopes || t.prefix;
    const bool few = qk::all_few(kv->type, with_terms, kv->head_dim);
    const qk::Splits wanted = qk::wanted_splits(plan_batch, heads, kv->kv_heads, kv->head_dim, few);
    // Splits of whole rounds of a workgroup's tiles.
    auto plan = [&](int kind, int splits, int round) {
        const int64_t n = std::min<int64_t>(splits, fit < 2 ? 1 : fit), rows = plan_batch.max_rows;
        const int64_t each = ((rows + n - 1) / n + round - 1) / round * round;
        a.split_rows[kind] = static_cast<int>(each);
        a.splits[kind] = static_cast<int>((rows + each - 1) / each);
    };
    a.few_rows = qk::few_rows(plan_batch, heads, kv->kv_heads, few);
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
    return qk::launch(a, with_terms, qk::S(stream));
}

}  // extern "C"
