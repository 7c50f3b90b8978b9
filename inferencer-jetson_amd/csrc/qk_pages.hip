// qk_pages.hip - a pool of cache pages: given out and taken back, forked, compacted,
// and copied, all on the device.
//
// A call is a few launches: one over the table's rows (a workgroup each) that says
// what each row gives back and lacks, one of a single workgroup that adds up what is
// lacking and lists as many free pages (or, compacting, pairs pages to move with
// free ones before them), one over the rows again that fills them in, and the copies
// of contents.  Pages are given in the order of table rows and their entries, lowest
// page first: what a call does depends on the table and the counts alone, and the
// atomics on the counts are sums of whole numbers.
#include "qk_paged.h"

#include <algorithm>

namespace qk {
namespace {

hipStream_t S(qk_stream s) { return static_cast<hipStream_t>(s); }

// ---------------------------------------------------------- workspace --

// What the launches of a call leave each other, in 32-bit numbers: how many pages
// are given (or moved), then for each table row what it lacks and the rank of its
// first page, the pages given, the sources of their copies, and the rows that a fork
// makes (or, compacting, the new number of each page).
struct Space {
    int32_t *counts, *need, *base, *list, *source, *next;
};
constexpr int kCounts = 16;   // counts[0]: pages given; [1]: pages moved; [2]: live pages

int64_t list_entries(const qk_page_pool &p) {
    return std::min<int64_t>(p.pages, static_cast<int64_t>(p.table_rows) * p.table_stride);
}
int64_t next_entries(const qk_page_pool &p) {
    return std::max<int64_t>(p.pages, static_cast<int64_t>(p.table_rows) * p.table_stride);
}
int64_t space_entries(const qk_page_pool &p) {
    return kCounts + 2 * static_cast<int64_t>(p.table_rows) + 2 * std::max<int64_t>(list_entries(p), p.pages / 2 + 1) +
           next_entries(p);
}
Space space_of(const qk_page_pool &p, void *workspace) {
    Space s;
    const int64_t list = std::max<int64_t>(list_entries(p), p.pages / 2 + 1);
    s.counts = static_cast<int32_t *>(workspace);
    s.need = s.counts + kCounts;
    s.base = s.need + p.table_rows;
    s.list = s.base + p.table_rows;
    s.source = s.list + list;
    s.next = s.source + list;
    return s;
}

struct Pool {
    int32_t *table, *refs;
    int rows, stride, pages, page_rows;
    __device__ __forceinline__ bool is_page(int32_t p) const { return p >= 0 && p < pages; }
    __device__ __forceinline__ int32_t *row(int r) const { return table + static_cast<int64_t>(r) * stride; }
};

// ------------------------------------------------------- sums in order --

typedef unsigned long long u64;

// A workgroup's exclusive sums of v in the order of its threads, and their total.
// (Four sums of 16 bits at once, as long as none passes 2^16.)
template <int WAVES>
__device__ __forceinline__ u64 block_sums(u64 v, u64 &total, u64 (&part)[WAVES]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u64 sum = v;
    #pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const u64 other = __shfl_up(sum, off);
        if (lane >= off) sum += other;
    }
    __syncthreads();   // the parts of the sums before have been read
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    u64 before = 0;
    total = 0;
    #pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) before += part[w];
        total += part[w];
    }
    return before + sum - v;
}

// A workgroup of 1024 looks over the counts of all pages in order, 16384 at a time,
// four runs of four neighbours a thread: which(count, page) says whether a page is
// one of those that are ranked, put(rank, page) takes it.  Ends once `most` are
// found.  65536 pages in 7 us: four rounds of a load's latency and of the sums.
constexpr int kScanThreads = 1024, kRuns = 4, kRound = kScanThreads * 4 * kRuns;
template <typename Which, typename Put>
__device__ __forceinline__ int rank_pages(const int32_t *refs, int pages, int most, u64 (&part)[kScanThreads / 64],
                                          Which which, Put put) {
    auto load = [&](int64_t at, int4 (&v)[kRuns]) {
        #pragma unroll
        for (int k = 0; k < kRuns; ++k) {
            const int64_t i = at + (static_cast<int64_t>(k) * kScanThreads + threadIdx.x) * 4;
            if (i + 4 <= pages) {
                v[k] = *reinterpret_cast<const int4 *>(refs + i);
            } else {
                v[k].x = i < pages ? refs[i] : 0;
                v[k].y = i + 1 < pages ? refs[i + 1] : 0;
                v[k].z = i + 2 < pages ? refs[i + 2] : 0;
                v[k].w = i + 3 < pages ? refs[i + 3] : 0;
            }
        }
    };
    int found = 0;
    int4 v[kRuns], next[kRuns];
    load(0, v);
    for (int64_t at = 0; at < pages && found < most; at += kRound) {
        if (at + kRound < pages) load(at + kRound, next);
        uint32_t flags = 0;
        u64 counts = 0;
        #pragma unroll
        for (int k = 0; k < kRuns; ++k) {
            const int64_t i = at + (static_cast<int64_t>(k) * kScanThreads + threadIdx.x) * 4;
            const int32_t c[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
            #pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < pages && which(c[e], static_cast<int>(i + e))) {
                    flags |= 1u << (4 * k + e);
                    counts += 1ull << (16 * k);
                }
        }
        u64 total;
        const u64 before = block_sums<kScanThreads / 64>(counts, total, part);
        int first = found;
        #pragma unroll
        for (int k = 0; k < kRuns; ++k) {
            int rank = first + static_cast<int>(before >> (16 * k) & 0xFFFF);
            #pragma unroll
            for (int e = 0; e < 4; ++e)
                if (flags >> (4 * k + e) & 1) {
                    if (rank < most)
                        put(rank, static_cast<int>(at + (static_cast<int64_t>(k) * kScanThreads + threadIdx.x) * 4 + e));
                    ++rank;
                }
            first += static_cast<int>(total >> (16 * k) & 0xFFFF);
        }
        found = first;
        #pragma unroll
        for (int k = 0; k < kRuns; ++k) v[k] = next[k];
    }
    return min(found, most);
}

// What the rows lack, in order, and the free pages for it.
__global__ __launch_bounds__(kScanThreads) void give_kernel(Pool p, Space s, int32_t *missing) {
    __shared__ u64 part[kScanThreads / 64];
    u64 need = 0, over = 0;   // entries; those that the table has no place for
    for (int r0 = 0; r0 < p.rows; r0 += kScanThreads) {
        const int r = r0 + threadIdx.x;
        u64 total;
        const u64 mine = r < p.rows ? static_cast<uint32_t>(s.need[r]) | static_cast<u64>(static_cast<uint32_t>(s.base[r])) << 32 : 0;
        const u64 before = block_sums<kScanThreads / 64>(mine & 0xFFFFFFFFull, total, part);
        if (r < p.rows) s.base[r] = static_cast<int32_t>(need + before);
        need += total;
        block_sums<kScanThreads / 64>(mine >> 32, total, part);
        over += total;
    }
    int32_t *const list = s.list;
    const int found = need == 0 ? 0 : rank_pages(
        p.refs, p.pages, static_cast<int>(need), part, [](int32_t count, int) { return count == 0; },
        [&](int rank, int page) { list[rank] = page; });
    if (threadIdx.x == 0) {
        s.counts[0] = found;
        if (missing) *missing = static_cast<int32_t>(min(need - found + over, u64(0x7FFFFFFF)));
    }
}

// ------------------------------------------------------------- resize --

constexpr int kRowThreads = 256;

// Entries first .. last - 1 are those that row r is to have (last may lie beyond the
// table); false: the row stays as it is.
__device__ __forceinline__ bool wanted(const Pool &p, const int32_t *begins, const int32_t *lengths, int r, int &first,
                                       int &last) {
    const int length = lengths[r];
    if (length < 0) return false;
    first = begins ? max(begins[r], 0) / p.page_rows : 0;
    last = static_cast<int>((static_cast<int64_t>(length) + p.page_rows - 1) / p.page_rows);
    return true;
}

__global__ __launch_bounds__(kRowThreads) void resize_look_kernel(Pool p, Space s, const int32_t *begins, const int32_t *lengths) {
    __shared__ int lacks;
    const int r = blockIdx.x;
    int first = 0, last = 0;
    const bool change = wanted(p, begins, lengths, r, first, last);
    if (threadIdx.x == 0) lacks = 0;
    __syncthreads();
    int lack = 0;
    if (change)
        for (int e = threadIdx.x; e < p.stride; e += kRowThreads) {
            const int32_t page = p.row(r)[e];
            const bool want = e >= first && e < last;
            if (p.is_page(page) && !want) {
                atomicSub(p.refs + page, 1);
                p.row(r)[e] = -1;
            }
            lack += want && !p.is_page(page);
        }
    if (lack) atomicAdd(&lacks, lack);
    __syncthreads();
    if (threadIdx.x == 0) {
        s.need[r] = lacks;
        s.base[r] = change ? max(last - max(first, p.stride), 0) : 0;
    }
}

__global__ __launch_bounds__(kRowThreads) void resize_fill_kernel(Pool p, Space s, const int32_t *begins, const int32_t *lengths) {
    __shared__ u64 part[kRowThreads / 64];
    const int r = blockIdx.x;
    if (s.need[r] == 0) return;
    int first = 0, last = 0;
    wanted(p, begins, lengths, r, first, last);
    const int given = s.counts[0];
    int rank = s.base[r];
    const int end = min(last, p.stride);
    for (int e0 = first; e0 < end; e0 += kRowThreads) {
        const int e = e0 + threadIdx.x;
        const bool lacks = e < end && !p.is_page(p.row(r)[e]);
        u64 total;
        const int k = rank + static_cast<int>(block_sums<kRowThreads / 64>(lacks, total, part));
        if (lacks) {
            const int32_t page = k < given ? s.list[k] : -1;
            p.row(r)[e] = page;
            if (page >= 0) p.refs[page] = 1;   // it was free, and is given once
        }
        rank += static_cast<int>(total);
    }
}

// --------------------------------------------------------------- fork --

__device__ __forceinline__ bool forks(const Pool &p, const int32_t *parents, int r) {
    return parents[r] >= 0 && parents[r] < p.rows && parents[r] != r;
}

// The rows of the forks as they will be but for fresh pages (parents may be forks
// themselves: all rows are read before any is written).
__global__ __launch_bounds__(kRowThreads) void fork_look_kernel(Pool p, Space s, const int32_t *parents, const int32_t *lengths) {
    const int r = blockIdx.x;
    if (!forks(p, parents, r)) {
        if (threadIdx.x == 0) s.need[r] = s.base[r] = 0;
        return;
    }
    const int length = max(lengths[r], 0), full = length / p.page_rows;
    const int32_t *from = p.row(parents[r]);
    if (threadIdx.x == 0) {
        s.need[r] = length % p.page_rows && full < p.stride && p.is_page(from[full]);
        s.base[r] = 0;
    }
    int32_t *next = s.next + static_cast<int64_t>(r) * p.stride;
    for (int e = threadIdx.x; e < p.stride; e += kRowThreads) {
        const int32_t page = from[e];
        next[e] = p.is_page(page) && (e < full || (e == full && length % p.page_rows)) ? page : -1;
    }
}

__global__ __launch_bounds__(kRowThreads) void fork_fill_kernel(Pool p, Space s, const int32_t *parents, const int32_t *lengths) {
    const int r = blockIdx.x;
    if (!forks(p, parents, r)) return;
    const int full = max(lengths[r], 0) / p.page_rows, k = s.base[r];
    const bool fresh = s.need[r] != 0;
    const int32_t *next = s.next + static_cast<int64_t>(r) * p.stride;
    for (int e = threadIdx.x; e < p.stride; e += kRowThreads) {
        const int32_t old = p.row(r)[e];
        int32_t page = next[e];
        if (fresh && e == full) {
            const int32_t source = page;
            page = k < s.counts[0] ? s.list[k] : -1;
            if (page >= 0) s.source[k] = source;
        }
        if (p.is_page(old)) atomicSub(p.refs + old, 1);
        if (page >= 0) atomicAdd(p.refs + page, 1);
        p.row(r)[e] = page;
    }
}

// ------------------------------------------------------------ compact --

// Of `live` pages held, those numbered live and more move, in order, to the free
// ones below.
__global__ __launch_bounds__(kScanThreads) void compact_look_kernel(Pool p, Space s, int32_t *moved) {
    __shared__ u64 part[kScanThreads / 64];
    auto nothing = [](int, int) {};
    const int live = rank_pages(p.refs, p.pages, p.pages, part, [](int32_t count, int) { return count > 0; }, nothing);
    int32_t *const list = s.list, *const source = s.source, *const next = s.next;
    const int holes = rank_pages(
        p.refs, live, live, part, [](int32_t count, int) { return count == 0; },
        [&](int rank, int page) { list[rank] = page; });
    // (As many as there are holes, if the counts are right.)
    const int movers = holes == 0 ? 0 : min(holes, rank_pages(
        p.refs, p.pages, p.pages, part,
        [&](int32_t count, int page) {
            if (page >= live) next[page] = page;
            return count > 0 && page >= live;
        },
        [&](int rank, int page) {
            if (rank < holes) source[rank] = page;
        }));
    __syncthreads();
    for (int k = threadIdx.x; k < movers; k += kScanThreads) {
        const int32_t from = source[k], to = list[k];
        next[from] = to;
        p.refs[to] = p.refs[from];
        p.refs[from] = 0;
    }
    if (threadIdx.x == 0) {
        s.counts[0] = movers;
        s.counts[2] = live;
        if (moved) *moved = movers;
    }
}

__global__ __launch_bounds__(256) void compact_table_kernel(Pool p, Space s) {
    const int64_t n = static_cast<int64_t>(p.rows) * p.stride, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= n || s.counts[0] == 0) return;
    const int32_t page = p.table[i];
    if (p.is_page(page) && page >= s.counts[2]) p.table[i] = s.next[page];
}

// ------------------------------------------------------------- copies --

// A launch copies what up to kParts arrays (keys, values and scales of layers) hold
// of each pair of pages, in pieces of kPiece bytes, a workgroup a piece.
constexpr int kParts = 128, kPieceLoads = 4, kPiece = 256 * 16 * kPieceLoads;
struct Copies {
    char *base[kParts];
    uint32_t bytes[kParts];         // of a page, a multiple of 16
    uint32_t first[kParts + 1];     // piece
    int parts, pages;
    const int32_t *source, *target, *count;   // count NULL: n pairs
    int n;
};

__global__ __launch_bounds__(256) void copy_pages_kernel(Copies c) {
    const int64_t per = c.first[c.parts], units = per * (c.count ? min(*c.count, c.n) : c.n);
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int pair = static_cast<int>(u / per);
        const uint32_t piece = static_cast<uint32_t>(u - pair * per);
        int lo = 0, hi = c.parts;   // the part that holds the piece
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            (c.first[mid] <= piece ? lo : hi) = mid;
        }
        const int64_t from = c.source[pair], to = c.target[pair];
        if (from < 0 || from >= c.pages || to < 0 || to >= c.pages || from == to) continue;
        const uint32_t bytes = c.bytes[lo], at = (piece - c.first[lo]) * kPiece + threadIdx.x * 16;
        const char *src = c.base[lo] + from * bytes;
        char *dst = c.base[lo] + to * bytes;
        uint4 v[kPieceLoads];
        #pragma unroll
        for (int k = 0; k < kPieceLoads; ++k)
            if (at + k * 4096 < bytes) v[k] = *reinterpret_cast<const uint4 *>(src + at + k * 4096);
        #pragma unroll
        for (int k = 0; k < kPieceLoads; ++k)
            if (at + k * 4096 < bytes) *reinterpret_cast<uint4 *>(dst + at + k * 4096) = v[k];
    }
}

// Copies of `n` pairs at most (as many as *count says) in all layers.
int copy_pages(const qk_paged_kv *layers, int n_layers, int64_t pages, const int32_t *source, const int32_t *target,
               const int32_t *count, int n, hipStream_t stream) {
    if (n < 1) return QK_OK;
    for (int layer = 0; layer < n_layers;) {
        Copies c{};
        c.pages = static_cast<int>(pages);
        c.source = source;
        c.target = target;
        c.count = count;
        c.n = n;
        auto add = [&](void *base, int64_t bytes) {
            c.base[c.parts] = static_cast<char *>(base);
            c.bytes[c.parts] = static_cast<uint32_t>(bytes);
            c.first[c.parts + 1] = c.first[c.parts] + static_cast<uint32_t>((bytes + kPiece - 1) / kPiece);
            ++c.parts;
        };
        for (; layer < n_layers && c.parts + 4 <= kParts; ++layer) {
            const qk_paged_kv &kv = layers[layer];
            const int64_t rows = static_cast<int64_t>(kv.kv_heads) * kv.page_rows;
            const int64_t code = rows * (kv.type == QK_TYPE_F16 ? 2 * kv.head_dim : kv.type == QK_TYPE_I4 ? kv.head_dim / 2 : kv.head_dim);
            add(kv.key, code);
            add(kv.value, code);
            if (kv.type != QK_TYPE_F16) {
                add(kv.key_scale, rows * (kv.type == QK_TYPE_I4 ? 8 : 4));
                add(kv.value_scale, rows * (kv.type == QK_TYPE_I4 ? 8 : 4));
            }
        }
        const int64_t units = static_cast<int64_t>(c.first[c.parts]) * n;
        hipLaunchKernelGGL(copy_pages_kernel, dim3(static_cast<unsigned>(std::min<int64_t>(units, 2048))), dim3(256), 0, stream, c);
        if (int s = launch_status("page copy launch")) return s;
    }
    return QK_OK;
}

// ------------------------------------------------------------- checks --

int check_layers(const char *where, const qk_paged_kv *layers, int n_layers, int64_t pages, int page_rows) {
    const std::string w(where);
    if (n_layers < 0 || (n_layers > 0 && !layers)) return fail(QK_ERR_INVALID_ARG, w + ": null layers or negative count");
    for (int i = 0; i < n_layers; ++i) {
        if (int s = check_paged_kv(where, layers + i)) return s;
        if (layers[i].pages != pages || layers[i].page_rows != page_rows)
            return fail(QK_ERR_SHAPE, w + ": layer " + std::to_string(i) + " has other pages than the pool");
        const int64_t page = static_cast<int64_t>(layers[i].kv_heads) * page_rows * layers[i].head_dim;
        if (page * 2 > 0x7FFFFFFF) return fail(QK_ERR_LIMIT, w + ": a page of more than 2^31 bytes");
    }
    return QK_OK;
}

int check_pool(const char *where, const qk_page_pool *p) {
    const std::string w(where);
    if (!p || !p->page_table || !p->refs) return fail(QK_ERR_INVALID_ARG, w + ": null pool pointer");
    if (p->table_rows < 1 || p->table_stride < 1 || p->pages < 1)
        return fail(QK_ERR_INVALID_ARG, w + ": empty page table or pool");
    if (p->page_rows < 16 || p->page_rows > 1024 || (p->page_rows & (p->page_rows - 1)))
        return fail(QK_ERR_LIMIT, w + ": page_rows must be a power of two from 16 to 1024");
    // (The launch over the table's entries has fewer than 2^32 threads.)
    if (p->pages > 1 << 30 || p->table_rows >= 1 << 24 || static_cast<int64_t>(p->table_rows) * p->table_stride > 1 << 30)
        return fail(QK_ERR_LIMIT, w + ": more than 2^30 pages or table entries, or 2^24 table rows");
    if (!aligned(p->refs, 16) || !aligned(p->page_table, 4))
        return fail(QK_ERR_ALIGN, w + ": refs must be 16-byte and page_table 4-byte aligned");
    return check_layers(where, p->layers, p->n_layers, p->pages, p->page_rows);
}

int check_space(const char *where, const qk_page_pool *p, const void *workspace, size_t bytes) {
    if (!workspace || bytes < static_cast<size_t>(space_entries(*p)) * 4)
        return fail(QK_ERR_INVALID_ARG, std::string(where) + ": workspace smaller than qk_pages_workspace_bytes");
    if (!aligned(workspace, 16)) return fail(QK_ERR_ALIGN, std::string(where) + ": workspace must be 16-byte aligned");
    return QK_OK;
}

Pool pool_of(const qk_page_pool &p) {
    return Pool{p.page_table, p.refs, p.table_rows, p.table_stride, static_cast<int>(p.pages), p.page_rows};
}

}  // namespace
}  // namespace qk

extern "C" {

size_t qk_pages_workspace_bytes(const qk_page_pool *pool) {
    if (qk::check_pool("qk_pages_workspace_bytes", pool)) return 0;
    return static_cast<size_t>(qk::space_entries(*pool)) * 4;
}

int qk_pages_resize(const qk_page_pool *pool, const int32_t *begins, const int32_t *lengths, int32_t *missing,
                    void *workspace, size_t workspace_bytes, qk_stream stream) {
    const char *where = "qk_pages_resize";
    if (int s = qk::check_pool(where, pool)) return s;
    if (!lengths) return qk::fail(QK_ERR_INVALID_ARG, "qk_pages_resize: null lengths");
    if (!qk::aligned(begins, 4) || !qk::aligned(lengths, 4) || !qk::aligned(missing, 4))
        return qk::fail(QK_ERR_ALIGN, "qk_pages_resize: begins, lengths and missing must be 4-byte aligned");
    if (int s = qk::check_space(where, pool, workspace, workspace_bytes)) return s;
    const qk::Pool p = qk::pool_of(*pool);
    const qk::Space s = qk::space_of(*pool, workspace);
    const dim3 rows(pool->table_rows);
    hipLaunchKernelGGL(qk::resize_look_kernel, rows, dim3(qk::kRowThreads), 0, qk::S(stream), p, s, begins, lengths);
    hipLaunchKernelGGL(qk::give_kernel, dim3(1), dim3(qk::kScanThreads), 0, qk::S(stream), p, s, missing);
    hipLaunchKernelGGL(qk::resize_fill_kernel, rows, dim3(qk::kRowThreads), 0, qk::S(stream), p, s, begins, lengths);
    return qk::launch_status("qk_pages_resize launch");
}

int qk_pages_fork(const qk_page_pool *pool, const int32_t *parents, const int32_t *lengths, int32_t *missing,
                  void *workspace, size_t workspace_bytes, qk_stream stream) {
    const char *where = "qk_pages_fork";
    if (int s = qk::check_pool(where, pool)) return s;
    if (!parents || !lengths) return qk::fail(QK_ERR_INVALID_ARG, "qk_pages_fork: null parents or lengths");
    if (!qk::aligned(parents, 4) || !qk::aligned(lengths, 4) || !qk::aligned(missing, 4))
        return qk::fail(QK_ERR_ALIGN, "qk_pages_fork: parents, lengths and missing must be 4-byte aligned");
    if (int s = qk::check_space(where, pool, workspace, workspace_bytes)) return s;
    const qk::Pool p = qk::pool_of(*pool);
    const qk::Space s = qk::space_of(*pool, workspace);
    const dim3 rows(pool->table_rows);
    hipLaunchKernelGGL(qk::fork_look_kernel, rows, dim3(qk::kRowThreads), 0, qk::S(stream), p, s, parents, lengths);
    hipLaunchKernelGGL(qk::give_kernel, dim3(1), dim3(qk::kScanThreads), 0, qk::S(stream), p, s, missing);
    hipLaunchKernelGGL(qk::fork_fill_kernel, rows, dim3(qk::kRowThreads), 0, qk::S(stream), p, s, parents, lengths);
    if (int status = qk::launch_status("qk_pages_fork launch")) return status;
    const int most = static_cast<int>(std::min<int64_t>(pool->table_rows, pool->pages));
    if (int status = qk::copy_pages(pool->layers, pool->n_layers, pool->pages, s.source, s.list, s.counts, most, qk::S(stream)))
        return status;
    return qk::ok();
}

int qk_pages_compact(const qk_page_pool *pool, int32_t *moved, void *workspace, size_t workspace_bytes, qk_stream stream) {
    const char *where = "qk_pages_compact";
    if (int s = qk::check_pool(where, pool)) return s;
    if (!qk::aligned(moved, 4)) return qk::fail(QK_ERR_ALIGN, "qk_pages_compact: moved must be 4-byte aligned");
    if (int s = qk::check_space(where, pool, workspace, workspace_bytes)) return s;
    const qk::Pool p = qk::pool_of(*pool);
    const qk::Space s = qk::space_of(*pool, workspace);
    const int64_t entries = static_cast<int64_t>(pool->table_rows) * pool->table_stride;
    hipLaunchKernelGGL(qk::compact_look_kernel, dim3(1), dim3(qk::kScanThreads), 0, qk::S(stream), p, s, moved);
    hipLaunchKernelGGL(qk::compact_table_kernel, dim3(static_cast<unsigned>((entries + 255) / 256)), dim3(256), 0,
                       qk::S(stream), p, s);
    if (int status = qk::launch_status("qk_pages_compact launch")) return status;
    if (int status = qk::copy_pages(pool->layers, pool->n_layers, pool->pages, s.source, s.list, s.counts,
                                    static_cast<int>(pool->pages / 2), qk::S(stream)))
        return status;
    return qk::ok();
}

int qk_pages_copy(const qk_paged_kv *layers, int n_layers, const int32_t *source, const int32_t *target, int n,
                  qk_stream stream) {
    if (n < 0 || n_layers < 0) return qk::fail(QK_ERR_INVALID_ARG, "qk_pages_copy: negative count");
    if (n_layers == 0 || n == 0) return qk::ok();
    if (!layers || !source || !target) return qk::fail(QK_ERR_INVALID_ARG, "qk_pages_copy: null pointer");
    if (int s = qk::check_layers("qk_pages_copy", layers, n_layers, layers->pages, layers->page_rows)) return s;
    if (!qk::aligned(source, 4) || !qk::aligned(target, 4))
        return qk::fail(QK_ERR_ALIGN, "qk_pages_copy: source and target must be 4-byte aligned");
    if (int s = qk::copy_pages(layers, n_layers, layers->pages, source, target, nullptr, n, qk::S(stream))) return s;
    return qk::ok();
}

}  // extern "C"
