// qk_pages.hip - a pool of cache pages: given out and taken back, forked, compacted,
// and copied, all on the device.
//
// A call is a few launches.  One over the table's rows (a wave each) says what each
// row gives back and lacks; one adds up what rows lack, in order, and writes down which
// pages are free, a bit each, and how many of each segment of the pool; one over the
// rows again in which a wave finds the free pages of its ranks and fills them in; and
// the copies of contents.
// (Compacting, one workgroup pairs pages to move with free ones before them.)  Pages
// are given in the order of table rows and their entries, lowest page first: what a
// call does depends on the table and the counts alone, and the atomics on the counts
// are sums of whole numbers.
#include "qk_paged.h"

#include <algorithm>

namespace qk {
namespace {

hipStream_t S(qk_stream s) { return static_cast<hipStream_t>(s); }

// ---------------------------------------------------------- workspace --

// What the launches of a call leave each other, in 32-bit numbers: how many pages
// are given (or moved), the free pages of each segment, and all of them a bit each
// (the counts change while pages are given), for each table row what it
// lacks and the rank of its first page, the pages given by rank, the sources of their
// copies, and the rows that a fork makes (or, compacting, the new number of each page).
struct Space {
    int32_t *counts, *free;
    uint64_t *bits;
    int32_t *need, *base, *list, *source, *next;
};
constexpr int kCounts = 16;   // counts[0]: pages given or moved; [1]: wanted; [2]: live pages

// Segments of the pool: 4096 pages, or as many times that as make 256 of them.
constexpr int kSegments = 256, kSegment = 4096;
constexpr int64_t segment_pages(int64_t pages) {
    return (pages + int64_t(kSegments) * kSegment - 1) / (int64_t(kSegments) * kSegment) * kSegment;
}

int64_t list_entries(const qk_page_pool &p) {
    return std::max<int64_t>(std::min<int64_t>(p.pages, static_cast<int64_t>(p.table_rows) * p.table_stride), p.pages / 2 + 1);
}
int64_t bit_words(const qk_page_pool &p) { return (p.pages + kSegment - 1) / kSegment * (kSegment / 64); }
int64_t next_entries(const qk_page_pool &p) {
    return std::max<int64_t>(p.pages, static_cast<int64_t>(p.table_rows) * p.table_stride);
}
int64_t space_entries(const qk_page_pool &p) {
    return kCounts + kSegments + 2 * bit_words(p) + 2 * static_cast<int64_t>(p.table_rows) + 2 * list_entries(p) + next_entries(p);
}
Space space_of(const qk_page_pool &p, void *workspace) {
    Space s;
    s.counts = static_cast<int32_t *>(workspace);
    s.free = s.counts + kCounts;
    s.bits = reinterpret_cast<uint64_t *>(s.free + kSegments);
    s.need = reinterpret_cast<int32_t *>(s.bits + bit_words(p));
    s.base = s.need + p.table_rows;
    s.list = s.base + p.table_rows;
    s.source = s.list + list_entries(p);
    s.next = s.source + list_entries(p);
    return s;
}

struct Pool {
    int32_t *table, *refs;
    int rows, stride, pages, page_rows, segment;
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

// Workgroup 0: the rank of each row's first page; the others: the free pages of a
// segment each.
__global__ __launch_bounds__(kScanThreads) void count_kernel(Pool p, Space s) {
    __shared__ u64 part[kScanThreads / 64];
    u64 total;
    if (blockIdx.x == 0) {
        u64 need = 0;
        for (int r0 = 0; r0 < p.rows; r0 += kScanThreads) {
            const int r = r0 + threadIdx.x;
            const u64 before = block_sums<kScanThreads / 64>(r < p.rows ? s.need[r] : 0, total, part);
            if (r < p.rows) s.base[r] = static_cast<int32_t>(need + before);
            need += total;
        }
        if (threadIdx.x == 0) s.counts[1] = static_cast<int32_t>(need);
        return;
    }
    // A wave 64 pages at a time, a bit a lane.
    const int segment = blockIdx.x - 1, lane = threadIdx.x & 63;
    const int64_t first = static_cast<int64_t>(segment) * p.segment, end = min(first + p.segment, int64_t(p.pages));
    int count = 0;
    constexpr int kLoads = 4;
    for (int64_t w0 = first + threadIdx.x - lane; w0 < end; w0 += kScanThreads * kLoads) {
        int32_t c[kLoads];
        #pragma unroll
        for (int k = 0; k < kLoads; ++k) c[k] = w0 + k * kScanThreads + lane < end ? p.refs[w0 + k * kScanThreads + lane] : 1;
        #pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            const uint64_t word = __builtin_amdgcn_ballot_w64(c[k] == 0);
            if (lane == 0 && w0 + k * kScanThreads < end) s.bits[(w0 + k * kScanThreads) / 64] = word;
            count += __popcll(word);
        }
    }
    block_sums<kScanThreads / 64>(lane == 0 ? static_cast<u64>(count) : 0, total, part);
    if (threadIdx.x == 0) s.free[segment] = static_cast<int32_t>(total);
}

// How many lanes before this one a mask holds.
__device__ __forceinline__ int lanes_before(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

// A wave lists the free pages of ranks base .. base + n - 1 (kFound at most), as far as
// there are, in `found` (LDS of its own); the number of free pages.  From the segment that holds the first one
// on it looks at 4096 pages at a time, a word of 64 a lane.
constexpr int kFound = 256;
__device__ __forceinline__ int find_pages(const Pool &p, const Space &s, int base, int n, int32_t *found) {
    const int lane = threadIdx.x & 63, segments = (p.pages + p.segment - 1) / p.segment;
    int all = 0, segment = 0, skipped = 0;   // the free pages of segments before `segment`
    for (int g0 = 0; g0 < segments; g0 += 64) {
        const int own = g0 + lane < segments ? s.free[g0 + lane] : 0;
        int upto = own;
        #pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int other = __shfl_up(upto, off);
            if (lane >= off) upto += other;
        }
        upto += all;
        const int whole = __popcll(__builtin_amdgcn_ballot_w64(g0 + lane < segments && upto <= base));   // (a run of lanes)
        if (whole > 0) segment = g0 + whole, skipped = __shfl(upto, whole - 1);
        all = __shfl(upto, 63);
    }
    int64_t at = static_cast<int64_t>(segment) * p.segment;
    for (int rank = skipped; at < p.pages && rank < base + n; at += kSegment) {
        const int64_t first = at + lane * 64;
        uint64_t word = first < p.pages ? s.bits[first / 64] : 0;
        const int own = __popcll(word);
        int upto = own;
        #pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int other = __shfl_up(upto, off);
            if (lane >= off) upto += other;
        }
        const int k = rank + upto - own;   // the rank of this lane's first
        if (k < base + n && k + own > base) {
            // Without the ones before rank base: where that many lower bits end, by halves.
            int skip = max(base - k, 0), at_bit = 0;
            const int from = max(k, base) - base, upto_here = min(k + own, base + n) - base;
            for (int width = 32; width > 0; width >>= 1) {
                const int lower = __popcll(word >> at_bit & ((1ull << width) - 1));
                if (skip >= lower) skip -= lower, at_bit += width;
            }
            word = word >> at_bit << at_bit;
            for (int i = from; i < upto_here; ++i, word &= word - 1) found[i] = static_cast<int32_t>(first + __builtin_ctzll(word));
        }
        rank += __shfl(upto, 63);
    }
    asm volatile("" ::: "memory");   // other lanes read it, in the order of the wave's LDS accesses
    return all;
}

// ------------------------------------------------------------- resize --

// Rows of a workgroup, a wave each.  256 rows of 512 entries over 65536 pages: 3.4 us to
// look, 4.3 to count, 4.8 to fill, all of them a launch and a chain of three or four
// loads.  (Bits walked one by one up to a row's first rank: 8.5 to fill.)
constexpr int kRowWaves = 4;

__device__ __forceinline__ int row_of_wave() {
    return blockIdx.x * kRowWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
}

// The row's entries in order, 256 at a time, four loads under way: use(entry, page)
// by the lane that has it, for all lanes at once (entry may be beyond the row).
template <typename Use>
__device__ __forceinline__ void each_entry(const int32_t *row, int first, int end, Use use) {
    const int lane = threadIdx.x & 63;
    constexpr int kLoads = 4;
    for (int e0 = first; e0 < end; e0 += 64 * kLoads) {
        int32_t page[kLoads];
        #pragma unroll
        for (int k = 0; k < kLoads; ++k) page[k] = e0 + k * 64 + lane < end ? row[e0 + k * 64 + lane] : -1;
        #pragma unroll
        for (int k = 0; k < kLoads; ++k) use(e0 + k * 64 + lane, page[k]);
    }
}

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

__global__ __launch_bounds__(64 * kRowWaves) void resize_look_kernel(Pool p, Space s, const int32_t *begins, const int32_t *lengths) {
    const int r = row_of_wave();
    if (r >= p.rows) return;
    int first = 0, last = 0, lacks = 0;
    if (wanted(p, begins, lengths, r, first, last))
        each_entry(p.row(r), 0, p.stride, [&](int e, int32_t page) {
            const bool want = e >= first && e < min(last, p.stride);
            if (p.is_page(page) && !want) {
                atomicSub(p.refs + page, 1);
                p.row(r)[e] = -1;
            }
            lacks += __popcll(__builtin_amdgcn_ballot_w64(want && !p.is_page(page)));
        });
    if ((threadIdx.x & 63) == 0) s.need[r] = lacks;
}

// (What row 0's wave says: the entries that got no page, and those that the table has
// no place for.)
__global__ __launch_bounds__(64 * kRowWaves) void resize_fill_kernel(Pool p, Space s, const int32_t *begins, const int32_t *lengths,
                                                                      int32_t *missing) {
    __shared__ int32_t pages[kRowWaves][kFound];
    int32_t *const found = pages[threadIdx.x >> 6];
    const int r = row_of_wave(), lane = threadIdx.x & 63;
    if (r >= p.rows) return;
    const int n = s.need[r];
    if (n == 0 && (r > 0 || !missing)) return;
    const int base = s.base[r];
    int all = find_pages(p, s, base, min(n, kFound), found);
    if (r == 0 && missing) {
        int64_t over = 0;
        for (int i = lane; i < p.rows; i += 64) {
            int first = 0, last = 0;
            if (wanted(p, begins, lengths, i, first, last)) over += max(last - max(first, p.stride), 0);
        }
        #pragma unroll
        for (int off = 32; off > 0; off >>= 1) over += __shfl_xor(over, off);
        if (lane == 0) *missing = static_cast<int32_t>(min(max(s.counts[1] - all, 0) + over, int64_t(0x7FFFFFFF)));
    }
    if (n == 0) return;
    int first = 0, last = 0;
    wanted(p, begins, lengths, r, first, last);
    int rank = 0, listed = 0;   // of the row's own; those before `listed` are no longer in LDS
    each_entry(p.row(r), first, min(last, p.stride), [&](int e, int32_t page) {
        const bool lacks = e < min(last, p.stride) && !p.is_page(page);
        const uint64_t mask = __builtin_amdgcn_ballot_w64(lacks);
        if (rank + __popcll(mask) > listed + kFound) {   // the next ones, from this entry on
            listed = rank;
            find_pages(p, s, base + listed, min(n - listed, kFound), found);
        }
        const int k = rank + lanes_before(mask);
        if (lacks) {
            const int32_t given = base + k < all ? found[k - listed] : -1;
            p.row(r)[e] = given;
            if (given >= 0) p.refs[given] = 1;   // it was free, and is given once
        }
        rank += __popcll(mask);
    });
}

// --------------------------------------------------------------- fork --

__device__ __forceinline__ bool forks(const Pool &p, const int32_t *parents, int r) {
    return parents[r] >= 0 && parents[r] < p.rows && parents[r] != r;
}

// The rows of the forks as they will be but for fresh pages (parents may be forks
// themselves: all rows are read before any is written).
__global__ __launch_bounds__(64 * kRowWaves) void fork_look_kernel(Pool p, Space s, const int32_t *parents, const int32_t *lengths) {
    const int r = row_of_wave(), lane = threadIdx.x & 63;
    if (r >= p.rows) return;
    int need = 0;
    if (forks(p, parents, r)) {
        const int length = max(lengths[r], 0), full = length / p.page_rows;
        const bool part = length % p.page_rows != 0;
        int32_t *next = s.next + static_cast<int64_t>(r) * p.stride;
        each_entry(p.row(parents[r]), 0, p.stride, [&](int e, int32_t page) {
            const bool held = p.is_page(page) && (e < full || (e == full && part));
            if (e < p.stride) next[e] = held ? page : -1;
            need += __builtin_amdgcn_ballot_w64(held && e == full) != 0;
        });
    }
    if (lane == 0) s.need[r] = need;
}

__global__ __launch_bounds__(64 * kRowWaves) void fork_fill_kernel(Pool p, Space s, const int32_t *parents, const int32_t *lengths,
                                                                    int32_t *missing) {
    const int r = row_of_wave(), lane = threadIdx.x & 63;
    if (r >= p.rows) return;
    const bool fork = forks(p, parents, r);
    if (!fork && r > 0) return;
    const int n = s.need[r], k = s.base[r];
    __shared__ int32_t pages[kRowWaves][kFound];
    int32_t *const found = pages[threadIdx.x >> 6];   // (n is 1 at most)
    int all = 0;
    if (n > 0 || r == 0) all = find_pages(p, s, k, n, found);
    if (r == 0 && lane == 0) {
        s.counts[0] = min(s.counts[1], all);   // pairs to copy
        if (missing) *missing = max(s.counts[1] - all, 0);
    }
    if (!fork) return;
    const int full = max(lengths[r], 0) / p.page_rows;
    const int32_t fresh = n > 0 && k < all ? found[0] : -1;
    const int32_t *next = s.next + static_cast<int64_t>(r) * p.stride;
    each_entry(p.row(r), 0, p.stride, [&](int e, int32_t old) {
        if (e >= p.stride) return;
        int32_t page = next[e];
        if (n > 0 && e == full) {
            if (fresh >= 0) s.source[k] = page, s.list[k] = fresh;
            page = fresh;
        }
        if (p.is_page(old)) atomicSub(p.refs + old, 1);
        if (page >= 0) atomicAdd(p.refs + page, 1);
        p.row(r)[e] = page;
    });
}

// ------------------------------------------------------------ compact --

// Of `live` pages held, those numbered live and more move, in order, to the free
// ones below.  Three looks at all counts: 5000 pages in 16 us, beside 900 of copies.
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
// of each pair of pages, in pieces of kPiece bytes, a workgroup a piece, 2048 of them
// at once.  4.7 GB in and out in 900 us, 5.2 TB/s (torch's copy 4.95); 47 MB, in pieces
// of 4 and 16 KB, in 21 (with 8192 workgroups 24, and 947 the former).
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

// Whether what a call writes (table, counts, its number, workspace) lies apart from all
// else that it takes: rows read their lengths while others write.
int check_apart(const char *where, const qk_page_pool &p, const int32_t *one, const int32_t *two, const int32_t *number,
                const void *workspace) {
    struct Span {
        const void *at;
        int64_t bytes;
    };
    const int64_t rows = static_cast<int64_t>(p.table_rows) * 4;
    const Span all[] = {{p.page_table, rows * p.table_stride}, {p.refs, p.pages * 4}, {number, 4},
                        {workspace, space_entries(p) * 4}, {one, rows}, {two, rows}};
    for (int i = 0; i < 4; ++i)
        for (int j = i + 1; j < 6; ++j) {
            const auto a = reinterpret_cast<uintptr_t>(all[i].at), b = reinterpret_cast<uintptr_t>(all[j].at);
            if (a && b && (a < b ? b - a < static_cast<uintptr_t>(all[i].bytes) : a - b < static_cast<uintptr_t>(all[j].bytes)))
                return fail(QK_ERR_INVALID_ARG, std::string(where) + ": page table, refs, number returned or workspace overlaps another argument");
        }
    return QK_OK;
}

Pool pool_of(const qk_page_pool &p) {
    return Pool{p.page_table, p.refs, p.table_rows, p.table_stride, static_cast<int>(p.pages), p.page_rows,
                static_cast<int>(segment_pages(p.pages))};
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
    if (int s = qk::check_apart(where, *pool, begins, lengths, missing, workspace)) return s;
    const qk::Pool p = qk::pool_of(*pool);
    const qk::Space s = qk::space_of(*pool, workspace);
    const dim3 rows((pool->table_rows + qk::kRowWaves - 1) / qk::kRowWaves), threads(64 * qk::kRowWaves);
    hipLaunchKernelGGL(qk::resize_look_kernel, rows, threads, 0, qk::S(stream), p, s, begins, lengths);
    hipLaunchKernelGGL(qk::count_kernel, dim3(1 + (p.pages - 1) / p.segment + 1), dim3(qk::kScanThreads), 0, qk::S(stream), p, s);
    hipLaunchKernelGGL(qk::resize_fill_kernel, rows, threads, 0, qk::S(stream), p, s, begins, lengths, missing);
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
    if (int s = qk::check_apart(where, *pool, parents, lengths, missing, workspace)) return s;
    const qk::Pool p = qk::pool_of(*pool);
    const qk::Space s = qk::space_of(*pool, workspace);
    const dim3 rows((pool->table_rows + qk::kRowWaves - 1) / qk::kRowWaves), threads(64 * qk::kRowWaves);
    hipLaunchKernelGGL(qk::fork_look_kernel, rows, threads, 0, qk::S(stream), p, s, parents, lengths);
    hipLaunchKernelGGL(qk::count_kernel, dim3(1 + (p.pages - 1) / p.segment + 1), dim3(qk::kScanThreads), 0, qk::S(stream), p, s);
    hipLaunchKernelGGL(qk::fork_fill_kernel, rows, threads, 0, qk::S(stream), p, s, parents, lengths, missing);
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
    if (int s = qk::check_apart(where, *pool, nullptr, nullptr, moved, workspace)) return s;
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
