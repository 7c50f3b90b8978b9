// qk_paged.h - the paged cache: argument checks, and the device helpers that
// find a sequence's rows (csrc/qk_paged_cache.hip, csrc/qk_paged_attention.hip).
#pragma once

#include "qk_internal.h"

namespace qk {

// Checks of a cache and of a batch over it; QK_OK or a status.
int check_paged_kv(const char *where, const qk_paged_kv *kv);
int check_paged_batch(const char *where, const qk_paged_batch *batch);

// Whether n rows of wa values, lda apart from a on, share one with n of wb, ldb apart.
bool rows_meet(const float *a, int64_t lda, int64_t wa, const float *b, int64_t ldb, int64_t wb, int64_t n);

// Whether a sequence of a batch takes part (qk.h).
__device__ __forceinline__ bool paged_seq_ok(const qk_paged_seq &s, const qk_paged_batch &b, int page_shift) {
    return s.first >= 0 && s.count >= 1 && s.pos >= 0 && s.table >= 0 && s.count <= b.max_count &&
           s.pos <= b.max_rows - s.count && s.first <= b.n_tokens - s.count && s.table < b.table_rows &&
           ((s.pos + s.count - 1) >> page_shift) < b.table_stride;
}

// The page that holds entry `index` of a table row, or -1.
__device__ __forceinline__ int64_t paged_page(const int32_t *table, int index, int64_t pages) {
    const int64_t page = table[index];
    return page >= 0 && page < pages ? page : -1;
}

}  // namespace qk
