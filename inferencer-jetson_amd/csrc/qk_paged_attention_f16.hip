// qk_paged_attention_f16.hip - attention over paged fp16 rows.
#include "qk_paged_attention.h"

namespace qk {

int attend_f16(const PagedAttn &a, bool terms, hipStream_t stream) {
    return attend_type<QK_TYPE_F16>(a, terms, stream);
}

}  // namespace qk
