// qk_paged_attention_i8.hip - attention over paged int8 rows.
#include "qk_paged_attention.h"

namespace qk {

int attend_i8(const PagedAttn &a, bool terms, hipStream_t stream) {
    return attend_type<QK_TYPE_I8>(a, terms, stream);
}

}  // namespace qk
