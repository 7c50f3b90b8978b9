// qk_paged_attention_i4.hip - attention over paged 4-bit rows.
#include "qk_paged_attention.h"

namespace qk {

int attend_i4(const PagedAttn &a, bool terms, hipStream_t stream) {
    return attend_type<QK_TYPE_I4>(a, terms, stream);
}

}  // namespace qk
