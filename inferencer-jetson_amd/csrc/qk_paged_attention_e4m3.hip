// qk_paged_attention_e4m3.hip - attention over paged float8 rows.
#include "qk_paged_attention.h"

namespace qk {

int attend_e4m3(const PagedAttn &a, bool terms, hipStream_t stream) {
    return attend_type<QK_TYPE_F8_E4M3>(a, terms, stream);
}

}  // namespace qk
