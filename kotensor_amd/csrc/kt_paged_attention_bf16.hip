// kt_paged_attention_bf16.hip -- attention over pages held in bf16 (kt_paged_attention.h).
#include "kt_paged_attention.h"

namespace kt {

int32_t launch_paged_attention_bf16(const PagedAttnArgs& a, const float* k, const float* v, hipStream_t st) { return paged::launch<KT_PAGED_BF16>(a, k, v, st); }

}  // namespace kt
