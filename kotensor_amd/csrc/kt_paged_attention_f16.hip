// kt_paged_attention_f16.hip -- attention over pages held in fp16 (kt_paged_attention.h).
#include "kt_paged_attention.h"

namespace kt {

int32_t launch_paged_attention_f16(const PagedAttnArgs& a, const float* k, const float* v, hipStream_t st) { return paged::launch<KT_PAGED_F16>(a, k, v, st); }

}  // namespace kt
