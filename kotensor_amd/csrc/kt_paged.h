// kt_paged.h -- the cache in pages that several sequences share: its memory, a call's batch and
// what the kernels of kt_paged.hip and kt_paged_attention.h read of both.
//
// Memory of a layer: keys and values [pages][kv_heads][page_tokens][head_dim] in fp32, fp16 or bf16;
// token x of a sequence lies in page table[x / page_tokens], row x % page_tokens. Sequence s holds
// lengths[s] tokens; its rows of a call are starts[s] .. starts[s + 1] - 1, row i of them token lengths[s] + i.
// Tables, lengths, starts, masks and depths are read on the device, so nothing of them can be refused
// there: a page outside the pool holds nothing, tokens outside the table are not there, starts that do not
// ascend within the call's rows are a call without rows. No kernel reads or writes outside the pool for any of their values.
#pragma once

#include "kt_common.h"
#include "kt_wave.h"

namespace kt {

struct PagedView {
    uint8_t* keys;  // of the layer
    uint8_t* values;
    int32_t fmt, pages, kv_heads, head_dim, page_shift;
};
struct BatchView {
    const int32_t* tables;
    const int32_t* lengths;
    const int32_t* starts;
    const int32_t* depths;  // NULL: text
    const uint32_t* masks;
    int32_t table_stride, sequences, rows, most_rows, key_bound, mask_words;
};

constexpr int element_bytes(int fmt) { return fmt == KT_PAGED_F32 ? 4 : 2; }

// The first row of sequence s (s up to sequences), held within the call's rows.
__device__ __forceinline__ int32_t start_of(const BatchView& b, int32_t s) { return min(max(b.starts[s], 0), b.rows); }
// Tokens that a sequence's table has room for.
__device__ __forceinline__ int64_t room_of(const PagedView& c, const BatchView& b) { return static_cast<int64_t>(b.table_stride) << c.page_shift; }
// Where token x of a sequence lies (in elements, of dim 0 of kv head g); negative where there is no such place.
__device__ __forceinline__ int64_t place_of(const PagedView& c, const BatchView& b, int32_t s, int64_t x, int32_t g) {
    if (x < 0 || x >= room_of(c, b)) return -1;
    const int32_t page = b.tables[static_cast<size_t>(s) * b.table_stride + (x >> c.page_shift)];
    if (page < 0 || page >= c.pages) return -1;
    const int64_t row = x & ((int64_t{1} << c.page_shift) - 1);
    return ((((static_cast<int64_t>(page) * c.kv_heads + g) << c.page_shift) + row)) * c.head_dim;
}

template <int FMT>
__device__ __forceinline__ float load_element(const uint8_t* p, int64_t at) {
    if constexpr (FMT == KT_PAGED_F32) return reinterpret_cast<const float*>(p)[at];
    else if constexpr (FMT == KT_PAGED_F16) return static_cast<float>(reinterpret_cast<const _Float16*>(p)[at]);
    else return __builtin_bit_cast(float, static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[at]) << 16);
}
// (to the nearest, ties to even: half a step, 2^-11 of the value in fp16, 2^-8 in bf16; fp16 takes
// magnitudes from 65520 on as infinities)
template <int FMT>
__device__ __forceinline__ void store_element(uint8_t* p, int64_t at, float x) {
    if constexpr (FMT == KT_PAGED_F32) reinterpret_cast<float*>(p)[at] = x;
    else if constexpr (FMT == KT_PAGED_F16) reinterpret_cast<_Float16*>(p)[at] = static_cast<_Float16>(x);
    else reinterpret_cast<__bf16*>(p)[at] = static_cast<__bf16>(x);
}

// Whether a launch of that many workgroups has 2^32 threads or more, which no launch has.
constexpr bool too_many(int64_t workgroups, int32_t threads) { return workgroups > UINT32_MAX / threads; }

// The checks of the entry points (kt_paged.hip).
int32_t view_paged(const kt_paged_cache* cache, int32_t layer, PagedView* v);
int32_t view_batch(const kt_paged_batch* batch, const kt_paged_cache* cache, BatchView* v);

// The attention of a batch (kt_paged_attention.h). k and v: NULL, or the projections of a step's tokens (at most one a
// sequence), which the launch rotates, as the queries, appends and attends to.
struct PagedAttnArgs {
    const float* q;
    const float* inv_freq;
    float* context;
    PagedView c;
    BatchView b;
    int32_t num_heads;
    float scale;
};
int32_t launch_paged_attention_f32(const PagedAttnArgs& a, const float* k, const float* v, hipStream_t st);
int32_t launch_paged_attention_f16(const PagedAttnArgs& a, const float* k, const float* v, hipStream_t st);
int32_t launch_paged_attention_bf16(const PagedAttnArgs& a, const float* k, const float* v, hipStream_t st);

}  // namespace kt
