// kt_paged_attention.hip -- attention over the cache in pages (kt_paged.h): of a decode step, prompts
// and trees of drafted tokens. No counterpart in the reference (K/Attention.kt:277-349 attends in one
// sequence's cache).
#include "kt_paged.h"

namespace kt {
namespace {

// A wave takes one row and query head, its lanes the dims: a key's score is a sum over the wave, the running
// maximum, sum and values are in registers.
template <int FMT, int HD>
__global__ void __launch_bounds__(256) attention_kernel(PagedAttnArgs a) {
    constexpr int DL = HD < 64 ? 1 : HD / 64;
    const PagedView& c = a.c;
    const BatchView& b = a.b;
    const int32_t lane = threadIdx.x & 63;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t row = static_cast<int32_t>(item / a.num_heads), h = static_cast<int32_t>(item % a.num_heads), g = h / (a.num_heads / c.kv_heads);
    if (row >= b.rows) return;
    int32_t s = 0;
    for (int32_t s0 = 0; s0 < b.sequences; s0 += 64) {
        const int32_t end = b.starts[min(s0 + lane, b.sequences - 1) + 1];
        s += __popcll(__ballot(s0 + lane < b.sequences && end <= row));
    }
    if (s >= b.sequences) return;
    const int32_t index = row - b.starts[s], n = start_of(b, s + 1) - start_of(b, s);
    if (index < 0) return;
    const int64_t length = b.lengths[s];
    const float* src = a.q + (static_cast<size_t>(row) * a.num_heads + h) * HD;
    float q[DL], o[DL], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int u = 0; u < DL; ++u) {
        const int32_t d = (lane + 64 * u) % HD, i = d % (HD / 2);
        q[u] = src[d];
        o[u] = 0.0f;
        if (a.inv_freq) {
            float cf, sf, y1, y2;
            rope_sin_cos(static_cast<int32_t>(length + (b.depths ? b.depths[row] : index)), a.inv_freq[i], cf, sf);
            rope_apply(src[i], src[i + HD / 2], cf, sf, y1, y2);
            q[u] = d < HD / 2 ? y1 : y2;
        }
        if (lane >= HD) q[u] = 0.0f;
    }
    const int64_t end = min(min(length + (b.masks ? n : index + 1), static_cast<int64_t>(b.key_bound)), room_of(c, b));
    for (int64_t x = 0; x < end; ++x) {
        if (b.masks && x >= length) {
            const int32_t j = static_cast<int32_t>(x - length);
            if (!(b.masks[static_cast<size_t>(row) * b.mask_words + (j >> 5)] >> (j & 31) & 1)) continue;
        }
        const int64_t at = place_of(c, b, s, x, g);
        if (at < 0) continue;
        float dot = 0.0f, v[DL];
#pragma unroll
        for (int u = 0; u < DL; ++u) {
            const int32_t d = (lane + 64 * u) % HD;
            dot = fmaf(q[u], load_element<FMT>(c.keys, at + d), dot);
            v[u] = load_element<FMT>(c.values, at + d);
        }
        const float score = wave_sum_dpp(dot) * a.scale, top = fmaxf(m, score);
        const float alpha = m == -INFINITY ? 0.0f : expf(m - top), p = expf(score - top);
        l = l * alpha + p;
#pragma unroll
        for (int u = 0; u < DL; ++u) o[u] = o[u] * alpha + p * v[u];
        m = top;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int u = 0; u < DL; ++u)
        if (lane < HD) a.context[(static_cast<size_t>(row) * a.num_heads + h) * HD + lane + 64 * u] = o[u] * inv;
}

template <int FMT>
int32_t launch_format(const PagedAttnArgs& a, hipStream_t st) {
    const int64_t grid = (static_cast<int64_t>(a.b.rows) * a.num_heads + 3) / 4;
    if (grid > INT32_MAX) return fail(KT_ERR_SHAPE, "too many rows and heads in one call");
    const auto kernel = a.c.head_dim == 32 ? attention_kernel<FMT, 32> : a.c.head_dim == 64 ? attention_kernel<FMT, 64>
                        : a.c.head_dim == 128 ? attention_kernel<FMT, 128> : attention_kernel<FMT, 256>;
    kernel<<<static_cast<uint32_t>(grid), 256, 0, st>>>(a);
    KT_LAUNCHED("paged attention kernel");
    return KT_OK;
}

}  // namespace

int32_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t st) {
    return a.c.fmt == KT_PAGED_F32 ? launch_format<KT_PAGED_F32>(a, st) : a.c.fmt == KT_PAGED_F16 ? launch_format<KT_PAGED_F16>(a, st) : launch_format<KT_PAGED_BF16>(a, st);
}

}  // namespace kt
