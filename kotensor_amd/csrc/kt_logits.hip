// kt_logits.hip -- control of the next token by the text so far: penalties for its tokens,
// biases, and a grammar's mask, on rows of logits. No counterpart in the reference, whose
// greedy choice takes the logits as they are (K/Transformer.kt:253-266).
//
//   y = x;  c = occurrences of the token in the row's text, o = those from output_start on
//   c > 0:  y = y > 0 ? y / repetition : y * repetition
//   o > 0:  y = y - (o * frequency + presence)
//   biased: y = y + bias
//   not allowed: y = -inf
#include <math.h>

#include "kt_common.h"
#include "kt_split.h"

namespace kt {
namespace {

constexpr int THREADS = 256;
constexpr int SEGMENT = 4096;  // logits of a workgroup
typedef float f4 __attribute__((ext_vector_type(4)));

struct LogitsArgs {
    const float* logits;
    float* out;
    int64_t stride, out_stride;
    int32_t n, text, mask;  // whether the text counts, whether there is a mask
    kt_logits_controls c;
};

// Workgroup (segment, row): counts the text's tokens of its segment in LDS, by integer
// atomics, whose order changes nothing, then reads, changes and writes its logits once. Of a token
// biased twice the later entry holds (the largest entry index).
__global__ void __launch_bounds__(THREADS) process_kernel(LogitsArgs a) {
    __shared__ uint32_t marks[SEGMENT];  // occurrences from output_start on; the top bit: any
    __shared__ int32_t entry[SEGMENT];   // the token's bias, or -1
    const kt_logits_controls& c = a.c;
    const int32_t r = blockIdx.y, first = blockIdx.x * SEGMENT, count = min(SEGMENT, a.n - first), tid = threadIdx.x;
    const bool biased = c.bias_count > 0;
    if (a.text) for (int32_t i = tid; i < count; i += THREADS) marks[i] = 0;
    if (biased) for (int32_t i = tid; i < count; i += THREADS) entry[i] = -1;
    __syncthreads();
    if (a.text) {
        const int32_t* text = c.history + r * c.history_stride;
        const int64_t length = min(max(static_cast<int64_t>(c.history_length[r]) + c.length_offset, int64_t{0}), static_cast<int64_t>(c.history_capacity));
        const int32_t start = c.output_start ? c.output_start[r] : 0;
        for (int64_t i = tid; i < length; i += THREADS) {
            const uint32_t at = static_cast<uint32_t>(text[i]) - static_cast<uint32_t>(first);
            if (text[i] < 0 || at >= static_cast<uint32_t>(count)) continue;
            atomicOr(&marks[at], 0x80000000u);
            if (i >= start) atomicAdd(&marks[at], 1u);
        }
    }
    if (biased) {
        const int32_t* tokens = c.bias_tokens + r * c.bias_stride;
        for (int64_t i = tid; i < c.bias_count; i += THREADS) {
            const uint32_t at = static_cast<uint32_t>(tokens[i]) - static_cast<uint32_t>(first);
            if (tokens[i] >= 0 && at < static_cast<uint32_t>(count)) atomicMax(&entry[at], static_cast<int32_t>(i));
        }
    }
    __syncthreads();
    const float* x = a.logits + r * a.stride + first;
    float* y = a.out + r * a.out_stride + first;
    for (int32_t i = tid; i < count; i += THREADS) {
        float v = x[i];
        if (a.text && marks[i]) {
            v = v > 0.0f ? v / c.repetition : v * c.repetition;
            const uint32_t o = marks[i] & 0x7FFFFFFFu;
            if (o) v -= static_cast<float>(o) * c.frequency + c.presence;
        }
        if (biased && entry[i] >= 0) v += c.bias_values[r * c.bias_stride + entry[i]];
        if (a.mask && !(c.allowed[r * c.allowed_stride + ((first + i) >> 5)] >> ((first + i) & 31) & 1u)) v = -INFINITY;
        y[i] = v;
    }
}

}  // namespace
}  // namespace kt

using namespace kt;

extern "C" {

int32_t kt_process_logits(const float* logits, int32_t rows, int32_t n, int64_t stride, const kt_logits_controls* controls, float* out,
                          int64_t out_stride, void* stream) {
    if (!logits || !controls || !out) return fail(KT_ERR_ARGUMENT, "logits, controls or out is NULL");
    if (rows < 0 || n <= 0) return fail(KT_ERR_SHAPE, "logits need rows >= 0 and a vocabulary, got %d x %d", rows, n);
    if (rows > 1 && (stride < n || out_stride < n)) return fail(KT_ERR_SHAPE, "a row of %d logits does not fit its stride", n);
    if (rows > 65535) return fail(KT_ERR_SHAPE, "%d rows in one call: at most 65535", rows);
    const kt_logits_controls& c = *controls;
    if (!(c.repetition > 0.0f) || !(c.repetition < INFINITY)) return fail(KT_ERR_ARGUMENT, "the repetition penalty must be positive and finite");
    if (!(fabsf(c.frequency) < INFINITY) || !(fabsf(c.presence) < INFINITY)) return fail(KT_ERR_ARGUMENT, "the frequency and presence penalties must be finite");
    const bool text = c.repetition != 1.0f || c.frequency != 0.0f || c.presence != 0.0f;
    if (text) {
        if (!c.history || !c.history_length) return fail(KT_ERR_ARGUMENT, "penalties need the history and its length");
        if (c.history_capacity < 0 || c.history_stride < 0 || (rows > 1 && c.history_stride != 0 && c.history_stride < c.history_capacity))
            return fail(KT_ERR_SHAPE, "a history of up to %d tokens does not fit its stride", c.history_capacity);
    }
    if (c.bias_count < 0) return fail(KT_ERR_SHAPE, "negative bias count");
    if (c.bias_count > 0) {
        if (!c.bias_tokens || !c.bias_values) return fail(KT_ERR_ARGUMENT, "bias_tokens or bias_values is NULL");
        if (c.bias_stride != 0 && c.bias_stride < c.bias_count) return fail(KT_ERR_SHAPE, "%d biases do not fit their stride", c.bias_count);
    }
    if (c.allowed && c.allowed_stride != 0 && c.allowed_stride < (static_cast<int64_t>(n) + 31) / 32)
        return fail(KT_ERR_SHAPE, "a mask of %d tokens does not fit its stride", n);
    if (rows == 0) return KT_OK;
    LogitsArgs a{logits, out, stride, out_stride, n, text, c.allowed != nullptr, c};
    process_kernel<<<dim3(static_cast<uint32_t>((n - 1) / SEGMENT + 1), static_cast<uint32_t>(rows)), THREADS, 0, static_cast<hipStream_t>(stream)>>>(a);
    KT_LAUNCHED("logits kernel");
    return KT_OK;
}

}  // extern "C"
