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

typedef float f4 __attribute__((ext_vector_type(4)));
typedef int32_t i4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct LogitsArgs {
    const float* logits;
    float* out;
    int64_t stride, out_stride;
    int32_t n, text, mask;  // whether the text counts, whether there is a mask
    kt_logits_controls c;
};

// Workgroup (segment of 4 THREADS VECS logits, row): its logits go into registers first; meanwhile it counts the text's
// tokens of its segment in LDS, by integer atomics, whose order changes nothing; then it changes and writes
// each logit once. Every workgroup of a row reads the row's whole text, from L2 after the first.
// Of a token biased twice the later entry holds (the largest entry index).
// Traced: 64 rows of 151936 with texts of up to 4096, 100 biases and masks 19.9 us, 80 MB at 4.0 TB/s (scalar
// accesses after the text: 48.7); one row of 32000 3.0, 5 of 49157 3.7: the launch and two memory round trips.
template <int THREADS, int VECS>
__global__ void __launch_bounds__(THREADS) process_kernel(LogitsArgs a) {
    constexpr int SEGMENT = 4 * THREADS * VECS;
    __shared__ __attribute__((aligned(16))) uint32_t marks[SEGMENT];  // occurrences from output_start on; the top bit: any
    extern __shared__ __attribute__((aligned(16))) int32_t entry[];   // [SEGMENT] with biases: the token's, or -1
    const kt_logits_controls& c = a.c;
    const int32_t r = blockIdx.y, first = blockIdx.x * SEGMENT, count = min(SEGMENT, a.n - first), tid = threadIdx.x;
    const bool biased = c.bias_count > 0;
    const float* x = a.logits + r * a.stride + first;
    float* y = a.out + r * a.out_stride + first;
    // (four logits at 4 (tid + 256 u); rows may begin at any float. A group that the row ends in goes one by one.)
    f4 v[VECS];
#pragma unroll
    for (int u = 0; u < VECS; ++u) {
        const int32_t at = 4 * (tid + u * THREADS);
        v[u] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        if (at + 4 <= count) {
            v[u] = load_any<f4>(x + at);
        } else {
            for (int i = 0; i < 4; ++i)
                if (at + i < count) v[u][i] = x[at + i];
        }
    }
    if (a.text || biased) {
#pragma unroll
        for (int u = 0; u < VECS; ++u) {
            reinterpret_cast<u4*>(marks)[tid + u * THREADS] = u4{0u, 0u, 0u, 0u};
            if (biased) reinterpret_cast<i4*>(entry)[tid + u * THREADS] = i4{-1, -1, -1, -1};
        }
        __syncthreads();
        if (a.text) {
            const int32_t* text = c.history + r * c.history_stride;
            const int64_t length = min(max(static_cast<int64_t>(c.history_length[r]) + c.length_offset, int64_t{0}), static_cast<int64_t>(c.history_capacity));
            const int32_t start = c.output_start ? c.output_start[r] : 0;
            auto mark = [&](int32_t token, int64_t i) {
                const uint32_t at = static_cast<uint32_t>(token) - static_cast<uint32_t>(first);
                if (token < 0 || at >= static_cast<uint32_t>(count)) return;
                atomicOr(&marks[at], 0x80000000u);
                if (i >= start) atomicAdd(&marks[at], 1u);
            };
            const int64_t whole = length / 4;
            for (int64_t i = tid; i < whole; i += THREADS) {
                const i4 t = load_any<i4>(text + 4 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) mark(t[e], 4 * i + e);
            }
            if (tid < length - 4 * whole) mark(text[4 * whole + tid], 4 * whole + tid);
        }
        if (biased) {
            const int32_t* tokens = c.bias_tokens + r * c.bias_stride;
            for (int64_t i = tid; i < c.bias_count; i += THREADS) {
                const uint32_t at = static_cast<uint32_t>(tokens[i]) - static_cast<uint32_t>(first);
                if (tokens[i] >= 0 && at < static_cast<uint32_t>(count)) atomicMax(&entry[at], static_cast<int32_t>(i));
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < VECS; ++u) {
        const int32_t at = 4 * (tid + u * THREADS);
        if (at >= count) break;
        if (a.text) {
            const u4 m = reinterpret_cast<const u4*>(marks)[tid + u * THREADS];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (!m[e]) continue;
                v[u][e] = v[u][e] > 0.0f ? v[u][e] / c.repetition : v[u][e] * c.repetition;
                const uint32_t o = m[e] & 0x7FFFFFFFu;
                if (o) v[u][e] -= static_cast<float>(o) * c.frequency + c.presence;
            }
        }
        if (biased) {
            const i4 b = reinterpret_cast<const i4*>(entry)[tid + u * THREADS];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (b[e] >= 0) v[u][e] += c.bias_values[r * c.bias_stride + b[e]];
        }
        if (a.mask) {
            const uint32_t bits = c.allowed[r * c.allowed_stride + ((first + at) >> 5)] >> ((first + at) & 31);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!(bits >> e & 1u)) v[u][e] = -INFINITY;
        }
        if (at + 4 <= count) {
            __builtin_memcpy(y + at, &v[u], sizeof(f4));
        } else {
            for (int i = 0; i < 4; ++i)
                if (at + i < count) y[at + i] = v[u][i];
        }
    }
}

template <int THREADS, int VECS>
int32_t launch(const LogitsArgs& a, int32_t rows, hipStream_t st) {
    constexpr int SEGMENT = 4 * THREADS * VECS;
    process_kernel<THREADS, VECS><<<dim3(static_cast<uint32_t>((a.n - 1) / SEGMENT + 1), static_cast<uint32_t>(rows)), THREADS,
                           a.c.bias_count > 0 ? SEGMENT * sizeof(int32_t) : 0, st>>>(a);
    KT_LAUNCHED("logits kernel");
    return KT_OK;
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
    hipStream_t st = static_cast<hipStream_t>(stream);
    // Segments of 1024 logits on 256 threads up to four for each CU, of 4096 on 512 (fewer readings of the text) beyond. Rows of
    // 151936, texts of 4096, short and long: 2 rows 4.8 and 5.3 us, 4 5.1 and 5.4, 8 6.2 and 6.2, 16 9.8 and 7.9, 64 25.2 and 20.3
    // (2048 on 256 threads 22.3, 8192 on 1024 19.8, and 16 rows 8.2).
    const int64_t short_ones = (static_cast<int64_t>(n - 1) / 1024 + 1) * rows;
    if (short_ones <= 4 * cu_count()) return launch<256, 1>(a, rows, st);
    return launch<512, 2>(a, rows, st);
}

}  // extern "C"
