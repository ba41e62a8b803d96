// kt_kv8.hip -- the KV cache held in 8 bits, with a scale for each block of tokens and head:
// RoPE and the append, the cached attention over it, its rows as fp32, and the copy of a
// prefix. No counterpart in the reference, whose cache is fp32 (K/KVCache.kt:3-59).
//
// Memory of a layer (kt_kv8_cache, include/kotensor_hip.h), slots = max_seq rounded up to whole
// blocks and to whole chunks of 64 tokens:
//   keys    [kv_heads][slots][head_dim] codes;
//   values  [kv_heads][slots / 64][head_dim][64] codes: the 64 tokens of a dim lie in the order
//           of the matrix products' operands (value_byte);
//   scales  [kv_heads][slots / block_tokens], one array for the keys, one for the values;
//   rows    [kv_heads][block_tokens][head_dim] fp32: the rows of the block that is not full yet.
// A block's scale is s = max(m / QMAX, 2^-120), m the largest magnitude of its rows so far (QMAX
// 127 for int8, 448 for e4m3), its codes the nearest to x * (1 / s), ties to even; a value that is
// not finite makes the scale NaN. An append that raises the scale of the open block encodes the
// block again from its fp32 rows, so what the cache holds depends on the rows alone, not on the
// calls they came in. A copy that ends inside the source's open block drops rows that the block's scale may
// come from: it sets the scale's sign bit (readers take the magnitude), and the next append makes the scale and
// the codes anew from the rows that stayed.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "kt_common.h"
#include "kt_split.h"
#include "kt_wave.h"

namespace kt {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

constexpr int THREADS = 256;
constexpr int CHUNK = 64;  // tokens whose values lie together
constexpr float MIN_SCALE = 0x1p-120f;  // a block of zeros: its reciprocal is finite

struct KV8View {
    uint8_t* keys;
    uint8_t* values;
    float* key_scales;
    float* value_scales;
    float* key_rows;
    float* value_rows;
    int32_t fmt, kv_heads, max_seq, head_dim, block, slots;
};

int32_t slots_of(int32_t max_seq, int32_t block) {
    const int32_t unit = block > CHUNK ? block : CHUNK;
    return (max_seq + unit - 1) / unit * unit;
}

int32_t check_shape(const kt_kv8_cache* c) {
    if (!c) return fail(KT_ERR_ARGUMENT, "cache is NULL");
    if (c->format != KT_KV8_INT8 && c->format != KT_KV8_E4M3) return fail(KT_ERR_ARGUMENT, "cache format %d: KT_KV8_INT8 or KT_KV8_E4M3", c->format);
    if (c->layers <= 0 || c->kv_heads <= 0 || c->max_seq <= 0)
        return fail(KT_ERR_ARGUMENT, "layers, key/value heads and maxSequenceLength must be positive");
    if (c->max_seq > INT32_MAX - 128) return fail(KT_ERR_ARGUMENT, "maxSequenceLength %d is too large", c->max_seq);
    if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(KT_ERR_ARGUMENT, "head dimension %d of an 8-bit cache: 32, 64, 128 or 256", c->head_dim);
    if (c->block_tokens != 32 && c->block_tokens != 64 && c->block_tokens != 128)
        return fail(KT_ERR_ARGUMENT, "%d tokens to a block: 32, 64 or 128", c->block_tokens);
    return KT_OK;
}

int32_t view_kv8(const kt_kv8_cache* c, int32_t layer, KV8View* v) {
    if (const int32_t status = check_shape(c)) return status;
    if (!c->keys || !c->values || !c->key_scales || !c->value_scales || !c->key_rows || !c->value_rows)
        return fail(KT_ERR_ARGUMENT, "a pointer of the cache is NULL");
    if (!aligned(c->keys, 16) || !aligned(c->values, 16) || !aligned(c->key_rows, 16) || !aligned(c->value_rows, 16) ||
        !aligned(c->key_scales, 4) || !aligned(c->value_scales, 4))
        return fail(KT_ERR_ARGUMENT, "the cache's codes and rows must be 16-byte aligned");
    if (layer < 0 || layer >= c->layers) return fail(KT_ERR_RANGE, "layer %d out of bounds %d", layer, c->layers);
    v->fmt = c->format;
    v->kv_heads = c->kv_heads;
    v->max_seq = c->max_seq;
    v->head_dim = c->head_dim;
    v->block = c->block_tokens;
    v->slots = slots_of(c->max_seq, c->block_tokens);
    const size_t heads = static_cast<size_t>(layer) * c->kv_heads;
    const size_t codes = heads * v->slots * c->head_dim, scales = heads * (v->slots / v->block);
    const size_t rows = heads * v->block * c->head_dim;
    v->keys = static_cast<uint8_t*>(c->keys) + codes;
    v->values = static_cast<uint8_t*>(c->values) + codes;
    v->key_scales = c->key_scales + scales;
    v->value_scales = c->value_scales + scales;
    v->key_rows = c->key_rows + rows;
    v->value_rows = c->value_rows + rows;
    return KT_OK;
}

// ---- codes ---------------------------------------------------------------------------
// int8 codes are stored + 128 (0x6400 | byte is then the fp16 number 1024 + byte).
template <int FMT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (FMT == KT_KV8_INT8) {
        auto code = [](float x) { return static_cast<uint32_t>(static_cast<int32_t>(fminf(fmaxf(rintf(x), -127.0f), 127.0f)) + 128); };
        return code(a) | code(b) << 8 | code(c) << 16 | code(d) << 24;
    } else {
        auto in = [](float x) { return fminf(fmaxf(x, -448.0f), 448.0f); };
        const int low = __builtin_amdgcn_cvt_pk_fp8_f32(in(a), in(b), 0, false);
        return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(in(c), in(d), low, true));
    }
}
template <int FMT>
__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
    if constexpr (FMT == KT_KV8_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(w >> (8 * i) & 0xFFu) - 128.0f;
    } else {
        x[0] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 0);
        x[1] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 1);
        x[2] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 2);
        x[3] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 3);
    }
}
template <int FMT>
constexpr float QMAX = FMT == KT_KV8_INT8 ? 127.0f : 448.0f;

// The scale of a block whose largest magnitude has these bits (past the largest finite number's
// for an infinity or a NaN).
template <int FMT>
__device__ __forceinline__ float scale_of(uint32_t magnitude) {
    if (magnitude >= 0x7F800000u) return __builtin_nanf("");
    return fmaxf(__builtin_bit_cast(float, magnitude) / QMAX<FMT>, MIN_SCALE);
}

// Where the values of the four tokens 4 quad .. + 3 of a dim lie in its 64 bytes of a chunk.
__device__ __forceinline__ int32_t value_byte(int32_t quad) {
    const int32_t h = quad >> 3, r = quad & 7;
    return (2 * (r >> 2) + (r & 1)) * 16 + h * 8 + ((r >> 1) & 1) * 4;
}

// ---- RoPE and the append ---------------------------------------------------------------
// Workgroup (block y of those the new tokens touch, kv head, keys or values) rotates and
// encodes its block through LDS; further workgroups rotate q. Traced, 32 query and 8 kv heads: one token 4.2 us, the
// launch and three memory round trips; 1024 tokens of heads of 64 9.4 us (22 MB moved: 4.3 at a copy's rate), 1501 of
// heads of 128 16.0 (65 MB, 13), bound by the double-precision cosines of the keys' workgroups, each of which makes
// its block's anew (a table of them would be another launch).
// The first block's earlier rows come from the fp32 rows of the open block, which the last
// block's rows replace: where the first block has earlier rows, one workgroup does both, in
// that order.
constexpr int Q_HEADS = 8;
struct AppendArgs {
    KV8View c;
    const float* q;
    const float* k;
    const float* v;
    float* q_out;
    const float* inv_freq;
    const int32_t* position;
    int32_t tokens, num_heads;
    int32_t blocks;  // most blocks the tokens may touch
};

__device__ __forceinline__ uint32_t block_max(uint32_t m, uint32_t (&part)[THREADS / 64]) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), o)));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
    m = max(max(part[0], part[1]), max(part[2], part[3]));
    __syncthreads();
    return m;
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }
// Whether a block's scale says that rows of it were dropped (a NaN may say so, too).
__device__ __forceinline__ bool shortened(float scale) { return __builtin_bit_cast(uint32_t, scale) >> 31; }

// The block b of a head, of whose rows 0 .. n - 1 those from lo on are new.
template <int FMT, bool KEYS>
__device__ void append_block(const AppendArgs& a, float* lds, uint32_t (&part)[THREADS / 64], int32_t g, int32_t b, int32_t p0, int32_t lo, int32_t n) {
    const KV8View& c = a.c;
    const int32_t HD = c.head_dim, B = c.block, LR = HD + 1, tid = threadIdx.x;
    float* rows = (KEYS ? c.key_rows : c.value_rows) + static_cast<size_t>(g) * B * HD;
    const int32_t t0 = b * B - p0;  // token of row 0 in this call
    const bool open = n < B;
    float* scale = (KEYS ? c.key_scales : c.value_scales) + static_cast<size_t>(g) * (c.slots / B) + b;
    const float held = lo > 0 ? *scale : 0.0f;
    uint32_t m = 0;
    constexpr int AHEAD = 4;  // pairs, or groups of four values, a thread loads at a time
    if constexpr (KEYS) {
        const int32_t half = HD >> 1, pairs = (n - lo) * half;
        for (int32_t e0 = tid; e0 < pairs; e0 += AHEAD * THREADS) {
            float x1[AHEAD], x2[AHEAD], f[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int32_t e = min(e0 + u * THREADS, pairs - 1), r = lo + e / half, i = e % half;
                const float* src = a.k + (static_cast<size_t>(t0 + r) * c.kv_heads + g) * HD + i;
                x1[u] = src[0];
                x2[u] = src[half];
                f[u] = a.inv_freq[i];
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int32_t e = e0 + u * THREADS, r = lo + e / half, i = e % half;
                if (e >= pairs) break;
                float cf, sf, y1, y2;
                rope_sin_cos(b * B + r, f[u], cf, sf);
                rope_apply(x1[u], x2[u], cf, sf, y1, y2);
                lds[r * LR + i] = y1;
                lds[r * LR + i + half] = y2;
                m = max(m, max(magnitude(y1), magnitude(y2)));
                if (open) {
                    rows[r * HD + i] = y1;
                    rows[r * HD + i + half] = y2;
                }
            }
        }
    } else {
        const int32_t quads = (n - lo) * (HD / 4);
        for (int32_t e0 = tid; e0 < quads; e0 += AHEAD * THREADS) {
            f4 y[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int32_t e = min(e0 + u * THREADS, quads - 1), r = lo + e / (HD / 4), d = 4 * (e % (HD / 4));
                y[u] = load_any<f4>(a.v + (static_cast<size_t>(t0 + r) * c.kv_heads + g) * HD + d);
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int32_t e = e0 + u * THREADS, r = lo + e / (HD / 4), d = 4 * (e % (HD / 4));
                if (e >= quads) break;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    lds[r * LR + d + i] = y[u][i];
                    m = max(m, magnitude(y[u][i]));
                }
                if (open) *reinterpret_cast<f4*>(rows + r * HD + d) = y[u];
            }
        }
    }
    m = block_max(m, part);
    int32_t from = lo;
    if (lo > 0 && shortened(held)) {  // the earlier rows that stayed, and the scale of all
        from = 0;
        for (int32_t e = tid; e < lo * HD; e += THREADS) {
            lds[e / HD * LR + e % HD] = rows[e];
            m = max(m, magnitude(rows[e]));
        }
        m = block_max(m, part);
    }
    float s = scale_of<FMT>(m);
    if (from > 0) {
        if (held != held || held >= s) {
            s = held;
        } else if (s == s) {  // raised: the earlier rows again
            from = 0;
            for (int32_t e = tid; e < lo * HD; e += THREADS) lds[e / HD * LR + e % HD] = rows[e];
        }
    }
    __syncthreads();  // the rows are in LDS, every thread has read the held scale
    if (tid == 0) *scale = s;
    const float inv = s == s ? 1.0f / s : 0.0f;
    auto at = [&](int32_t r, int32_t d) { return s == s ? lds[r * LR + d] * inv : 0.0f; };
    if constexpr (KEYS) {
        uint8_t* dst = c.keys + (static_cast<size_t>(g) * c.slots + static_cast<size_t>(b) * B) * HD;
        for (int32_t e = tid; e < (n - from) * (HD / 4); e += THREADS) {
            const int32_t r = from + e / (HD / 4), d = 4 * (e % (HD / 4));
            reinterpret_cast<uint32_t*>(dst + r * HD)[d / 4] = encode4<FMT>(at(r, d), at(r, d + 1), at(r, d + 2), at(r, d + 3));
        }
    } else {
        uint8_t* dst = c.values + static_cast<size_t>(g) * c.slots * HD;
        const int32_t q0 = from >> 2, quads = ((n + 3) >> 2) - q0;
        for (int32_t e = tid; e < quads * HD; e += THREADS) {
            const int32_t r = 4 * (q0 + e % quads), d = e / quads, tok = b * B + r;
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = r + i >= from && r + i < n ? at(r + i, d) : 0.0f;
            const uint32_t w = encode4<FMT>(x[0], x[1], x[2], x[3]);
            uint8_t* to = dst + (static_cast<size_t>(tok / CHUNK) * HD + d) * CHUNK + value_byte(tok % CHUNK / 4);
            if (r >= from && r + 4 <= n) {
                *reinterpret_cast<uint32_t*>(to) = w;
            } else {  // other tokens' bytes stay as they are
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (r + i >= from && r + i < n) to[i] = static_cast<uint8_t>(w >> (8 * i));
            }
        }
    }
}

template <int FMT>
__global__ void __launch_bounds__(THREADS) append_kernel(AppendArgs a) {
    extern __shared__ float append_lds[];
    __shared__ uint32_t part[THREADS / 64];
    const KV8View& c = a.c;
    const int32_t HD = c.head_dim, B = c.block;
    const int32_t p0 = *a.position;
    int32_t id = blockIdx.x;
    const int32_t roles = a.blocks * c.kv_heads * 2;
    if (id < roles) {
        if (p0 < 0 || p0 >= c.max_seq) return;  // the host checks capacity; never write outside the cache
        const int32_t end = p0 + min(a.tokens, c.max_seq - p0);
        const int32_t g = id / 2 % c.kv_heads, y = id / 2 / c.kv_heads;
        const bool keys = id % 2 == 0;
        const int32_t b0 = p0 / B, b1 = (end - 1) / B;
        const bool both = p0 % B != 0 && b1 > b0;  // workgroup 0 does the last block after the first
        if (y > b1 - b0 || (both && y == b1 - b0)) return;
        for (int32_t b = b0 + y;; b = b1) {
            const int32_t lo = max(p0 - b * B, 0), n = min(B, end - b * B);
            if (keys) append_block<FMT, true>(a, append_lds, part, g, b, p0, lo, n);
            else append_block<FMT, false>(a, append_lds, part, g, b, p0, lo, n);
            if (y > 0 || !both || b == b1) return;
            __syncthreads();  // the first block's rows are read
        }
    }
    // q: a thread's pair of a token, Q_HEADS heads whose loads go out together
    const int32_t half = HD >> 1, per = THREADS / half, groups = (a.num_heads + Q_HEADS - 1) / Q_HEADS;
    id -= roles;
    const int32_t i = threadIdx.x % half, t = id / groups * per + threadIdx.x / half, h0 = id % groups * Q_HEADS;
    if (t >= a.tokens) return;
    const size_t row = static_cast<size_t>(t) * a.num_heads * HD + i;
    float x1[Q_HEADS], x2[Q_HEADS], cf, sf;
#pragma unroll
    for (int u = 0; u < Q_HEADS; ++u) {
        const size_t at = row + static_cast<size_t>(min(h0 + u, a.num_heads - 1)) * HD;
        x1[u] = a.q[at];
        x2[u] = a.q[at + half];
    }
    rope_sin_cos(p0 + t, a.inv_freq[i], cf, sf);
#pragma unroll
    for (int u = 0; u < Q_HEADS; ++u) {
        if (h0 + u >= a.num_heads) break;
        float y1, y2;
        rope_apply(x1[u], x2[u], cf, sf, y1, y2);
        a.q_out[row + (h0 + u) * HD] = y1;
        a.q_out[row + (h0 + u) * HD + half] = y2;
    }
}

// ---- the cached attention -----------------------------------------------------------------
// Rows: the (token, query head) pairs of a kv head, token t's G heads side by side; a workgroup
// (kv head, tile of R rows, key split) holds its rows as matrix operands and its waves take the
// split's chunks of 64 keys in turn. Codes are exact in fp16, and a query is the sum of two fp16
// numbers to 2^-22 of its row's largest element (the row scaled by a power of two to 2^13 .. 2^14), so
// two fp16 products with fp32 sums give a score in fp32 precision; likewise a weight for the values.
//   S^T = K Q^T: a lane ends with scores of one row (its column), so that the running maximum and sum of a
//     row stay inside the lanes of a column; the exponentials are v_exp_f32 of one multiply-add.
//   O^T += V^T P^T: the values lie in memory such that the scores' lanes are the operand's.
// A wave's maximum follows a row's lazily: a larger score moves it only once it is 2^8 above (the weights
// then stay below 2^15 in fp16, being taken times 2^6), so that the sums are seldom rescaled.
// A block's value scale 2^e mu joins the exponent as log2(mu) and e less the row's own exponent, that of its largest
// contribution (weight times scale) so far, likewise moved lazily: weights include it, and the sum of weights takes it out
// again, with one product a set of 32 keys. So a weight's parts end 2^-30 below the row's largest contribution, whatever
// the loudness of blocks that the row hardly attends to or does not see.
// Waves' sums meet in LDS; key splits' through memory, where the last workgroup of a tile to arrive (a counter,
// which it returns to zero) merges all in their order: no workgroup waits for another, and the bits do not depend on
// who is last.
// Traced, 32 query and 8 kv heads: a step with its append at 131072 keys of 128 dims (e4m3) 54.8 us, 269 MB at
// 4.9 TB/s, the rate of a large copy; at 8192 keys of 64 (int8) 11.6 us, of which the cache's 8.4 MB are 1.7: latencies
// of the launch, the position, the keys (3.6 us to the end of the scores' work), the append in the last split (1.4) and
// the splits' meeting (4); at 544 keys of 2 kv heads, a bound at the length, 8.8. Seven tokens after 4000 (e4m3) 12.1. A prompt
// of 1024 tokens 21.7 us; 301 tokens after 7000 (heads of 128, int8) 118: 300 Tflop/s, 600 in the products of two parts, bound by the
// vector work beside them (592 instructions a wave and 64 keys, 256 of them the codes' conversion, for 64 products).
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));

struct AttnArgs {
    // (what the first loads need comes first: it arrives with the wave)
    const int32_t* position;
    const float* q;
    // one token with RoPE and the append inside: its projections before RoPE
    const float* k_new;
    const float* v_new;
    const float* inv_freq;
    int32_t tokens, num_heads;
    float scale;
    KV8View c;
    float* context;
    // key splits: most of them, and their rows' averages [kv_heads][tiles][splits][R][head_dim], maxima and
    // sums [..][R][2], and a counter for each (kv head, tile), zero between launches
    int32_t max_splits;
    float* averages;
    float* stats;
    uint32_t* counters;
};

constexpr float LAZY = 8.0f;      // how far a score may pass the maximum, in powers of two
constexpr float WEIGHT_UP = 6.0f; // weights are taken times 2^6
constexpr float MOST_QUIET = 40.0f; // how far below the row's a value scale's exponent goes into the exponentials
constexpr float NO_EXPONENT = -1000.0f; // of a row without a contribution so far

// Eight codes as fp16.
template <int FMT>
__device__ __forceinline__ half8 to_half8(u2 w) {
    half8 out;
    half2v* o = reinterpret_cast<half2v*>(&out);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (FMT == KT_KV8_INT8) {  // 0x6400 | byte is 1024 + byte
            const half2v low = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
            o[2 * i] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w[i], 0x04010400u)) + low;
            o[2 * i + 1] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w[i], 0x04030402u)) + low;
        } else {
            o[2 * i] = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w[i]), 1.0f, false));
            o[2 * i + 1] = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w[i]), 1.0f, true));
        }
    }
    return out;
}
__device__ __forceinline__ u2 half_of(u4 v, int i) { return i ? u2{v[2], v[3]} : u2{v[0], v[1]}; }

// Eight numbers as the sum of two fp16 operands.
__device__ __forceinline__ void split2(const float (&v)[8], half8& hi, half8& lo) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const half2v h = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(v[2 * i], v[2 * i + 1]));
        float a, b;  // what is left of the two: one mixed multiply-add each (the compiler converts and subtracts)
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(a) : "v"(h), "v"(v[2 * i]));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(b) : "v"(h), "v"(v[2 * i + 1]));
        // (to the nearest, so that what weights below fp16's normal numbers lose has no sign)
        const half2v l = __builtin_convertvector((f2v{a, b}), half2v);
        hi[2 * i] = h[0];
        hi[2 * i + 1] = h[1];
        lo[2 * i] = l[0];
        lo[2 * i + 1] = l[1];
    }
}

// The maximum is a rounded product; at sizes where its rounding is a power of two and more, the
// exponent is the difference of rounded products, so that it stays below LAZY.
constexpr float HUGE_SCORE = 65536.0f;
__device__ __forceinline__ float weight_of_huge(float x, float f, float m, float shift) {
#pragma clang fp contract(off)
    const float s = x * f;
    return __builtin_amdgcn_exp2f((s - m) - shift);
}
// A score as the maxima hold it: rounded, also where the next step subtracts one.
__device__ __forceinline__ float rounded_score(float x, float f) {
#pragma clang fp contract(off)
    return x * f;
}

// The largest of a value over the lanes of a column (lanes apart by 16 or 32).
struct Swapped {
    float a, b;  // of two lanes apart by 16 (32): the value of the one and of the other, in both
};
// (the compiler's builtins for these gave the first result in the place of the second, too; the wait states
// are those between a vector write and the swap's read)
__device__ __forceinline__ Swapped swap16(float v) {
    Swapped s{v, v};
    asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(s.a), "+v"(s.b));
    return s;
}
__device__ __forceinline__ Swapped swap32(float v) {
    Swapped s{v, v};
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(s.a), "+v"(s.b));
    return s;
}
template <int R>
__device__ __forceinline__ float column_max(float v) {
    if constexpr (R == 16) {
        const Swapped s = swap16(v);
        v = fmaxf(s.a, s.b);
    }
    const Swapped s = swap32(v);
    return fmaxf(s.a, s.b);
}
template <int R>
__device__ __forceinline__ float column_sum(float v) {
    if constexpr (R == 16) {
        const Swapped s = swap16(v);
        v = s.a + s.b;
    }
    const Swapped s = swap32(v);
    return s.a + s.b;
}

// What a part with the maximum m and the sum l counts beside parts with the maximum mx: a part without keys
// (l = 0) nothing, one with a NaN a NaN.
__device__ __forceinline__ float share_of(float m, float l, float mx) {
    return l == 0.0f ? 0.0f : l * __builtin_amdgcn_exp2f((m == -INFINITY ? mx : m) - (mx == -INFINITY ? 0.0f : mx));
}
constexpr int MAX_SPLITS = 128;
constexpr int THROUGH = 1 | 16;  // buffer cache bits sc0 sc1: past the caches

// The shapes of the products: R = 16 rows on 16x16x32, or R = 32 CT on 32x32x16.
template <int HD, int R>
struct Shape {
    static constexpr bool SMALL = R == 16;
    static constexpr int CT = SMALL ? 1 : R / 32;         // column tiles
    static constexpr int E = SMALL ? 8 : 16;              // scores of a lane in a set of 32 keys
    static constexpr int QS = SMALL ? HD / 32 : HD / 16;  // steps of a score
    static constexpr int KL = SMALL ? (HD + 63) / 64 : HD / 32;  // 16-byte loads of a key's share (HD 32 and R 16: 8 bytes used)
    static constexpr int KT = SMALL ? 4 : 2;              // groups of keys with loads of their own in a chunk
    static constexpr int DB = SMALL ? HD / 16 : HD / 32;  // dim blocks of the output
    static constexpr int VL = SMALL ? 1 : 2;              // 16-byte loads of a dim
    static constexpr int OE = SMALL ? 4 : 16;
    static constexpr bool QREG = SMALL && HD < 256;       // a row's operands stay in registers
    static constexpr int J = SMALL ? 2 : 1;               // sets of 32 keys that share a maximum's check
};

// Splits of a tile's keys, from the number of chunks alone.
__host__ __device__ __forceinline__ int32_t splits_of(int32_t chunks, int32_t waves, int32_t most) {
    const int32_t s = (chunks + waves - 1) / waves;
    return s < 1 ? 1 : s < most ? s : most;
}

// What a workgroup that appends the step's token shares: the rotation, and the token's codes.
template <int HD, bool STEP>
struct StepShared {
    __attribute__((aligned(16))) float cosines[HD / 2], sines[HD / 2];
    __attribute__((aligned(16))) uint8_t key[HD], value[HD];
    uint32_t top[4];
    uint32_t rest[2][8];
};
template <int HD>
struct StepShared<HD, false> {};

// The append of a step's token at pos in the workgroup whose keys end with it: threads 0 .. 127 hold the pairs (i, i + half) of
// its key, the next 128 those of its value (y1, y2, `on` where there is one; each wave's largest magnitude
// in sh.top); held: the scales of its block. Returns whether earlier rows of the block changed (their codes are in memory when the
// workgroup's next barrier has passed); the token's codes are in sh, and the block's scales in held.
template <int FMT, int HD, int NT>
__device__ bool append_token(const KV8View& c, StepShared<HD, true>& sh, int32_t g, int32_t pos, bool on, float y1, float y2, float (&held)[2]) {
    constexpr int HALF = HD / 2;
    const int32_t tid = threadIdx.x, B = c.block, b = pos / B, r = pos % B, i = tid & 127;
    const bool is_key = tid < 128;
    uint32_t most[2] = {max(sh.top[0], sh.top[1]), max(sh.top[2], sh.top[3])};
    float* rows[2] = {c.key_rows + static_cast<size_t>(g) * B * HD, c.value_rows + static_cast<size_t>(g) * B * HD};
    const bool remake[2] = {r > 0 && shortened(held[0]), r > 0 && shortened(held[1])};
    if (remake[0] || remake[1]) {  // the earlier rows that stayed count for the scale
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            uint32_t m = 0;
            for (int32_t e = tid; e < r * (HD / 4); e += NT) {
                const f4 x = *reinterpret_cast<const f4*>(rows[w] + 4 * e);
                m = max(max(m, max(magnitude(x[0]), magnitude(x[1]))), max(magnitude(x[2]), magnitude(x[3])));
            }
            for (int o = 32; o > 0; o >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), o)));
            if ((tid & 63) == 0) sh.rest[w][tid >> 6] = m;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 2; ++w)
            for (int i = 0; remake[w] && i < NT / 64; ++i) most[w] = max(most[w], sh.rest[w][i]);
    }
    bool raised[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const float own = scale_of<FMT>(most[w]);
        raised[w] = r > 0 && (remake[w] ? own == own : held[w] < own);  // (below: neither of them NaN)
        if (r == 0 || raised[w] || remake[w] || own != own) held[w] = own;
    }
    uint8_t* kdst = c.keys + (static_cast<size_t>(g) * c.slots + static_cast<size_t>(b) * B) * HD;
    uint8_t* vdst = c.values + static_cast<size_t>(g) * c.slots * HD;
    auto value_to = [&](int32_t tok, int32_t d) { return vdst + (static_cast<size_t>(tok / CHUNK) * HD + d) * CHUNK + value_byte(tok % CHUNK / 4) + tok % 4; };
    if (on) {
        const float s = is_key ? held[0] : held[1], inv = s == s ? 1.0f / s : 0.0f;
        const uint32_t w = encode4<FMT>(s == s ? y1 * inv : 0.0f, s == s ? y2 * inv : 0.0f, 0.0f, 0.0f);
        const uint8_t c1 = static_cast<uint8_t>(w), c2 = static_cast<uint8_t>(w >> 8);
        (is_key ? sh.key : sh.value)[i] = c1;
        (is_key ? sh.key : sh.value)[i + HALF] = c2;
        if (is_key) {
            kdst[r * HD + i] = c1;
            kdst[r * HD + i + HALF] = c2;
        } else {
            *value_to(pos, i) = c1;
            *value_to(pos, i + HALF) = c2;
        }
        if (r + 1 < B) {
            float* row = (is_key ? rows[0] : rows[1]) + r * HD + i;
            row[0] = y1;
            row[HALF] = y2;
        }
        if (i == 0) (is_key ? c.key_scales : c.value_scales)[static_cast<size_t>(g) * (c.slots / B) + b] = s;
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        if (!raised[w]) continue;
        const float inv = 1.0f / held[w];
        for (int32_t e = tid; e < r * (HD / 4); e += NT) {
            const int32_t row = e / (HD / 4), d = 4 * (e % (HD / 4));
            const f4 x = *reinterpret_cast<const f4*>(rows[w] + row * HD + d);
            const uint32_t codes = encode4<FMT>(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
            if (w == 0) {
                reinterpret_cast<uint32_t*>(kdst)[e] = codes;
            } else {
#pragma unroll
                for (int u = 0; u < 4; ++u) *value_to(b * B + row, d + u) = static_cast<uint8_t>(codes >> (8 * u));
            }
        }
    }
    const bool again = raised[0] || raised[1];
    if (again) __threadfence();
    return again;
}

template <int FMT, int HD, int R, int NW, bool STEP>
__global__ void __launch_bounds__(64 * NW, R > 16 ? 2 : 1) attention_kernel(AttnArgs a) {
    using X = Shape<HD, R>;
    constexpr int LR = HD + 4;  // padded row of the waves' averages
    extern __shared__ __attribute__((aligned(16))) float attn_lds[];
    float* avg = attn_lds;               // [NW][R][LR]
    float* ms = avg + NW * R * LR;       // [NW][R]
    float* ls = ms + NW * R;             // [NW][R]
    __shared__ float fr_s[R];
    const KV8View& c = a.c;
    const int32_t g = blockIdx.x, tile = gridDim.y - 1 - blockIdx.y, split = blockIdx.z;
    const int32_t G = a.num_heads / c.kv_heads, rows = a.tokens * G;
    const int32_t tid = threadIdx.x, lane = tid & 63;
    const int32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int32_t col = X::SMALL ? lane & 15 : lane & 31, grp = X::SMALL ? lane >> 4 : lane >> 5;

    // The rows' queries, sixteen lanes to a row (four dims each, or 64 apart; for the rotation those of the dims'
    // pairs, too), go out ahead of the position, as does a step's token.
    constexpr int RW = R / (4 * NW) > 0 ? R / (4 * NW) : 1, DL = HD / 64 > 0 ? HD / 64 : 1;
    const int32_t held = min(R, rows - tile * R);  // rows of this tile
    const int32_t lr = lane >> 4, lc = lane & 15;
    f4 qv[RW][DL], qo[STEP ? RW : 1][STEP ? DL : 1];
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        const int32_t row = tile * R + min(4 * (wave + i * NW) + lr, held - 1), t = STEP ? 0 : row / G;
        const float* src = a.q + (static_cast<size_t>(t) * a.num_heads + g * G + (row - t * G)) * HD;
#pragma unroll
        for (int u = 0; u < DL; ++u) {
            const int32_t d = (4 * lc + 64 * u) % HD;
            qv[i][u] = *reinterpret_cast<const f4*>(src + d);
            if constexpr (STEP) qo[i][u] = *reinterpret_cast<const f4*>(src + (d + HD / 2) % HD);
        }
    }
    __shared__ StepShared<HD, STEP> sh;
    constexpr int HALF = HD / 2;
    const bool on = STEP && tid < 256 && (tid & 127) < HALF;  // threads with a pair of the key or the value
    float x1 = 0.0f, x2 = 0.0f, ifr = 0.0f;
    if constexpr (STEP) {
        if (on) {
            const float* src = (tid < 128 ? a.k_new : a.v_new) + g * HD + (tid & 127);
            x1 = src[0];
            x2 = src[HALF];
            ifr = a.inv_freq[tid & 127];
        }
    }
    const int32_t P0 = *a.position;
    const int32_t t_first = tile * R / G, t_last = min((tile * R + R - 1) / G, a.tokens - 1);
    auto last_key = [&](int32_t t) { return min(P0 + t, c.max_seq - 1); };  // negative: none; never read outside the cache
    const int32_t n_keys = last_key(t_last) + 1, n_all = last_key(t_first) + 1;  // keys of any row, of every row
    const int32_t chunks = n_keys > 0 ? (n_keys + CHUNK - 1) / CHUNK : 0;
    const int32_t splits = splits_of(chunks, NW, a.max_splits);
    if (split >= splits) return;
    // (a block's chunks stay together: a step that changes its codes is the only one to read them)
    const int32_t per = c.block > CHUNK ? c.block / CHUNK : 1, units = (chunks + per - 1) / per;
    // (fewer than 2^25 units, at most 2^7 splits)
    const int32_t c0 = per * static_cast<int32_t>(static_cast<uint32_t>(units) * split / static_cast<uint32_t>(splits));
    const int32_t c1 = min(per * static_cast<int32_t>(static_cast<uint32_t>(units) * (split + 1) / static_cast<uint32_t>(splits)), chunks);

    const uint8_t* kbase = c.keys + static_cast<size_t>(g) * c.slots * HD;
    const uint8_t* vbase = c.values + static_cast<size_t>(g) * c.slots * HD;
    const float* kscale = c.key_scales + static_cast<size_t>(g) * (c.slots / c.block);
    const float* vscale = c.value_scales + static_cast<size_t>(g) * (c.slots / c.block);
    u4 kr[X::KT][X::KL], vr[X::DB][X::VL];
    float sk[2], sv[2];
    auto load_keys = [&](int32_t ch) {
        const uint8_t* p = kbase + static_cast<size_t>(ch) * CHUNK * HD;
#pragma unroll
        for (int t = 0; t < X::KT; ++t) {
            // the key of the operand's row: R 16: set t / 2, its quads 0 1 4 5 or 2 3 6 7
            const int32_t x = col >> 2;
            const int32_t key = X::SMALL ? 32 * (t / 2) + 4 * (4 * (x >> 1) + 2 * (t % 2) + (x & 1)) + (col & 3) : 32 * t + col;
#pragma unroll
            for (int i = 0; i < X::KL; ++i) {
                const uint8_t* q = p + key * HD + (X::SMALL ? (HD == 32 ? 8 * grp : 64 * i + 16 * grp) : 32 * i + 16 * grp);
                if constexpr (HD == 32 && X::SMALL) {
                    const u2 two = *reinterpret_cast<const u2*>(q);
                    kr[t][i] = u4{two[0], two[1], 0u, 0u};
                } else {
                    kr[t][i] = *reinterpret_cast<const u4*>(q);
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int32_t b = (ch * CHUNK + 32 * h) / c.block;
            sk[h] = kscale[b];
            sv[h] = vscale[b];
        }
    };
    auto load_values = [&](int32_t ch) {
        const uint8_t* p = vbase + static_cast<size_t>(ch) * CHUNK * HD;
#pragma unroll
        for (int db = 0; db < X::DB; ++db)
#pragma unroll
            for (int s = 0; s < X::VL; ++s) {
                const int32_t d = (X::SMALL ? 16 : 32) * db + col, piece = X::SMALL ? grp : 2 * s + grp;
                vr[db][s] = *reinterpret_cast<const u4*>(p + d * CHUNK + 16 * piece);
            }
    };
    // a step: the scales of the new token's block, where this workgroup's keys end with it
    const bool holder = STEP && split == splits - 1 && P0 >= 0 && P0 < c.max_seq;
    float block_scales[2] = {0.0f, 0.0f};
    if constexpr (STEP) {
        if (holder && P0 % c.block != 0) {
            block_scales[0] = kscale[P0 / c.block];
            block_scales[1] = vscale[P0 / c.block];
        }
    }
    // the new token's codes and its block's scales in the chunk that holds it, whatever the loads saw
    auto patch = [&]() {
        if constexpr (STEP) {
            const int32_t at = P0 % CHUNK;
#pragma unroll
            for (int t = 0; t < X::KT; ++t) {
                const int32_t x = col >> 2, key = 32 * (t / 2) + 4 * (4 * (x >> 1) + 2 * (t % 2) + (x & 1)) + (col & 3);
                if (key == at) {
#pragma unroll
                    for (int i = 0; i < X::KL; ++i) {
                        if constexpr (HD == 32) {
                            const u2 two = *reinterpret_cast<const u2*>(sh.key + 8 * grp);
                            kr[t][i] = u4{two[0], two[1], 0u, 0u};
                        } else {
                            kr[t][i] = *reinterpret_cast<const u4*>(sh.key + 64 * i + 16 * grp);
                        }
                    }
                }
            }
            const int32_t h = at >> 5, u = at >> 3 & 1, piece = 2 * (at >> 4 & 1) + (at >> 2 & 1), byte = 8 * (at & 3);
#pragma unroll
            for (int db = 0; db < X::DB; ++db) {
                const uint32_t code = static_cast<uint32_t>(sh.value[16 * db + col]) << byte;
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    if (grp == piece && w == 2 * h + u) vr[db][0][w] = (vr[db][0][w] & ~(0xFFu << byte)) | code;
            }
#pragma unroll
            for (int w = 0; w < 2; ++w)
                if ((P0 / CHUNK * CHUNK + 32 * w) / c.block == P0 / c.block) {
                    sk[w] = block_scales[0];
                    sv[w] = block_scales[1];
                }
        }
    };
    if (c0 + wave < c1) {
        load_keys(c0 + wave);
        load_values(c0 + wave);
    }
    if constexpr (STEP) {
        if (on) {  // cosines by the key's threads, sines by the value's
            if (tid < 128) sh.cosines[tid] = rope_cos(P0, ifr);
            else sh.sines[tid - 128] = rope_sin(P0, ifr);
        }
        __syncthreads();
    }

    // the rows' parts through LDS
    _Float16* qs = reinterpret_cast<_Float16*>(attn_lds);  // [2][R][HD + 8]
    constexpr int QR = HD + 8;
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        if (4 * (wave + i * NW) >= held) break;
        const int32_t r = 4 * (wave + i * NW) + lr;
        uint32_t top = 0;
#pragma unroll
        for (int u = 0; u < DL; ++u) {
            if constexpr (STEP) {
                const int32_t d = (4 * lc + 64 * u) % HD;
                const bool upper = d >= HALF;
                const f4 cf = *reinterpret_cast<const f4*>(&sh.cosines[d % HALF]), sf = *reinterpret_cast<const f4*>(&sh.sines[d % HALF]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float y1, y2;
                    rope_apply(upper ? qo[i][u][e] : qv[i][u][e], upper ? qv[i][u][e] : qo[i][u][e], cf[e], sf[e], y1, y2);
                    qv[i][u][e] = upper ? y2 : y1;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, magnitude(qv[i][u][e]));
        }
        // the row's largest magnitude (bits below an infinity's, whose order is the floats')
        float most = __builtin_bit_cast(float, min(top, 0x7F7FFFFFu));
        most = fmaxf(most, dpp_move<0xB1>(most));
        most = fmaxf(most, dpp_move<0x4E>(most));
        most = fmaxf(most, dpp_move<0x141>(most));
        most = fmaxf(most, dpp_move<0x140>(most));
        const int32_t up = 13 - max(static_cast<int32_t>(__builtin_bit_cast(uint32_t, most) >> 23) - 127, -100);
        const float by = ldexpf(1.0f, up);
        if (r < held) {
#pragma unroll
            for (int u = 0; u < DL; ++u) {
                half4 hi, lo;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = qv[i][u][e] * by;
                    hi[e] = static_cast<_Float16>(x);
                    lo[e] = static_cast<_Float16>(x - static_cast<float>(hi[e]));
                }
                if (4 * lc + 64 * u < HD) {
                    *reinterpret_cast<half4*>(qs + r * QR + 4 * lc + 64 * u) = hi;
                    *reinterpret_cast<half4*>(qs + (R + r) * QR + 4 * lc + 64 * u) = lo;
                }
            }
            if (lc == 0) fr_s[r] = ldexpf(a.scale * 1.4426950408889634f, -up);
        }
    }
    if constexpr (STEP) {
        if (holder) {
            if (on && tid < 128) {
                const float k1 = x1, k2 = x2;
                rope_apply(k1, k2, sh.cosines[tid], sh.sines[tid], x1, x2);
            }
            uint32_t m = on ? max(magnitude(x1), magnitude(x2)) : 0;
            if (tid < 256) {
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), o)));
                if (lane == 0) sh.top[wave] = m;
            }
        }
    }
    __syncthreads();
    // A row's operands: in registers for 16 rows of up to 128 dims, else read from LDS for each set of keys (64 registers
    // of heads of 128: without them two waves share a SIMD, one's products beside the other's softmax).
    half8 qh[X::QREG ? X::QS : 1], ql[X::QREG ? X::QS : 1];
    const _Float16* qrow[X::CT];
    float fr[X::CT];
    int32_t last[X::CT];
#pragma unroll
    for (int ct = 0; ct < X::CT; ++ct) {
        const int32_t r = min(32 * ct + col, held - 1);  // (columns past the rows repeat the last)
        fr[ct] = fr_s[r];
        last[ct] = last_key(STEP ? 0 : (tile * R + r) / G);
        qrow[ct] = qs + r * QR + (HD == 32 && X::SMALL ? 8 : 16) * grp;
    }
    auto query = [&](int ct, int s, int part) {  // step s of column tile ct's operand
        const int32_t d = HD == 32 && X::SMALL ? 0 : (X::SMALL ? 64 : 32) * (s / 2) + 8 * (s % 2);
        return *reinterpret_cast<const half8*>(qrow[ct] + part * R * QR + d);
    };
    if constexpr (X::QREG) {
#pragma unroll
        for (int s = 0; s < X::QS; ++s) {
            qh[s] = query(0, s, 0);
            ql[s] = query(0, s, 1);
        }
    }
    if constexpr (STEP) {
        if (holder) {
            const bool again = append_token<FMT, HD, 64 * NW>(c, sh, g, P0, on, x1, x2, block_scales);
            __syncthreads();
            // the new token in the chunk that its wave loaded ahead of the append; earlier rows that changed
            // are loaded again
            const int32_t mine = chunks - 1 - c0;  // (this workgroup's last chunk)
            if (c0 + wave < c1) {
                if (again) {
                    __threadfence();
                    load_keys(c0 + wave);
                    load_values(c0 + wave);
                }
                if (wave == mine % NW && mine < NW) patch();
            }
        }
    }

    // the key of a lane's score i in its set
    auto key_of = [&](int i) { return X::SMALL ? 16 * (grp >> 1) + 4 * (grp & 1) + 8 * (i >> 2) + (i & 3) : 8 * (i >> 2) + 4 * grp + (i & 3); };

    typedef typename std::conditional<X::SMALL, f4, f16v>::type acc_t;
    acc_t o[X::CT][X::DB];
    // a row's maximum, sum of weights, largest contribution (its exponent, relative to the maximum) and that exponent as a
    // whole number, whose power of two o is held in
    float m[X::CT], l[X::CT], reach[X::CT], ex[X::CT];
#pragma unroll
    for (int ct = 0; ct < X::CT; ++ct) {
        m[ct] = -INFINITY;
        l[ct] = 0.0f;
        reach[ct] = ex[ct] = NO_EXPONENT;
#pragma unroll
        for (int db = 0; db < X::DB; ++db)
#pragma unroll
            for (int e = 0; e < X::OE; ++e) o[ct][db][e] = 0.0f;
    }
    // (two forms of the loop's body: only chunks that not every row sees whole compare keys with rows)
    auto attend_chunk = [&](auto masked_form, const int32_t ch) {
        constexpr bool masked = decltype(masked_form)::value;
        const int32_t next = min(ch + NW, c1 - 1);  // (past the end the last chunk again, unused)
        const float ks[2] = {sk[0], sk[1]}, vs[2] = {sv[0], sv[1]};
        if (masked && FMT == KT_KV8_E4M3 && ch * CHUNK + CHUNK > n_keys) {  // tokens not held: bytes that may be NaNs
#pragma unroll
            for (int db = 0; db < X::DB; ++db)
#pragma unroll
                for (int s = 0; s < X::VL; ++s)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int32_t piece = X::SMALL ? grp : 2 * s + grp;
                        const int32_t held = n_keys - (ch * CHUNK + 32 * (w >> 1) + 16 * (piece >> 1) + 8 * (w & 1) + 4 * (piece & 1));
                        vr[db][s][w] &= held >= 4 ? 0xFFFFFFFFu : held <= 0 ? 0u : (1u << (8 * held)) - 1u;
                    }
        }
#pragma unroll
        for (int h0 = 0; h0 < 2; h0 += X::J) {  // J sets of 32 keys at a time
        if (masked && X::J == 1 && ch * CHUNK + 32 * h0 >= n_keys) break;
        acc_t sc[X::J][X::CT][X::SMALL ? 2 : 1];
#pragma unroll
        for (int j = 0; j < X::J; ++j)
#pragma unroll
            for (int t = 0; t < (X::SMALL ? 2 : 1); ++t) {
#pragma unroll
                for (int ct = 0; ct < X::CT; ++ct)
#pragma unroll
                    for (int e = 0; e < X::OE; ++e) sc[j][ct][t][e] = 0.0f;
#pragma unroll
                for (int s = 0; s < X::QS; ++s) {
                    const half8 k = to_half8<FMT>(half_of(kr[X::SMALL ? 2 * (h0 + j) + t : h0 + j][s / 2], s % 2));
#pragma unroll
                    for (int ct = 0; ct < X::CT; ++ct) {
                        if constexpr (X::SMALL) {
                            sc[j][ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, X::QREG ? ql[X::QREG ? s : 0] : query(ct, s, 1), sc[j][ct][t], 0, 0, 0);
                            sc[j][ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, X::QREG ? qh[X::QREG ? s : 0] : query(ct, s, 0), sc[j][ct][t], 0, 0, 0);
                        } else {
                            sc[j][ct][t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, query(ct, s, 1), sc[j][ct][t], 0, 0, 0);
                            sc[j][ct][t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, query(ct, s, 0), sc[j][ct][t], 0, 0, 0);
                        }
                    }
                }
            }
        if (h0 + X::J == 2) load_keys(next);
        // the sets' value scales 2^e mu (past the last key the first's again)
        float ks_h[X::J], e_h[X::J], shift_h[X::J], unscale_h[X::J];
#pragma unroll
        for (int h = 0; h < X::J; ++h) {
            const bool there = !masked || h == 0 || ch * CHUNK + 32 < n_keys;
            ks_h[h] = fabsf(there ? ks[h0 + h] : ks[0]);
            const uint32_t vs_h = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(magnitude(there ? vs[h0 + h] : vs[0]))));
            const int32_t e = static_cast<int32_t>(vs_h >> 23) - 127;  // (of a NaN any)
            const float mu = ldexpf(__builtin_bit_cast(float, vs_h), -e);
            e_h[h] = static_cast<float>(e);
            shift_h[h] = -__builtin_amdgcn_logf(mu) - WEIGHT_UP;
            unscale_h[h] = __builtin_amdgcn_rcpf(mu);  // (off by one unit at most, as a weight's rounding)
        }
        half8 ph[X::J][X::CT][X::VL], pl[X::J][X::CT][X::VL];
#pragma unroll
        for (int ct = 0; ct < X::CT; ++ct) {
            // a set's scores, the largest, and how far above the row's exponent (where it is) its value scale's is
            float x[X::J][X::E], f[X::J], most[X::J], above = -INFINITY;
#pragma unroll
            for (int h = 0; h < X::J; ++h) {
                f[h] = ks_h[h] * fr[ct];
                most[h] = -INFINITY;
#pragma unroll
                for (int i = 0; i < X::E; ++i) {
                    x[h][i] = X::SMALL ? sc[h][ct][X::SMALL ? i >> 2 : 0][X::SMALL ? i & 3 : i] : sc[h][ct][0][i];
                    if (masked && ch * CHUNK + 32 * (h0 + h) + key_of(i) > last[ct]) x[h][i] = -INFINITY;
                    most[h] = fmaxf(most[h], x[h][i]);
                }
                most[h] = rounded_score(most[h], f[h]);
                above = fmaxf(above, (most[h] - m[ct]) + fmaxf(e_h[h] - ex[ct], 0.0f));
            }
            if (__ballot(above > LAZY)) {
                const float m_new = fmaxf(m[ct], column_max<R>(fmaxf(most[0], most[X::J - 1])));
                float r = NO_EXPONENT;
#pragma unroll
                for (int h = 0; h < X::J; ++h) r = fmaxf(r, (most[h] - m_new) + e_h[h]);
                const bool first = m[ct] == -INFINITY;
                const float fall = first ? 0.0f : m[ct] - m_new, alpha = first ? 0.0f : __builtin_amdgcn_exp2f(fall);
                reach[ct] = fmaxf(reach[ct] + fall, column_max<R>(r));
                const float ex_new = rintf(fmaxf(reach[ct], NO_EXPONENT));
                const float beta = first ? 0.0f : __builtin_amdgcn_exp2f(fall + (ex[ct] - ex_new));
                l[ct] *= alpha;
#pragma unroll
                for (int db = 0; db < X::DB; ++db) o[ct][db] *= beta;
                m[ct] = m_new;
                ex[ct] = ex_new;
            }
            const float at = m[ct] == -INFINITY ? 0.0f : m[ct];
            const bool huge = __ballot(fabsf(at) > HUGE_SCORE);  // (one-hot rows)
#pragma unroll
            for (int h = 0; h < X::J; ++h) {
                float quiet = ex[ct] - e_h[h];
                const float in_exp = quiet <= MOST_QUIET ? quiet : 0.0f, shift = in_exp + shift_h[h];
                quiet -= in_exp;
                if (huge) {
#pragma unroll
                    for (int i = 0; i < X::E; ++i) x[h][i] = weight_of_huge(x[h][i], f[h], at, shift);
                } else {
                    const float both = at + shift;
#pragma unroll
                    for (int i = 0; i < X::E; ++i) x[h][i] = __builtin_amdgcn_exp2f(fmaf(x[h][i], f[h], -both));
                }
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < X::E; ++i) {
                    if (masked && ch * CHUNK + 32 * (h0 + h) + key_of(i) > last[ct]) x[h][i] = 0.0f;
                    sum += x[h][i];
                }
                // (0 * NaN: a row that sees none of the block)
                l[ct] += sum == 0.0f ? 0.0f : sum * ldexpf(unscale_h[h], static_cast<int32_t>(in_exp));
                if (quiet != 0.0f) {
                    const float down = ldexpf(1.0f, static_cast<int32_t>(fmaxf(-quiet, -200.0f)));
#pragma unroll
                    for (int i = 0; i < X::E; ++i) x[h][i] *= down;
                }
#pragma unroll
                for (int s = 0; s < X::VL; ++s) {
                    float w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) w[i] = x[h][8 * s + i];
                    split2(w, ph[h][ct][s], pl[h][ct][s]);
                }
            }
        }
#pragma unroll
        for (int db = 0; db < X::DB; ++db)
#pragma unroll
            for (int s = 0; s < X::VL; ++s)
#pragma unroll
                for (int h = 0; h < X::J; ++h) {
                    const half8 v = to_half8<FMT>(half_of(vr[db][s], h0 + h));
#pragma unroll
                    for (int ct = 0; ct < X::CT; ++ct) {
                        if constexpr (X::SMALL) {
                            o[ct][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl[h][ct][s], o[ct][db], 0, 0, 0);
                            o[ct][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[h][ct][s], o[ct][db], 0, 0, 0);
                        } else {
                            o[ct][db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[h][ct][s], o[ct][db], 0, 0, 0);
                            o[ct][db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[h][ct][s], o[ct][db], 0, 0, 0);
                        }
                    }
                }
        }
        load_values(next);
        if constexpr (STEP) {
            if (holder && next == chunks - 1) patch();
        }
    };
    int32_t ch = c0 + wave;
    for (; ch < c1 && ch * CHUNK + CHUNK <= n_all; ch += NW) attend_chunk(std::false_type{}, ch);
    for (; ch < c1; ch += NW) attend_chunk(std::true_type{}, ch);

    // each wave's averages, maxima and sums, then all waves' through LDS
    const int32_t used = min(NW, c1 - c0);  // waves with keys
    __syncthreads();                        // (the queries' parts are read)
    if (wave < used) {
#pragma unroll
        for (int ct = 0; ct < X::CT; ++ct) {
            l[ct] = column_sum<R>(l[ct]);
            const float inv = l[ct] == 0.0f ? 0.0f : 1.0f / l[ct];
            if (32 * ct + col >= held) continue;
            float* row = avg + (wave * R + 32 * ct + col) * LR;
#pragma unroll
            for (int db = 0; db < X::DB; ++db)
#pragma unroll
                for (int e = 0; e < X::OE; e += 4) {
                    f4 v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = ldexpf(o[ct][db][e + i] * inv, static_cast<int32_t>(ex[ct]));
                    *reinterpret_cast<f4*>(row + (X::SMALL ? 16 * db + 4 * grp : 32 * db + 2 * e + 4 * grp)) = v;
                }
            if (grp == 0) {
                ms[wave * R + 32 * ct + col] = m[ct];
                ls[wave * R + 32 * ct + col] = l[ct];
            }
        }
    }
    __syncthreads();
    const size_t part = ((static_cast<size_t>(g) * gridDim.y + tile) * a.max_splits + split) * R;
    const __amdgpu_buffer_rsrc_t averages = __builtin_amdgcn_make_buffer_rsrc(a.averages + part * HD, 0, R * HD * 4, 0x00020000);
    for (int32_t e = tid; e < held * (HD / 4); e += 64 * NW) {  // (every thread weighs its row's parts itself: no further barrier)
        const int32_t r = e / (HD / 4), d = 4 * (e % (HD / 4)), row = tile * R + r;
        float mx = -INFINITY, sum = 0.0f;
        f4 x = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int32_t w = 0; w < used; ++w) mx = fmaxf(mx, ms[w * R + r]);
        for (int32_t w = 0; w < used; ++w) {
            const float by = share_of(ms[w * R + r], ls[w * R + r], mx);
            const f4 v = *reinterpret_cast<const f4*>(avg + (w * R + r) * LR + d);
            sum += by;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = fmaf(by, v[i], x[i]);
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] *= inv;
        if (splits == 1) {
            const int32_t t = STEP ? 0 : row / G;
            *reinterpret_cast<f4*>(a.context + (static_cast<size_t>(t) * a.num_heads + g * G + (row - t * G)) * HD + d) = x;
        } else {  // written through to memory: the reader may be on another die
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, x), averages, (r * HD + d) * 4, 0, THROUGH);
            if (d == 0) {
                const u2 both = {__builtin_bit_cast(uint32_t, mx), __builtin_bit_cast(uint32_t, sum)};
                __hip_atomic_store(reinterpret_cast<uint64_t*>(a.stats) + part + r, __builtin_bit_cast(uint64_t, both), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            }
        }
    }
    if (splits == 1) return;
    // the last workgroup of the tile to arrive merges the splits, in their order
    __shared__ uint32_t arrived;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
        uint32_t* counter = a.counters + g * gridDim.y + tile;
        arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        if (arrived == static_cast<uint32_t>(splits) - 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    }
    __syncthreads();
    if (arrived != static_cast<uint32_t>(splits) - 1) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    const size_t first = part - static_cast<size_t>(split) * R;
    float* weight = attn_lds;                  // [R][MAX_SPLITS]
    float* total = weight + R * MAX_SPLITS;    // [R]
    f4* shares = reinterpret_cast<f4*>(total + R);  // [64 NW]
    // thread (four dims of a row, phase): every phases-th split, eight loads in flight together, the first eight with the
    // maxima and sums
    constexpr int BATCH = 8;
    const __amdgpu_buffer_rsrc_t all = __builtin_amdgcn_make_buffer_rsrc(a.averages + first * HD, 0, splits * R * HD * 4, 0x00020000);
    const int32_t items = held * (HD / 4), phases = max(1, 64 * NW / items);
    const int32_t phase = phases > 1 ? tid / items : 0;
    u4 v[BATCH];
    auto load_batch = [&](int32_t item, int32_t s0) {
        const int32_t at = (min(item, items - 1) / (HD / 4)) * HD + 4 * (min(item, items - 1) % (HD / 4));
#pragma unroll
        for (int u = 0; u < BATCH; ++u) v[u] = __builtin_amdgcn_raw_buffer_load_b128(all, (min(s0 + u * phases, splits - 1) * R * HD + at) * 4, 0, THROUGH);
    };
    load_batch(phases > 1 ? tid % items : tid, phase);
    for (int32_t r = wave; r < held; r += NW) {  // a row's weights: lane = split
        float ml[MAX_SPLITS / 64], ll[MAX_SPLITS / 64], mx = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < MAX_SPLITS / 64; ++i) {
            const int32_t s = lane + 64 * i;
            const uint64_t both = __hip_atomic_load(reinterpret_cast<uint64_t*>(a.stats) + first + static_cast<size_t>(min(s, splits - 1)) * R + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            ml[i] = s < splits ? __builtin_bit_cast(float, static_cast<uint32_t>(both)) : -INFINITY;
            ll[i] = s < splits ? __builtin_bit_cast(float, static_cast<uint32_t>(both >> 32)) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < MAX_SPLITS / 64; ++i) mx = fmaxf(mx, wave_max_dpp(ml[i]));
#pragma unroll
        for (int i = 0; i < MAX_SPLITS / 64; ++i) {
            const float by = share_of(ml[i], ll[i], mx);
            weight[r * MAX_SPLITS + lane + 64 * i] = by;
            sum += wave_sum_dpp(by);
        }
        if (lane == 0) total[r] = sum;
    }
    __syncthreads();
    for (int32_t i0 = 0; i0 < items; i0 += 64 * NW) {
        const int32_t item = phases > 1 ? tid % items : i0 + tid;
        const bool on = item < items && phase < phases;
        const int32_t r = min(item, items - 1) / (HD / 4), d = 4 * (min(item, items - 1) % (HD / 4));
        f4 x = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int32_t s0 = phase; on && s0 < splits; s0 += BATCH * phases) {
            if (i0 > 0 || s0 > phase) load_batch(item, s0);
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const int32_t s = s0 + u * phases;
                const float by = s < splits ? weight[r * MAX_SPLITS + s] : 0.0f;
                const f4 y = __builtin_bit_cast(f4, v[u]);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = s < splits ? fmaf(by, y[i], x[i]) : x[i];
            }
        }
        if (phases > 1) {
            shares[tid] = x;
            __syncthreads();
        }
        if (on && phase == 0) {
            for (int32_t p = 1; p < phases; ++p)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] += shares[item + p * items][i];
            const float inv = total[r] == 0.0f ? 0.0f : 1.0f / total[r];
            const int32_t row = tile * R + r, t = STEP ? 0 : row / G;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] *= inv;
            *reinterpret_cast<f4*>(a.context + (static_cast<size_t>(t) * a.num_heads + g * G + (row - t * G)) * HD + d) = x;
        }
    }
}

// ---- rows as fp32, and the copy of a prefix ------------------------------------------------
// Workgroup (chunk, kv head, 64 dims of the keys or of the values): the chunk's rows in [first, first + count) as code *
// scale, sixteen codes a thread; the values turn through LDS. One memory round trip and the stores: a block of 64 tokens
// of 8 heads of 64 3.2 us traced, 1501 tokens of heads of 128 6.6 (12.3 MB written and 3.1 read: 2.3 TB/s).
template <int FMT>
__global__ void __launch_bounds__(THREADS) read_kernel(KV8View c, int32_t first, int32_t count, float* keys, float* values) {
    __shared__ float turned[CHUNK][65];
    const int32_t HD = c.head_dim, g = blockIdx.y, tid = threadIdx.x, d0 = blockIdx.z / 2 * 64, nd = min(64, HD - d0);
    const int32_t tok0 = (first / CHUNK + static_cast<int32_t>(blockIdx.x)) * CHUNK;
    const bool is_key = blockIdx.z % 2 == 0;
    float* out = is_key ? keys : values;
    if (!out) return;
    out += static_cast<size_t>(g) * count * HD + d0;
    const float* scales = (is_key ? c.key_scales : c.value_scales) + static_cast<size_t>(g) * (c.slots / c.block);
    const uint8_t* src = (is_key ? c.keys : c.values) + (static_cast<size_t>(g) * c.slots + tok0) * HD;
    auto inside = [&](int32_t tok) { return tok >= first && tok < first + count; };
    if (is_key) {
        const int32_t per = nd / 16, r = tid / per, d = 16 * (tid % per), tok = tok0 + r;
        if (r >= CHUNK || !inside(tok)) return;
        const u4 w = *reinterpret_cast<const u4*>(src + r * HD + d0 + d);
        const float s = fabsf(scales[tok / c.block]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x[4];
            decode4<FMT>(w[i], x);
            *reinterpret_cast<float4*>(out + static_cast<size_t>(tok - first) * HD + d + 4 * i) = make_float4(x[0] * s, x[1] * s, x[2] * s, x[3] * s);
        }
        return;
    }
    constexpr int OUT = 4;  // groups of four dims a thread writes: 64 x 16 of them
    const int32_t groups = nd / 4;
    float s[OUT];
#pragma unroll
    for (int u = 0; u < OUT; ++u) {
        const int32_t tok = tok0 + min((tid + u * THREADS) / groups, CHUNK - 1);
        s[u] = inside(tok) ? fabsf(scales[tok / c.block]) : 0.0f;
    }
    if (tid < 4 * nd) {  // (dim, piece)
        const int32_t d = tid / 4, piece = tid % 4;
        const u4 w = *reinterpret_cast<const u4*>(src + (d0 + d) * CHUNK + 16 * piece);
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // four tokens from 32 (i / 2) + 16 (piece / 2) + 8 (i % 2) + 4 (piece % 2)
            float x[4];
            decode4<FMT>(w[i], x);
            const int32_t t = 32 * (i >> 1) + 16 * (piece >> 1) + 8 * (i & 1) + 4 * (piece & 1);
#pragma unroll
            for (int e = 0; e < 4; ++e) turned[t + e][d] = x[e];
        }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < OUT; ++u) {
        const int32_t e = tid + u * THREADS, r = e / groups, d = 4 * (e % groups), tok = tok0 + r;
        if (r >= CHUNK || !inside(tok)) continue;
        f4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = turned[r][d + i] * s[u];
        __builtin_memcpy(out + static_cast<size_t>(tok - first) * HD + d, &x, sizeof(x));
    }
}

// Workgroup (chunk, kv head): the chunk's codes and scales; the workgroups of chunk 0 also the open block's
// rows, from the source's rows where it is the source's open block too, else from its codes. Where the source's
// open block loses rows, its scale says so. (The cache may be the source: a thread writes a scale that
// it alone has read, and codes and rows as they are.) Traced, 16 layers of 8 heads of 64: 1000 tokens 12.8 us (in place 14.9), 30000 181 (187):
// 491 MB read and written, 5.4 TB/s.
template <int FMT>
__global__ void __launch_bounds__(THREADS) copy_kernel(KV8View to, KV8View from, int32_t length, int32_t source_length) {
    const int32_t HD = to.head_dim, B = to.block, g = blockIdx.y, tid = threadIdx.x;
    const int32_t layer = blockIdx.z;
    const size_t head_to = static_cast<size_t>(layer) * to.kv_heads + g;
    const size_t at_to = head_to * to.slots * HD, at_from = head_to * from.slots * HD;
    const size_t chunk = static_cast<size_t>(blockIdx.x) * CHUNK * HD;
    for (int32_t e = tid; e < CHUNK * HD / 16; e += THREADS) {
        reinterpret_cast<uint4*>(to.keys + at_to + chunk)[e] = reinterpret_cast<const uint4*>(from.keys + at_from + chunk)[e];
        reinterpret_cast<uint4*>(to.values + at_to + chunk)[e] = reinterpret_cast<const uint4*>(from.values + at_from + chunk)[e];
    }
    const float* ks = from.key_scales + head_to * (from.slots / B);
    const float* vs = from.value_scales + head_to * (from.slots / B);
    const int32_t per = max(1, CHUNK / B), blocks = (length + B - 1) / B;
    const int32_t b = B > CHUNK ? (blockIdx.x % 2 == 0 ? blockIdx.x / 2 : blocks) : blockIdx.x * per + tid;
    const int32_t open = length / B;
    const bool same = open == source_length / B;
    if (tid < per && b < blocks) {
        const bool drops = same && b == open && length < source_length;
        to.key_scales[head_to * (to.slots / B) + b] = drops ? -fabsf(ks[b]) : ks[b];
        to.value_scales[head_to * (to.slots / B) + b] = drops ? -fabsf(vs[b]) : vs[b];
    }
    if (blockIdx.x != 0 || length % B == 0) return;
    const size_t rows = head_to * B * HD;
    for (int32_t e = tid; e < length % B * HD; e += THREADS) {
        if (same) {
            to.key_rows[rows + e] = from.key_rows[rows + e];
            to.value_rows[rows + e] = from.value_rows[rows + e];
            continue;
        }
        const int32_t tok = open * B + e / HD, d = e % HD;
        float x[4];
        decode4<FMT>(from.keys[at_from + static_cast<size_t>(tok) * HD + d], x);
        to.key_rows[rows + e] = x[0] * ks[open];
        decode4<FMT>(from.values[at_from + (static_cast<size_t>(tok / CHUNK) * HD + d) * CHUNK + value_byte(tok % CHUNK / 4) + tok % 4], x);
        to.value_rows[rows + e] = x[0] * vs[open];
    }
}

int32_t check_heads(int32_t num_heads, int32_t kv_heads) {
    if (num_heads <= 0 || num_heads % kv_heads != 0)
        return fail(KT_ERR_ARGUMENT, "numHeads %d must be a multiple of numKeyValueHeads %d", num_heads, kv_heads);
    return KT_OK;
}

int32_t append_args(const float* q, const float* k, const float* v, int32_t tokens, int32_t num_heads, const float* inv_freq, const int32_t* position,
                    const kt_kv8_cache* cache, int32_t layer, float* q_out, AppendArgs* a) {
    if (const int32_t status = view_kv8(cache, layer, &a->c)) return status;
    if (!k || !v || !inv_freq || !position || !q != !q_out) return fail(KT_ERR_ARGUMENT, "a pointer argument is NULL");
    if (const int32_t status = check_heads(num_heads, a->c.kv_heads)) return status;
    if (tokens < 0 || tokens > a->c.max_seq) return fail(KT_ERR_ARGUMENT, "%d tokens do not fit maxSequenceLength %d", tokens, a->c.max_seq);
    a->q = q;
    a->k = k;
    a->v = v;
    a->q_out = q_out;
    a->inv_freq = inv_freq;
    a->position = position;
    a->tokens = tokens;
    a->num_heads = num_heads;
    a->blocks = (tokens + a->c.block - 2) / a->c.block + 1;
    return KT_OK;
}

int32_t launch_append(const AppendArgs& a, hipStream_t st) {
    const int32_t per = THREADS / (a.c.head_dim / 2);
    const int64_t grid = static_cast<int64_t>(a.blocks) * a.c.kv_heads * 2 +
                         (a.q ? static_cast<int64_t>((a.tokens + per - 1) / per) * ((a.num_heads + Q_HEADS - 1) / Q_HEADS) : 0);
    if (grid > INT32_MAX) return fail(KT_ERR_SHAPE, "too many tokens and heads in one call");
    const size_t lds = static_cast<size_t>(a.c.block) * (a.c.head_dim + 1) * sizeof(float);
    if (const int32_t ls = a.c.fmt == KT_KV8_INT8 ? allow_lds<&append_kernel<KT_KV8_INT8>, 144 << 10>(lds) : allow_lds<&append_kernel<KT_KV8_E4M3>, 144 << 10>(lds)) return ls;
    const auto kernel = a.c.fmt == KT_KV8_INT8 ? append_kernel<KT_KV8_INT8> : append_kernel<KT_KV8_E4M3>;
    kernel<<<static_cast<uint32_t>(grid), THREADS, lds, st>>>(a);
    KT_LAUNCHED("8-bit cache append kernel");
    return KT_OK;
}

int32_t attention_args(const float* q, int32_t tokens, const int32_t* position, int32_t key_bound, const kt_kv8_cache* cache, int32_t layer,
                       int32_t num_heads, float* context, AttnArgs* a) {
    if (const int32_t status = view_kv8(cache, layer, &a->c)) return status;
    if (!q || !position || !context) return fail(KT_ERR_ARGUMENT, "a pointer argument is NULL");
    if (const int32_t status = check_heads(num_heads, a->c.kv_heads)) return status;
    if (tokens < 0 || key_bound < tokens || key_bound > a->c.max_seq)
        return fail(KT_ERR_ARGUMENT, "key bound %d must cover the %d tokens and fit maxSequenceLength %d", key_bound, tokens, a->c.max_seq);
    if (static_cast<int64_t>(tokens) * (num_heads / a->c.kv_heads) > 65535 * 16)
        return fail(KT_ERR_SHAPE, "%d tokens of %d query heads a key/value head in one call: at most %d rows", tokens, num_heads / a->c.kv_heads, 65535 * 16);
    if (!aligned(q, 16) || !aligned(context, 16)) return fail(KT_ERR_ARGUMENT, "attention: q and the context must be 16-byte aligned");
    a->q = q;
    a->position = position;
    a->context = context;
    a->tokens = tokens;
    a->num_heads = num_heads;
    a->scale = 1.0f / sqrtf(static_cast<float>(a->c.head_dim));
    return KT_OK;
}

// Up to so many keys one workgroup of 8 waves takes them without splits. The rule reads key_bound, for a recorded step
// all that the host knows: in Transformer the cache's capacity, so a short text in a long cache takes the splits' form, and the
// same text in caches on both sides of the limit has sums in another order. Steps of 32 heads of 64 traced, bound 1024 (8192):
// 200 keys 7.8 us (8.0), 500 8.9 (10.6), 1000 11.2 (10.9); 14 heads, 2 kv heads, 543 8.6 (10.6). With the call, and a bound
// at the length: heads of 64 after 500 keys 8.8 us (with splits 10.6), 1000 10.2 (10.4), 1500 11.8 (10.5); of 128 500 11.9
// (12.6), 760 13.0 (12.5).
constexpr int direct_keys(int hd) { return hd <= 64 ? 16 * CHUNK : 10 * CHUNK; }

template <int FMT, int HD, int R, int WAVES, bool STEP = false>
int32_t launch_rows(AttnArgs a, int32_t key_bound, hipStream_t st, AppendArgs* append) {
    constexpr bool DIRECT = WAVES > 4;  // no splits
    const int32_t tiles = ceil_div(a.tokens * (a.num_heads / a.c.kv_heads), R);
    const int64_t wgs = static_cast<int64_t>(a.c.kv_heads) * tiles;
    // Key splits: as many as two workgroups for each CU hold, which is what fits at once (24 tokens of 32 heads after
    // 4000, rounded up to 528 workgroups: 16.9 us for 12.6).
    const int32_t fill = static_cast<int32_t>(std::min<int64_t>(MAX_SPLITS, std::max<int64_t>(1, 2 * cu_count() / wgs)));
    a.max_splits = splits_of(ceil_div(key_bound, CHUNK), WAVES, DIRECT ? 1 : wgs < static_cast<int64_t>(MAX_COUNTERS) ? fill : 1);
    CallScratch turned;  // the rotated query of a step whose append is a launch of its own
    if (append && !STEP) {
        const size_t bytes = static_cast<size_t>(a.num_heads) * HD * sizeof(float);
        if (const int32_t status = turned.take(CALL_SLICES, st, bytes)) return status;
        append->q_out = static_cast<float*>(turned.ptr);
    }
    // The workspace: the splits' averages and sums, behind room for that query, which a capture begun by other means takes
    // (no scratch to have there) and an eager call reserves: it sizes what a recording of its shapes needs.
    size_t q = 0;
    if (append && !STEP) {
        hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
        if (turned.ptr) KT_HIP(hipStreamIsCapturing(st, &capture));
        if (capture == hipStreamCaptureStatusNone) q = static_cast<size_t>(a.num_heads) * HD;
    }
    if (a.max_splits > 1 || q > 0) {
        const size_t rows = a.max_splits > 1 ? static_cast<size_t>(wgs) * a.max_splits * R : 0;
        void* ws = nullptr;
        if (const int32_t status = workspace_counters(st, (rows * (HD + 2) + q) * sizeof(float) + 16, a.max_splits > 1 ? static_cast<size_t>(wgs) : 0, &ws, &a.counters)) return status;
        ws = reinterpret_cast<void*>((reinterpret_cast<uintptr_t>(ws) + 15) & ~uintptr_t{15});  // (it begins at any dword)
        a.averages = static_cast<float*>(ws) + q;
        a.stats = a.averages + rows * HD;
        if (append && !STEP && !turned.ptr) append->q_out = static_cast<float*>(ws);
    }
    if (append && !STEP) {
        a.q = append->q_out;
        if (const int32_t status = launch_append(*append, st)) return status;
    }
    constexpr size_t lds = sizeof(float) * std::max(std::max(static_cast<size_t>(WAVES) * R * (HD + 6), static_cast<size_t>(R) * (HD + 8)), static_cast<size_t>(R) * (MAX_SPLITS + 1) + 4 * 64 * WAVES);
    if (const int32_t ls = allow_lds<&attention_kernel<FMT, HD, R, WAVES, STEP>, lds>(lds)) return ls;
    attention_kernel<FMT, HD, R, WAVES, STEP><<<dim3(static_cast<uint32_t>(a.c.kv_heads), static_cast<uint32_t>(tiles), static_cast<uint32_t>(a.max_splits)), 64 * WAVES, lds, st>>>(a);
    KT_LAUNCHED("8-bit cache attention kernel");
    return KT_OK;
}

template <int FMT, int HD>
int32_t launch_dims(const AttnArgs& a, int32_t key_bound, hipStream_t st, AppendArgs* append) {
    const int32_t rows = a.tokens * (a.num_heads / a.c.kv_heads);
    if constexpr (HD < 256) {  // (of 256 dims the step's form would not fit the registers)
        if (append && rows <= 16) {  // a step of up to 16 query heads a kv head: one launch
            if (key_bound <= direct_keys(HD)) return launch_rows<FMT, HD, 16, 8, true>(a, key_bound, st, append);
            return launch_rows<FMT, HD, 16, 4, true>(a, key_bound, st, append);
        }
        // Tiles of 16 rows while two workgroups for each CU hold them, of 32 beyond. 32 heads of 64, 8 kv heads, with the call,
        // 16 (32): 16 tokens after 1000 8.0 us (12.6), 256 after 1000 13.4 (18.6), after 4000 32.4 (32.6), 512 after 4000 61
        // (48), a prompt of 1024 28.5 (19.3); heads of 128, 64 tokens after 4000 23.0 (25.1), 300 76 (66).
        if (static_cast<int64_t>(a.c.kv_heads) * ceil_div(rows, 16) > 2 * cu_count()) return launch_rows<FMT, HD, 32, 4>(a, key_bound, st, append);
        if (key_bound <= direct_keys(HD)) return launch_rows<FMT, HD, 16, 8>(a, key_bound, st, append);
    }
    return launch_rows<FMT, HD, 16, 4>(a, key_bound, st, append);
}

template <int FMT>
int32_t launch_format(const AttnArgs& a, int32_t key_bound, hipStream_t st, AppendArgs* append) {
    switch (a.c.head_dim) {
        case 32: return launch_dims<FMT, 32>(a, key_bound, st, append);
        case 64: return launch_dims<FMT, 64>(a, key_bound, st, append);
        case 128: return launch_dims<FMT, 128>(a, key_bound, st, append);
        default: return launch_dims<FMT, 256>(a, key_bound, st, append);
    }
}

int32_t launch_attention(const AttnArgs& a, int32_t key_bound, hipStream_t st, AppendArgs* append = nullptr) {
    return a.c.fmt == KT_KV8_INT8 ? launch_format<KT_KV8_INT8>(a, key_bound, st, append) : launch_format<KT_KV8_E4M3>(a, key_bound, st, append);
}

}  // namespace
}  // namespace kt

using namespace kt;

extern "C" {

int32_t kt_kv8_layout(const kt_kv8_cache* cache, int64_t* out3) {
    if (const int32_t status = check_shape(cache)) return status;
    if (!out3) return fail(KT_ERR_ARGUMENT, "out3 is NULL");
    const int64_t heads = static_cast<int64_t>(cache->layers) * cache->kv_heads, slots = slots_of(cache->max_seq, cache->block_tokens);
    out3[0] = heads * slots * cache->head_dim;
    out3[1] = heads * (slots / cache->block_tokens);
    out3[2] = heads * cache->block_tokens * cache->head_dim;
    return KT_OK;
}

int32_t kt_rope_kv8(const float* q, const float* k, const float* v, int32_t tokens, int32_t num_heads, const float* inv_freq, const int32_t* position,
                    const kt_kv8_cache* cache, int32_t layer, float* q_out, void* stream) {
    AppendArgs a{};
    if (const int32_t status = append_args(q, k, v, tokens, num_heads, inv_freq, position, cache, layer, q_out, &a)) return status;
    return tokens == 0 ? KT_OK : launch_append(a, static_cast<hipStream_t>(stream));
}

int32_t kt_attention_kv8(const float* q, int32_t tokens, const int32_t* position, int32_t key_bound, const kt_kv8_cache* cache, int32_t layer,
                         int32_t num_heads, float* context, void* stream) {
    AttnArgs a{};
    if (const int32_t status = attention_args(q, tokens, position, key_bound, cache, layer, num_heads, context, &a)) return status;
    return tokens == 0 ? KT_OK : launch_attention(a, key_bound, static_cast<hipStream_t>(stream));
}

int32_t kt_rope_attention_kv8(float* q, const float* k, const float* v, const float* inv_freq, int32_t tokens, const int32_t* position, int32_t key_bound,
                              const kt_kv8_cache* cache, int32_t layer, int32_t num_heads, float* context, void* stream) {
    AppendArgs p{};
    AttnArgs a{};
    if (const int32_t status = append_args(q, k, v, tokens, num_heads, inv_freq, position, cache, layer, q, &p)) return status;
    if (const int32_t status = attention_args(q, tokens, position, key_bound, cache, layer, num_heads, context, &a)) return status;
    if (tokens == 0) return KT_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (tokens == 1) {  // q stays as it is
        a.k_new = k;
        a.v_new = v;
        a.inv_freq = inv_freq;
        return launch_attention(a, key_bound, st, &p);
    }
    if (const int32_t status = launch_append(p, st)) return status;
    return launch_attention(a, key_bound, st);
}

int32_t kt_kv8_read(const kt_kv8_cache* cache, int32_t layer, int32_t first, int32_t count, float* keys, float* values, void* stream) {
    KV8View c;
    if (const int32_t status = view_kv8(cache, layer, &c)) return status;
    if (first < 0 || count < 0 || count > c.max_seq - first) return fail(KT_ERR_RANGE, "tokens %d + %d out of bounds %d", first, count, c.max_seq);
    if (!aligned(keys, 16)) return fail(KT_ERR_ARGUMENT, "keys must be 16-byte aligned");
    if (count == 0 || (!keys && !values)) return KT_OK;
    const dim3 grid(static_cast<uint32_t>((first + count - 1) / CHUNK - first / CHUNK + 1), static_cast<uint32_t>(c.kv_heads), 2u * static_cast<uint32_t>(ceil_div(c.head_dim, 64)));
    const auto kernel = c.fmt == KT_KV8_INT8 ? read_kernel<KT_KV8_INT8> : read_kernel<KT_KV8_E4M3>;
    kernel<<<grid, THREADS, 0, static_cast<hipStream_t>(stream)>>>(c, first, count, keys, values);
    KT_LAUNCHED("8-bit cache read kernel");
    return KT_OK;
}

int32_t kt_kv8_copy(const kt_kv8_cache* source, int32_t source_length, const kt_kv8_cache* cache, int32_t length, void* stream) {
    KV8View from, to;
    if (const int32_t status = view_kv8(source, 0, &from)) return status;
    if (const int32_t status = view_kv8(cache, 0, &to)) return status;
    if (source->layers != cache->layers || from.kv_heads != to.kv_heads || from.head_dim != to.head_dim || from.fmt != to.fmt || from.block != to.block)
        return fail(KT_ERR_SHAPE, "the caches differ in layers, heads, dims, format or block");
    if (source_length < 0 || source_length > from.max_seq || length < 0 || length > source_length)
        return fail(KT_ERR_RANGE, "Cannot copy %d positions from a cache holding %d", length, source_length);
    if (length > to.max_seq) return fail(KT_ERR_RANGE, "Cannot copy %d positions into a cache of %d", length, to.max_seq);
    if (length == 0) return KT_OK;
    const dim3 grid(static_cast<uint32_t>(ceil_div(length, CHUNK)), static_cast<uint32_t>(to.kv_heads), static_cast<uint32_t>(cache->layers));
    const auto kernel = to.fmt == KT_KV8_INT8 ? copy_kernel<KT_KV8_INT8> : copy_kernel<KT_KV8_E4M3>;
    kernel<<<grid, THREADS, 0, static_cast<hipStream_t>(stream)>>>(to, from, length, source_length);
    KT_LAUNCHED("8-bit cache copy kernel");
    return KT_OK;
}

}  // extern "C"
