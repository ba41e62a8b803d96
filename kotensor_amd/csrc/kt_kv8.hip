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
// calls they came in.
#include <math.h>

#include <atomic>

#include "kt_common.h"
#include "kt_wave.h"

namespace kt {
namespace {

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
// encodes its block through LDS; further workgroups rotate q. Bound by the launch for one
// token, by reading the rows and (keys, q) the double-precision cosines for a prompt.
// The first block's earlier rows come from the fp32 rows of the open block, which the last
// block's rows replace: where the first block has earlier rows, one workgroup does both, in
// that order.
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

// The block b of a head, of whose rows 0 .. n - 1 those from lo on are new.
template <int FMT, bool KEYS>
__device__ void append_block(const AppendArgs& a, float* lds, uint32_t (&part)[THREADS / 64], int32_t g, int32_t b, int32_t p0, int32_t lo, int32_t n) {
    const KV8View& c = a.c;
    const int32_t HD = c.head_dim, B = c.block, LR = HD + 1, tid = threadIdx.x;
    float* rows = (KEYS ? c.key_rows : c.value_rows) + static_cast<size_t>(g) * B * HD;
    const int32_t t0 = b * B - p0;  // token of row 0 in this call
    const bool open = n < B;
    uint32_t m = 0;
    if constexpr (KEYS) {
        const int32_t half = HD >> 1;
        for (int32_t e = tid; e < (n - lo) * half; e += THREADS) {
            const int32_t r = lo + e / half, i = e % half;
            const float* src = a.k + (static_cast<size_t>(t0 + r) * c.kv_heads + g) * HD + i;
            float cf, sf, y1, y2;
            rope_cos_sin(b * B + r, a.inv_freq[i], cf, sf);
            rope_apply(src[0], src[half], cf, sf, y1, y2);
            lds[r * LR + i] = y1;
            lds[r * LR + i + half] = y2;
            m = max(m, max(magnitude(y1), magnitude(y2)));
            if (open) {
                rows[r * HD + i] = y1;
                rows[r * HD + i + half] = y2;
            }
        }
    } else {
        for (int32_t e = tid; e < (n - lo) * HD; e += THREADS) {
            const int32_t r = lo + e / HD, d = e % HD;
            const float y = a.v[(static_cast<size_t>(t0 + r) * c.kv_heads + g) * HD + d];
            lds[r * LR + d] = y;
            m = max(m, magnitude(y));
            if (open) rows[r * HD + d] = y;
        }
    }
    m = block_max(m, part);
    float* scale = (KEYS ? c.key_scales : c.value_scales) + static_cast<size_t>(g) * (c.slots / B) + b;
    float s = scale_of<FMT>(m);
    int32_t from = lo;
    if (lo > 0) {
        const float held = *scale;
        if (held != held || held >= s) {
            s = held;
        } else if (s == s) {  // raised: the earlier rows again
            from = 0;
            for (int32_t e = tid; e < lo * HD; e += THREADS) lds[e / HD * LR + e % HD] = rows[e];
        }
    }
    __syncthreads();  // the rows are in LDS, the held scale is read
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
    if (p0 < 0 || p0 >= c.max_seq) return;  // the host checks capacity; never write outside the cache
    const int32_t end = p0 + min(a.tokens, c.max_seq - p0);
    int32_t id = blockIdx.x;
    const int32_t roles = a.blocks * c.kv_heads * 2;
    if (id < roles) {
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
    // q: a thread's pair of a token, all heads
    const int32_t half = HD >> 1, per = THREADS / half;
    const int32_t i = threadIdx.x % half, t = (id - roles) * per + threadIdx.x / half;
    if (t >= end - p0) return;
    float cf, sf;
    rope_cos_sin(p0 + t, a.inv_freq[i], cf, sf);
    const size_t row = static_cast<size_t>(t) * a.num_heads * HD + i;
    for (int32_t h = 0; h < a.num_heads; ++h) {
        float y1, y2;
        rope_apply(a.q[row + h * HD], a.q[row + h * HD + half], cf, sf, y1, y2);
        a.q_out[row + h * HD] = y1;
        a.q_out[row + h * HD + half] = y2;
    }
}

// ---- the cached attention -----------------------------------------------------------------
struct AttnArgs {
    KV8View c;
    const float* q;
    const int32_t* position;
    float* context;
    int32_t tokens, num_heads;
    float scale;
};

// Workgroup (token, query head): a wave takes every fourth key, its lanes the dims. 32 keys' sums join
// the running ones as one (one by one, the many small weights of a long context would be lost).
template <int FMT>
__global__ void __launch_bounds__(THREADS) attention_kernel(AttnArgs a) {
    const KV8View& c = a.c;
    constexpr int MAXD = 4;
    __shared__ float part[THREADS / 64][MAXD * 64], pm[THREADS / 64], pl[THREADS / 64];
    const int32_t HD = c.head_dim, t = blockIdx.y, h = blockIdx.x, g = h / (a.num_heads / c.kv_heads);
    const int32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int32_t n = min(max(*a.position + t + 1, 0), c.max_seq);
    const float* q = a.q + (static_cast<size_t>(t) * a.num_heads + h) * HD;
    float qd[MAXD], acc[MAXD] = {};
    for (int i = 0; i < MAXD; ++i) qd[i] = lane + 64 * i < HD ? q[lane + 64 * i] : 0.0f;
    float m = -INFINITY, l = 0.0f, l_part = 0.0f, part_acc[MAXD] = {};
    int32_t held = 0;
    for (int32_t j = wave; j < n; j += THREADS / 64) {
        const uint8_t* key = c.keys + (static_cast<size_t>(g) * c.slots + j) * HD;
        const uint8_t* value = c.values + (static_cast<size_t>(g) * c.slots / CHUNK + j / CHUNK) * HD * CHUNK + value_byte(j % CHUNK / 4) + j % 4;
        const size_t block = static_cast<size_t>(g) * (c.slots / c.block) + j / c.block;
        float d = 0.0f, v[MAXD];
        for (int i = 0; i < MAXD; ++i) {
            const int32_t at = lane + 64 * i;
            float x[4] = {}, y[4] = {};
            if (at < HD) {
                decode4<FMT>(key[at], x);
                decode4<FMT>(value[at * CHUNK], y);
            }
            d = fmaf(qd[i], x[0], d);
            v[i] = y[0];
        }
        d = wave_sum_dpp(d) * c.key_scales[block] * a.scale;
        const float m_new = fmaxf(m, d), alpha = m == -INFINITY ? 0.0f : expf(m - m_new);
        const float p = expf(d - m_new), pv = p * c.value_scales[block];
        l *= alpha;
        l_part = l_part * alpha + p;
        for (int i = 0; i < MAXD; ++i) {
            acc[i] *= alpha;
            part_acc[i] = part_acc[i] * alpha + pv * v[i];
        }
        m = m_new;
        if (++held == 32 || j + THREADS / 64 >= n) {
            l += l_part;
            l_part = 0.0f;
            for (int i = 0; i < MAXD; ++i) {
                acc[i] += part_acc[i];
                part_acc[i] = 0.0f;
            }
            held = 0;
        }
    }
    for (int i = 0; i < MAXD; ++i) part[wave][lane + 64 * i] = acc[i];
    if (lane == 0) {
        pm[wave] = m;
        pl[wave] = l;
    }
    __syncthreads();
    const int32_t d = threadIdx.x;
    if (d >= HD) return;
    float mx = -INFINITY, x = 0.0f, sum = 0.0f;
    for (int w = 0; w < THREADS / 64; ++w) mx = fmaxf(mx, pm[w]);
    for (int w = 0; w < THREADS / 64; ++w) {
        const float e = pl[w] == 0.0f ? 0.0f : expf(pm[w] - mx);
        x += part[w][d] * e;
        sum += pl[w] * e;
    }
    a.context[(static_cast<size_t>(t) * a.num_heads + h) * HD + d] = n > 0 ? x / sum : 0.0f;
}

// ---- rows as fp32, and the copy of a prefix ------------------------------------------------
// Workgroup (chunk, kv head, keys or values): the chunk's rows in [first, first + count) as
// code * scale; the values turn through LDS.
template <int FMT>
__global__ void __launch_bounds__(THREADS) read_kernel(KV8View c, int32_t first, int32_t count, float* keys, float* values) {
    __shared__ float turned[CHUNK][65];
    const int32_t HD = c.head_dim, g = blockIdx.y, tid = threadIdx.x;
    const int32_t tok0 = (first / CHUNK + static_cast<int32_t>(blockIdx.x)) * CHUNK;
    const bool is_key = blockIdx.z == 0;
    float* out = is_key ? keys : values;
    if (!out) return;
    out += static_cast<size_t>(g) * count * HD;
    const float* scales = (is_key ? c.key_scales : c.value_scales) + static_cast<size_t>(g) * (c.slots / c.block);
    const uint8_t* src = (is_key ? c.keys : c.values) + (static_cast<size_t>(g) * c.slots + tok0) * HD;
    auto inside = [&](int32_t tok) { return tok >= first && tok < first + count; };
    if (is_key) {
        for (int32_t e = tid; e < CHUNK * HD / 4; e += THREADS) {
            const int32_t r = e / (HD / 4), d = 4 * (e % (HD / 4)), tok = tok0 + r;
            if (!inside(tok)) continue;
            float x[4];
            decode4<FMT>(reinterpret_cast<const uint32_t*>(src)[e], x);
            const float s = scales[tok / c.block];
            *reinterpret_cast<float4*>(out + static_cast<size_t>(tok - first) * HD + d) = make_float4(x[0] * s, x[1] * s, x[2] * s, x[3] * s);
        }
        return;
    }
    for (int32_t d0 = 0; d0 < HD; d0 += 64) {  // 64 dims at a time
        const int32_t nd = min(64, HD - d0);
        for (int32_t e = tid; e < nd * 16; e += THREADS) {
            const int32_t quad = e % 16, d = e / 16;
            float x[4];
            decode4<FMT>(*reinterpret_cast<const uint32_t*>(src + (d0 + d) * CHUNK + value_byte(quad)), x);
#pragma unroll
            for (int i = 0; i < 4; ++i) turned[4 * quad + i][d] = x[i];
        }
        __syncthreads();
        for (int32_t e = tid; e < CHUNK * nd; e += THREADS) {
            const int32_t tok = tok0 + e / nd, d = e % nd;
            if (inside(tok)) out[static_cast<size_t>(tok - first) * HD + d0 + d] = turned[e / nd][d] * scales[tok / c.block];
        }
        __syncthreads();
    }
}

// Workgroup (chunk, kv head): the chunk's codes and scales; the workgroups of chunk 0 also the open block's
// rows, from the source's rows where it is the source's open block too, else from its codes.
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
    if (tid < per && b < blocks) {
        to.key_scales[head_to * (to.slots / B) + b] = ks[b];
        to.value_scales[head_to * (to.slots / B) + b] = vs[b];
    }
    if (blockIdx.x != 0 || length % B == 0) return;
    const int32_t open = length / B;
    const size_t rows = head_to * B * HD;
    const bool same = open == source_length / B;
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
    const int64_t grid = static_cast<int64_t>(a.blocks) * a.c.kv_heads * 2 + (a.q ? (a.tokens + per - 1) / per : 0);
    if (grid > INT32_MAX) return fail(KT_ERR_SHAPE, "too many tokens and heads in one call");
    const size_t lds = static_cast<size_t>(a.c.block) * (a.c.head_dim + 1) * sizeof(float);
    if (lds > (64u << 10)) {  // beyond the default dynamic LDS limit (160 KB per CU on gfx950)
        static std::atomic<bool> raised{false};
        if (!raised) {
            KT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&append_kernel<KT_KV8_INT8>), hipFuncAttributeMaxDynamicSharedMemorySize, 144 << 10));
            KT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&append_kernel<KT_KV8_E4M3>), hipFuncAttributeMaxDynamicSharedMemorySize, 144 << 10));
            raised = true;
        }
    }
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
    if (tokens > 65535) return fail(KT_ERR_ARGUMENT, "%d tokens in one call: at most 65535", tokens);
    if (!aligned(q, 16) || !aligned(context, 16)) return fail(KT_ERR_ARGUMENT, "attention: q and the context must be 16-byte aligned");
    a->q = q;
    a->position = position;
    a->context = context;
    a->tokens = tokens;
    a->num_heads = num_heads;
    a->scale = 1.0f / sqrtf(static_cast<float>(a->c.head_dim));
    return KT_OK;
}

int32_t launch_attention(const AttnArgs& a, hipStream_t st) {
    const auto kernel = a.c.fmt == KT_KV8_INT8 ? attention_kernel<KT_KV8_INT8> : attention_kernel<KT_KV8_E4M3>;
    kernel<<<dim3(static_cast<uint32_t>(a.num_heads), static_cast<uint32_t>(a.tokens)), THREADS, 0, st>>>(a);
    KT_LAUNCHED("8-bit cache attention kernel");
    return KT_OK;
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
    return tokens == 0 ? KT_OK : launch_attention(a, static_cast<hipStream_t>(stream));
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
        void* ws = nullptr;
        if (const int32_t status = workspace(st, static_cast<size_t>(num_heads) * a.c.head_dim * sizeof(float), &ws)) return status;
        p.q_out = static_cast<float*>(ws);
        a.q = p.q_out;
    }
    if (const int32_t status = launch_append(p, st)) return status;
    return launch_attention(a, st);
}

int32_t kt_kv8_read(const kt_kv8_cache* cache, int32_t layer, int32_t first, int32_t count, float* keys, float* values, void* stream) {
    KV8View c;
    if (const int32_t status = view_kv8(cache, layer, &c)) return status;
    if (first < 0 || count < 0 || count > c.max_seq - first) return fail(KT_ERR_RANGE, "tokens %d + %d out of bounds %d", first, count, c.max_seq);
    if (!aligned(keys, 16)) return fail(KT_ERR_ARGUMENT, "keys must be 16-byte aligned");
    if (count == 0 || (!keys && !values)) return KT_OK;
    const dim3 grid(static_cast<uint32_t>((first + count - 1) / CHUNK - first / CHUNK + 1), static_cast<uint32_t>(c.kv_heads), 2);
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
