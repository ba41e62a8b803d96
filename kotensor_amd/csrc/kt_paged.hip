// kt_paged.hip -- the cache in pages that several sequences share, and trees of drafted tokens:
// RoPE and the append, the trees' masks, the walk that accepts drafted tokens, the move of what is
// kept, rows as fp32. No counterpart in the reference, whose cache holds one sequence (K/KVCache.kt:3-59).
// The attention is in kt_paged_attention.h.
#include <math.h>

#include "kt_paged.h"

namespace kt {
namespace {

constexpr int THREADS = 256;

// ---- RoPE and the append ---------------------------------------------------------------
// A wave takes one row and HEADS heads a lane of it: a lane has four pairs of a head, as many heads as fit lie side by side in the wave. Each
// lane makes one pair's cosine and sine (of 256 dims two), which those that need it take from there; they serve all its heads, whose loads go
// out together. Waves of query heads write the rotated query, waves of kv heads the key and the value. Bound by its bytes: five prompts
// of up to 1001 tokens, 32 and 8 heads of 128, fp32: 200 MB in 31 us where the last cache has them, 40 from memory; one token of 16
// sequences by its launch and three loads that wait for each other (starts, lengths, table): 4 us. (One float of a pair a lane and eight
// heads: 44 us; four heads of four pairs 32.)
constexpr int HEADS = 2;
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4_any __attribute__((ext_vector_type(4), aligned(4)));  // (k, v and q lie at any float)
struct AppendArgs {
    const float* q;  // NULL: only the append
    const float* k;
    const float* v;
    float* q_out;
    const float* inv_freq;
    PagedView c;
    BatchView b;
    int32_t num_heads, q_groups, groups;  // groups of heads a wave takes: of q, of all
};

// The sequence that row `row` belongs to; `sequences` for a row behind them all. All lanes of the wave active.
__device__ __forceinline__ int32_t sequence_of(const BatchView& b, int32_t row) {
    const int32_t lane = threadIdx.x & 63;
    int32_t s = 0;
    for (int32_t s0 = 0; s0 < b.sequences; s0 += 64) {
        const int32_t end = b.starts[min(s0 + lane, b.sequences - 1) + 1];
        s += __popcll(__ballot(s0 + lane < b.sequences && end <= row));
    }
    return s;
}

// Four elements as the cache holds them (store_element).
template <int FMT>
__device__ __forceinline__ void store_four(uint8_t* p, int64_t at, f4 x) {
    if constexpr (FMT == KT_PAGED_F32) {
        *reinterpret_cast<f4*>(p + 4 * at) = x;
    } else {
        uint2 both;
#pragma unroll
        for (int e = 0; e < 4; ++e) store_element<FMT>(reinterpret_cast<uint8_t*>(&both), e, x[e]);
        *reinterpret_cast<uint2*>(p + 2 * at) = both;
    }
}

template <int FMT>
__global__ void __launch_bounds__(THREADS) append_kernel(AppendArgs a) {
    const PagedView& c = a.c;
    const int32_t HD = c.head_dim, half = HD >> 1, lane = threadIdx.x & 63;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * (THREADS / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t row = static_cast<int32_t>(item / a.groups), group = static_cast<int32_t>(item % a.groups);
    if (row >= a.b.rows) return;
    const int32_t per_head = half >> 2, side = 64 / per_head, mine = lane % per_head;  // lanes of a head, heads side by side
    const bool is_q = group < a.q_groups;
    const int32_t heads = is_q ? a.num_heads : c.kv_heads;
    const int32_t h0 = (is_q ? group : group - a.q_groups) * HEADS * side + lane / per_head;
    const int32_t s = sequence_of(a.b, row);
    if (s >= a.b.sequences) return;  // behind the last sequence
    const int32_t index = row - a.b.starts[s];
    if (index < 0) return;
    const int64_t slot = static_cast<int64_t>(a.b.lengths[s]) + index;
    const int32_t pos = static_cast<int32_t>(a.b.depths ? static_cast<int64_t>(a.b.lengths[s]) + a.b.depths[row] : slot);
    const float* src = (is_q ? a.q : a.k) + static_cast<size_t>(row) * heads * HD + 4 * mine;
    const float* vsrc = a.v + static_cast<size_t>(row) * heads * HD + 4 * mine;
    f4 x1[HEADS], x2[HEADS], v1[HEADS], v2[HEADS];
#pragma unroll
    for (int u = 0; u < HEADS; ++u) {
        const size_t at = static_cast<size_t>(min(h0 + u * side, heads - 1)) * HD;
        x1[u] = *reinterpret_cast<const f4_any*>(src + at);
        x2[u] = *reinterpret_cast<const f4_any*>(src + at + half);
        if (!is_q) {
            v1[u] = *reinterpret_cast<const f4_any*>(vsrc + at);
            v2[u] = *reinterpret_cast<const f4_any*>(vsrc + at + half);
        }
    }
    float own_cos, own_sin, far_cos = 0.0f, far_sin = 0.0f, cf[4], sf[4];
    rope_sin_cos(pos, a.inv_freq[lane % half], own_cos, own_sin);
    if (half > 64) rope_sin_cos(pos, a.inv_freq[64 + lane], far_cos, far_sin);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int32_t pair = 4 * mine + e;
        cf[e] = __shfl(own_cos, pair & 63);
        sf[e] = __shfl(own_sin, pair & 63);
        if (half > 64) {
            const float other_cos = __shfl(far_cos, pair & 63), other_sin = __shfl(far_sin, pair & 63);
            cf[e] = pair < 64 ? cf[e] : other_cos;
            sf[e] = pair < 64 ? sf[e] : other_sin;
        }
    }
    const int64_t place = is_q ? 0 : place_of(c, a.b, s, slot, 0);
#pragma unroll
    for (int u = 0; u < HEADS; ++u) {
        const int32_t h = h0 + u * side;
        if (h >= heads) continue;
        f4 y1, y2;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float low, high;
            rope_apply(x1[u][e], x2[u][e], cf[e], sf[e], low, high);
            y1[e] = low;
            y2[e] = high;
        }
        if (is_q) {
            float* out = a.q_out + (static_cast<size_t>(row) * heads + h) * HD + 4 * mine;
            *reinterpret_cast<f4_any*>(out) = y1;
            *reinterpret_cast<f4_any*>(out + half) = y2;
        } else if (place >= 0) {
            const int64_t at = place + (static_cast<int64_t>(h) << c.page_shift) * HD + 4 * mine;
            store_four<FMT>(c.keys, at, y1);
            store_four<FMT>(c.keys, at + half, y2);
            store_four<FMT>(c.values, at, v1[u]);
            store_four<FMT>(c.values, at + half, v2[u]);
        }
    }
}

int32_t launch_append(AppendArgs a, hipStream_t st) {
    const int32_t heads = HEADS * (512 / a.c.head_dim);  // of a wave
    a.q_groups = a.q ? ceil_div(a.num_heads, heads) : 0;
    a.groups = a.q_groups + ceil_div(a.c.kv_heads, heads);
    const int64_t grid = (static_cast<int64_t>(a.b.rows) * a.groups + THREADS / 64 - 1) / (THREADS / 64);
    if (too_many(grid, THREADS)) return fail(KT_ERR_SHAPE, "too many rows and heads in one call");
    const auto kernel = a.c.fmt == KT_PAGED_F32 ? append_kernel<KT_PAGED_F32> : a.c.fmt == KT_PAGED_F16 ? append_kernel<KT_PAGED_F16> : append_kernel<KT_PAGED_BF16>;
    kernel<<<static_cast<uint32_t>(grid), THREADS, 0, st>>>(a);
    KT_LAUNCHED("paged cache append kernel");
    return KT_OK;
}

// ---- trees -------------------------------------------------------------------------------
// Workgroup: a sequence; thread: a row of it, which walks from parent to parent. A parent comes before its
// row (any other is none), so the walk ends, and meets the words of its mask in descending order. Latencies: 2 to 5 us.
constexpr int32_t TREE_LDS = 4096;  // parents held in LDS
__global__ void __launch_bounds__(THREADS) masks_kernel(const int32_t* parents, BatchView b, int32_t* depths, uint32_t* masks) {
    __shared__ int32_t held[TREE_LDS];
    const int32_t s = blockIdx.x, first = start_of(b, s), n = min(start_of(b, s + 1) - first, 32 * b.mask_words);
    const bool in_lds = n <= TREE_LDS;
    if (in_lds) {
        for (int32_t i = threadIdx.x; i < n; i += THREADS) held[i] = parents[first + i];
        __syncthreads();
    }
    for (int32_t i = threadIdx.x; i < n; i += THREADS) {
        uint32_t* row = masks + static_cast<size_t>(first + i) * b.mask_words;
        int32_t at = i, depth = 0, word = b.mask_words - 1;
        uint32_t bits = 0;
        for (;;) {
            for (; word > at >> 5; --word, bits = 0) row[word] = bits;
            bits |= 1u << (at & 31);
            const int32_t up = in_lds ? held[at] : parents[first + at];
            if (up < 0 || up >= at) break;
            at = up;
            ++depth;
        }
        for (; word >= 0; --word, bits = 0) row[word] = bits;
        depths[first + i] = depth;
    }
}

constexpr int32_t ACCEPT_LDS = 1024;  // rows whose numbers are held in LDS (a step of the walk reads three, one after another: 2.0 us for 4.0 from memory)
// One wave a sequence: from row 0 to the first row whose parent is the last one kept and whose token is
// the one chosen after that, as long as there is one.
__global__ void __launch_bounds__(64) accept_kernel(const int32_t* tokens, const int32_t* chosen, const int32_t* parents, BatchView b,
                                                    int32_t* kept, int32_t kept_stride, int32_t* counts, int32_t* next) {
    __shared__ int32_t held[3][ACCEPT_LDS];
    const int32_t s = blockIdx.x, lane = threadIdx.x, first = start_of(b, s), n = min(start_of(b, s + 1) - first, kept_stride);
    int32_t* out = kept + static_cast<size_t>(s) * kept_stride;
    const bool in_lds = n <= ACCEPT_LDS;
    if (in_lds) {
        for (int32_t i = lane; i < n; i += 64) {
            held[0][i] = parents[first + i];
            held[1][i] = tokens[first + i];
            held[2][i] = chosen[first + i];
        }
        __syncthreads();
    }
    auto parent_of = [&](int32_t r) { return in_lds ? held[0][r] : parents[first + r]; };
    auto token_of = [&](int32_t r) { return in_lds ? held[1][r] : tokens[first + r]; };
    auto chosen_after = [&](int32_t r) { return in_lds ? held[2][r] : chosen[first + r]; };
    int32_t count = 0, last = 0;
    if (n > 0) {
        count = 1;
        if (lane == 0) out[0] = 0;
        for (int32_t i0 = 1; i0 < n;) {  // rows from i0 on may follow `last`
            const int32_t want = chosen_after(last);
            int32_t found = -1;
            for (int32_t r0 = i0; r0 < n && found < 0; r0 += 64) {
                const int32_t r = min(r0 + lane, n - 1);
                const uint64_t hit = __ballot(r0 + lane < n && parent_of(r) == last && token_of(r) == want);
                if (hit) found = r0 + __builtin_ctzll(hit);
            }
            if (found < 0) break;
            if (lane == 0) out[count] = found;
            ++count;
            last = found;
            i0 = found + 1;
        }
    }
    for (int32_t i = count + lane; i < kept_stride; i += 64) out[i] = -1;
    if (lane == 0) {
        counts[s] = count;
        if (n > 0) next[s] = chosen_after(last);
    }
}

// ---- what is kept ------------------------------------------------------------------------
// How many of a sequence's kept rows count: up to the first that does not ascend or is none of its rows. All lanes of the
// wave active: each looks at an entry and the one before it.
__device__ __forceinline__ int32_t kept_count(const int32_t* kept, int32_t count, int32_t n) {
    const int32_t lane = threadIdx.x & 63;
    for (int32_t m0 = 0; m0 < count; m0 += 64) {
        const int32_t m = m0 + lane;
        const int32_t r = m < count ? kept[m] : -1, before = m > 0 && m < count ? kept[m - 1] : -1;
        const uint64_t odd = __ballot(r <= before || r >= n);  // (past the count too)
        if (odd) return m0 + __builtin_ctzll(odd);
    }
    return max(count, 0);
}

// Thread: 16 bytes of a head's keys or values in one layer, which it moves for every kept row in turn (a row
// moves down or stays, so no row is overwritten before it is read), several loads ahead. Latencies (counts, kept rows, table,
// rows): 4.6 us for one tree of 15 in two layers, 6.0 for 16 of up to 64 in eight.
constexpr int AHEAD = 8;
template <int BYTES>
__global__ void __launch_bounds__(THREADS) keep_kernel(PagedView c, size_t layer_bytes, int32_t pieces, BatchView b, const int32_t* kept, int32_t kept_stride,
                                                       const int32_t* counts, int32_t* new_lengths) {
    const int32_t s = blockIdx.y;
    const int32_t first = start_of(b, s), n = start_of(b, s + 1) - first, length = b.lengths[s];
    const int32_t* rows = kept + static_cast<size_t>(s) * kept_stride;
    const int32_t count = kept_count(rows, min(counts[s], kept_stride), n);
    if (blockIdx.x == 0 && threadIdx.x == 0 && new_lengths != b.lengths) new_lengths[s] = length + count;
    const int32_t per_row = c.head_dim * BYTES / 16;
    const int32_t e = blockIdx.x * THREADS + threadIdx.x;
    if (e >= pieces) return;
    const int32_t piece = e % per_row, g = e / per_row % c.kv_heads, which = e / per_row / c.kv_heads;
    uint8_t* base = (which % 2 ? c.values : c.keys) + static_cast<size_t>(which / 2) * layer_bytes + 16 * piece;
    for (int32_t m0 = 0; m0 < count; m0 += AHEAD) {
        uint4 x[AHEAD];
        int64_t to[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            to[u] = -1;
            const int32_t m = m0 + u;
            if (m >= count || rows[m] == m) continue;
            const int64_t from = place_of(c, b, s, static_cast<int64_t>(length) + rows[m], g);
            to[u] = from < 0 ? -1 : place_of(c, b, s, static_cast<int64_t>(length) + m, g);
            if (to[u] >= 0) x[u] = *reinterpret_cast<const uint4*>(base + from * BYTES);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (to[u] >= 0) *reinterpret_cast<uint4*>(base + to[u] * BYTES) = x[u];
    }
}

// lengths += what was kept: a wave a sequence
__global__ void __launch_bounds__(THREADS) kept_lengths_kernel(BatchView b, const int32_t* kept, int32_t kept_stride, const int32_t* counts, int32_t* lengths) {
    const int32_t s = blockIdx.x * (THREADS / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (s >= b.sequences) return;
    const int32_t count = kept_count(kept + static_cast<size_t>(s) * kept_stride, min(counts[s], kept_stride), start_of(b, s + 1) - start_of(b, s));
    if ((threadIdx.x & 63) == 0) lengths[s] += count;
}

// lengths += the rows of the call
__global__ void __launch_bounds__(THREADS) advance_kernel(BatchView b, int32_t* lengths) {
    const int32_t s = blockIdx.x * THREADS + threadIdx.x;
    if (s < b.sequences) lengths[s] += max(start_of(b, s + 1) - start_of(b, s), 0);
}

// ---- rows as fp32 --------------------------------------------------------------------------
template <int FMT>
__global__ void __launch_bounds__(THREADS) read_kernel(PagedView c, BatchView b, int32_t first, int32_t count, float* keys, float* values) {
    const int32_t HD = c.head_dim;
    const int64_t e = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x, per_head = static_cast<int64_t>(count) * HD;
    if (e >= per_head * c.kv_heads) return;
    const int32_t g = static_cast<int32_t>(e / per_head), x = static_cast<int32_t>(e % per_head / HD), d = static_cast<int32_t>(e % HD);
    const int64_t at = place_of(c, b, 0, static_cast<int64_t>(first) + x, g);
    if (keys) keys[e] = at < 0 ? __builtin_nanf("") : load_element<FMT>(c.keys, at + d);
    if (values) values[e] = at < 0 ? __builtin_nanf("") : load_element<FMT>(c.values, at + d);
}

int32_t check_heads(int32_t num_heads, int32_t kv_heads) {
    if (num_heads <= 0 || num_heads % kv_heads != 0)
        return fail(KT_ERR_ARGUMENT, "numHeads %d must be a multiple of numKeyValueHeads %d", num_heads, kv_heads);
    return KT_OK;
}

int32_t check_shape(const kt_paged_cache* c) {
    if (!c) return fail(KT_ERR_ARGUMENT, "cache is NULL");
    if (c->format != KT_PAGED_F32 && c->format != KT_PAGED_F16 && c->format != KT_PAGED_BF16)
        return fail(KT_ERR_ARGUMENT, "cache format %d: KT_PAGED_F32, KT_PAGED_F16 or KT_PAGED_BF16", c->format);
    if (c->layers <= 0 || c->pages <= 0 || c->kv_heads <= 0) return fail(KT_ERR_ARGUMENT, "layers, pages and key/value heads must be positive");
    if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(KT_ERR_ARGUMENT, "head dimension %d of a paged cache: 32, 64, 128 or 256", c->head_dim);
    if (c->page_tokens < 16 || c->page_tokens > 256 || (c->page_tokens & (c->page_tokens - 1)))
        return fail(KT_ERR_ARGUMENT, "%d tokens to a page: 16, 32, 64, 128 or 256", c->page_tokens);
    if (c->kv_heads > 65535 || c->layers > 65535) return fail(KT_ERR_SHAPE, "%d layers of %d key/value heads: at most 65535 each", c->layers, c->kv_heads);
    if (static_cast<__int128>(c->layers) * c->pages * c->kv_heads * c->page_tokens * c->head_dim * 4 > INT64_MAX) return fail(KT_ERR_SHAPE, "the pool is too large");
    return KT_OK;
}

int64_t layer_elements(const kt_paged_cache* c) { return static_cast<int64_t>(c->pages) * c->kv_heads * c->page_tokens * c->head_dim; }

}  // namespace

int32_t view_paged(const kt_paged_cache* c, int32_t layer, PagedView* v) {
    if (const int32_t status = check_shape(c)) return status;
    if (!c->keys || !c->values) return fail(KT_ERR_ARGUMENT, "a pointer of the cache is NULL");
    if (!aligned(c->keys, 16) || !aligned(c->values, 16)) return fail(KT_ERR_ARGUMENT, "the cache's keys and values must be 16-byte aligned");
    if (layer < 0 || layer >= c->layers) return fail(KT_ERR_RANGE, "layer %d out of bounds %d", layer, c->layers);
    const size_t at = static_cast<size_t>(layer) * layer_elements(c) * element_bytes(c->format);
    v->keys = static_cast<uint8_t*>(c->keys) + at;
    v->values = static_cast<uint8_t*>(c->values) + at;
    v->fmt = c->format;
    v->pages = c->pages;
    v->kv_heads = c->kv_heads;
    v->head_dim = c->head_dim;
    v->page_shift = __builtin_ctz(c->page_tokens);
    return KT_OK;
}

// (cache: NULL for a call that needs only the rows)
int32_t view_batch(const kt_paged_batch* b, const kt_paged_cache* cache, BatchView* v) {
    if (!b) return fail(KT_ERR_ARGUMENT, "batch is NULL");
    if (!b->starts || (cache && (!b->tables || !b->lengths))) return fail(KT_ERR_ARGUMENT, "a pointer of the batch is NULL");
    if (b->sequences < 0 || b->sequences > 65535) return fail(KT_ERR_ARGUMENT, "%d sequences: 0 to 65535", b->sequences);
    if (b->rows < 0 || b->most_rows < 0 || b->most_rows > b->rows)
        return fail(KT_ERR_ARGUMENT, "at most %d rows a sequence of %d rows in all", b->most_rows, b->rows);
    if (b->rows >= 1 << 24) return fail(KT_ERR_SHAPE, "%d rows in one call: at most %d", b->rows, (1 << 24) - 1);
    if (!b->masks != !b->depths) return fail(KT_ERR_ARGUMENT, "a tree has masks and depths, a text neither");
    if (b->masks && (b->mask_words <= 0 || b->mask_words > INT32_MAX / 32 || 32 * static_cast<int64_t>(b->mask_words) < b->most_rows))
        return fail(KT_ERR_SHAPE, "%d mask words do not hold %d rows", b->mask_words, b->most_rows);
    if (cache) {
        if (b->table_stride <= 0) return fail(KT_ERR_ARGUMENT, "table_stride must be positive");
        const int64_t room = static_cast<int64_t>(b->table_stride) * cache->page_tokens;
        if (b->key_bound > 1 << 30) return fail(KT_ERR_SHAPE, "key bound %d: at most %d", b->key_bound, 1 << 30);  // (chunks' ends are 32-bit)
        if (b->key_bound < b->most_rows || b->key_bound > room)
            return fail(KT_ERR_ARGUMENT, "key bound %d must cover the %d rows of a sequence and fit its table's %lld tokens", b->key_bound, b->most_rows, static_cast<long long>(room));
    }
    v->tables = b->tables;
    v->lengths = b->lengths;
    v->starts = b->starts;
    v->depths = b->depths;
    v->masks = b->masks;
    v->table_stride = b->table_stride;
    v->sequences = b->sequences;
    v->rows = b->rows;
    v->most_rows = b->most_rows;
    v->key_bound = b->key_bound;
    v->mask_words = b->mask_words;
    return KT_OK;
}

}  // namespace kt

using namespace kt;

namespace {

// Nothing to do for any sequence (rows that belong to none may be there).
bool no_rows(const BatchView& b) { return b.rows == 0 || b.sequences == 0 || b.most_rows == 0; }

int32_t append_args(const float* q, const float* k, const float* v, int32_t num_heads, const float* inv_freq, const kt_paged_cache* cache, int32_t layer,
                    const kt_paged_batch* batch, float* q_out, AppendArgs* a) {
    if (const int32_t status = view_paged(cache, layer, &a->c)) return status;
    if (const int32_t status = view_batch(batch, cache, &a->b)) return status;
    if (!k || !v || !inv_freq || !q != !q_out) return fail(KT_ERR_ARGUMENT, "a pointer argument is NULL");
    if (const int32_t status = check_heads(num_heads, a->c.kv_heads)) return status;
    a->q = q;
    a->k = k;
    a->v = v;
    a->q_out = q_out;
    a->inv_freq = inv_freq;
    a->num_heads = num_heads;
    return KT_OK;
}

int32_t launch_attention(const PagedAttnArgs& a, hipStream_t st, const float* k = nullptr, const float* v = nullptr) {
    const auto launch = a.c.fmt == KT_PAGED_F32 ? launch_paged_attention_f32 : a.c.fmt == KT_PAGED_F16 ? launch_paged_attention_f16 : launch_paged_attention_bf16;
    return launch(a, k, v, st);
}

int32_t attention_args(const float* q, int32_t num_heads, const kt_paged_cache* cache, int32_t layer, const kt_paged_batch* batch, float* context,
                       PagedAttnArgs* a) {
    if (const int32_t status = view_paged(cache, layer, &a->c)) return status;
    if (const int32_t status = view_batch(batch, cache, &a->b)) return status;
    if (!q || !context) return fail(KT_ERR_ARGUMENT, "a pointer argument is NULL");
    if (const int32_t status = check_heads(num_heads, a->c.kv_heads)) return status;
    if (!aligned(q, 16) || !aligned(context, 16)) return fail(KT_ERR_ARGUMENT, "attention: q and the context must be 16-byte aligned");
    a->q = q;
    a->context = context;
    a->num_heads = num_heads;
    a->scale = 1.0f / sqrtf(static_cast<float>(a->c.head_dim));
    return KT_OK;
}

}  // namespace

extern "C" {

int32_t kt_paged_layout(const kt_paged_cache* cache, int64_t* bytes) {
    if (const int32_t status = check_shape(cache)) return status;
    if (!bytes) return fail(KT_ERR_ARGUMENT, "bytes is NULL");
    *bytes = cache->layers * layer_elements(cache) * element_bytes(cache->format);
    return KT_OK;
}

int32_t kt_rope_paged(const float* q, const float* k, const float* v, int32_t num_heads, const float* inv_freq, const kt_paged_cache* cache, int32_t layer,
                      const kt_paged_batch* batch, float* q_out, void* stream) {
    AppendArgs a{};
    if (const int32_t status = append_args(q, k, v, num_heads, inv_freq, cache, layer, batch, q_out, &a)) return status;
    return no_rows(a.b) ? KT_OK : launch_append(a, static_cast<hipStream_t>(stream));
}

int32_t kt_attention_paged(const float* q, int32_t num_heads, const kt_paged_cache* cache, int32_t layer, const kt_paged_batch* batch, float* context,
                           void* stream) {
    PagedAttnArgs a{};
    if (const int32_t status = attention_args(q, num_heads, cache, layer, batch, context, &a)) return status;
    return no_rows(a.b) ? KT_OK : launch_attention(a, static_cast<hipStream_t>(stream));
}

int32_t kt_rope_attention_paged(const float* q, const float* k, const float* v, const float* inv_freq, int32_t num_heads, const kt_paged_cache* cache,
                                int32_t layer, const kt_paged_batch* batch, float* context, void* stream) {
    AppendArgs p{};
    PagedAttnArgs a{};
    if (const int32_t status = append_args(q, k, v, num_heads, inv_freq, cache, layer, batch, context, &p)) return status;
    if (const int32_t status = attention_args(q, num_heads, cache, layer, batch, context, &a)) return status;
    if (no_rows(a.b)) return KT_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    // A step of up to 16 query heads a kv head: one launch.
    if (a.b.most_rows == 1 && num_heads / a.c.kv_heads <= 16) {
        a.inv_freq = inv_freq;
        return launch_attention(a, st, k, v);
    }
    // Otherwise the rotated queries wait in the context: a tile's are read by its own parts alone, all of them before
    // the last writes what becomes of them there.
    if (const int32_t status = launch_append(p, st)) return status;
    a.q = context;
    return launch_attention(a, st);
}

int32_t kt_tree_masks(const int32_t* parents, const kt_paged_batch* batch, int32_t* depths, uint32_t* masks, void* stream) {
    BatchView b;
    if (const int32_t status = view_batch(batch, nullptr, &b)) return status;
    if (!parents || !depths || !masks) return fail(KT_ERR_ARGUMENT, "a pointer argument is NULL");
    if (!b.masks) return fail(KT_ERR_ARGUMENT, "the batch has no masks");
    if (b.rows == 0 || b.sequences == 0) return KT_OK;
    masks_kernel<<<static_cast<uint32_t>(b.sequences), THREADS, 0, static_cast<hipStream_t>(stream)>>>(parents, b, depths, masks);
    KT_LAUNCHED("tree masks kernel");
    return KT_OK;
}

int32_t kt_tree_accept(const int32_t* tokens, const int32_t* chosen, const int32_t* parents, const kt_paged_batch* batch, int32_t* kept, int32_t kept_stride,
                       int32_t* counts, int32_t* next, void* stream) {
    BatchView b;
    if (const int32_t status = view_batch(batch, nullptr, &b)) return status;
    if (!tokens || !chosen || !parents || !kept || !counts || !next) return fail(KT_ERR_ARGUMENT, "a pointer argument is NULL");
    if (kept_stride <= 0 || kept_stride < b.most_rows) return fail(KT_ERR_SHAPE, "kept_stride %d does not hold %d rows", kept_stride, b.most_rows);
    if (b.sequences == 0) return KT_OK;
    accept_kernel<<<static_cast<uint32_t>(b.sequences), 64, 0, static_cast<hipStream_t>(stream)>>>(tokens, chosen, parents, b, kept, kept_stride, counts, next);
    KT_LAUNCHED("tree accept kernel");
    return KT_OK;
}

int32_t kt_paged_keep(const kt_paged_cache* cache, const kt_paged_batch* batch, const int32_t* kept, int32_t kept_stride, const int32_t* counts,
                      int32_t* new_lengths, void* stream) {
    PagedView c;
    BatchView b;
    if (const int32_t status = view_paged(cache, 0, &c)) return status;
    if (const int32_t status = view_batch(batch, cache, &b)) return status;
    if (!kept || !counts || !new_lengths) return fail(KT_ERR_ARGUMENT, "a pointer argument is NULL");
    if (kept_stride <= 0) return fail(KT_ERR_SHAPE, "kept_stride must be positive");
    if (b.sequences == 0) return KT_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int32_t bytes = element_bytes(c.fmt);
    const int64_t pieces = 2 * static_cast<int64_t>(cache->layers) * c.kv_heads * (c.head_dim * bytes / 16);
    if (pieces > INT32_MAX - THREADS) return fail(KT_ERR_SHAPE, "too many layers and heads in one call");
    const dim3 grid(static_cast<uint32_t>((pieces + THREADS - 1) / THREADS), static_cast<uint32_t>(b.sequences));
    const auto kernel = bytes == 4 ? keep_kernel<4> : keep_kernel<2>;
    kernel<<<grid, THREADS, 0, st>>>(c, static_cast<size_t>(layer_elements(cache)) * bytes, static_cast<int32_t>(pieces), b, kept, kept_stride, counts, new_lengths);
    KT_LAUNCHED("paged cache keep kernel");
    if (new_lengths == b.lengths) {  // (the move reads the lengths from before)
        kept_lengths_kernel<<<static_cast<uint32_t>(ceil_div(b.sequences, THREADS / 64)), THREADS, 0, st>>>(b, kept, kept_stride, counts, new_lengths);
        KT_LAUNCHED("paged cache lengths kernel");
    }
    return KT_OK;
}

int32_t kt_paged_advance(int32_t* lengths, const kt_paged_batch* batch, void* stream) {
    BatchView b;
    if (const int32_t status = view_batch(batch, nullptr, &b)) return status;
    if (!lengths) return fail(KT_ERR_ARGUMENT, "a pointer argument is NULL");
    if (b.sequences == 0) return KT_OK;
    advance_kernel<<<static_cast<uint32_t>(ceil_div(b.sequences, THREADS)), THREADS, 0, static_cast<hipStream_t>(stream)>>>(b, lengths);
    KT_LAUNCHED("paged cache lengths kernel");
    return KT_OK;
}

int32_t kt_paged_read(const kt_paged_cache* cache, int32_t layer, const int32_t* table, int32_t entries, int32_t first, int32_t count, float* keys, float* values,
                      void* stream) {
    PagedView c;
    if (const int32_t status = view_paged(cache, layer, &c)) return status;
    if (!table) return fail(KT_ERR_ARGUMENT, "a pointer argument is NULL");
    const int64_t room = static_cast<int64_t>(entries) * cache->page_tokens;
    if (entries <= 0 || first < 0 || count < 0 || static_cast<int64_t>(first) + count > room)
        return fail(KT_ERR_RANGE, "tokens %d + %d out of bounds %lld", first, count, static_cast<long long>(entries > 0 ? room : 0));
    if (count == 0 || (!keys && !values)) return KT_OK;
    const int64_t grid = (static_cast<int64_t>(count) * c.kv_heads * c.head_dim + THREADS - 1) / THREADS;
    if (too_many(grid, THREADS)) return fail(KT_ERR_SHAPE, "too many tokens and heads in one call");
    BatchView b{};
    b.tables = table;
    b.table_stride = entries;
    const auto kernel = c.fmt == KT_PAGED_F32 ? read_kernel<KT_PAGED_F32> : c.fmt == KT_PAGED_F16 ? read_kernel<KT_PAGED_F16> : read_kernel<KT_PAGED_BF16>;
    kernel<<<static_cast<uint32_t>(grid), THREADS, 0, static_cast<hipStream_t>(stream)>>>(c, b, first, count, keys, values);
    KT_LAUNCHED("paged cache read kernel");
    return KT_OK;
}

}  // extern "C"
