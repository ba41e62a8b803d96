// kt_paged_attention.h -- attention over the cache in pages (kt_paged.h): decode steps, prompts and
// trees of drafted tokens of several sequences in one launch. No counterpart in the reference
// (K/Attention.kt:277-349 attends in one sequence's cache). One translation unit a format includes it.
//
// Rows: the (row, query head) pairs of a sequence and kv head, a row's G heads side by side, in tiles of R. A
// tile's keys are cut into parts of about the same number of chunks for all sequences of the launch, whatever
// their lengths: every workgroup reads the sequences' rows and lengths, from which follow the parts'
// size and its own place among them, so that one long sequence beside short ones fills the card. A workgroup holds
// its rows' queries as matrix operands and goes through its part's chunks of keys:
//   S^T = K Q^T: a lane ends with scores of one row (its column), so that the running maximum and sum of a
//     row stay inside the lanes of a column.
//   O^T += V^T P^T: the weights are operands where they are.
// Products in fp32 precision: numbers held in fp16 are one operand and queries and weights two fp16 ones (to
// 2^-22 of a row's largest query, 2^-30 of its largest weight); held in bf16 one operand and three bf16 ones (exact);
// fp32 three each, of whose nine products the six down to 2^-17 are formed (kt_split.h).
// A row's maximum follows its scores lazily: a larger one moves it only once it is 2^8 above, so that the sums are
// seldom rescaled. Parts meet through memory: of tiles of 16 rows the last workgroup of a tile to arrive (a counter, which it
// returns to zero) merges all in their order, so that no workgroup waits for another and the bits do not depend on who
// is last; of larger tiles a launch of its own does.
// Two kernels: attention_kernel for few rows, bound by the cache's bytes (64 steps over 2048 tokens on average, 128 dims, bf16: 111 us,
// 4.9 TB/s; one of 131000 beside seven shorter, fp16: 84 us, 5.2 TB/s; a large copy runs at 4.8), with short texts by the chain of loads from
// the lengths to the merge (11.5 us); tile_kernel for many, bound by the vector and matrix instructions of two waves a SIMD that wait for
// each other's chunks (a prompt of 2048, 128 dims, bf16, pages of 64: 94 us, 365 TFLOP/s of attention, 1095 of matrix products, of which a
// large library product reaches 1112), with few chunks by a part's beginning, 7 to 10 us.
#pragma once

#include <algorithm>
#include <type_traits>

#include "kt_paged.h"
#include "kt_split.h"

namespace kt {
namespace paged {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

constexpr int CHUNK = 32;        // keys a wave takes at a time
constexpr float LAZY = 8.0f;     // how far a score may pass the maximum, in powers of two
constexpr int THROUGH = 1 | 16;  // buffer cache bits sc0 sc1: past the caches

// ---- operands ------------------------------------------------------------------------------
// QP parts of a query or weight, KP of a key or value; weights are taken times 2^UP.
template <int FMT>
struct Format {
    typedef bf16x8 op;
    static constexpr int QP = 3, KP = FMT == KT_PAGED_F32 ? 3 : 1, E = element_bytes(FMT);
    static constexpr float UP = 0.0f;
};
template <>
struct Format<KT_PAGED_F16> {
    typedef half8 op;
    static constexpr int QP = 2, KP = 1, E = 2;
    static constexpr float UP = 6.0f;  // (so that their second parts are normal numbers down to 2^-20)
};

__device__ __forceinline__ f4 product(bf16x8 a, bf16x8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 product(half8 a, half8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// Several sums at once, product by product: neighbours do not wait for each other.
template <int N, int KP, int QP, typename OP>
__device__ __forceinline__ void products_of(const OP (&k)[N][KP], const OP (&q)[QP], f4 (&c)[N]) {
#pragma unroll
    for (int w = QP - 1; w >= 0; --w)
#pragma unroll
        for (int i = KP - 1; i >= 0; --i)
#pragma unroll
            for (int t = 0; t < N; ++t)
                if (w - i >= 0) c[t] = product(k[t][i], q[w - i], c[t]);
}
// The sum of the parts' products down to 2^-17 of the largest, the small ones first.
template <int KP, int QP, typename OP>
__device__ __forceinline__ f4 products(const OP (&k)[KP], const OP (&q)[QP], f4 c) {
#pragma unroll
    for (int w = QP - 1; w >= 0; --w)
#pragma unroll
        for (int i = KP - 1; i >= 0; --i)
            if (w - i >= 0) c = product(k[i], q[w - i], c);
    return c;
}

__device__ __forceinline__ void split_weights(const float (&v)[8], bf16x8 (&part)[3]) { split3_nearest(v, part); }
__device__ __forceinline__ void split_weights(const float (&v)[8], half8 (&part)[2]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const half2v h = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(v[2 * i], v[2 * i + 1]));
        // (to the nearest, so that what weights below fp16's normal numbers lose has no sign)
        const half2v l = __builtin_convertvector((f32x2{v[2 * i] - static_cast<float>(h[0]), v[2 * i + 1] - static_cast<float>(h[1])}), half2v);
        part[0][2 * i] = h[0];
        part[0][2 * i + 1] = h[1];
        part[1][2 * i] = l[0];
        part[1][2 * i + 1] = l[1];
    }
}

__device__ __forceinline__ void split_query(const float (&v)[8], bf16x8 (&part)[3]) { split3_nearest(v, part); }
__device__ __forceinline__ void split_query(const float (&v)[8], half8 (&part)[2]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        part[0][i] = static_cast<_Float16>(v[i]);
        part[1][i] = static_cast<_Float16>(v[i] - static_cast<float>(part[0][i]));
    }
}

// Eight consecutive elements (registers of a row) as operands.
template <int FMT>
__device__ __forceinline__ void to_operands(const uint32_t* w, typename Format<FMT>::op (&part)[Format<FMT>::KP]) {
    if constexpr (FMT == KT_PAGED_F32) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(float, w[i]);
        split3_nearest(v, part);
    } else {
        part[0] = __builtin_bit_cast(typename Format<FMT>::op, u4{w[0], w[1], w[2], w[3]});
    }
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }

// ---- exchanges over the lanes of a column (apart by 16 or 32) --------------------------------
struct Swapped {
    float a, b;  // of two lanes apart by 16 (32): the value of the one and of the other, in both
};
// (the wait states are those between a vector write and the swap's read)
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
__device__ __forceinline__ float column_max(float v) {
    const Swapped near = swap16(v), far = swap32(fmaxf(near.a, near.b));
    return fmaxf(far.a, far.b);
}
__device__ __forceinline__ float column_sum(float v) {
    const Swapped near = swap16(v), far = swap32(near.a + near.b);
    return far.a + far.b;
}

// The maximum is a rounded product; at sizes where its rounding is a power of two and more, the
// exponent is the difference of rounded products, so that it stays below LAZY.
constexpr float HUGE_SCORE = 65536.0f;
__device__ __forceinline__ float weight_of_huge(float x, float f, float m, float up) {
#pragma clang fp contract(off)
    const float s = x * f;
    return __builtin_amdgcn_exp2f((s - m) + up);
}
// A score as the maxima hold it: rounded, also where the next step subtracts one.
__device__ __forceinline__ float rounded_score(float x, float f) {
#pragma clang fp contract(off)
    return x * f;
}
// What a part with the maximum m and the sum l counts beside parts with the maximum mx: a part without keys
// (l = 0) nothing, one with a NaN a NaN.
__device__ __forceinline__ float share_of(float m, float l, float mx) {
    return l == 0.0f ? 0.0f : l * __builtin_amdgcn_exp2f((m == -INFINITY ? mx : m) - (mx == -INFINITY ? 0.0f : mx));
}
// The weight of a part's average: with keys (l) it is above zero, so that infinities count (2^-149 of a finite average is nothing
// beside the 2^-30 of the weights' parts).
__device__ __forceinline__ float weight_of_part(float share, float l) { return share < 0x1p-149f && l != 0.0f ? 0x1p-149f : share; }

// A chunk's scores x of one row (a lane's share of them) into weights; m and l: the row's running maximum and the sum of this
// lane's weights; rescale: what the maximum's move does to the sums. Tokens that the row does not see come with -infinity.
template <int FMT, int E, typename RESCALE>
__device__ __forceinline__ void to_weights(float (&x)[E], float f, float& m, float& l, RESCALE rescale) {
    constexpr float UP = Format<FMT>::UP;
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < E; ++i) most = fmaxf(most, x[i]);
    most = rounded_score(most, f);
    if (__ballot(most - m > LAZY)) {
        const float m_new = fmaxf(m, column_max(most));
        const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
        l *= alpha;
        rescale(alpha);
        m = m_new;
    }
    const float at = m == -INFINITY ? 0.0f : m;
    if (__ballot(fabsf(at) > HUGE_SCORE)) {  // (one-hot rows)
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = weight_of_huge(x[i], f, at, UP);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], f, UP - at));
    }
#pragma unroll
    for (int i = 0; i < E; ++i) l += x[i];
}

// The tokens x0 .. x0 + 31 that row `index` of a sequence's rows sees, a bit each.
__device__ __forceinline__ uint32_t seen_bits(const BatchView& b, int32_t first, int32_t index, int64_t length, int32_t x0, uint32_t there) {
    const int64_t below = length - x0;  // tokens of the chunk before the new ones
    uint32_t bits = below >= 32 ? 0xFFFFFFFFu : below <= 0 ? 0u : (1u << below) - 1u;
    if (b.masks) {
        const uint32_t* mask = b.masks + static_cast<size_t>(first + index) * b.mask_words;
        auto word = [&](int64_t w) { return w >= 0 && w < b.mask_words ? mask[w] : 0u; };
        if (below < 32) {  // the mask's bits from -below on
            const int64_t from = -below, w = from >> 5;
            const int32_t by = static_cast<int32_t>(from & 31);
            bits |= word(w) >> by | (by ? word(w + 1) << (32 - by) : 0u);
        }
    } else {
        const int64_t upto = below + index + 1;
        bits = upto >= 32 ? 0xFFFFFFFFu : upto <= 0 ? 0u : (1u << upto) - 1u;
    }
    return bits & there;
}

// ---- the parts of a launch ---------------------------------------------------------------------
// Parts of a tile at most.
constexpr int MOST_PARTS = 128;
struct Args {
    PagedAttnArgs p;
    const float* k_new;  // STEP: the step's projections before RoPE
    const float* v_new;
    int32_t target;      // workgroups among which the launch's chunks are shared out
    float* averages;     // [slots][R][head_dim]: the parts' averages
    float* stats;        // [slots][R][2]: their maxima and sums
    uint32_t* counters;  // [slots], zero between launches
    int32_t slots;       // 0: every tile is one part
};

__device__ __forceinline__ int32_t held_keys(const PagedView& c, const BatchView& b, int32_t length, int32_t n) {
    const int64_t most = min(room_of(c, b), static_cast<int64_t>(b.key_bound));
    return static_cast<int32_t>(min(max(static_cast<int64_t>(length) + n, int64_t{0}), most));
}
// Sums over the lanes up to each lane, without LDS: by DPP inside rows of 16 lanes, then the rows' totals passed on.
template <int CTRL, int ROWS>
__device__ __forceinline__ int32_t dpp_add(int32_t v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int32_t lanes_upto(int32_t v) {
    v = dpp_add<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);  // lane 15 of a row to the next one (rows 1 and 3), lane 31 to rows 2 and 3
    return dpp_add<0x143, 0xC>(v);
}
__device__ __forceinline__ int32_t lane_int(int32_t v, int32_t lane) { return __builtin_amdgcn_readlane(v, lane); }
// A number that every lane has, as a scalar (divisions leave it in vector registers, and what follows from it too).
__device__ __forceinline__ int32_t uniform(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int32_t>(v))); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    return static_cast<int64_t>(static_cast<uint64_t>(uniform(static_cast<uint32_t>(v >> 32))) << 32 | uniform(static_cast<uint32_t>(v)));
}

struct Part {
    int32_t sequence, first, n, length;  // its rows and tokens
    int32_t tile, head, split, splits;
    int32_t keys;   // tokens that rows of the sequence may see
    int32_t per;    // chunks a part may have
    int32_t slot;   // of the tile's first part
    __device__ __forceinline__ void make_uniform() {  // (they meet behind branches that look divergent)
        for (int32_t* v : {&sequence, &first, &n, &length, &tile, &head, &split, &splits, &keys, &per, &slot}) *v = uniform(*v);
    }
};

// Which part of the launch workgroup `at` has (BY_SLOT: whose slot `at` is); false: none. Every lane is a sequence. A part's size is at least
// the chunks over target, so a launch has at most target + (its tiles of all kv heads) parts, and at most 2 target that share a
// tile. Tiles of many rows (FINE): where that size is above LONG tokens and tiles are fewer than 2 target, whose rounds would leave
// workgroups idle, but not a round of whole tiles, the chunks over 2 target: at most 4 target parts that share a tile. (us at target, at 2 target,
// 128 dims, bf16: 300 rows after 8000 tokens 185, 122; 1300 after 8000 597, 495; 16 sequences with trees of 64 after 3000 120, 117; with 64 rows
// after 1000 each 58, 75: a round of whole tiles. Everywhere: a tree of 60 after 4000 38, 46.)
constexpr int LONG = 1024;
constexpr bool fine(int R) { return R > 16; }
template <int R, int LEAST, int CHUNK, bool BY_SLOT = false>
__device__ __forceinline__ bool find_part(const Args& a, int32_t at, Part& out) {
    const PagedView& c = a.p.c;
    const BatchView& b = a.p.b;
    const int32_t lane = threadIdx.x & 63, G = a.p.num_heads / c.kv_heads;
    int32_t first = 0, n = 0, length = 0;
    auto load = [&](int32_t s0) {
        const int32_t s = min(s0 + lane, b.sequences - 1);
        first = start_of(b, s);
        n = start_of(b, s + 1) - first;
        length = b.lengths[s];
        if (s0 + lane >= b.sequences) n = 0;
        n = min(max(n, 0), b.most_rows);
    };
    auto tiles_of = [&]() { return static_cast<int32_t>((static_cast<int64_t>(n) * G + R - 1) / R); };
    auto chunks_of = [&]() { return (held_keys(c, b, length, n) + CHUNK - 1) / CHUNK; };
    // (whole numbers up to 2^24 are exact in fp32; of larger totals a little more)
    float total = 0.0f, rows = 0.0f, all_tiles = 0.0f;
    int32_t most = 0;
    for (int32_t s0 = 0; s0 < b.sequences; s0 += 64) {
        load(s0);
        const float tiles = static_cast<float>(tiles_of()) * static_cast<float>(c.kv_heads);
        total += tiles * static_cast<float>(max(chunks_of(), 1));
        all_tiles += tiles;
        rows += static_cast<float>(n);
        most = max(most, n > 0 ? chunks_of() : 0);
    }
    total = wave_sum_dpp(total);
    if (wave_sum_dpp(rows) > static_cast<float>(b.rows)) return false;  // starts that do not ascend
    if (total >= 0x1p24f) total *= 1.0f + 0x1p-16f;
    auto size_for = [&](float target) {
        int32_t size = static_cast<int32_t>(fminf(total / target, 0x1p30f));
        if (static_cast<float>(size) * target < total) ++size;
        return uniform((max(size, 1) + LEAST - 1) / LEAST * LEAST);
    };
    const float target = static_cast<float>(a.target);
    int32_t per = a.slots == 0 ? 1 << 26 : size_for(target);
    if constexpr (fine(R)) {
        if (a.slots > 0 && total > target * (LONG / CHUNK)) {
            all_tiles = wave_sum_dpp(all_tiles);
            if (all_tiles < 2.0f * target && (all_tiles > target || __ballot(most > per))) per = size_for(2.0f * target);
        }
    }
    int32_t before = 0, slots = 0;
    for (int32_t s0 = 0; s0 < b.sequences; s0 += 64) {
        if (b.sequences > 64) load(s0);
        const int32_t tiles = tiles_of(), chunks = chunks_of();
        const int32_t size = max(per, (chunks + MOST_PARTS - 1) / MOST_PARTS);
        const int32_t splits = max((chunks + size - 1) / size, 1), parts = tiles * c.kv_heads * splits;
        const int32_t mine = splits > 1 ? parts : 0;
        const int32_t upto = lanes_upto(parts), slots_upto = lanes_upto(mine);
        const int32_t passed = uniform(static_cast<int32_t>(__popcll(__ballot((BY_SLOT ? slots + slots_upto : before + upto) <= at))));
        if (passed < 64) {
            const int32_t slot0 = uniform(slots) + lane_int(slots_upto, passed) - lane_int(mine, passed);
            const int32_t local = BY_SLOT ? at - slot0 : at - before - (lane_int(upto, passed) - lane_int(parts, passed));
            out.sequence = uniform(s0 + passed);
            out.first = lane_int(first, passed);
            out.n = lane_int(n, passed);
            out.length = lane_int(length, passed);
            out.splits = lane_int(splits, passed);
            out.per = lane_int(size, passed);
            if constexpr (BY_SLOT) {
                const int32_t rest = uniform(local / out.splits);
                out.split = uniform(local % out.splits);
                out.head = uniform(rest % c.kv_heads);
                out.tile = uniform(rest / c.kv_heads);
            } else {
                out.head = uniform(local % c.kv_heads);  // (workgroups go round the eight dies: a head's stay on few of them)
                const int32_t rest = uniform(local / c.kv_heads);
                out.split = uniform(rest % out.splits);
                out.tile = lane_int(tiles, passed) - 1 - uniform(rest / out.splits);  // (a text's last tiles see the most)
            }
            out.keys = uniform(held_keys(c, b, out.length, out.n));
            out.slot = slot0 + (out.tile * c.kv_heads + out.head) * out.splits;
            return true;
        }
        before += lane_int(upto, 63);
        slots += lane_int(slots_upto, 63);
    }
    return false;
}

// A tile's keys: tokens below n_keys that some row sees, below n_all that all see; the part's chunks c0 .. c1 - 1.
struct Keys {
    int32_t n_keys, n_all, splits, c0, c1;
};
template <int R, int CHUNK>
__device__ __forceinline__ Keys keys_of(const Args& a, const Part& part, int32_t held) {
    const int32_t G = a.p.num_heads / a.p.c.kv_heads, t_first = uniform(part.tile * R / G), t_last = uniform((part.tile * R + held - 1) / G);
    const int64_t length = part.length;
    const bool tree = a.p.b.masks != nullptr;
    Keys k;
    k.n_keys = tree ? part.keys : uniform(static_cast<int32_t>(min(static_cast<int64_t>(part.keys), max(length + t_last + 1, int64_t{0}))));
    k.n_all = uniform(static_cast<int32_t>(min(static_cast<int64_t>(k.n_keys), max(length + (tree ? 0 : t_first + 1), int64_t{0}))));
    const int32_t chunks = (k.n_keys + CHUNK - 1) / CHUNK;
    k.splits = uniform(max(1, min(part.splits, (chunks + part.per - 1) / part.per)));
    const uint32_t whole = static_cast<uint32_t>(chunks) / static_cast<uint32_t>(k.splits), rest = static_cast<uint32_t>(chunks) - whole * k.splits;
    k.c0 = uniform(static_cast<int32_t>(whole * part.split + rest * part.split / static_cast<uint32_t>(k.splits)));
    k.c1 = uniform(static_cast<int32_t>(whole * (part.split + 1) + rest * (part.split + 1) / static_cast<uint32_t>(k.splits)));
    return k;
}

// A chunk's runs of 16 tokens, each in one page: their pages, then where they begin (bytes from the layer's keys or values)
// and which tokens there are, a bit each. WHOLE: pages hold whole chunks, so that one look into the table is enough.
template <int CHUNK, bool WHOLE>
struct Pages {
    int32_t page[WHOLE ? 1 : CHUNK / 16];
};
template <int CHUNK, bool WHOLE>
struct Where {
    size_t base[WHOLE ? 1 : CHUNK / 16];
    uint32_t there[CHUNK / 32];
    // where run `run` begins (selects between the scalars: an index would go through scratch memory)
    __device__ __forceinline__ size_t of_run(int32_t run) const {
        static_assert(!WHOLE, "one run");
        const size_t low = pick(run & 1, base[0], base[1]);
        if constexpr (CHUNK == 32) return low;
        else return pick(run & 2, low, pick(run & 1, base[2], base[3]));
    }
    static __device__ __forceinline__ size_t pick(int32_t second, size_t a, size_t b) {
        const uint32_t low = second ? static_cast<uint32_t>(b) : static_cast<uint32_t>(a), high = second ? static_cast<uint32_t>(b >> 32) : static_cast<uint32_t>(a >> 32);
        return static_cast<size_t>(high) << 32 | low;
    }
};
template <int CHUNK, bool WHOLE>
struct PageReader {
    typedef const __attribute__((address_space(4))) int32_t* table_t;  // (read-only, by uniform indexes)
    table_t table;
    size_t page_bytes, head_bytes;
    int32_t pages, page_shift, n_keys, last_entry, row_bytes;
    __device__ __forceinline__ PageReader(const PagedView& c, const BatchView& b, const Part& part, int32_t keys, int32_t element)
        : table((table_t)(b.tables + static_cast<size_t>(part.sequence) * b.table_stride)), pages(c.pages), page_shift(c.page_shift), n_keys(keys),
          last_entry(keys > 0 ? (keys - 1) >> c.page_shift : 0), row_bytes(c.head_dim * element) {
        head_bytes = (static_cast<size_t>(part.head) << page_shift) * row_bytes;
        page_bytes = (static_cast<size_t>(c.kv_heads) << page_shift) * row_bytes;
    }
    __device__ __forceinline__ Pages<CHUNK, WHOLE> pages_of(int32_t ch) const {
        Pages<CHUNK, WHOLE> p;
#pragma unroll
        for (int h = 0; h < (WHOLE ? 1 : CHUNK / 16); ++h) p.page[h] = table[min((ch * CHUNK + 16 * h) >> page_shift, last_entry)];
        return p;
    }
    __device__ __forceinline__ Where<CHUNK, WHOLE> where_of(int32_t ch, const Pages<CHUNK, WHOLE>& p) const {
        constexpr int RUN = WHOLE ? CHUNK : 16;
        Where<CHUNK, WHOLE> w;
#pragma unroll
        for (int h = 0; h < CHUNK / RUN; ++h) {
            const int32_t x = ch * CHUNK + RUN * h;
            const bool fine = static_cast<uint32_t>(p.page[h]) < static_cast<uint32_t>(pages);
            const size_t page = fine ? p.page[h] : 0;  // (any memory of the pool)
            w.base[h] = page * page_bytes + head_bytes + static_cast<uint32_t>((x & ((1 << page_shift) - 1)) * row_bytes);
            if constexpr (WHOLE) {
                const int32_t left = fine ? n_keys - x : 0;
#pragma unroll
                for (int i = 0; i < CHUNK / 32; ++i) w.there[i] = left >= 32 * i + 32 ? 0xFFFFFFFFu : left <= 32 * i ? 0u : (1u << (left - 32 * i)) - 1u;
            } else {
                const int32_t m = min(max(n_keys - x, 0), 16);
                if (h % 2 == 0) w.there[h / 2] = 0;
                w.there[h / 2] |= (fine ? (1u << m) - 1u : 0u) << (16 * (h % 2));
            }
        }
        return w;
    }
};

// ---- where the parts of a tile meet ----------------------------------------------------------------
// A part's averages and its rows' maxima and sums, written through to memory: the reader may be on another die.
__device__ __forceinline__ void store_average(const __amdgpu_buffer_rsrc_t& averages, int32_t at, f4 y) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, y), averages, at * 4, 0, THROUGH);
}
__device__ __forceinline__ void store_stats(const Args& a, size_t row, float m, float l) {
    const uint64_t both = __builtin_bit_cast(uint32_t, m) | static_cast<uint64_t>(__builtin_bit_cast(uint32_t, l)) << 32;
    __hip_atomic_store(reinterpret_cast<uint64_t*>(a.stats) + row, both, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}
template <int HD, int R>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t averages_of(const Args& a, size_t slot, int32_t slots) {
    return __builtin_amdgcn_make_buffer_rsrc(a.averages + slot * R * HD, 0, slots * R * HD * 4, 0x00020000);
}
constexpr size_t merge_lds(int R, int NW) { return sizeof(float) * (2 * R * MOST_PARTS + R + 4 * 64 * NW); }

// Called by all threads of a workgroup once its part is stored. The last workgroup of the tile to arrive merges the
// parts, in their order, into the context; row_at: where a row of the tile lies there.
template <int HD, int R, int NW, typename ROW>
__device__ __forceinline__ void meet(const Args& a, const Part& part, int32_t splits, int32_t held, float* lds, ROW row_at) {
    constexpr int T = 64 * NW, BATCH = 8;
    const int32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    __shared__ uint32_t arrived;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
        uint32_t* counter = a.counters + part.slot;
        arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        if (arrived == static_cast<uint32_t>(splits) - 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    }
    __syncthreads();
    if (uniform(arrived) != static_cast<uint32_t>(splits) - 1) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    const size_t slot0 = static_cast<size_t>(part.slot) * R;
    float* maxima = lds;                          // [R][splits]: then the parts' weights
    float* sums = maxima + R * MOST_PARTS;     // [R][splits]
    float* total = sums + R * MOST_PARTS;      // [R]
    f4* shares = reinterpret_cast<f4*>(total + R);  // [T]
    const __amdgpu_buffer_rsrc_t all = averages_of<HD, R>(a, part.slot, splits);
    // A thread sums its items (four dims of a row) over the parts; where there are fewer items than threads, phases of
    // threads share an item's parts. Eight loads are in flight while eight others are summed.
    const int32_t items = held * (HD / 4), phases = uniform(max(1, T / items));
    const int32_t phase = phases > 1 ? tid / items : 0, step = phases > 1 ? items : T;
    struct Cursor {
        int32_t item, part;
    };
    Cursor ahead{phases > 1 ? tid % items : tid, phase}, now = ahead;
    u4 v[2][BATCH];
    auto load = [&](u4 (&to)[BATCH]) {  // (past the last item or part: the last, unused)
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            to[u] = __builtin_amdgcn_raw_buffer_load_b128(all, (min(ahead.part, splits - 1) * (R * HD) + 4 * min(ahead.item, items - 1)) * 4, 0, THROUGH);
            ahead.part += phases;
            if (ahead.part >= splits) {
                ahead.item += step;
                ahead.part = phase;
            }
        }
    };
    load(v[0]);
    for (int32_t e = tid; e < held * splits; e += T) {
        const int32_t s = e / held, r = e % held;
        const uint64_t both = __hip_atomic_load(reinterpret_cast<uint64_t*>(a.stats) + slot0 + static_cast<size_t>(s) * R + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        maxima[r * splits + s] = __builtin_bit_cast(float, static_cast<uint32_t>(both));
        sums[r * splits + s] = __builtin_bit_cast(float, static_cast<uint32_t>(both >> 32));
    }
    __syncthreads();
    // a row's weights: as many lanes as hold its parts (128 parts: two a lane)
    int32_t width = 1;
    while (width < splits && width < 64) width <<= 1;
    for (int32_t r0 = wave * (64 / width); r0 < held; r0 += NW * (64 / width)) {
        const int32_t r = r0 + lane / width, at = min(r, held - 1) * splits;
        constexpr int PER = (MOST_PARTS + 63) / 64;
        float ml[PER], ll[PER], mx = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int32_t s = lane % width + 64 * i;
            ml[i] = s < splits ? maxima[at + s] : -INFINITY;
            ll[i] = s < splits ? sums[at + s] : 0.0f;
            mx = fmaxf(mx, ml[i]);
        }
        for (int32_t o = 1; o < width; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const float share = share_of(ml[i], ll[i], mx);
            sum += share;
            ll[i] = weight_of_part(share, ll[i]);
        }
        for (int32_t o = 1; o < width; o <<= 1) sum += __shfl_xor(sum, o);
        if (r < held) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (lane % width + 64 * i < splits) maxima[at + lane % width + 64 * i] = ll[i];
            if (lane % width == 0) total[r] = sum;
        }
    }
    __syncthreads();
    f4 y = {0.0f, 0.0f, 0.0f, 0.0f};
    auto write = [&](int32_t item, const f4& z) {
        const int32_t r = item / (HD / 4), d = 4 * (item % (HD / 4));
        const float inv = total[r] == 0.0f ? 0.0f : 1.0f / total[r];
        *reinterpret_cast<f4*>(a.p.context + row_at(r) + d) = z * inv;
    };
    const int32_t mine = (splits - phase + phases - 1) / phases;  // parts of an item that this thread sums
    const int32_t entries = phases > 1 ? (phase < phases ? mine : 0) : (items - tid + T - 1) / T * splits;
    auto sum_batch = [&](const u4 (&from)[BATCH], int32_t e0) {
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            if (e0 + u >= entries) break;
            const float by = maxima[now.item / (HD / 4) * splits + now.part];
            const f4 z = __builtin_bit_cast(f4, from[u]);
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = fmaf(by, z[i], y[i]);
            now.part += phases;
            if (now.part >= splits) {
                if (phases == 1) {
                    write(now.item, y);
                    y = f4{0.0f, 0.0f, 0.0f, 0.0f};
                }
                now.item += step;
                now.part = phase;
            }
        }
    };
    for (int32_t e0 = 0; e0 < entries; e0 += 2 * BATCH) {
        load(v[1]);
        sum_batch(v[0], e0);
        if (e0 + 2 * BATCH < entries) load(v[0]);
        sum_batch(v[1], e0 + BATCH);
    }
    if (phases > 1) {
        shares[tid] = y;
        __syncthreads();
        if (tid < items) {
            for (int32_t p = 1; p < phases; ++p) y += shares[tid + p * items];
            write(tid, y);
        }
    }
}

// The same as a launch of its own, for tiles of many rows, whose merge is more than one workgroup's work: the workgroups of a
// slot take their shares of the tile's rows (two a tile of 128: four, with as many empty ones beside them, cost every call 1 us).
constexpr int merge_shares(int R) { return R / 64; }
template <int HD, int R, int LEAST, int CHUNK>
__global__ void __launch_bounds__(256) merge_kernel(Args a) {
    __shared__ float maxima[64 + MOST_PARTS], sums[64 + MOST_PARTS], weights[64 + MOST_PARTS];
    Part part;
    if (!find_part<R, LEAST, CHUNK, true>(a, blockIdx.x, part)) return;
    part.make_uniform();
    const int32_t H = a.p.num_heads, G = H / a.p.c.kv_heads, row0 = part.tile * R, held = min(R, part.n * G - row0);
    const Keys keys = keys_of<R, CHUNK>(a, part, held);
    const int32_t splits = keys.splits, tid = threadIdx.x;
    if (splits == 1) return;
    const int32_t shares = part.splits * merge_shares(R), share = part.split * merge_shares(R) + blockIdx.y;
    const int32_t r0 = uniform(held * share / shares), rows = uniform(held * (share + 1) / shares) - r0;
    if (rows == 0) return;
    const size_t slot0 = static_cast<size_t>(part.slot) * R;
    // (fewer than held / shares + 1 rows, of at most part.splits parts: 64 + MOST_PARTS weights at most)
    for (int32_t e = tid; e < rows * splits; e += 256) {
        const int32_t s = e / rows, r = e % rows;
        const float2 both = reinterpret_cast<const float2*>(a.stats)[slot0 + static_cast<size_t>(s) * R + r0 + r];
        maxima[r * splits + s] = both.x;
        sums[r * splits + s] = both.y;
    }
    __syncthreads();
    for (int32_t e = tid; e < rows * splits; e += 256) {  // a part's share of its row, over all of them
        const int32_t r = e / splits;
        float mx = -INFINITY, sum = 0.0f;
        for (int32_t s = 0; s < splits; ++s) mx = fmaxf(mx, maxima[r * splits + s]);
        for (int32_t s = 0; s < splits; ++s) sum += share_of(maxima[r * splits + s], sums[r * splits + s], mx);
        weights[e] = sum == 0.0f ? 0.0f : weight_of_part(share_of(maxima[e], sums[e], mx) / sum, sums[e]);
    }
    __syncthreads();
    constexpr int BATCH = 8;
    for (int32_t item = tid; item < rows * (HD / 4); item += 256) {
        const int32_t r = item / (HD / 4), d = 4 * (item % (HD / 4));
        const float* from = a.averages + (slot0 + r0 + r) * HD + d;
        f4 y = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int32_t s0 = 0; s0 < splits; s0 += BATCH) {
            f4 v[BATCH];
#pragma unroll
            for (int u = 0; u < BATCH; ++u) v[u] = *reinterpret_cast<const f4*>(from + static_cast<size_t>(min(s0 + u, splits - 1)) * (R * HD));
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const float by = s0 + u < splits ? weights[r * splits + s0 + u] : 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = s0 + u < splits ? fmaf(by, v[u][i], y[i]) : y[i];
            }
        }
        const int32_t t = (row0 + r0 + r) / G;
        *reinterpret_cast<f4*>(a.p.context + (static_cast<size_t>(part.first + t) * H + part.head * G + (row0 + r0 + r - t * G)) * HD + d) = y;
    }
}

// ---- few rows, and few keys --------------------------------------------------------------------------
// R = 16 rows a workgroup on 16x16x32. Its four waves take the part's chunks of 32 keys in turn, straight from memory into registers,
// no LDS and no barrier in the loop: a lane loads its dims of the tokens whose weights it will hold, and turns them there. The
// next chunk's keys are on their way while a chunk's weights and output are formed, its values while the next scores are.
// Registers: 106 scalars are too few for what the loop and its surroundings need; 6 to 132 of them (of 256 dims up to 264) wait in vector registers, and
// a chunk reads up to four back. From 256 dims on (fp32: 128) sums lie in accumulators and move 88 to 263 times a chunk.
// STEP: the tokens are rotated, appended and attended to in this launch: every workgroup makes its own rotated query, key and
// value, the last part's also writes them to the cache, and its wave with the token's chunk takes them from LDS.
template <int FMT, int HD>
struct Shape {
    static constexpr int R = 16, NW = 4, LEAST = NW;          // a part has a chunk for each wave
    static constexpr int QS = HD / 32;                        // steps of a score
    static constexpr int DB = HD / 16;                        // dim blocks of the output: consecutive dims of a lane
    static constexpr int KW = 8 * Format<FMT>::E / 4;         // dwords of a key tile's step
    static constexpr int VW = DB * Format<FMT>::E / 4;        // dwords of a token's dims
    static constexpr bool QREG = HD < 256;                    // a row's operands stay in registers
};

// What a step's workgroups share: the rotation, and the new token as the cache holds it.
template <int HD, bool STEP>
struct StepShared {
    __attribute__((aligned(16))) float cosines[HD / 2], sines[HD / 2];
    __attribute__((aligned(16))) uint8_t key[4 * HD], value[4 * HD];
};
template <int HD>
struct StepShared<HD, false> {};

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        if constexpr (N >= 4) {
            const u4 v = *reinterpret_cast<const u4*>(p + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[i + e] = v[e];
        } else if constexpr (N == 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x;
            w[1] = v.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        }
    }
}

template <int FMT>
__device__ __forceinline__ bool any_not_finite(uint32_t w) {
    if constexpr (FMT == KT_PAGED_F32) return (w & 0x7F800000u) == 0x7F800000u;
    constexpr uint32_t x = FMT == KT_PAGED_F16 ? 0x7C00u : 0x7F80u;
    return (w & x) == x || (w >> 16 & x) == x;
}
template <int FMT>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {
    if constexpr (FMT == KT_PAGED_F32) return (w & 0x7F800000u) == 0x7F800000u ? 0u : w;
    constexpr uint32_t x = FMT == KT_PAGED_F16 ? 0x7C00u : 0x7F80u;
    return ((w & x) == x ? 0u : w & 0xFFFFu) | ((w >> 16 & x) == x ? 0u : w & 0xFFFF0000u);
}

// ---- values that are not finite --------------------------------------------------------------------
// The weight of a token that a row sees is above zero, so an infinite value makes the row's average of its dim infinite
// (infinities of both signs and NaNs: NaN), whatever the weight. The products do not give that: a weight's lower parts
// are zero or of the other sign, fp32 values' parts are NaN, weights and rescaled sums get too small for fp32. So the loops only find
// out that something is not finite: chunks that not all rows see whole come without such values and leave a flag, other chunks'
// make sums that are not finite. Then a wave looks at all values that its rows see: 1 bit a number of a lane. (An infinity that all rows
// see: a prompt of 1024 in fp16 at 64 dims 268 us for 27, a step of eight sequences of 2000 in bf16 at 128 dims 44 for 31.)
struct Odd {
    uint64_t up, down;  // infinities above and below zero; of a NaN both
};
// Tokens that a lane loads its numbers of together.
template <int FMT, int DB>
constexpr int together() {
    return std::clamp(64 / (DB * element_bytes(FMT)), 1, 8);
}
// The lane's numbers of N tokens: DB groups of four, `stride` elements apart, from at(u) on; seen: a bit a token.
template <int FMT, int DB, int N, typename AT>
__device__ __forceinline__ void look_at(Odd& odd, uint32_t seen, AT at, int32_t stride) {
    constexpr int E = element_bytes(FMT);
    uint32_t w[N][DB][E];
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
        for (int i = 0; i < DB; ++i) load_words(at(u) + i * stride * E, w[u][i]);
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
        for (int i = 0; i < DB; ++i) {
            bool any = false;
#pragma unroll
            for (int j = 0; j < E; ++j) any |= any_not_finite<FMT>(w[u][i][j]);
            if (!any || !(seen >> u & 1)) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v;
                if constexpr (FMT == KT_PAGED_F32) v = __builtin_bit_cast(float, w[u][i][e]);
                else if constexpr (FMT == KT_PAGED_F16) v = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[u][i][e / 2] >> 16 * (e % 2))));
                else v = __builtin_bit_cast(float, w[u][i][e / 2] >> 16 * (e % 2) << 16);
                if (fabsf(v) < INFINITY) continue;
                odd.up |= static_cast<uint64_t>(!(v < 0.0f)) << (4 * i + e);
                odd.down |= static_cast<uint64_t>(!(v > 0.0f)) << (4 * i + e);
            }
        }
}
// What such values make of number i of the lane.
__device__ __forceinline__ float or_odd(const Odd& odd, int i, float x) {
    const bool up = odd.up >> i & 1, down = odd.down >> i & 1;
    return up ? (down ? __builtin_nanf("") : INFINITY) : down ? -INFINITY : x;
}

template <int FMT, int HD, bool STEP>
__global__ void __launch_bounds__((64 * Shape<FMT, HD>::NW), (HD == 256 || (FMT == KT_PAGED_F32 && HD == 128) ? 1 : 2)) attention_kernel(Args a) {
    using F = Format<FMT>;
    using X = Shape<FMT, HD>;
    using op = typename F::op;
    constexpr int R = X::R, NW = X::NW;
    constexpr int LR = HD + 4;  // padded row of the waves' averages
    constexpr int QR = HD + 8;  // padded row of a query's parts
    extern __shared__ __attribute__((aligned(16))) float lds[];
    float* avg = lds;               // [NW][R][LR]
    float* ms = avg + NW * R * LR;  // [NW][R]
    float* ls = ms + NW * R;        // [NW][R]
    __shared__ float fr_s[R];
    __shared__ StepShared<HD, STEP> sh;
    const PagedView& c = a.p.c;
    const BatchView& b = a.p.b;
    const int32_t tid = threadIdx.x, lane = tid & 63;
    const int32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int32_t col = lane & 15, grp = lane >> 4;
    const int32_t H = a.p.num_heads, G = H / c.kv_heads;
    Part part;
    if (!find_part<R, X::LEAST, CHUNK>(a, blockIdx.x, part)) return;
    part.make_uniform();
    const int32_t g = part.head, row0 = part.tile * R, held = min(R, part.n * G - row0);  // rows of this tile
    // where row r of the tile lies in q and context
    auto row_at = [&](int32_t r) {
        const int32_t t = (row0 + r) / G;
        return (static_cast<size_t>(part.first + t) * H + g * G + (row0 + r - t * G)) * HD;
    };

    // The rows' queries, sixteen lanes to a row (four dims each, or 64 apart; for the rotation those of the dims'
    // pairs, too).
    constexpr int DL = HD / 64 > 0 ? HD / 64 : 1, HALF = HD / 2;
    const int32_t lr = lane >> 4, lc = lane & 15;
    static_assert(R == 4 * NW, "a wave brings four rows");
    f4 qv[DL], qo[STEP ? DL : 1];
    {
        const float* src = a.p.q + row_at(min(4 * wave + lr, held - 1));
#pragma unroll
        for (int u = 0; u < DL; ++u) {
            const int32_t d = (4 * lc + 64 * u) % HD;
            qv[u] = *reinterpret_cast<const f4*>(src + d);
            if constexpr (STEP) qo[u] = *reinterpret_cast<const f4*>(src + (d + HALF) % HD);
        }
    }
    // a step: the new token's pairs, those of the key in threads 0 .. 127, of the value in the next 128
    const bool on = STEP && tid < 256 && (tid & 127) < HALF;
    float x1 = 0.0f, x2 = 0.0f, ifr = 0.0f;
    int32_t pos = 0;
    if constexpr (STEP) {
        pos = part.length + (b.depths ? b.depths[part.first] : 0);
        if (on) {
            const float* src = (tid < 128 ? a.k_new : a.v_new) + (static_cast<size_t>(part.first) * c.kv_heads + g) * HD + (tid & 127);
            x1 = src[0];
            x2 = src[HALF];
            ifr = a.p.inv_freq[tid & 127];
        }
    }

    const Keys keys = keys_of<R, CHUNK>(a, part, held);
    if (part.split >= keys.splits) return;
    const int32_t splits = keys.splits, c0 = keys.c0, c1 = keys.c1, n_all = keys.n_all;
    const int64_t new_first = part.length;
    const PageReader<CHUNK, false> reader(c, b, part, keys.n_keys, F::E);

    uint32_t kr[2][X::QS][X::KW], vr[8][X::VW];
    auto load_keys = [&](const Where<CHUNK, false>& w) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint8_t* p = c.keys + w.base[t] + (col * HD + 8 * grp) * F::E;
#pragma unroll
            for (int s = 0; s < X::QS; ++s) load_words(p + 32 * s * F::E, kr[t][s]);
        }
    };
    // the token of a lane's value (or weight) e
    auto token_of = [&](int e) { return 16 * (e >> 2) + 4 * grp + (e & 3); };
    auto load_values = [&](const Where<CHUNK, false>& w) {
#pragma unroll
        for (int e = 0; e < 8; ++e) load_words(c.values + w.base[e >> 2] + ((token_of(e) & 15) * HD + col * X::DB) * F::E, vr[e]);
    };
    // a step's token in its chunk's registers, whatever the loads saw
    const bool holder = STEP && part.split == splits - 1;
    auto patch = [&]() {
        if constexpr (STEP) {
            const int32_t at = part.length & (CHUNK - 1);
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (16 * t + col == at)
#pragma unroll
                    for (int s = 0; s < X::QS; ++s) load_words(sh.key + (32 * s + 8 * grp) * F::E, kr[t][s]);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (token_of(e) == at) load_words(sh.value + col * X::DB * F::E, vr[e]);
        }
    };
    int32_t ch = c0 + wave;
    Where<CHUNK, false> here{};
    Pages<CHUNK, false> pages{};
    if (ch < c1) {
        here = reader.where_of(ch, reader.pages_of(ch));
        load_keys(here);
        load_values(here);
        pages = reader.pages_of(min(ch + NW, c1 - 1));
    }
    if constexpr (STEP) {
        if (on) {  // cosines by the key's threads, sines by the value's
            if (tid < 128) sh.cosines[tid] = rope_cos(pos, ifr);
            else sh.sines[tid - 128] = rope_sin(pos, ifr);
        }
        __syncthreads();
    }

    // the rows' parts through LDS
    typedef typename std::conditional<FMT == KT_PAGED_F16, _Float16, __bf16>::type element;
    element* qs = reinterpret_cast<element*>(lds);  // [QP][R][QR]
    if (4 * wave < held) {
        const int32_t r = 4 * wave + lr;
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
                    rope_apply(upper ? qo[u][e] : qv[u][e], upper ? qv[u][e] : qo[u][e], cf[e], sf[e], y1, y2);
                    qv[u][e] = upper ? y2 : y1;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, magnitude(qv[u][e]));
        }
        int32_t up = 0;
        if constexpr (FMT == KT_PAGED_F16) {
            // the row scaled by a power of two to 2^13 .. 2^14 (bits below an infinity's, whose order is the floats')
            float most = __builtin_bit_cast(float, min(top, 0x7F7FFFFFu));
            most = fmaxf(most, dpp_move<0xB1>(most));
            most = fmaxf(most, dpp_move<0x4E>(most));
            most = fmaxf(most, dpp_move<0x141>(most));
            most = fmaxf(most, dpp_move<0x140>(most));
            up = 13 - max(static_cast<int32_t>(__builtin_bit_cast(uint32_t, most) >> 23) - 127, -100);
        }
        if (r < held) {
#pragma unroll
            for (int u = 0; u < DL; ++u) {
                if (4 * lc + 64 * u >= HD) continue;
                float rest[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) rest[e] = FMT == KT_PAGED_F16 ? ldexpf(qv[u][e], up) : qv[u][e];
#pragma unroll
                for (int w = 0; w < F::QP; ++w) {
                    element part4[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        part4[e] = static_cast<element>(rest[e]);
                        rest[e] -= static_cast<float>(part4[e]);
                    }
                    __builtin_memcpy(__builtin_assume_aligned(qs + (w * R + r) * QR + 4 * lc + 64 * u, 8), part4, sizeof(part4));
                }
            }
            if (lc == 0) fr_s[r] = ldexpf(a.p.scale * 1.4426950408889634f, -up);
        }
    }
    if constexpr (STEP) {
        if (on) {  // the new token as the cache holds it
            const int32_t i = tid & 127;
            if (tid < 128) {
                const float k1 = x1, k2 = x2;
                rope_apply(k1, k2, sh.cosines[i], sh.sines[i], x1, x2);
            }
            uint8_t* mine = tid < 128 ? sh.key : sh.value;
            store_element<FMT>(mine, i, x1);
            store_element<FMT>(mine, i + HALF, x2);
            if (holder) {
                const int64_t at = place_of(c, b, part.sequence, part.length, g);
                if (at >= 0) {
                    store_element<FMT>(tid < 128 ? c.keys : c.values, at + i, x1);
                    store_element<FMT>(tid < 128 ? c.keys : c.values, at + i + HALF, x2);
                }
            }
        }
    }
    __syncthreads();
    op qreg[X::QREG ? X::QS : 1][F::QP];
    const int32_t own_row = min(col, held - 1), token = (row0 + own_row) / G;  // (columns past the rows repeat the last)
    const float fr = fr_s[own_row];
    auto query = [&](int s, op (&q)[F::QP]) {
#pragma unroll
        for (int w = 0; w < F::QP; ++w) q[w] = *reinterpret_cast<const op*>(qs + (w * R + own_row) * QR + 8 * grp + 32 * s);
    };
    if constexpr (X::QREG) {
#pragma unroll
        for (int s = 0; s < X::QS; ++s) query(s, qreg[s]);
    }
    if constexpr (STEP) {
        if (holder && ch < c1 && ch == part.length / CHUNK) patch();
    }

    f4 o[X::DB];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int db = 0; db < X::DB; ++db) o[db] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    // the operands of dim block db: the tokens' elements of the lane's dim
    auto value_operand = [&](int db, op (&v)[F::KP]) {
        if constexpr (FMT == KT_PAGED_F32) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = vr[e][db];
            to_operands<FMT>(w, v);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(vr[2 * i + 1][db / 2], vr[2 * i][db / 2], db % 2 ? 0x07060302u : 0x05040100u);
            to_operands<FMT>(w, v);
        }
    };
    bool not_finite = false;  // some values were left out
    // (masked: not every row sees the chunk whole)
    auto attend_chunk = [&](bool masked) {
        const Where<CHUNK, false> now = here;
        f4 sc[2] = {f4{0.0f, 0.0f, 0.0f, 0.0f}, f4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int s = 0; s < X::QS; ++s) {
            op k[2][F::KP];
#pragma unroll
            for (int t = 0; t < 2; ++t) to_operands<FMT>(kr[t][s], k[t]);
            if constexpr (X::QREG) {
#pragma unroll
                for (int t = 0; t < 2; ++t) sc[t] = products(k[t], qreg[s], sc[t]);
            } else {
                op q[F::QP];
                query(s, q);
#pragma unroll
                for (int t = 0; t < 2; ++t) sc[t] = products(k[t], q, sc[t]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // (loads ahead of their registers' last use would cost others)
        const int32_t next = min(ch + NW, c1 - 1);  // (past the end the last chunk again, unused)
        here = reader.where_of(next, pages);
        load_keys(here);
        pages = reader.pages_of(min(ch + 2 * NW, c1 - 1));
        __builtin_amdgcn_sched_barrier(0);
        op p[F::QP];
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = sc[i >> 2][i & 3];
        if (masked) {  // (a score of -infinity has no weight)
            const uint32_t vis = seen_bits(b, part.first, token, new_first, ch * CHUNK, now.there[0]);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!(vis >> token_of(i) & 1)) x[i] = -INFINITY;
        }
        to_weights<FMT>(x, fr, m, l, [&](float alpha) {
#pragma unroll
            for (int db = 0; db < X::DB; ++db) o[db] *= alpha;
        });
        split_weights(x, p);
        if (__builtin_expect(masked, 0)) {  // (as likely as not 1 to 4% of a step more)
            // values of tokens that are not there count for nothing, nor does here what is not finite
            bool odd = false;
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int w = 0; w < X::VW; ++w) {
                    if (!(now.there[0] >> token_of(e) & 1)) vr[e][w] = 0;
                    odd |= any_not_finite<FMT>(vr[e][w]);
                }
            if (__ballot(odd)) {
                not_finite = true;
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int w = 0; w < X::VW; ++w) vr[e][w] = finite_only<FMT>(vr[e][w]);
            }
        }
#pragma unroll
        for (int db = 0; db < X::DB; ++db) {
            op v[F::KP];
            value_operand(db, v);
            o[db] = products(v, p, o[db]);
        }
        __builtin_amdgcn_sched_barrier(0);  // (loads ahead of their registers' last use would cost others)
        load_values(here);
        if constexpr (STEP) {
            if (holder && next == part.length / CHUNK) patch();
        }
    };
    for (; ch < c1; ch += NW) {
        attend_chunk(ch * CHUNK + CHUNK > n_all || here.there[0] != 0xFFFFFFFFu);
    }
    f4 none = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int db = 0; db < X::DB; ++db) none += o[db] * 0.0f;  // (NaN of what is not finite)
    if (not_finite || __ballot(!(none[0] + none[1] + none[2] + none[3] == 0.0f))) {
        Odd odd{0, 0};
        for (ch = c0 + wave; ch < c1; ch += NW) {
            here = reader.where_of(ch, reader.pages_of(ch));
            uint32_t vis = seen_bits(b, part.first, token, new_first, ch * CHUNK, here.there[0]);
            if constexpr (STEP) {
                const uint32_t own = holder && ch == part.length / CHUNK ? 1u << (part.length & (CHUNK - 1)) : 0u;  // (the new token is in LDS)
                if (vis & own) look_at<FMT, X::DB, 1>(odd, 1, [&](int) { return sh.value + 4 * grp * X::DB * F::E; }, 4);
                vis &= ~own;
            }
            constexpr int N = together<FMT, X::DB>();
            for (int32_t tok = 0; tok < CHUNK; tok += N) {
                const uint8_t* rows = c.values + (tok < 16 ? here.base[0] : here.base[1]) + ((tok & 15) * HD + 4 * grp * X::DB) * F::E;
                look_at<FMT, X::DB, N>(odd, vis >> tok, [&](int u) { return rows + u * HD * F::E; }, 4);
            }
        }
#pragma unroll
        for (int i = 0; i < HD / 4; ++i) o[i % X::DB][i / X::DB] = or_odd(odd, i, o[i % X::DB][i / X::DB]);
    }

    // each wave's averages, maxima and sums, then all waves' through LDS
    const int32_t used = min(NW, c1 - c0);  // waves with keys
    __syncthreads();                        // (the queries' parts are read)
    if (wave < used) {
        l = column_sum(l);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (col < held) {
            float* row = avg + (wave * R + col) * LR;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int db = 0; db < X::DB; ++db) row[(4 * grp + e) * X::DB + db] = o[db][e] * inv;
            if (grp == 0) {
                ms[wave * R + col] = m;
                ls[wave * R + col] = l;
            }
        }
    }
    __syncthreads();
    const size_t at_slot = static_cast<size_t>(part.slot + part.split) * R;
    const __amdgpu_buffer_rsrc_t averages = averages_of<HD, R>(a, part.slot + part.split, 1);
    for (int32_t e = tid; e < held * (HD / 4); e += 64 * NW) {  // (every thread weighs its row's parts itself: no further barrier)
        const int32_t r = e / (HD / 4), d = 4 * (e % (HD / 4));
        float mx = -INFINITY, sum = 0.0f;
        f4 y = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int32_t w = 0; w < used; ++w) mx = fmaxf(mx, ms[w * R + r]);
        for (int32_t w = 0; w < used; ++w) {
            const float by = weight_of_part(share_of(ms[w * R + r], ls[w * R + r], mx), ls[w * R + r]);
            const f4 v = *reinterpret_cast<const f4*>(avg + (w * R + r) * LR + d);
            sum += by;
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = fmaf(by, v[i], y[i]);
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] *= inv;
        if (splits == 1) {
            *reinterpret_cast<f4*>(a.p.context + row_at(r) + d) = y;
        } else {
            store_average(averages, r * HD + d, y);
            if (d == 0) store_stats(a, at_slot + r, mx, sum);
        }
    }
    if (splits == 1) return;
    meet<HD, R, NW>(a, part, splits, held, lds, row_at);
}

// ---- many rows ---------------------------------------------------------------------------------------
// 16 rows a wave on 16x16x32. The workgroup's threads load a chunk of keys ahead and lay it out in LDS, where all its waves
// read it: the keys as rows, the values as dims with their tokens in the order of the operands; fp32 ones split into their
// parts once for all waves. Queries stay in registers; operands of the next step are on their way from LDS while a step's products run.
template <int FMT, int HD, int WAVES>
struct Tile {
    static constexpr int NW = WAVES, R = 16 * NW, THREADS = 64 * NW;
    // waves a SIMD that leave a wave the registers it needs (of 256 dims with two: 352 bytes and more in scratch memory)
    static constexpr int MW = NW == 8 ? 2 : HD == 256 ? 1 : HD <= 64 && FMT != KT_PAGED_F32 ? 3 : 2;
    static constexpr int KP = Format<FMT>::KP, QP = Format<FMT>::QP, E = Format<FMT>::E;
    // keys of a chunk: half the barriers with 64 (against 32, pages of 64: at 64 dims a prompt of 1024 in fp16 23 us for 28, of 2048 in fp32 98 for
    // 110, in bf16 58 for 63; at 128 dims in fp16 79 for 86), where the registers and LDS allow it
    static constexpr int CH = HD == 256 || (FMT == KT_PAGED_F32 && HD == 128) ? 32 : 64, SETS = CH / 32;
    static constexpr int QS = HD / 32, DB = HD / 16;
    static constexpr int KR = HD + 8, VR = CH + 8;  // padded rows: of a key, of a dim (2-byte elements)
    static constexpr int KSIZE = CH * KR, VSIZE = HD * VR, SIZE = KP * (KSIZE + VSIZE);
    static constexpr int BUFFERS = 2 * SIZE * 2 <= (150 << 10) / (4 * MW / NW) ? 2 : 1;
    static constexpr int PIECES = HD * E / 16;  // 16-byte pieces of a key
    static constexpr int KN = (CH * PIECES + THREADS - 1) / THREADS;
    static constexpr int VN = (CH / 4 * (HD / 4) + THREADS - 1) / THREADS;  // 4 tokens x 4 dims
    static constexpr size_t LDS = size_t{2} * SIZE * BUFFERS;
    static constexpr int LEAST = 128 / CH;
    static constexpr int TARGET = NW == 4 && HD < 256 ? 2 : 1;  // workgroups a CU among which the launch's chunks are shared out
    static constexpr int VGROUP = FMT != KT_PAGED_F32 ? 4 : HD == 128 ? 1 : 2;  // (fp32 at 128 dims: a prompt of 2048 171 us with one, 176 with two)
};

template <int FMT, int HD, int WAVES, bool WHOLE>
__global__ void __launch_bounds__((Tile<FMT, HD, WAVES>::THREADS), (Tile<FMT, HD, WAVES>::MW)) tile_kernel(Args a) {
    using F = Format<FMT>;
    using X = Tile<FMT, HD, WAVES>;
    using op = typename F::op;
    constexpr int R = X::R, E = F::E, CH = X::CH;
    typedef typename std::conditional<FMT == KT_PAGED_F16, _Float16, __bf16>::type element;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    __shared__ int32_t not_finite;  // some values were left out
    const PagedView& c = a.p.c;
    const BatchView& b = a.p.b;
    const int32_t tid = threadIdx.x, lane = tid & 63;
    const int32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int32_t col = lane & 15, grp = lane >> 4;
    const int32_t H = a.p.num_heads, G = H / c.kv_heads;
    Part part;
    if (!find_part<R, X::LEAST, CH>(a, blockIdx.x, part)) return;
    part.make_uniform();
    const int32_t g = part.head, row0 = part.tile * R, held = min(R, part.n * G - row0);
    auto row_at = [&](int32_t r) {
        const int32_t t = (row0 + r) / G;
        return (static_cast<size_t>(part.first + t) * H + g * G + (row0 + r - t * G)) * HD;
    };
    const Keys keys = keys_of<R, CH>(a, part, held);
    if (part.split >= keys.splits) return;
    const int32_t c0 = keys.c0, c1 = keys.c1;
    const PageReader<CH, WHOLE> reader(c, b, part, keys.n_keys, E);
    if (tid == 0) not_finite = 0;

    // the chunk ahead: a thread's pieces of keys, and its four tokens of four dims
    u4 kr[X::KN];
    uint32_t vr[X::VN][4][E];
    auto key_item = [&](int i, int32_t& key, int32_t& piece) {
        const int32_t e = tid + i * X::THREADS;
        key = e / X::PIECES;
        piece = e % X::PIECES;
        return CH * X::PIECES % X::THREADS == 0 || e < CH * X::PIECES;
    };
    auto value_item = [&](int i, int32_t& quad, int32_t& dims) {
        const int32_t e = tid + i * X::THREADS;
        quad = e / (HD / 4);
        dims = 4 * (e % (HD / 4));
        return CH / 4 * (HD / 4) % X::THREADS == 0 || e < CH / 4 * (HD / 4);
    };
    auto load_chunk = [&](const Where<CH, WHOLE>& w) {
#pragma unroll
        for (int i = 0; i < X::KN; ++i) {
            int32_t key, piece;
            if (!key_item(i, key, piece)) break;
            if constexpr (WHOLE) kr[i] = *reinterpret_cast<const u4*>(c.keys + w.base[0] + static_cast<uint32_t>(key * HD * E + 16 * piece));
            else kr[i] = *reinterpret_cast<const u4*>(c.keys + w.of_run(uniform(key >> 4)) + static_cast<uint32_t>((key & 15) * HD * E + 16 * piece));
        }
#pragma unroll
        for (int i = 0; i < X::VN; ++i) {
            int32_t quad, dims;
            if (!value_item(i, quad, dims)) break;
            const uint8_t* p;
            if constexpr (WHOLE) p = c.values + w.base[0] + static_cast<uint32_t>((4 * quad * HD + dims) * E);
            else p = c.values + w.of_run(HD >= 64 ? uniform(quad >> 2) : quad >> 2) + static_cast<uint32_t>(((4 * quad & 15) * HD + dims) * E);
#pragma unroll
            for (int j = 0; j < 4; ++j) load_words(p + j * HD * E, vr[i][j]);
        }
    };
    auto all_there = [&](const Where<CH, WHOLE>& w) { return w.there[0] == 0xFFFFFFFFu && w.there[X::SETS - 1] == 0xFFFFFFFFu; };
    // whether every row of the tile sees the chunk whole
    auto whole = [&](int32_t ch, const Where<CH, WHOLE>& w) { return ch * CH + CH <= keys.n_all && all_there(w); };
    // where the 8 tokens of (set of 32, lane group) lie among a dim's: blocks turned by the dim's block of 16, so that the lanes that write
    // every fourth dim meet different banks, and those that read a block's dims still do
    auto block_of = [&](int32_t block, int32_t dim) { return 8 * (block ^ ((dim >> 4) & (CH / 8 - 1))); };
    auto store_chunk = [&](int32_t ch, const Where<CH, WHOLE>& where) {
        element* kl = reinterpret_cast<element*>(lds) + (X::BUFFERS == 2 ? (ch & 1) * X::SIZE : 0);
        element* vl = kl + X::KP * X::KSIZE;
        // four numbers' parts
        auto store_parts = [&](float (&rest)[4], element* to, int32_t size) {
#pragma unroll
            for (int w = 0; w < 3; ++w) {
                const uint32_t low = nearest_halves(rest[0], rest[1]), high = nearest_halves(rest[2], rest[3]);
                *reinterpret_cast<uint2*>(to + w * size) = make_uint2(low, high);
                rest[0] -= __builtin_bit_cast(float, low << 16);
                rest[1] -= __builtin_bit_cast(float, low & 0xFFFF0000u);
                rest[2] -= __builtin_bit_cast(float, high << 16);
                rest[3] -= __builtin_bit_cast(float, high & 0xFFFF0000u);
            }
        };
#pragma unroll
        for (int i = 0; i < X::KN; ++i) {
            int32_t key, piece;
            if (!key_item(i, key, piece)) break;
            if constexpr (FMT == KT_PAGED_F32) {
                float rest[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w = kr[i][e];
                    rest[e] = __builtin_bit_cast(float, w);
                }
                store_parts(rest, kl + key * X::KR + 4 * piece, X::KSIZE);
            } else {
                *reinterpret_cast<u4*>(kl + key * X::KR + 8 * piece) = kr[i];
            }
        }
#pragma unroll
        for (int i = 0; i < X::VN; ++i) {
            int32_t quad, dims;
            if (!value_item(i, quad, dims)) break;
            if (!whole(ch, where)) {  // values of tokens that are not there count for nothing, nor does here what is not finite
                const uint32_t there = (quad < 8 ? where.there[0] : where.there[X::SETS - 1]) >> (4 * quad & 31);
                bool odd = false;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int w = 0; w < E; ++w) {
                        if (!(there >> j & 1)) vr[i][j][w] = 0;
                        odd |= any_not_finite<FMT>(vr[i][j][w]);
                        vr[i][j][w] = finite_only<FMT>(vr[i][j][w]);
                    }
                if (odd) not_finite = 1;
            }
            const int32_t block = quad >> 3 << 2 | (quad & 3), at = block_of(block, dims) + (quad & 4);  // (tokens 16 t + 4 grp + i of a set: 8 grp + 4 t + i)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                element* to = vl + (dims + d) * X::VR + at;
                if constexpr (FMT == KT_PAGED_F32) {
                    float rest[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) rest[j] = __builtin_bit_cast(float, vr[i][j][d]);
                    store_parts(rest, to, X::VSIZE);
                } else {
                    const uint32_t pick = d % 2 ? 0x07060302u : 0x05040100u;
                    *reinterpret_cast<uint2*>(to) = make_uint2(__builtin_amdgcn_perm(vr[i][1][d / 2], vr[i][0][d / 2], pick), __builtin_amdgcn_perm(vr[i][3][d / 2], vr[i][2][d / 2], pick));
                }
            }
        }
    };

    Where<CH, WHOLE> next{};
    Pages<CH, WHOLE> pages{};
    if (c0 < c1) {
        next = reader.where_of(c0, reader.pages_of(c0));
        load_chunk(next);
        pages = reader.pages_of(min(c0 + 1, c1 - 1));
    }
    // the wave's queries: a lane's dims of its row, as operands
    const bool active = 16 * wave < held;  // waves with rows
    const int32_t r = min(16 * wave + col, held - 1), token = (row0 + r) / G;
    op q[X::QS][F::QP];
    float f = a.p.scale * 1.4426950408889634f;
    if (active) {
        const float* src = a.p.q + row_at(r) + 8 * grp;
        float x[X::QS][8];
#pragma unroll
        for (int s = 0; s < X::QS; ++s) {
            const f4 low = *reinterpret_cast<const f4*>(src + 32 * s), high = *reinterpret_cast<const f4*>(src + 32 * s + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[s][e] = low[e];
                x[s][4 + e] = high[e];
            }
        }
        if constexpr (FMT == KT_PAGED_F16) {
            // the row scaled by a power of two to 2^13 .. 2^14 (bits below an infinity's, whose order is the floats')
            uint32_t top = 0;
#pragma unroll
            for (int s = 0; s < X::QS; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = max(top, magnitude(x[s][e]));
            const float most = column_max(__builtin_bit_cast(float, min(top, 0x7F7FFFFFu)));
            const int32_t up = 13 - max(static_cast<int32_t>(magnitude(most) >> 23) - 127, -100);
#pragma unroll
            for (int s = 0; s < X::QS; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[s][e] = ldexpf(x[s][e], up);
            f = ldexpf(f, -up);
        }
#pragma unroll
        for (int s = 0; s < X::QS; ++s) split_query(x[s], q[s]);
    }
    __syncthreads();  // (not_finite)
    if (c0 < c1) store_chunk(c0, next);

    constexpr int VG = X::DB < X::VGROUP ? X::DB : X::VGROUP, GROUPS = X::DB / VG;  // dim blocks whose operands are loaded together
    f4 o[GROUPS][VG];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int db = 0; db < X::DB; ++db)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[db / VG][db % VG][e] = 0.0f;
    // the token of a lane's score i in its set of 32
    auto token_of = [&](int i) { return 16 * (i >> 2) + 4 * grp + (i & 3); };
    const int32_t first_token = uniform((row0 + 16 * wave) / G), last_token = uniform((row0 + min(16 * wave + 15, held - 1)) / G);
    // what the wave's rows see: tokens below all of them, from none on nothing
    const int64_t see_all = b.masks ? static_cast<int64_t>(part.length) : static_cast<int64_t>(part.length) + first_token + 1;
    const int64_t see_none = b.masks ? INT64_MAX - CH : static_cast<int64_t>(part.length) + last_token + 1;
    const int32_t all_upto = uniform(static_cast<int32_t>(min(max(see_all, int64_t{0}) / CH, int64_t{c1})));              // chunks before which all is seen
    const int32_t none_from = uniform(active ? static_cast<int32_t>(min((max(see_none, int64_t{0}) + CH - 1) / CH, int64_t{c1})) : 0);  // and from which nothing is
    auto attend_chunk = [&](bool masked, int32_t ch, const Where<CH, WHOLE>& where) {
        const element* kl = reinterpret_cast<const element*>(lds) + (X::BUFFERS == 2 ? (ch & 1) * X::SIZE : 0);
        const element* vl = kl + X::KP * X::KSIZE;
        // (operands of the next step are on their way from LDS while a step's products run)
        constexpr int T = 2 * X::SETS;
        op k[2][T][F::KP];
        auto load_keys = [&](int s) {
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int w = 0; w < F::KP; ++w) k[s & 1][t][w] = *reinterpret_cast<const op*>(kl + w * X::KSIZE + (16 * t + col) * X::KR + 32 * s + 8 * grp);
        };
        load_keys(0);
        f4 sc[T];
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[t][e] = 0.0f;
#pragma unroll
        for (int s = 0; s < X::QS; ++s) {
            if (s + 1 < X::QS) load_keys(s + 1);
            __builtin_amdgcn_sched_barrier(0);
            products_of(k[s & 1], q[s], sc);
            __builtin_amdgcn_sched_barrier(0);
        }
        op v[2][VG][F::KP];
        auto load_values = [&](int i) {
#pragma unroll
            for (int u = 0; u < VG; ++u) {
                const int32_t dim = 16 * (i % GROUPS * VG + u) + col;
#pragma unroll
                for (int w = 0; w < F::KP; ++w) v[i & 1][u][w] = *reinterpret_cast<const op*>(vl + w * X::VSIZE + dim * X::VR + block_of(4 * (i / GROUPS) + grp, dim));
            }
        };
        load_values(0);
        __builtin_amdgcn_sched_barrier(0);  // (the first values are on their way from LDS while the weights are made)
        float x[8 * X::SETS];
#pragma unroll
        for (int i = 0; i < 8 * X::SETS; ++i) x[i] = sc[i >> 2][i & 3];
        if (masked) {  // (a score of -infinity has no weight)
#pragma unroll
            for (int h = 0; h < X::SETS; ++h) {
                const uint32_t vis = seen_bits(b, part.first, token, part.length, ch * CH + 32 * h, where.there[h]);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (!(vis >> token_of(i) & 1)) x[8 * h + i] = -INFINITY;
            }
        }
        to_weights<FMT>(x, f, m, l, [&](float alpha) {
#pragma unroll
            for (int db = 0; db < X::DB; ++db) o[db / VG][db % VG] *= alpha;
        });
        op p[F::QP];
#pragma unroll
        for (int i = 0; i < X::SETS * GROUPS; ++i) {
            if (i % GROUPS == 0) {
                float w8[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w8[e] = x[8 * (i / GROUPS) + e];
                split_weights(w8, p);
            }
            if (i + 1 < X::SETS * GROUPS) load_values(i + 1);
            __builtin_amdgcn_sched_barrier(0);
            products_of(v[i & 1], p, o[i % GROUPS]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (int32_t ch = c0; ch < c1; ++ch) {
        const Where<CH, WHOLE> now = next;
        if (ch + 1 < c1) {
            next = reader.where_of(ch + 1, pages);
            load_chunk(next);
            pages = reader.pages_of(min(ch + 2, c1 - 1));
        }
        __syncthreads();  // the chunk is in LDS
        if (ch < none_from) {
            attend_chunk(ch >= all_upto || !all_there(now), ch, now);
        }
        if constexpr (X::BUFFERS == 1) __syncthreads();  // (and read by all)
        if (ch + 1 < c1) store_chunk(ch + 1, next);
    }

    f4 none = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int db = 0; db < X::DB; ++db) none += o[db / VG][db % VG] * 0.0f;  // (NaN of what is not finite)
    if (active && (not_finite || __ballot(!(none[0] + none[1] + none[2] + none[3] == 0.0f)))) {
        Odd odd{0, 0};
        for (int32_t ch = c0; ch < min(c1, none_from); ++ch) {
            next = reader.where_of(ch, reader.pages_of(ch));
#pragma unroll
            for (int h = 0; h < X::SETS; ++h) {
                const uint32_t vis = seen_bits(b, part.first, token, part.length, ch * CH + 32 * h, next.there[h]);
                constexpr int N = together<FMT, X::DB>();
                for (int32_t tok = 0; tok < 32; tok += N) {
                    const uint8_t* rows = c.values + 4 * grp * E;
                    if constexpr (WHOLE) rows += next.base[0] + (32 * h + tok) * HD * E;
                    else rows += next.of_run(2 * h + (tok >> 4)) + (tok & 15) * HD * E;
                    look_at<FMT, X::DB, N>(odd, vis >> tok, [&](int u) { return rows + u * HD * E; }, 16);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < HD / 4; ++i) o[i / 4 / VG][i / 4 % VG][i % 4] = or_odd(odd, i, o[i / 4 / VG][i / 4 % VG][i % 4]);
    }

    l = column_sum(l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (16 * wave + col < held) {
        const size_t at_slot = static_cast<size_t>(part.slot + part.split) * R + r;
        float* out = keys.splits == 1 ? a.p.context + row_at(r) : a.averages + at_slot * HD;
#pragma unroll
        for (int db = 0; db < X::DB; ++db) *reinterpret_cast<f4*>(out + 16 * db + 4 * grp) = o[db / VG][db % VG] * inv;
        if (keys.splits > 1 && grp == 0) reinterpret_cast<float2*>(a.stats)[at_slot] = make_float2(m, l);
    }
}

// ---- launches ---------------------------------------------------------------------------------------
// The grid (of workgroups of `threads`) and the workspace of a launch of tiles of R rows whose parts have at least LEAST chunks of CHUNK keys.
template <int HD, int R, int LEAST, int CHUNK>
int32_t prepare(Args& a, int32_t target, int32_t threads, int64_t* grid, hipStream_t st) {
    const BatchView& b = a.p.b;
    const int64_t G = a.p.num_heads / a.p.c.kv_heads;
    const int64_t tiles = std::min(b.sequences * ((b.most_rows * G + R - 1) / R), b.rows * G / R + b.sequences) * a.p.c.kv_heads;  // at most
    const int64_t chunks = (static_cast<int64_t>(b.key_bound) + CHUNK - 1) / CHUNK, most_splits = std::min<int64_t>(MOST_PARTS, (chunks + LEAST - 1) / LEAST);
    a.target = target;
    const int64_t most = fine(R) ? 2 * target : target;  // (find_part)
    *grid = std::min(tiles + most, tiles * most_splits);
    if (too_many(*grid, threads)) return fail(KT_ERR_SHAPE, "too many rows and heads in one call");
    // One sequence whose tiles are target and more by themselves is not cut (find_part would not, were its rows fewer than the call says it
    // could): no merge to launch. A prompt of 1024 (fp16, 64 dims): 33 us, with one 36; of 2048 63 and 67.
    const bool finer = fine(R) && tiles * chunks > int64_t{target} * (LONG / CHUNK) && tiles < 2 * int64_t{target};
    const bool whole = b.sequences == 1 && tiles >= target && !finer;
    if (whole) *grid = tiles;
    if (most_splits <= 1 || whole) return KT_OK;
    const size_t slots = static_cast<size_t>(std::min<int64_t>(2 * most, *grid));
    a.slots = static_cast<int32_t>(slots);
    void* ws = nullptr;
    if (const int32_t status = workspace_counters(st, slots * R * (HD + 2) * sizeof(float) + 16, R == 16 ? slots : 0, &ws, &a.counters)) return status;
    ws = reinterpret_cast<void*>((reinterpret_cast<uintptr_t>(ws) + 15) & ~uintptr_t{15});  // (it begins at any dword)
    a.averages = static_cast<float*>(ws);
    a.stats = a.averages + slots * R * HD;
    return KT_OK;
}

template <int HD, int R, int LEAST, int CHUNK>
int32_t launch_merge(const Args& a, hipStream_t st) {
    if (a.slots == 0) return KT_OK;
    merge_kernel<HD, R, LEAST, CHUNK><<<dim3(static_cast<uint32_t>(a.slots), merge_shares(R)), 256, 0, st>>>(a);
    KT_LAUNCHED("paged attention merge kernel");
    return KT_OK;
}

template <int FMT, int HD, bool STEP>
int32_t launch_rows(Args a, hipStream_t st) {
    using X = Shape<FMT, HD>;
    int64_t grid = 0;
    // four parts a CU (64 steps over 2048 tokens on average, 128 dims, bf16 / one of 131000 beside seven, 64 dims, fp16: 2 parts 115 / 95 us,
    // 3 110 / 91, 4 111 / 84, 6 112 / 86, 8 112 / 87). One to four rounds of them, as registers leave a CU five to one of these workgroups:
    // of texts of 1000 tokens two or three parts take 5 to 13% less (64 of them, from the last cache, at 2, 3, 4, 6: 64 dims in fp16 30, 30, 34,
    // 33; 128 54, 52, 59, 59; 256 126, 129, 139, 145; fp32 128 126, 129, 141, 150).
    if (const int32_t status = prepare<HD, X::R, X::LEAST, CHUNK>(a, 4 * cu_count(), 64 * X::NW, &grid, st)) return status;
    constexpr size_t lds = std::max(std::max(sizeof(float) * X::NW * X::R * (HD + 6), size_t{2} * Format<FMT>::QP * X::R * (HD + 8)), merge_lds(X::R, X::NW));
    if (const int32_t ls = allow_lds<&attention_kernel<FMT, HD, STEP>, lds>(lds)) return ls;
    attention_kernel<FMT, HD, STEP><<<static_cast<uint32_t>(grid), 64 * X::NW, lds, st>>>(a);
    KT_LAUNCHED("paged attention kernel");
    return KT_OK;
}

template <int FMT, int HD, int WAVES>
int32_t launch_tiles(Args a, hipStream_t st) {
    using X = Tile<FMT, HD, WAVES>;
    int64_t grid = 0;
    if (const int32_t status = prepare<HD, X::R, X::LEAST, X::CH>(a, X::TARGET * cu_count(), X::THREADS, &grid, st)) return status;
    const auto kernel = [&](auto whole) -> int32_t {
        constexpr bool WHOLE = decltype(whole)::value;
        if (const int32_t ls = allow_lds<&tile_kernel<FMT, HD, WAVES, WHOLE>, X::LDS>(X::LDS)) return ls;
        tile_kernel<FMT, HD, WAVES, WHOLE><<<static_cast<uint32_t>(grid), X::THREADS, X::LDS, st>>>(a);
        KT_LAUNCHED("paged attention kernel");
        return KT_OK;
    };
    // pages that hold whole chunks have a form of their own (a prompt of 2048, pages of 64, with and without it: bf16 at 128 dims 94 and 100 us, fp32 at 64 dims 98 and 108)
    if (const int32_t status = 1 << a.p.c.page_shift >= X::CH ? kernel(std::true_type{}) : kernel(std::false_type{})) return status;
    return launch_merge<HD, X::R, X::LEAST, X::CH>(a, st);
}

// Which kernel (us here: head dims of 128 unless said, 32 heads on 8 kv heads, one sequence, pages of 32, of trees 64; the kernel taken first):
//   up to 16 rows of a kv head: tiles of 16. (A tree of 4 tokens has no use for more.)
//   up to 128 keys: the same for any number of rows, as its waves have a chunk each: no parts to merge, and four
//     times the workgroups. A prompt of 128: fp16 9.2 against 12.7, fp32 12.6 against 16.8, fp16 at 64 dims 6.9 against 7.9, fp32
//     at 256 dims 24 against 26.
//   up to 64 rows: tiles of 64, so that no wave is idle, two workgroups a CU: 16 sequences with trees of 15 after 2000 tokens 36
//     against 46 with tiles of 128 (fp32 54 against 79); one tree of 15 after 4000 in fp32 30 and 29.
//   up to 64 dims in 16 bits: tiles of 64 for any number of rows, of which three workgroups share a CU: a prompt of 1024 26
//     against 31, of 2048 54 against 64 (fp16).
//   else: tiles of 128, as the chunk that eight waves share is half the loads and LDS writes a row: a prompt of 2048 86 against 96 (fp16), 100
//     against 110 (bf16), 171 against 211 (fp32); a tree of 60 in fp32 43 against 46.
//   256 dims: tiles of 64 whose waves have a SIMD's registers each: a prompt of 512 36 against 38 with tiles of
//     128 (bf16 40 against 42, fp32 72 against 97; 16 trees of 15 78 against 67).
template <int FMT, int HD>
int32_t launch_dims(const Args& a, hipStream_t st) {
    const int64_t rows = static_cast<int64_t>(a.p.b.most_rows) * (a.p.num_heads / a.p.c.kv_heads);
    if (a.k_new) return launch_rows<FMT, HD, true>(a, st);
    if (rows <= 16 || a.p.b.key_bound <= 128) return launch_rows<FMT, HD, false>(a, st);
    if constexpr (HD == 256 || (HD <= 64 && FMT != KT_PAGED_F32)) {
        return launch_tiles<FMT, HD, 4>(a, st);
    } else {
        if (rows <= 64) return launch_tiles<FMT, HD, 4>(a, st);
        return launch_tiles<FMT, HD, 8>(a, st);
    }
}

template <int FMT>
int32_t launch(const PagedAttnArgs& p, const float* k, const float* v, hipStream_t st) {
    Args a{};
    a.p = p;
    a.k_new = k;
    a.v_new = v;
    switch (p.c.head_dim) {
        case 32: return launch_dims<FMT, 32>(a, st);
        case 64: return launch_dims<FMT, 64>(a, st);
        case 128: return launch_dims<FMT, 128>(a, st);
        default: return launch_dims<FMT, 256>(a, st);
    }
}

}  // namespace paged
}  // namespace kt
