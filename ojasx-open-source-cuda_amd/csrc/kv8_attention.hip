// kv8_attention.hip -- causal attention of the newest tokens over the 8-bit paged cache
// (layout: include/ojasx_e8t.h).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m)
//
// over the visible keys j of a row (a token's query head), with k_j = kcode_j * kscale(block),
// v_j likewise: the scales of a block multiply the score and the weight, not the elements.

#include <hip/hip_runtime.h>

#include <type_traits>

#include "serve.h"

namespace ojx {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// ---------------------------------------------------------------- items

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;

// Where each wave has rows of its own, a workgroup has 128 or 64.  Heads of up to 128 leave the
// registers for two 16-row columns in each of four waves, or one (how a call is cut says when).
// Larger ones have one: four waves at up to 192 (22 requests of up to 1796 tokens 170 us, 192 with
// eight), eight over that (13 of up to 2038 tokens 249 us, 397 with four).
constexpr int row_columns(int dc, int rows) { return dc <= 2 && rows == 128 ? 2 : 1; }
constexpr int row_waves(int dc, int rows) { return rows / (16 * row_columns(dc, rows)); }
constexpr float kFixed = 32512.f;  // largest fixed-point value: 127 * 256 with its low part 0
constexpr float kMagic = 12582912.f + 128.f;  // 1.5 * 2^23: the sum's low bits are the integer
constexpr float kLeastScale = 0x1p-100f;

// How a launch cuts its work.  An item is a tile of rows of one request (tok tokens of it, or
// part of one token's heads where a key head has more than a tile's rows) and one key head.  Items
// of more than `per` 64-key tiles are done in parts by several workgroups, joined by a second
// launch; of the two kinds, the last items may be cut finer than the first `whole`.
struct Cut {
    int rows;      // rows of a tile
    int tok;       // tokens of a tile
    int subs;      // tiles of one token's heads of a key head
    int64_t tiles; // tiles (upper bound), without subs and key heads
    int each;      // tiles of a request where every one has as many (few rows)
    int small;     // requests of at most so many tokens belong to the launch that splits keys
    int items, whole;
    int joins;     // workgroups that join an item's parts
    int per[2];    // 64-key tiles of a part, at most
    int parts[2];  // parts of an item, at most (the launch's workgroups for each)
    float* part;   // [stored parts][rows][dp]
    float2* ml;    // [stored parts][rows]
};

struct Item {
    int id, split;       // of the launch: the item, and which of its parts
    int head, sub, tile;
    int r, tok0, ntok;   // request, the tile's tokens in it
    int q0;              // first row of q of the request
    int group;           // query heads of a key head
    int rows;            // rows in use
    int len;             // the request's tokens, newest included
    int before;          // the tile's first token's place
    int parts;
    int t0, t1;          // 64-key tiles of the part
    int end_key;         // end of the keys that any of its rows sees
    int64_t stored;      // first row of the part's results, of several
};

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Zeros in n rows from `first` on, as in rows that see nothing: a thread takes every `step`-th
// element from `at` on.
template <int DT>
__device__ __forceinline__ void clear(const AttnArgs& a, int64_t first, int64_t n, int64_t at,
                                      int64_t step) {
    for (int64_t i = first * a.shape.d + at; i < (first + n) * a.shape.d; i += step)
        store_from_f32<DT>(a.out, i, 0.f);
    if (a.lse)
        for (int64_t i = first + at; i < first + n; i += step) a.lse[i] = -INFINITY;
}

// The workgroup's heads of tokens [from, to).
template <int DT>
__device__ __forceinline__ void clear_heads(const AttnArgs& a, const Item& it, int from, int to) {
    for (int t = from; t < to; ++t)
        clear<DT>(a, (int64_t)t * a.shape.heads + it.head * it.group, it.group, threadIdx.x, blockDim.x);
}

// The item `id` in its part `split`; false: none.  CLEAR: rows that no item has are cleared by the
// workgroup of a first item beside them, which has read where they are: of tokens past a request's
// max_query, of those before the first request (further loads would cost small calls 0.4 us).
template <bool ROWS, int DT, bool CLEAR>
__device__ __forceinline__ bool find_item(const AttnArgs& a, const Cut& c, int id, int split, Item& it) {
    it.id = id;
    it.split = split;
    it.head = id % a.shape.kv_heads;
    id /= a.shape.kv_heads;
    it.sub = id % c.subs;
    it.tile = id / c.subs;
    it.group = a.shape.heads / a.shape.kv_heads;
    int q0, q1;
    if constexpr (!ROWS) {
        it.r = it.tile / c.each;
        q0 = a.query_starts ? a.query_starts[it.r] : it.r;
        q1 = a.query_starts ? a.query_starts[it.r + 1] : it.r + 1;
        it.tok0 = (it.tile - it.r * c.each) * c.tok;
    } else {
        // request r's tiles begin at query_starts[r] / tok + r: room for each one's last, partly
        // filled tile without a sum over the requests; 64 requests are looked at at a time
        int lo = 0, n = a.shape.requests;
        const int lane = threadIdx.x & 63;
        while (n > 0) {
            const int step = (n + 63) >> 6;
            const int i = lo + lane * step;
            const bool at = lane * step < n && a.query_starts[i] / c.tok + i <= it.tile;
            const int last = 63 - __builtin_clzll(__ballot(at) | 1);
            lo += last * step;
            n = step == 1 ? 0 : min(step, n - last * step);
        }
        it.r = lo;
        q0 = a.query_starts[lo];
        q1 = a.query_starts[lo + 1];
        it.tok0 = (it.tile - (q0 / c.tok + lo)) * c.tok;
    }
    const int tokens = a.shape.tokens;
    const bool first_of = CLEAR && it.sub == 0 && split == 0;
    if (__builtin_expect(first_of && it.tile == 0 && q0 > 0, 0))
        clear_heads<DT>(a, it, 0, min(q0, tokens));
    const int newest = q1 - q0;
    if (ROWS ? newest <= c.small || it.tok0 < 0 : newest > c.small) return false;
    // no rows outside q, whatever query_starts says
    if (q0 < 0 || q0 >= tokens) return false;
    if (__builtin_expect(first_of && it.tok0 == 0 && newest > a.shape.max_query, 0))
        clear_heads<DT>(a, it, q0 + a.shape.max_query, min(q1, tokens));
    it.ntok = min(min(min(newest, a.shape.max_query), tokens - q0) - it.tok0, c.tok);
    if (it.ntok <= 0) return false;
    it.q0 = q0;
    it.rows = c.subs > 1 ? min(it.group - it.sub * c.rows, c.rows) : it.ntok * it.group;
    it.len = max(0, min(a.seq_lens[it.r], a.shape.max_seq));
    it.before = a.seq_lens[it.r] - newest + it.tok0;
    const int first = a.shape.window ? max(0, it.before + 1 - a.shape.window) : 0;
    it.end_key = max(0, min(it.before + it.ntok, it.len));
    const int kind = it.id < c.whole ? 0 : 1;
    const int from = first >> 6, to = max(from, (it.end_key + 63) >> 6);
    it.parts = max(1, min(c.parts[kind], (to - from + c.per[kind] - 1) / c.per[kind]));
    if (it.split >= it.parts) return false;
    const int per = (to - from + it.parts - 1) / it.parts;
    it.t0 = from + it.split * per;
    it.t1 = min(to, it.t0 + per);
    const int64_t at = kind == 0 ? (int64_t)it.split * c.whole + it.id
                                 : (c.parts[0] > 1 ? (int64_t)c.parts[0] * c.whole : 0) +
                                       (int64_t)it.split * (c.items - c.whole) + it.id - c.whole;
    it.stored = at * c.rows;
    return true;
}

// The item and part of a workgroup: parts of an item lie apart, so they run at the same time.
template <bool ROWS, int DT>
__device__ __forceinline__ bool block_item(const AttnArgs& a, const Cut& c, int block, Item& it) {
    const int first = c.whole * c.parts[0];
    if (block < first) return find_item<ROWS, DT, true>(a, c, block % c.whole, block / c.whole, it);
    block -= first;
    const int rest = c.items - c.whole;
    return find_item<ROWS, DT, true>(a, c, c.whole + block % rest, block / rest, it);
}

// Token (within the tile) and query head of a row of an item.
__device__ __forceinline__ void row_at(const AttnArgs& a, const Cut& c, const Item& it, int row,
                                       int& tok, int& head) {
    tok = c.subs > 1 ? 0 : row / it.group;
    head = it.head * it.group + (c.subs > 1 ? it.sub * c.rows + row : row - tok * it.group);
}

template <int DT> __device__ __forceinline__ void load8(const void* p, int64_t e, float (&x)[8]) {
    const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + e);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = DT == kBF16 ? bf16_bits_to_f32(u[i] & 0xFFFFu) : f16_bits_to_f32(u[i] & 0xFFFFu);
        x[2 * i + 1] = DT == kBF16 ? bf16_bits_to_f32(u[i] >> 16) : f16_bits_to_f32(u[i] >> 16);
    }
}

// The high and low bytes of four fixed-point values, each the low 16 bits of a float kMagic was
// added to: value = 256 * high + low, both signed bytes.
__device__ __forceinline__ void limbs(const float (&t)[4], int& high, int& low) {
    const uint32_t t0 = __float_as_uint(t[0]), t1 = __float_as_uint(t[1]);
    const uint32_t t2 = __float_as_uint(t[2]), t3 = __float_as_uint(t[3]);
    const uint32_t a = __builtin_amdgcn_perm(t1, t0, 0x05010400u);  // t0.b0 t1.b0 t0.b1 t1.b1
    const uint32_t b = __builtin_amdgcn_perm(t3, t2, 0x05010400u);
    low = (int)(__builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u);
    high = (int)__builtin_amdgcn_perm(b, a, 0x07060302u);
}

__device__ __forceinline__ v4i times256(v4i x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (int)((uint32_t)x[i] << 8);
    return x;
}

__device__ __forceinline__ v4i product(v4i a, v4i b, v4i c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ void store_row4(void* out, int64_t e, int n, bool vec, const float (&v)[4]) {
    if (vec && n >= 4) {
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            b[i] = DT == kBF16 ? f32_to_bf16_bits(v[i]) : f32_to_f16_bits(v[i]);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + e) =
            make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) store_from_f32<DT>(out, e + i, v[i]);
}

__device__ __forceinline__ bool out_vector(const AttnArgs& a) {
    return a.shape.d % 4 == 0 && ((uintptr_t)a.out & 15) == 0;
}

// The query rows of a lane's columns: fixed-point operands of the score products, bounds of the
// keys that a row sees.
template <int DC, int NQ> struct Rows {
    int hi[NQ], lo[NQ];
    float qs[NQ];  // a row's unit times scale * log2(e): a whole-number score times it and the
                   // key scale is the exponent
    bool live[NQ], bad[NQ];
    v4i qh[NQ][DC], ql[NQ][DC];

    template <int DT>
    __device__ __forceinline__ void load(const AttnArgs& a, const Cut& c, const Item& it, int row0,
                                         int g, int n) {
        const bool vec = a.shape.d % 8 == 0 && ((uintptr_t)a.q.p & 15) == 0 &&
                         a.q.token % 8 == 0 && a.q.head % 8 == 0;
        const float to_log2 = a.scale * kLog2e;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const int row = row0 + 16 * q + n;
            live[q] = row < it.rows;
            int tok, head;
            row_at(a, c, it, live[q] ? row : 0, tok, head);
            const int pos = it.before + tok;
            hi[q] = max(0, min(pos + 1, it.len));
            lo[q] = a.shape.window ? max(0, pos + 1 - a.shape.window) : 0;
            const int64_t e = (int64_t)(it.q0 + it.tok0 + tok) * a.q.token + head * a.q.head;
            float x[DC][16], m = 0.f;
#pragma unroll
            for (int k = 0; k < DC; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int d = 64 * k + 16 * g + 8 * h;
                    float y[8];
                    if (vec && d < a.shape.d) {
                        load8<DT>(a.q.p, e + d, y);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            y[i] = d + i < a.shape.d ? load_as_f32<DT>(a.q.p, e + d + i) : 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[k][8 * h + i] = y[i] * to_log2;
                        m = __builtin_elementwise_maximum(m, fabsf(x[k][8 * h + i]));  // keeps NaN
                    }
                }
            m = col_max(m < INFINITY ? m : INFINITY);
            // also where only the product with the scale overflows: so far out only NaN is right
            bad[q] = m == INFINITY;
            const float up = m >= kLeastScale && !bad[q] ? kFixed / m : 0.f;
            qs[q] = up > 0.f ? m * (1.f / kFixed) : 0.f;
#pragma unroll
            for (int k = 0; k < DC; ++k)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    float t[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        t[i] = bad[q] ? kMagic : __builtin_fmaf(x[k][4 * w + i], up, kMagic);
                    int high, low;
                    limbs(t, high, low);
                    qh[q][k][w] = high;
                    ql[q][k][w] = low;
                }
        }
    }

    // Whether every row sees the 64 keys from j0 on.
    __device__ __forceinline__ bool see_all(int j0) const {
        bool all = true;
#pragma unroll
        for (int q = 0; q < NQ; ++q) all &= !live[q] || (lo[q] <= j0 && hi[q] >= j0 + 64);
        return all;
    }

    // Those of the 16 keys from `key` on that row q sees, from bit 0 on.
    __device__ __forceinline__ uint32_t seen(int q, int key) const {
        const int h = hi[q] - key, w = lo[q] - key;
        const uint32_t below = h <= 0 ? 0u : h >= 16 ? 0xFFFFu : (1u << h) - 1u;
        return below & (w <= 0 ? 0xFFFFu : w >= 16 ? 0u : ~((1u << w) - 1u));
    }
};

// A lane's 16 whole-number scores as floats, and -inf in the place of those without a bit in
// `seen`: a step of its own for the tiles that need it, so the weights' code is the same for all.
__device__ __forceinline__ void to_float(const v4i (&s)[4], v4f (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[i][r] = (float)s[i][r];
}
__device__ __forceinline__ void hide(v4f (&x)[4], uint32_t seen) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[i][r] = seen >> (4 * i + r) & 1 ? x[i][r] : -INFINITY;
}
__device__ __forceinline__ float largest(const v4f (&x)[4]) {
    float top = x[0][0];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, x[i][r]);
    return top;
}

// A reference below every score (and no infinity, whose differences would be NaN), the score that
// larger ones count as, and the least and the largest factor of a score: times -inf it stays -inf,
// times 0 it is 0.
constexpr float kNone = -1e30f;
constexpr float kFar = 9e29f;
constexpr float kLeastFactor = 0x1p-120f;
constexpr float kLargestFactor = 0x1p120f;

__device__ __forceinline__ float score_factor(float q_unit, float key_scale) {
    return __builtin_amdgcn_fmed3f(q_unit * key_scale, kLeastFactor, kLargestFactor);
}

// The exponent of a lane's largest score `top` (-inf: it sees none): top * f + lv, within kFar.
__device__ __forceinline__ float far_or(float top, float f, float lv) {
    const float m = __builtin_amdgcn_fmed3f(__builtin_fmaf(top, f, lv), -kFar, kFar);
    return top == -INFINITY ? top : m;
}

// The block of a group of 16 keys (-1: none) and its bytes' offset.
struct Pages {
    const int32_t* table;
    int width, log_block, blocks, heads, head, end;
    int64_t head_bytes;

    __device__ __forceinline__ Pages(const AttnArgs& a, const Item& it)
        : table(a.tables + it.r * a.table_ld), width(a.width), log_block(a.cache.log_block),
          blocks(a.cache.blocks), heads(a.cache.heads), head(it.head), end(it.end_key),
          head_bytes(a.cache.head_bytes()) {}
    __device__ __forceinline__ int block(int key) const {
        const int i = key >> log_block;
        return key < end && i < width ? table[i] : -1;
    }
    __device__ __forceinline__ bool valid(int b) const { return b >= 0 && b < blocks; }
    __device__ __forceinline__ int64_t index(int b) const {  // of (block, head)
        return (int64_t)(valid(b) ? b : 0) * heads + head;
    }
    __device__ __forceinline__ int64_t at(int b, int key, int dp) const {
        return index(b) * head_bytes + ((key & ((1 << log_block) - 1)) >> 4) * (16 * dp);
    }
};

// Few rows over many keys, on the matrix unit in whole numbers: a score is 256 (qh.k) + (ql.k)
// with the row's q in 16-bit fixed point against its own largest element, 64 keys at a time;
// the weights of 64 keys are 16-bit fixed point against their largest weight * (value scale), so
// codes of keys and values enter as they lie in memory: what the cache costs is its bytes.
// Tile t of the four score products takes 4 keys of each group of 16: a lane then holds the 16
// scores of one group (one block: one pair of scales), and their weights are the second operand
// of the value products as they come.  The workgroup's waves take turns at 64 keys of a 16-row tile
// and join their results in LDS.  (Two tiles of rows for one pass over the keys would need more
// than half of a SIMD's registers: two workgroups that share the keys in L2 are faster.)
// The roundings are a choice: 2^-16 of the largest element for q (a bf16 element has 2^-9 of itself;
// an fp16 one, 2^-11, loses bits of its own from 1/32 of the largest on), 2^-16 of the largest of 64
// for weights, beside values that are held in 8 bits; all sums are 32-bit.
// Memory bounds it where there are many keys (64 tokens over 500 to 16000 tokens, 631 MB: 123 us
// and 5 for the join, 4.9 TB/s; heads off the grid of 64 read their padding too: 132 us for heads of
// 80, whose own bytes are 409 of 654 MB), launches and latency where there are few (one over 2048
// tokens: 6.6 us and 3 for the join).
template <int DC, int WAVES> struct KeyShared {
    static constexpr int kLd = 64 * DC + 4;
    float joined[WAVES * 16 * kLd];
    float m[WAVES][16], l[WAVES][16];
};

template <int DT, int DC, int WAVES>
__device__ __forceinline__ void key_item(const AttnArgs& a, const Cut& c, int block,
                                         KeyShared<DC, WAVES>& sh) {
    constexpr int NQ = 1, DP = 64 * DC, DM = DP / 16, LD = KeyShared<DC, WAVES>::kLd;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, n = lane & 15;
    Item it;
    if (!block_item<false, DT>(a, c, block, it)) return;
    const int t0 = it.t0 + wave, t1 = it.t1;

    // the first keys and values are on their way before the queries
    const Pages pages(a, it);
    const int key_k = (n >> 2) * 16, key_v = g * 16;
    const int in_k = g * 64 + (n & 3) * 16, in_v = n * 16;
    v4i kf[4][DC], vf[DM];
    float2 sc = make_float2(0.f, 0.f);
    auto load_keys = [&](int b, int j0) {
        const int8_t* p = a.cache.k + pages.at(b, j0 + key_k, DP) + in_k;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int k = 0; k < DC; ++k)
                kf[t][k] = *reinterpret_cast<const v4i*>(p + (4 * k + t) * 256);
    };
    auto load_values = [&](int b, int j0) {
        const int8_t* p = a.cache.v + pages.at(b, j0 + key_v, DP) + in_v;
#pragma unroll
        for (int i = 0; i < DM; ++i) vf[i] = *reinterpret_cast<const v4i*>(p + i * 256);
    };
    auto load_scales = [&](int b) {
        return *reinterpret_cast<const float2*>(a.cache.scales + 2 * pages.index(b));
    };
    int bv = -1, bk_next = -1, bv_next = -1;
    if (t0 < t1) {
        const int bk = pages.block(t0 * 64 + key_k);
        bv = pages.block(t0 * 64 + key_v);
        bk_next = pages.block((t0 + WAVES) * 64 + key_k);
        bv_next = pages.block((t0 + WAVES) * 64 + key_v);
        load_keys(bk, t0 * 64);
        sc = load_scales(bv);
        load_values(bv, t0 * 64);
    }
    Rows<DC, NQ> rows;
    rows.template load<DT>(a, c, it, 0, g, n);

    v4f o[NQ][DM];
    float m_run[NQ], l_run[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        m_run[q] = kNone;
        l_run[q] = 0.f;
#pragma unroll
        for (int i = 0; i < DM; ++i) o[q][i] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    for (int t = t0; t < t1; t += WAVES) {
        const int j0 = t * 64;
        v4i s[NQ][4];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[q][i] = v4i{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < DC; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[q][i] = product(kf[i][k], rows.qh[q][k], s[q][i]);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[q][i] = times256(s[q][i]);
#pragma unroll
            for (int k = 0; k < DC; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[q][i] = product(kf[i][k], rows.ql[q][k], s[q][i]);
        }
        const bool valid = pages.valid(bv);
        const float ks = sc.x, v_scale = fmaxf(sc.y, kLeastScale);
        const bool more = t + WAVES < t1;
        const int bv_now = bv_next;
        if (more) {
            load_keys(bk_next, j0 + 64 * WAVES);
            sc = load_scales(bv_next);
            bv = bv_next;
            bk_next = pages.block(j0 + 128 * WAVES + key_k);
            bv_next = pages.block(j0 + 128 * WAVES + key_v);
        }
        const float lv = __builtin_amdgcn_logf(v_scale), rv = __builtin_amdgcn_rcpf(v_scale);
        v4f x[NQ][4];
#pragma unroll
        for (int q = 0; q < NQ; ++q) to_float(s[q], x[q]);
        if (!__all(valid && rows.see_all(j0))) {
#pragma unroll
            for (int q = 0; q < NQ; ++q) hide(x[q], valid ? rows.seen(q, j0 + key_v) : 0u);
        }
        v4i ph[NQ], pl[NQ];
        float beta[NQ];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            // Exponents as differences from the lane's largest score, which are exact: x * f + (lv -
            // m) is off by m's rounding, and a weight over 1 does not fit its 16 bits.
            const float f = score_factor(rows.qs[q], ks), top = largest(x[q]);
            const float mine = far_or(top, f, lv);
            const float m = fmaxf(col_max(mine), kNone);
            const float from = fmaxf(top, -0x1p31f), base = mine - m;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float p[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float e = fast_exp2(__builtin_fmaf(x[q][i][r] - from, f, base));
                    sum += e;
                    p[r] = __builtin_fmaf(e, kFixed, kMagic);
                }
                int high, low;
                limbs(p, high, low);
                ph[q][i] = high;
                pl[q][i] = low;
            }
            const float next = fmaxf(m_run[q], m);
            const float keep = fast_exp2(m_run[q] - next), part = fast_exp2(m - next);
            l_run[q] = __builtin_fmaf(l_run[q], keep, sum * rv * part);
            beta[q] = part * (1.f / kFixed);
            if (!__all(m_run[q] == next)) {
#pragma unroll
                for (int i = 0; i < DM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[q][i][r] *= keep;
            }
            m_run[q] = next;
        }
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int i0 = 0; i0 < DM; i0 += 4) {
                v4i w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = product(vf[i0 + i], ph[q], v4i{0, 0, 0, 0});
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = product(vf[i0 + i], pl[q], times256(w[i]));
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        o[q][i0 + i][r] = __builtin_fmaf((float)w[i][r], beta[q], o[q][i0 + i][r]);
            }
        if (more) load_values(bv_now, j0 + 64 * WAVES);
    }

    const bool out_vec = out_vector(a);
    const float nan = __uint_as_float(0x7FC00000u);
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        l_run[q] = col_sum(l_run[q]);
        if (g == 0) {
            sh.m[wave][16 * q + n] = m_run[q];
            sh.l[wave][16 * q + n] = l_run[q];
        }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const int row = 16 * q + n;
        float m = sh.m[0][row];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) m = fmaxf(m, sh.m[w][row]);
        const float keep = fast_exp2(m_run[q] - m);
        if (rows.live[q]) {
            float* p = sh.joined + (wave * 16 * NQ + row) * LD + 4 * g;
#pragma unroll
            for (int i = 0; i < DM; ++i) *reinterpret_cast<v4f*>(p + 16 * i) = o[q][i] * keep;
        }
        // the joined sum, in every wave
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
            l = __builtin_fmaf(sh.l[w][row], fast_exp2(sh.m[w][row] - m), l);
        l_run[q] = l;
        m_run[q] = m;
    }
    __syncthreads();
    if (wave == 0 && g == 0) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            sh.m[0][16 * q + n] = rows.bad[q] && l_run[q] > 0.f ? nan : m_run[q];
            sh.l[0][16 * q + n] = l_run[q];
        }
    }
    __syncthreads();
    for (int u = threadIdx.x; u < it.rows * (DP / 4); u += 64 * WAVES) {
        const int row = u / (DP / 4), d = (u - row * (DP / 4)) * 4;
        const float m = sh.m[0][row], l = sh.l[0][row];
        v4f sum = *reinterpret_cast<const v4f*>(sh.joined + row * LD + d);
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
            sum += *reinterpret_cast<const v4f*>(sh.joined + (w * 16 * NQ + row) * LD + d);
        if (it.parts > 1) {
            if (d == 0) c.ml[it.stored + row] = make_float2(m, l);
            if (l > 0.f) *reinterpret_cast<v4f*>(c.part + (it.stored + row) * DP + d) = sum;
            continue;
        }
        int tok, head;
        row_at(a, c, it, row, tok, head);
        const int64_t at = (int64_t)(it.q0 + it.tok0 + tok) * a.shape.heads + head;
        const float inv = l > 0.f ? 1.f / l : 0.f;
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = m != m ? nan : sum[r] * inv;
        if (d < a.shape.d) store_row4<DT>(a.out, at * a.shape.d + d, a.shape.d - d, out_vec, v);
        if (a.lse && d == 0)
            a.lse[at] = !(l > 0.f) ? -INFINITY : m != m ? nan : (m + log2f(l)) * kLn2;
    }
}

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// Four codes as fp16, exactly: the byte with its sign flipped is code + 128, under the exponent
// of 1024 it reads 1152 + code.
__device__ __forceinline__ void halves_of(uint32_t codes, uint32_t& a, uint32_t& b) {
    const uint32_t u = codes ^ 0x80808080u;
    const v2h bias = {(_Float16)1152.f, (_Float16)1152.f};
    const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
    const uint32_t hi = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    a = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, lo) - bias);
    b = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, hi) - bias);
}

// Many rows: each wave has 32 or 16 of its own, and the workgroup goes through the keys together,
// 64 at a time through two buffers in LDS.  Vector instructions bound it, so they are what the
// layout saves: scores as for few rows (no conversion of keys; q's second byte costs matrix
// instructions, which are not the bound), but the weights as fp16 on fp16 values, converted once
// for the workgroup on their way into LDS: the products then add up in fp32 in the matrix unit,
// where whole-number products would cost three vector instructions for every result of every 64
// keys.  The reference of the weights is raised only when one would pass 2^kHeadroom times it, so
// the sums are scaled again rarely.  A weight's rounding to fp16 is 2^-11 of it, under 2^-14 of
// the reference 2^-25 of that; the sum takes it unrounded.  Four chunks of 900 to 2048 tokens over
// up to 8000 (321 GF): 423 us a call with 11 for the join, 760 Tflop/s of the two products; the
// matrix unit is busy for a third of the time, q's second byte included, vector instructions for
// most of the rest: 12 for a score.  The two hardly overlap.
constexpr float kHeadroom = 8.f;
// References up to which the weights' exponents are x * f + (lv - ref): that difference's rounding
// is under 2^-12 then.  Beyond, they are formed from differences of scores, in the step that also
// raises the reference, so that other rows do not pay an instruction a score for it.
constexpr float kNearReference = 0x1p12f;

template <int DC> struct RowShared {
    // bytes of 16 keys: groups begin in different banks
    static constexpr int kGroup = 16 * 64 * DC + 64;
    int8_t keys[2][4 * kGroup];
    _Float16 values[2][64 * 64 * DC];
};

template <int DT, int DC, int ROWS>
__device__ __forceinline__ void row_item(const AttnArgs& a, const Cut& c, int block,
                                         RowShared<DC>& sh) {
    constexpr int NQ = row_columns(DC, ROWS), DP = 64 * DC, DM = DP / 16, kGroup = RowShared<DC>::kGroup;
    constexpr int kStep = 64 * row_waves(DC, ROWS);    // threads
    // a thread's pieces of 16 bytes of 64 keys (some threads have one less where they do not come
    // out even)
    constexpr int kPieces = (4 * DP + kStep - 1) / kStep;
    auto has_piece = [&](int i) {
        return 4 * DP % kStep == 0 || (int)threadIdx.x + kStep * i < 4 * DP;
    };
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, n = lane & 15;
    Item it;
    if (!block_item<true, DT>(a, c, block, it)) return;
    const int t0 = it.t0, t1 = it.t1;
    const Pages pages(a, it);

    // Thread's pieces (16 bytes) of a tile: piece u of DP a group of 16 keys.
    v4i kr[kPieces], vr[kPieces];
    int next_block[kPieces];
    auto piece_key = [&](int i) { return (int)(threadIdx.x + kStep * i) / DP * 16; };
    auto piece_in = [&](int i) { return (int)(threadIdx.x + kStep * i) % DP; };
    auto find = [&](int t) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) next_block[i] = pages.block(t * 64 + piece_key(i));
    };
    auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (!has_piece(i)) continue;
            const int64_t at = pages.at(next_block[i], t * 64 + piece_key(i), DP) + piece_in(i) * 16;
            kr[i] = *reinterpret_cast<const v4i*>(a.cache.k + at);
            vr[i] = *reinterpret_cast<const v4i*>(a.cache.v + at);
        }
    };
    // values: [d / 16][half of the group's 16 keys][group][d % 16][8 keys]
    auto put = [&](int buf) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (!has_piece(i)) continue;
            const int group = piece_key(i) >> 4, in = piece_in(i);
            *reinterpret_cast<v4i*>(sh.keys[buf] + group * kGroup + in * 16) = kr[i];
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) halves_of((uint32_t)vr[i][j], w[2 * j], w[2 * j + 1]);
            uint4* p = reinterpret_cast<uint4*>(sh.values[buf]) + (in >> 4) * 128 + group * 16 + (in & 15);
            p[0] = make_uint4(w[0], w[1], w[2], w[3]);
            p[64] = make_uint4(w[4], w[5], w[6], w[7]);
        }
    };
    int bv = -1, bv_next = -1;
    float2 sc = make_float2(0.f, 0.f), sc_next = sc;
    auto load_scales = [&](int b) {
        return *reinterpret_cast<const float2*>(a.cache.scales + 2 * pages.index(b));
    };
    const int key_v = g * 16;
    if (t0 < t1) {
        find(t0);
        bv = pages.block(t0 * 64 + key_v);
        fetch(t0);
        sc = load_scales(bv);
        find(t0 + 1);
        bv_next = pages.block((t0 + 1) * 64 + key_v);
    }
    const int row0 = wave * 16 * NQ;
    Rows<DC, NQ> rows;
    rows.template load<DT>(a, c, it, row0, g, n);
    // tiles that this wave's rows see
    int w0 = t1, w1 = t0;
    {
        const int here = min(it.rows - row0, 16 * NQ);
        if (here > 0) {
            int ta, tb, unused;
            row_at(a, c, it, row0, ta, unused);
            row_at(a, c, it, row0 + here - 1, tb, unused);
            w0 = a.shape.window ? max(0, it.before + ta + 1 - a.shape.window) >> 6 : t0;
            w1 = (max(0, min(it.before + tb + 1, it.len)) + 63) >> 6;
        }
    }

    v4f o[NQ][DM];
    // `step`: exponents above it take the step below
    float ref[NQ], step[NQ], l_run[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        ref[q] = kNone;
        step[q] = -INFINITY;
        l_run[q] = 0.f;
#pragma unroll
        for (int i = 0; i < DM; ++i) o[q][i] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    if (t0 < t1) put(0);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1, j0 = t * 64;
        const bool more = t + 1 < t1;
        if (more) {
            fetch(t + 1);
            sc_next = load_scales(bv_next);
            find(t + 2);
        }
        if (t >= w0 && t < w1) {
            v4i s[NQ][4];
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[q][i] = v4i{0, 0, 0, 0};
            const int8_t* kp = sh.keys[buf] + (n >> 2) * kGroup + g * 64 + (n & 3) * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v4i kf[DC];
#pragma unroll
                for (int k = 0; k < DC; ++k) kf[k] = *reinterpret_cast<const v4i*>(kp + (4 * k + i) * 256);
#pragma unroll
                for (int k = 0; k < DC; ++k)
#pragma unroll
                    for (int q = 0; q < NQ; ++q) s[q][i] = product(kf[k], rows.qh[q][k], s[q][i]);
#pragma unroll
                for (int q = 0; q < NQ; ++q) s[q][i] = times256(s[q][i]);
#pragma unroll
                for (int k = 0; k < DC; ++k)
#pragma unroll
                    for (int q = 0; q < NQ; ++q) s[q][i] = product(kf[k], rows.ql[q][k], s[q][i]);
            }
            __builtin_amdgcn_sched_barrier(0);
            const bool valid = pages.valid(bv);
            const float ks = sc.x, v_scale = fmaxf(sc.y, kLeastScale);
            const float lv = __builtin_amdgcn_logf(v_scale), rv = __builtin_amdgcn_rcpf(v_scale);
            v4f x[NQ][4];
#pragma unroll
            for (int q = 0; q < NQ; ++q) to_float(s[q], x[q]);
            if (!__all(valid && rows.see_all(j0))) {
#pragma unroll
                for (int q = 0; q < NQ; ++q) hide(x[q], valid ? rows.seen(q, j0 + key_v) : 0u);
            }
            v8h p[NQ][2];
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                const float f = score_factor(rows.qs[q], ks), top = largest(x[q]);
                float base = lv - ref[q];
                if (!__all(__builtin_fmaf(top, f, lv) <= step[q])) {
                    const float mine = far_or(top, f, lv);
                    const float m = col_max(mine);
                    // the difference is exact where the sum may round up to twice the headroom
                    const float next = m - ref[q] > kHeadroom ? m : ref[q];
                    const float keep = fast_exp2(ref[q] - next);
                    l_run[q] *= keep;
#pragma unroll
                    for (int i = 0; i < DM; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[q][i][r] *= keep;
                    ref[q] = next;
                    const bool near = fabsf(next) < kNearReference;
                    step[q] = near ? next + kHeadroom : -INFINITY;
                    const float from = near ? 0.f : fmaxf(top, -0x1p31f);
                    base = near ? lv - next : mine - next;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) x[q][i][r] -= from;
                }
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float e = fast_exp2(__builtin_fmaf(x[q][i][r], f, base));
                        sum += e;
                        p[q][i >> 1][4 * (i & 1) + r] = (_Float16)e;
                    }
                l_run[q] = __builtin_fmaf(sum, rv, l_run[q]);
            }
            __builtin_amdgcn_sched_barrier(0);
            const v8h* vp = reinterpret_cast<const v8h*>(sh.values[buf]) + lane;
#pragma unroll
            for (int i = 0; i < DM; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const v8h v = vp[(2 * i + h) * 64];
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
                        o[q][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[q][h], o[q][i], 0, 0, 0);
                }
        }
        if (more) {
            put(buf ^ 1);
            sc = sc_next;
            bv = bv_next;
            bv_next = pages.block((t + 2) * 64 + key_v);
        }
        __syncthreads();
    }

    const bool out_vec = out_vector(a);
    const float nan = __uint_as_float(0x7FC00000u);
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const float l = col_sum(l_run[q]);
        if (!rows.live[q]) continue;
        const int row = row0 + 16 * q + n;
        if (it.parts > 1) {
            if (g == 0)
                c.ml[it.stored + row] = make_float2(rows.bad[q] && l > 0.f ? nan : ref[q], l);
            if (!(l > 0.f)) continue;
            float* p = c.part + (it.stored + row) * DP + 4 * g;
#pragma unroll
            for (int i = 0; i < DM; ++i) *reinterpret_cast<v4f*>(p + 16 * i) = o[q][i];
            continue;
        }
        int tok, head;
        row_at(a, c, it, row, tok, head);
        const int64_t at = (int64_t)(it.q0 + it.tok0 + tok) * a.shape.heads + head;
        const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
        for (int i = 0; i < DM; ++i) {
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = rows.bad[q] && l > 0.f ? nan : o[q][i][r] * inv;
            const int d = 16 * i + 4 * g;
            if (d < a.shape.d)
                store_row4<DT>(a.out, at * a.shape.d + d, a.shape.d - d, out_vec, v);
        }
        if (a.lse && g == 0)
            a.lse[at] = !(l > 0.f) ? -INFINITY : rows.bad[q] ? nan : (ref[q] + log2f(l)) * kLn2;
    }
}

// First token past the last request's: read where a kernel begins, beside its other first loads.
__device__ __forceinline__ int last_start(const AttnArgs& a) {
    return a.query_starts ? a.query_starts[a.shape.requests] : a.shape.tokens;
}

// The launch's share of the rows of tokens from `end` on, which belong to no request (a padded batch).
template <int DT> __device__ __forceinline__ void no_request(const AttnArgs& a, int end) {
    if (end >= a.shape.tokens) return;
    const int64_t first = (int64_t)max(end, 0) * a.shape.heads;
    clear<DT>(a, first, (int64_t)a.shape.tokens * a.shape.heads - first,
              (int64_t)blockIdx.x * blockDim.x + threadIdx.x, (int64_t)gridDim.x * blockDim.x);
}

// What a launch does: every block of a batch whose requests all have few rows or all have many is
// of one kind; in a mixed batch the first `row_blocks` take the requests of many rows, the others
// those of up to 16.
enum class Mix { Few, Many, Both };

constexpr int waves_of(int dc, Mix mix, int rows) {
    return mix == Mix::Few ? kWaves : row_waves(dc, rows);
}

template <int DT, int DC, Mix MIX, int ROWS>
__global__ __launch_bounds__(64 * waves_of(DC, MIX, ROWS), DC <= 2 || MIX != Mix::Few ? 2 : 1)
void attend_kernel(AttnArgs a, Cut key, Cut row, int row_blocks) {
    constexpr int waves = waves_of(DC, MIX, ROWS);
    constexpr size_t few = MIX == Mix::Many ? 0 : sizeof(KeyShared<DC, waves>);
    constexpr size_t many = MIX == Mix::Few ? 0 : sizeof(RowShared<DC>);
    __shared__ __align__(16) char lds[few > many ? few : many];
    const int end = last_start(a);
    if (MIX == Mix::Many || (MIX == Mix::Both && (int)blockIdx.x < row_blocks)) {
        if constexpr (MIX != Mix::Few)
            row_item<DT, DC, ROWS>(a, row, blockIdx.x, *reinterpret_cast<RowShared<DC>*>(lds));
    } else if constexpr (MIX != Mix::Many) {
        key_item<DT, DC, waves>(a, key, blockIdx.x - row_blocks,
                                *reinterpret_cast<KeyShared<DC, waves>*>(lds));
    }
    no_request<DT>(a, end);
}

// ---------------------------------------------------------------- fp32 rows

// Queries in fp32 keep their 24 bits, which the int8 products do not hold: fp32 sums on the vector
// units.  A workgroup has up to four rows of a key head, so a converted code serves all of them;
// its waves take every fourth 64-key tile and are joined at the end.  For the scores a lane has a
// key and q comes from scalar registers; for the values it has up to four d, and the weights pass
// through LDS.  Vector products bound it: 4 x 512 tokens over 2048 (60 GF) 1191 us, 50 Tflop/s; 64
// tokens over 9000 315 us (3.7 TB/s); one over 32768 42 us.
constexpr int kFloatRows = kWaves;  // at the end a wave has a row
constexpr float kLargest = 3e38f;

template <int DC> struct FloatShared {
    float p[kWaves][kFloatRows][64];
    float o[kWaves][kFloatRows][64 * DC];
    float m[kWaves][kFloatRows], l[kWaves][kFloatRows];
};

typedef const float __attribute__((address_space(4)))* scalar_floats;  // read by all lanes alike

template <int DC, bool ROWS>
__device__ __forceinline__ void float_item(const AttnArgs& a, const Cut& c, FloatShared<DC>& sh) {
    constexpr int DP = 64 * DC, NR = kFloatRows;
    const KvCache& kv = a.cache;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Item it;
    if (!block_item<ROWS, kF32>(a, c, blockIdx.x, it)) return;
    const float to_log2 = a.scale * kLog2e;
    int hi[NR], lo[NR];
    scalar_floats q[NR];
    float m[NR], l[NR], acc[NR][DC];
    int64_t at[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        int tok, head;
        row_at(a, c, it, r < it.rows ? r : 0, tok, head);
        const int place = it.before + tok;
        hi[r] = max(0, min(place + 1, it.len));
        lo[r] = a.shape.window ? max(0, place + 1 - a.shape.window) : 0;
        const int64_t token = it.q0 + it.tok0 + tok;
        q[r] = (scalar_floats)(static_cast<const float*>(a.q.p) + token * a.q.token + head * a.q.head);
        at[r] = token * a.shape.heads + head;
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int i = 0; i < DC; ++i) acc[r][i] = 0.f;
    }
    const int32_t* pages = a.tables + it.r * a.table_ld;
    const int inside = (1 << kv.log_block) - 1;
    for (int t = it.t0 + wave; t < it.t1; t += kWaves) {
        const int j = 64 * t + lane;
        int b = j < it.end_key ? pages[j >> kv.log_block] : -1;
        const bool have = b >= 0 && b < kv.blocks;
        const uint64_t there = __ballot(have);
        if (!there) continue;
        if (!have) b = 0;  // read, not used
        const int tok = j & inside;
        const int8_t* k = kv.k + kv.at(b, it.head) + (tok >> 4) * 16 * DP + ((tok & 15) >> 2) * 256 +
                          (tok & 3) * 16;
        const float2 scales = *reinterpret_cast<const float2*>(kv.scales + kv.scale_at(b, it.head));
        float s[NR] = {};
        for (int d0 = 0; d0 < a.shape.d; d0 += 16) {
            const uint4 w4 = *reinterpret_cast<const uint4*>(k + (d0 >> 6) * 1024 + (d0 & 63) * 4);
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3)));
            if (d0 + 16 <= a.shape.d) {
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[r] = __builtin_fmaf(x[i], q[r][d0 + i], s[r]);
            } else {
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (d0 + i < a.shape.d) s[r] = __builtin_fmaf(x[i], q[r][d0 + i], s[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const bool sees = have && j >= lo[r] && j < hi[r];
            // finite, so a row that sees a key has a weight of 1; NaN becomes so too, and the row's
            // end writes NaN
            const float x = sees ? __builtin_amdgcn_fmed3f(s[r] * scales.x * to_log2, -kLargest, kLargest)
                                 : -INFINITY;
            const float next = fmaxf(m[r], wave_max(x));
            const bool none = next == -INFINITY;
            const float keep = none ? 1.f : exp2f(m[r] - next);
            const float w = none ? 0.f : exp2f(x - next);
            m[r] = next;
            l[r] = __builtin_fmaf(l[r], keep, w);
            sh.p[wave][r][lane] = w * scales.y;
#pragma unroll
            for (int i = 0; i < DC; ++i) acc[r][i] *= keep;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int g = 0; g < 4; ++g) {
            // the 16 tokens share a block, whichever of them is there
            const uint64_t those = there >> (16 * g) & 0xFFFFu;
            if (!those) continue;
            const int from = __builtin_amdgcn_readlane(b, 16 * g + __builtin_ctzll(those));
            const int8_t* v = kv.v + kv.at(from, it.head) + (((64 * t + 16 * g) & inside) >> 4) * 16 * DP;
            uint4 code[DC];
#pragma unroll
            for (int i = 0; i < DC; ++i)
                code[i] = *reinterpret_cast<const uint4*>(v + (lane + 64 * i) * 16);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                float4 p[NR];
#pragma unroll
                for (int r = 0; r < NR; ++r)
                    p[r] = *reinterpret_cast<const float4*>(&sh.p[wave][r][16 * g + 4 * n]);
#pragma unroll
                for (int i = 0; i < DC; ++i) {
                    const uint32_t w = n == 0 ? code[i].x : n == 1 ? code[i].y
                                     : n == 2 ? code[i].z : code[i].w;
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        acc[r][i] = __builtin_fmaf(p[r].x, (float)(int8_t)w, acc[r][i]);
                        acc[r][i] = __builtin_fmaf(p[r].y, (float)(int8_t)(w >> 8), acc[r][i]);
                        acc[r][i] = __builtin_fmaf(p[r].z, (float)(int8_t)(w >> 16), acc[r][i]);
                        acc[r][i] = __builtin_fmaf(p[r].w, (float)(int8_t)(w >> 24), acc[r][i]);
                    }
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const float sum = wave_sum(l[r]);
        if (lane == 0) {
            sh.m[wave][r] = m[r];
            sh.l[wave][r] = sum;
        }
#pragma unroll
        for (int i = 0; i < DC; ++i) sh.o[wave][r][lane + 64 * i] = acc[r][i];
    }
    __syncthreads();
    if (wave >= it.rows) return;
    // row `wave`
    int64_t mine = at[0];
    scalar_floats mine_q = q[0];
#pragma unroll
    for (int r = 1; r < NR; ++r)
        if (wave == r) {
            mine = at[r];
            mine_q = q[r];
        }
    bool bad = false;
    for (int d = lane; d < a.shape.d; d += 64) bad |= !(fabsf(mine_q[d] * to_log2) < INFINITY);
    bad = __any(bad);
    float top = -INFINITY, sum = 0.f, o[DC] = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, sh.m[w][wave]);
    const bool some = top != -INFINITY;
    if (some) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = exp2f(sh.m[w][wave] - top);
            sum = __builtin_fmaf(f, sh.l[w][wave], sum);
#pragma unroll
            for (int i = 0; i < DC; ++i) o[i] = __builtin_fmaf(f, sh.o[w][wave][lane + 64 * i], o[i]);
        }
    }
    const float nan = __uint_as_float(0x7FC00000u);
    if (it.parts > 1) {
        if (lane == 0) c.ml[it.stored + wave] = make_float2(bad && some ? nan : top, sum);
        if (!some) return;
#pragma unroll
        for (int i = 0; i < DC; ++i) c.part[(it.stored + wave) * DP + lane + 64 * i] = o[i];
        return;
    }
#pragma unroll
    for (int i = 0; i < DC; ++i) {
        const int d = lane + 64 * i;
        if (d < a.shape.d)
            static_cast<float*>(a.out)[mine * a.shape.d + d] = !some ? 0.f : bad ? nan : o[i] / sum;
    }
    if (a.lse && lane == 0) a.lse[mine] = !some ? -INFINITY : bad ? nan : (top + log2f(sum)) * kLn2;
}

template <int DC, bool ROWS>
__global__ __launch_bounds__(kThreads) void float_kernel(AttnArgs a, Cut c) {
    __shared__ __align__(16) FloatShared<DC> sh;
    const int end = last_start(a);
    float_item<DC, ROWS>(a, c, sh);
    no_request<kF32>(a, end);
}

// ---------------------------------------------------------------- the parts' join

// Joins the parts of an item's rows from `first` on, a wave per row: lane s has part s's maximum
// and sum.
template <int DT, int DC, bool ROWS>
__device__ __forceinline__ void join_item(const AttnArgs& a, const Cut& c, int id, int first, int step) {
    constexpr int DP = 64 * DC;
    const int lane = threadIdx.x & 63;
    Item it;
    if (!find_item<ROWS, DT, false>(a, c, id, 0, it) || it.parts <= 1) return;
    const int64_t stride = (int64_t)(id < c.whole ? c.whole : c.items - c.whole) * c.rows;
    const float nan = __uint_as_float(0x7FC00000u);
    for (int row = first + (threadIdx.x >> 6); row < it.rows; row += step) {
        const int64_t at0 = it.stored + row;
        float2 ml = make_float2(-INFINITY, 0.f);
        if (lane < it.parts) ml = c.ml[at0 + lane * stride];
        const bool some = ml.y > 0.f;
        const bool bad = __any(some && ml.x != ml.x);
        // a part with a key has a finite reference, in fp32 also one under kNone
        const float m = wave_max(some && !bad ? ml.x : -INFINITY);
        const float keep = some && !bad ? fast_exp2(ml.x - m) : 0.f;
        const float l = wave_sum(keep * ml.y);
        float sum[DC];
#pragma unroll
        for (int i = 0; i < DC; ++i) sum[i] = 0.f;
        const uint64_t used = __ballot(some && !bad);
        const float* p = c.part + at0 * DP + lane;
        // four parts' loads at a time; where a part has no key for a row it has written nothing
        for (int s0 = 0; s0 < it.parts; s0 += 4) {
            float v[4][DC];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < DC; ++i)
                    v[j][i] = used >> (s0 + j) & 1 ? p[(s0 + j) * stride * DP + 64 * i] : 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float f = __shfl(keep, s0 + j);
#pragma unroll
                for (int i = 0; i < DC; ++i) sum[i] = __builtin_fmaf(v[j][i], f, sum[i]);
            }
        }
        int tok, head;
        row_at(a, c, it, row, tok, head);
        const int64_t at = (int64_t)(it.q0 + it.tok0 + tok) * a.shape.heads + head;
        const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
        for (int i = 0; i < DC; ++i) {
            const int d = lane + 64 * i;
            if (d < a.shape.d) store_from_f32<DT>(a.out, at * a.shape.d + d, bad ? nan : sum[i] * inv);
        }
        if (a.lse && lane == 0)
            a.lse[at] = bad ? nan : l > 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
    }
}

template <int DT, int DC>
__global__ __launch_bounds__(kThreads) void join_kernel(AttnArgs a, Cut key, Cut row, int row_blocks) {
    const int b = blockIdx.x;
    // items that can have parts: all, or the last ones
    if (b < row_blocks)
        return join_item<DT, DC, true>(a, row, (row.parts[0] > 1 ? 0 : row.whole) + b / row.joins,
                                       b % row.joins * kWaves, row.joins * kWaves);
    join_item<DT, DC, false>(a, key, (key.parts[0] > 1 ? 0 : key.whole) + b - row_blocks, 0, kWaves);
}

// ---------------------------------------------------------------- how a call is cut

// Rows of a request and key head up to which it is done in tiles of 16 with the keys split over
// the waves, each tile reading the keys again (50 requests of up to 36 rows over up to 7700 keys:
// 91 us, 156 with rows split over the waves; 16 requests of 64 rows over 2000 keys: 52 to 36).
constexpr int kFewRows = 48;
constexpr int kMaxParts = 64;
constexpr int kUncut = 1 << 30;

struct Plan {
    Mix mix;
    Cut key, row;
    bool has_key, has_row;
};

// 64-key tiles of the longest range that rows of `tok` tokens see.
int64_t key_tiles(const AttnShape& s, int tok) {
    int64_t keys = s.max_seq;
    if (s.window && (int64_t)s.window + tok < keys) keys = s.window + tok;
    return (keys + 63) / 64 + 1;
}

// each: tiles of every request; 0: as many as its tokens need.
void set_cut(Cut& c, const AttnShape& s, int rows, int each) {
    const int group = s.heads / s.kv_heads;
    c.rows = rows;
    c.tok = group <= rows ? rows / group : 1;
    c.subs = group <= rows ? 1 : (group + rows - 1) / rows;
    c.joins = rows < 32 ? 1 : rows / 16;
    c.each = each;
    c.tiles = each ? (int64_t)s.requests * each : (int64_t)s.requests + s.tokens / c.tok;
}

void set_parts(Cut& c, int kind, int64_t per, int64_t tiles) {
    if (per * kMaxParts < tiles) per = (tiles + kMaxParts - 1) / kMaxParts;
    const int64_t n = (tiles + per - 1) / per;
    c.per[kind] = (int)per;
    c.parts[kind] = n < 1 ? 1 : (int)n;
}

int64_t at_least(int64_t a, int64_t b) { return a < b ? b : a; }

// false: more items than a launch can number
bool plan_of(const AttnShape& s, Plan& p) {
    const int group = s.heads / s.kv_heads;
    const int64_t most = (int64_t)s.max_query * group;  // rows of a request and key head
    p.mix = most <= kFewRows || s.max_query <= 1 ? Mix::Few
            // all requests of the longest length?
            : (int64_t)s.requests * s.max_query == s.tokens ? Mix::Many
                                                            : Mix::Both;
    p.has_key = p.mix != Mix::Many;
    p.has_row = p.mix != Mix::Few;
    auto count = [&](Cut& c) {
        const int64_t n = (int64_t)c.subs * s.kv_heads;
        c.items = (int)(c.tiles * n);
        return c.tiles <= INT32_MAX / n;
    };
    if (s.dtype == kF32) {
        // Parts for some waves on every SIMD, of a tile a wave at least.
        const bool single = s.max_query <= 1;
        p.mix = single ? Mix::Few : Mix::Many;
        p.has_key = single;
        p.has_row = !single;
        Cut& c = single ? p.key : p.row;
        set_cut(c, s, kFloatRows, single ? 1 : 0);
        c.small = single ? INT32_MAX : 0;
        if (!count(c)) return false;
        const int64_t tiles = key_tiles(s, c.tok);
        set_parts(c, 1, at_least((c.items * tiles + 2047) / 2048, kWaves), tiles);
        c.parts[0] = 1;
        c.per[0] = kUncut;
        return true;
    }
    if (p.has_key) {
        Cut& c = p.key;
        const int tok = group <= 16 ? 16 / group : 1;
        set_cut(c, s, 16, p.mix == Mix::Both || s.max_query < 1 ? 1 : (s.max_query + tok - 1) / tok);
        c.small = p.mix == Mix::Both ? c.tok : INT32_MAX;
        if (!count(c)) return false;
        // Parts down to one tile a wave where the batch is too small to fill the GPU (one token
        // over 2048 keys: 9.7 us at 4 tiles a part, 12.6 at 16, 17.2 uncut), eight a wave where it
        // does (64 tokens over up to 16000: 132 us at 32, 157 at 4, whose waves mostly start up
        // and join).
        const int64_t tiles = key_tiles(s, c.tok);
        int64_t per = (c.items * tiles + 4095) / 4096;
        per = per < 4 ? 4 : per > 32 ? 32 : per;
        set_parts(c, 1, per, tiles);
        c.parts[0] = 1;
        c.per[0] = kUncut;
    }
    if (p.has_row) {
        Cut& c = p.row;
        // Workgroups at a time: two on each CU, one where a head needs more of its LDS.
        const int64_t slots = s.d <= 192 ? 512 : 256;
        // Tiles of 128 rows read and convert the keys for more rows (four chunks of up to 2048
        // tokens: 411 us, 535 at 64 rows, both on inputs used before); those of 64 are through theirs
        // sooner, so they are for batches of few tiles a slot (7 requests of 62 to 550 tokens: 14.8
        // us, 30.2 at 128).
        // Around 16 tiles a slot both come out alike.
        int64_t tiles = 0;
        for (int rows = s.d > 192 || (s.d <= 128 && most > 64) ? 128 : 64;; rows = 64) {
            set_cut(c, s, rows, 0);
            if (!count(c)) return false;
            tiles = key_tiles(s, c.tok);
            if (rows == 64 || s.d > 192 || c.items * tiles >= 16 * slots) break;
        }
        c.small = p.has_key ? p.key.small : 0;
        // Items of over half a slot's share are cut, which costs a store and a load of their rows
        // in fp32; small batches down to a few tiles, each of which takes over a microsecond.
        const int64_t share = at_least((c.items * tiles + 2 * slots - 1) / (2 * slots), 4);
        set_parts(c, 0, share, tiles);
        // The items that are left when the others have filled the slots some times over would leave
        // part of them idle: they are cut into as many parts as fill them best.
        c.whole = (int)(c.items >= slots ? c.items - c.items % slots : 0);
        const int64_t rest = c.items - c.whole;
        double best = 1e9;
        int64_t cuts = 1;
        for (int64_t n = 1; n <= 8; ++n) {
            const double cost = (double)((rest * n + slots - 1) / slots) / n + 0.03 * n;
            if (cost < best - 1e-9) {
                best = cost;
                cuts = n;
            }
        }
        const int64_t finer = at_least((tiles + cuts - 1) / cuts, 16);
        set_parts(c, 1, c.whole && finer < share ? finer : share, tiles);
    }
    return true;
}

int64_t blocks_of(const Cut& c) {
    return (int64_t)c.whole * c.parts[0] + (int64_t)(c.items - c.whole) * c.parts[1];
}

int64_t items_in_parts(const Cut& c) {
    return (c.parts[0] > 1 ? c.whole : 0) + (c.parts[1] > 1 ? c.items - c.whole : 0);
}

size_t stored_rows(const Cut& c) {
    return ((c.parts[0] > 1 ? (size_t)c.whole * c.parts[0] : 0) +
            (c.parts[1] > 1 ? (size_t)(c.items - c.whole) * c.parts[1] : 0)) * c.rows;
}

size_t row_bytes(const AttnShape& s) { return (s.d + 63) / 64 * 64 * sizeof(float); }

size_t cut_bytes(const Cut& c, const AttnShape& s) {
    return stored_rows(c) * (row_bytes(s) + sizeof(float2));
}

// The cut's part of the workspace, which it moves past; as many parts as fit.  (Fewer than the
// workspace was asked for may be needed and more: a longer max_seq_len than the table's makes longer
// parts.  One token over 16128 keys under a max_seq_len of 131072, 64 parts of 4 tiles where 63 fit:
// 16.0 us, 69.9 uncut.)
void place(Cut& c, const AttnShape& s, char*& ws, size_t& left) {
    size_t need = cut_bytes(c, s);
    while (need > left && items_in_parts(c) > 0) {
        const int kind = c.parts[0] > c.parts[1] ? 0 : 1;
        const int64_t tiles = (int64_t)c.per[kind] * c.parts[kind];
        const int fewer = c.parts[kind] - 1;
        c.per[kind] = fewer > 1 ? (int)((tiles + fewer - 1) / fewer) : kUncut;
        c.parts[kind] = fewer;
        need = cut_bytes(c, s);
    }
    c.part = reinterpret_cast<float*>(ws);
    c.ml = reinterpret_cast<float2*>(ws + stored_rows(c) * row_bytes(s));
    ws += need;
    left -= need;
}

template <int DT, int DC, int ROWS>
void attend(const AttnArgs& a, const Plan& p, int row_blocks, int key_blocks, hipStream_t stream) {
    constexpr int few = 64 * waves_of(DC, Mix::Few, ROWS), many = 64 * waves_of(DC, Mix::Many, ROWS);
    bool both = p.mix == Mix::Both;
    if constexpr (DC <= 2) {
        if (both)
            attend_kernel<DT, DC, Mix::Both, ROWS>
                <<<row_blocks + key_blocks, many, 0, stream>>>(a, p.key, p.row, row_blocks);
    } else if (both) {
        both = false;  // of large heads the few rows' code takes more registers: a launch each
    }
    if (!both && p.has_row)
        attend_kernel<DT, DC, Mix::Many, ROWS>
            <<<row_blocks, many, 0, stream>>>(a, p.key, p.row, row_blocks);
    if (!both && p.has_key)
        attend_kernel<DT, DC, Mix::Few, 0><<<key_blocks, few, 0, stream>>>(a, p.key, p.row, 0);
}

template <int DT, int DC>
hipError_t run(const AttnArgs& a, const Plan& p, hipStream_t stream) {
    const int64_t row_blocks = p.has_row ? blocks_of(p.row) : 0;
    const int64_t key_blocks = p.has_key ? blocks_of(p.key) : 0;
    if (row_blocks + key_blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
    const int rb = (int)row_blocks, kb = (int)key_blocks;
    if constexpr (DT == kF32) {
        if (p.has_row)
            float_kernel<DC, true><<<rb, kThreads, 0, stream>>>(a, p.row);
        else
            float_kernel<DC, false><<<kb, kThreads, 0, stream>>>(a, p.key);
    } else {
        if constexpr (DC <= 2) {
            if (p.has_row && p.row.rows == 64) attend<DT, DC, 64>(a, p, rb, kb, stream);
            else attend<DT, DC, 128>(a, p, rb, kb, stream);
        } else {
            attend<DT, DC, DC == 3 ? 64 : 128>(a, p, rb, kb, stream);
        }
    }
    const int64_t row_joins = p.has_row ? items_in_parts(p.row) * p.row.joins : 0;
    const int64_t key_joins = p.has_key ? items_in_parts(p.key) : 0;
    if (row_joins + key_joins > 0x7FFFFFFF) return hipErrorInvalidValue;
    if (row_joins + key_joins > 0)
        join_kernel<DT, DC><<<(unsigned)(row_joins + key_joins), kThreads, 0, stream>>>(
            a, p.key, p.row, (int)row_joins);
    return hipGetLastError();
}

template <int DT> hipError_t run(const AttnArgs& a, const Plan& p, hipStream_t stream) {
    switch (a.cache.dp / 64) {
        case 1: return run<DT, 1>(a, p, stream);
        case 2: return run<DT, 2>(a, p, stream);
        case 3: return run<DT, 3>(a, p, stream);
        default: return run<DT, 4>(a, p, stream);
    }
}

}  // namespace

size_t kv8_attention_bytes(const AttnShape& s) {
    Plan p{};
    if (s.tokens == 0 || s.requests == 0 || !plan_of(s, p)) return 0;
    return (p.has_key ? cut_bytes(p.key, s) : 0) + (p.has_row ? cut_bytes(p.row, s) : 0);
}

hipError_t launch_kv8_attention(const AttnArgs& args, void* ws, size_t ws_bytes,
                                hipStream_t stream) {
    AttnArgs a = args;
    if (a.cache.blocks == 0) a.shape.max_seq = 0;  // nothing to see
    Plan p{};
    if (!plan_of(a.shape, p)) return hipErrorInvalidValue;
    char* at = static_cast<char*>(ws);
    size_t left = ws ? ws_bytes : 0;
    if (p.has_key) place(p.key, a.shape, at, left);
    if (p.has_row) place(p.row, a.shape, at, left);
    switch (a.shape.dtype) {
        case kF32: return run<kF32>(a, p, stream);
        case kF16: return run<kF16>(a, p, stream);
        default: return run<kBF16>(a, p, stream);
    }
}

}  // namespace ojx
