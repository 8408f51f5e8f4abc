// kv8_cache.hip -- the 8-bit paged key / value cache: block tables and slots of a step (plan),
// new tokens into the cache (append, also with positions rotated into keys and queries), blocks out
// of it (read).  Layout: include/ojasx_e8t.h.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "rotary_heads.h"

namespace ojx {

namespace {

constexpr int kWave = 64;

// ---------------------------------------------------------------- plan

constexpr int kPlanThreads = 1024;
constexpr int kPlanItems = 4;                            // requests per thread and pass
constexpr int kPlanChunk = kPlanThreads * kPlanItems;    // requests per pass
constexpr int kPlanTokens = kPlanThreads;                // tokens per workgroup

__device__ __forceinline__ int sat32(int64_t v) { return v > 0x7FFFFFFF ? 0x7FFFFFFF : (int)v; }

// Sums saturate: what lies past 2^32 - 1 is past every token and block anyway.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
    return __builtin_elementwise_add_sat(a, b);
}

// Exclusive sum of v over the workgroup; *total: the sum over all of it.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* totals, uint32_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const uint32_t up = __shfl_up(s, o);
        s = add_sat(s, lane >= o ? up : 0u);
    }
    uint32_t before = __shfl_up(s, 1);
    before = lane ? before : 0u;
    if (lane == 63) totals[wave] = s;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / kWave; ++w) {
        const uint32_t t = totals[w];
        before = add_sat(before, w < wave ? t : 0u);
        all = add_sat(all, t);
    }
    __syncthreads();
    *total = all;
    return before;
}

// Every workgroup sums up the requests by itself (a pass over kPlanChunk lengths is a few
// microseconds of latency, less than a second launch) and then maps its own tokens; the first
// one also writes the requests' results.  Latency bounds it: 5 us for 64 requests, 8.7 for 4096
// with 214000 tokens (3.4 MB written).
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a) {
    __shared__ int starts[kPlanChunk], held[kPlanChunk], firsts[kPlanChunk];
    __shared__ uint32_t totals[kPlanThreads / kWave];
    const int block = 1 << a.log_block;
    const int64_t t0 = (int64_t)blockIdx.x * kPlanTokens, t1 = t0 + kPlanTokens;
    const uint32_t tokens = a.tokens;
    const int nf = *a.num_free < a.capacity ? *a.num_free : a.capacity;
    uint32_t q_base = 0, need_base = 0;
    for (int64_t c = 0; c < a.requests; c += kPlanChunk) {
        int now[kPlanItems], old[kPlanItems];
        uint32_t q = 0, need = 0, total;
        const int64_t r0 = c + (int64_t)threadIdx.x * kPlanItems;
#pragma unroll
        for (int i = 0; i < kPlanItems; ++i) {
            const bool in = r0 + i < a.requests;
            now[i] = in ? max(a.new_lens[r0 + i], 0) : 0;
            old[i] = in ? max(a.seq_lens[r0 + i], 0) : 0;
            q = add_sat(q, now[i]);
        }
        uint32_t start = add_sat(q_base, block_scan(q, totals, &total));
        const uint32_t q_next = add_sat(q_base, total);
#pragma unroll
        for (int i = 0; i < kPlanItems; ++i) {
            // no more tokens than there is room for
            const uint32_t at = min(start, tokens);
            const int64_t fit = min((uint32_t)now[i], tokens - at);
            const int64_t have = ((int64_t)old[i] + block - 1) >> a.log_block;
            const int64_t want = (old[i] + fit + block - 1) >> a.log_block;
            const int k = threadIdx.x * kPlanItems + i;
            starts[k] = (int)at;
            held[k] = old[i];
            if (blockIdx.x == 0 && r0 + i < a.requests) {
                a.query_starts[r0 + i] = (int)at;
                a.seq_lens_out[r0 + i] = sat32(old[i] + fit);
            }
            start = add_sat(start, now[i]);
            now[i] = (int)((want < a.width ? want : a.width) - (have < a.width ? have : a.width));
            need = add_sat(need, now[i]);
        }
        uint32_t first = add_sat(need_base, block_scan(need, totals, &total));
        need_base = add_sat(need_base, total);
#pragma unroll
        for (int i = 0; i < kPlanItems; ++i) {
            firsts[threadIdx.x * kPlanItems + i] = (int)min(first, 0x7FFFFFFFu);
            first = add_sat(first, now[i]);
        }
        __syncthreads();
        // this workgroup's tokens among the pass's requests
        const int64_t lo = q_base > t0 ? q_base : t0;
        int64_t hi = q_next < t1 ? q_next : t1;
        hi = hi < a.tokens ? hi : a.tokens;
        const int count = (int)(a.requests - c < kPlanChunk ? a.requests - c : kPlanChunk);
        for (int64_t t = lo + threadIdx.x; t < hi; t += kPlanThreads) {
            int l = 0, h = count;  // the last request that begins at or before t
            while (h - l > 1) {
                const int m = (l + h) >> 1;
                if (starts[m] <= t) l = m; else h = m;
            }
            const int64_t pos = held[l] + (t - starts[l]);
            const int64_t j = pos >> a.log_block;
            int64_t have = ((int64_t)held[l] + block - 1) >> a.log_block;
            int32_t* row = a.tables + (c + l) * a.table_ld;
            int entry = -1;
            if (j < a.width) {
                if (j < have) {
                    entry = row[j];
                } else {
                    const int64_t at = nf - 1 - (firsts[l] + (j - have));
                    entry = at >= 0 ? a.free_blocks[at] : -1;
                    // the block's first token enters it in the table
                    if ((pos & (block - 1)) == 0) row[j] = entry;
                }
            }
            a.slots[t] = entry < 0 ? -1 : ((int64_t)entry << a.log_block) + (pos & (block - 1));
            a.positions[t] = sat32(pos);
            a.request_ids[t] = (int)(c + l);
        }
        __syncthreads();
        q_base = q_next;
        if (blockIdx.x != 0 && q_base >= t1) return;
    }
    const int64_t end = q_base < a.tokens ? q_base : a.tokens;
    for (int64_t t = (end > t0 ? end : t0) + threadIdx.x; t < t1 && t < a.tokens;
         t += kPlanThreads) {
        a.slots[t] = -1;
        a.positions[t] = -1;
        a.request_ids[t] = -1;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.query_starts[a.requests] = (int)end;
        const int64_t left = (int64_t)nf - need_base;
        a.num_free_out[0] = left < -0x7FFFFFFF ? -0x7FFFFFFF : (int)left;
    }
}

// ---------------------------------------------------------------- append

constexpr int kAppendWaves = 4;
constexpr int64_t kAppendBlocks = 1024;
constexpr float kTinyAmax = 0x1p-100f;
constexpr int64_t kAngles = 4096;  // of a workgroup that rotates keys
constexpr int kHalfStepHeads = 4;  // of a thread that rotates queries by 8 bytes

template <int DT> __device__ __forceinline__ float elem(const void* p, int64_t i) {
    return load_as_f32<DT>(p, i);
}

// 16 elements from e (a multiple of 16 bytes when VEC), those from n on as zeros
template <int DT, bool VEC>
__device__ __forceinline__ void load16(const void* p, int64_t e, int n, float (&x)[16]) {
    if constexpr (VEC && DT != kF32) {
        if (n >= 16) {
            const uint4* w = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + e);
            const uint4 lo = w[0], hi = w[1];
            const uint32_t u[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[2 * i] = DT == kBF16 ? bf16_bits_to_f32(u[i] & 0xFFFFu)
                                       : f16_bits_to_f32(u[i] & 0xFFFFu);
                x[2 * i + 1] = DT == kBF16 ? bf16_bits_to_f32(u[i] >> 16)
                                           : f16_bits_to_f32(u[i] >> 16);
            }
            return;
        }
    }
    if constexpr (VEC && DT == kF32) {
        if (n >= 16) {
            const float4* w = reinterpret_cast<const float4*>(static_cast<const float*>(p) + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 f = w[i];
                x[4 * i] = f.x; x[4 * i + 1] = f.y; x[4 * i + 2] = f.z; x[4 * i + 3] = f.w;
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = i < n ? elem<DT>(p, e + i) : 0.f;
}

// Largest finite |element|.
__device__ __forceinline__ float amax16(float m, const float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float a = fabsf(x[i]);
        m = a < INFINITY ? fmaxf(m, a) : m;  // false for NaN
    }
    return m;
}

// The code of x: nearest integer to x / scale within +-127; NaN (also inf * 0) is 0.
__device__ __forceinline__ int code_of(float x, float inverse) {
    const float f = x * inverse;
    return f == f ? (int)fminf(fmaxf(rintf(f), -127.f), 127.f) : 0;
}

__device__ __forceinline__ int recode(int code, float ratio) {
    return (int)rintf((float)code * ratio);
}

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 |
           (uint32_t)d << 24;
}

__device__ __forceinline__ int byte_of(uint32_t w, int i) { return (int8_t)(w >> (8 * i)); }

// byte offset of key chunk c (16 elements) of token t within its block and head
__device__ __forceinline__ int key_at(int t, int c, int dp) {
    return (t >> 4) * 16 * dp + (c >> 2) * 1024 + ((t & 15) >> 2) * 256 + (c & 3) * 64 +
           (t & 3) * 16;
}

// One wave writes one run (the call's tokens of one block) for one head, keys or values: a
// pass over the run for its largest element, one over it (now in the cache) for the codes.  For
// rows that append_held does not take: fp32, off the 16-byte grid, blocks of over 32768 elements.
template <int DT, bool VEC>
__device__ void append_run(const KvCache& c, const KvRows& src, bool values, int head, int64_t t0,
                           int n, int block, int off, int lane) {
    const void* x0 = src.p;
    const int64_t e0 = t0 * src.token + head * src.head;
    const int chunks = (c.d + 15) >> 4;
    float m = 0.f;
    for (int i = lane; i < n * chunks; i += kWave) {
        const int t = i / chunks, ch = i - t * chunks;
        float x[16];
        load16<DT, VEC>(x0, e0 + t * src.token + ch * 16, c.d - ch * 16, x);
        m = amax16(m, x);
    }
    m = wave_max(m);
    m = m < kTinyAmax ? 0.f : m;
    float* sp = c.scales + c.scale_at(block, head) + values;
    const float before = off > 0 ? *sp : 0.f;
    const float scale = fmaxf(before, m * (1.f / 127.f));
    const float inverse = scale > 0.f ? 1.f / scale : 0.f;
    const float ratio = scale > 0.f ? before / scale : 0.f;
    const bool again = off > 0 && scale > before;  // earlier codes are rounded again
    if (lane == 0) *sp = scale;
    int8_t* base = (values ? c.v : c.k) + c.at(block, head);
    if (!values) {
        if (again) {
            for (int i = lane; i < off * chunks; i += kWave) {
                const int t = i / chunks, ch = i - t * chunks;
                uint4* p = reinterpret_cast<uint4*>(base + key_at(t, ch, c.dp));
                const uint4 o = *p;
                uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    w[j] = pack4(recode(byte_of(w[j], 0), ratio), recode(byte_of(w[j], 1), ratio),
                                 recode(byte_of(w[j], 2), ratio), recode(byte_of(w[j], 3), ratio));
                *p = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        for (int i = lane; i < n * chunks; i += kWave) {
            const int t = i / chunks, ch = i - t * chunks;
            float x[16];
            load16<DT, VEC>(x0, e0 + t * src.token + ch * 16, c.d - ch * 16, x);
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = pack4(code_of(x[4 * j], inverse), code_of(x[4 * j + 1], inverse),
                             code_of(x[4 * j + 2], inverse), code_of(x[4 * j + 3], inverse));
            *reinterpret_cast<uint4*>(base + key_at(off + t, ch, c.dp)) =
                make_uint4(w[0], w[1], w[2], w[3]);
        }
        return;
    }
    // 16 tokens of one d are 16 bytes: a lane has a d, and reads what the run does not fill
    const int end = off + n;
    for (int g = again ? 0 : off >> 4; g <= (end - 1) >> 4; ++g) {
        const int first = g * 16;
        const bool whole = first >= off && first + 16 <= end;
        for (int d = lane; d < c.d; d += kWave) {
            uint4* p = reinterpret_cast<uint4*>(base + (int64_t)g * 16 * c.dp + d * 16);
            const uint4 o = whole ? make_uint4(0, 0, 0, 0) : *p;
            uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                int b[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = first + 4 * j + i;
                    b[i] = byte_of(w[j], i);
                    if (t < off) {
                        if (again) b[i] = recode(b[i], ratio);
                    } else if (t < end) {
                        b[i] = code_of(elem<DT>(x0, e0 + (t - off) * src.token + d), inverse);
                    }
                }
                w[j] = pack4(b[0], b[1], b[2], b[3]);
            }
            *p = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                  __builtin_bit_cast(u16x2, b)));
}

template <int DT> __device__ __forceinline__ float half_to_f32(uint32_t bits) {
    return DT == kBF16 ? bf16_bits_to_f32(bits) : f16_bits_to_f32(bits);
}

// x times the inverse scale, rounded, as the low byte of a float: 1.5 * 2^23 is added to the
// rounded product (not fused with it), whose nearest integer then is the sum's low bits.
__device__ __forceinline__ uint32_t byte_float(float x, float inverse) {
#pragma clang fp contract(off)
    const float f = x * inverse;
    return __float_as_uint(f + 12582912.f);
}

// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t ab = __builtin_amdgcn_perm(b, a, 0x0C0C0400u);
    const uint32_t cd = __builtin_amdgcn_perm(d, c, 0x04000C0Cu);
    return ab | cd;
}

// Codes of eight elements; `plain`: all of the run's are finite.
__device__ __forceinline__ uint2 codes8(const float* x, float inverse, bool plain) {
    if (!plain)
        return make_uint2(pack4(code_of(x[0], inverse), code_of(x[1], inverse),
                                code_of(x[2], inverse), code_of(x[3], inverse)),
                          pack4(code_of(x[4], inverse), code_of(x[5], inverse),
                                code_of(x[6], inverse), code_of(x[7], inverse)));
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = byte_float(x[i], inverse);
    return make_uint2(low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7]));
}

template <int DT>
__device__ __forceinline__ uint2 codes8(const uint4& q, float inverse, bool plain) {
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = half_to_f32<DT>(u[i] & 0xFFFFu);
        x[2 * i + 1] = half_to_f32<DT>(u[i] >> 16);
    }
    return codes8(x, inverse, plain);
}

__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio) {
    return pack4(recode(byte_of(w, 0), ratio), recode(byte_of(w, 1), ratio),
                 recode(byte_of(w, 2), ratio), recode(byte_of(w, 3), ratio));
}

// u / d for u < 2^16: `inverse` is 2^32 / d rounded up.
__device__ __forceinline__ uint32_t inverse_of(int d) { return 0xFFFFFFFFu / (uint32_t)d + 1u; }
__device__ __forceinline__ int quotient(int u, uint32_t inverse, int d) {
    return d == 1 ? u : (int)__umulhi((uint32_t)u, inverse);
}

// Earlier codes of a block and head for its new scale, a few loads of 16 bytes in flight: keys
// of `off` tokens, or values of whole groups of 16 tokens (units have those of the run's first one).
__device__ __forceinline__ void recode_keys(int8_t* base, int off, int d, int dp, float ratio,
                                            int first, int step) {
    const int chunks = (d + 15) >> 4, total = off * chunks;
    const uint32_t inv = inverse_of(chunks);
    for (int i0 = first; i0 < total; i0 += 4 * step) {
        uint4* p[4];
        uint4 o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = min(i0 + j * step, total - 1), t = quotient(i, inv, chunks);
            p[j] = reinterpret_cast<uint4*>(base + key_at(t, i - t * chunks, dp));
            o[j] = *p[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + j * step < total)
                *p[j] = make_uint4(recode4(o[j].x, ratio), recode4(o[j].y, ratio),
                                   recode4(o[j].z, ratio), recode4(o[j].w, ratio));
    }
}

__device__ __forceinline__ void recode_values(int8_t* base, int groups, int d, int dp, float ratio,
                                              int first, int step) {
    const int total = groups * d;
    const uint32_t inv = inverse_of(d);
    for (int i0 = first; i0 < total; i0 += 4 * step) {
        uint4* p[4];
        uint4 o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = min(i0 + j * step, total - 1), g = quotient(i, inv, d);
            p[j] = reinterpret_cast<uint4*>(base + g * 16 * dp + (i - g * d) * 16);
            o[j] = *p[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + j * step < total)
                *p[j] = make_uint4(recode4(o[j].x, ratio), recode4(o[j].y, ratio),
                                   recode4(o[j].z, ratio), recode4(o[j].w, ratio));
    }
}

// append_run for 16-bit rows on a 16-byte grid, with the run held in registers between its
// maximum and its codes: HOLD loads of eight elements a lane, all in flight at once.  `waves`
// waves share a run (their maxima meet in LDS).  Lanes are laid out as the cache is, so that a
// store instruction fills whole stretches of it (a word in each of 40 lines took 37 us for
// 21500 tokens of 8 x 80 fp16 where reads and writes alone take 17): a key unit is 16 d of one
// token, lanes going through the 4 tokens of a quad first; a value unit is 8 d of a quad of
// tokens, lanes going through the 4 quads of a group first, and its bytes become 8 words of 4
// tokens.  Words that the run does not fill are read first.  What bounds it is the latency of one
// load, one maximum and one store after the other: 29 us for 21500 tokens of 8 x 80 fp16 (83 MB of
// rows and codes, 2.8 TB/s), 5 to 7 us for a token of each of 64 requests.
template <int DT, int HOLD, int WAVES>
__device__ __forceinline__ void append_held(const KvCache& c, const KvRows& src, bool values, int head,
                                            int64_t t0, int n, int block, int off, int lane, int wave,
                                            uint32_t* shared) {
    const uint16_t* x0 = static_cast<const uint16_t*>(src.p) + t0 * src.token + head * src.head;
    const int d8 = c.d >> 3, chunks = (c.d + 15) >> 4, first = wave * 64 + lane;
    const int wide = values ? d8 : chunks;
    const uint32_t inv = inverse_of(wide);
    // quads of the block that units cover: for keys the run's, for values whole groups
    const int q0 = values ? off >> 4 << 2 : off >> 2;
    const int quads = (values ? ((off + n - 1) >> 4 << 2) + 4 : ((off + n - 1) >> 2) + 1) - q0;
    const int units = quads * wide * (values ? 1 : 4);
    float* sp = c.scales + c.scale_at(block, head) + values;
    const float before = off > 0 ? *sp : 0.f;
    int8_t* base = (values ? c.v : c.k) + c.at(block, head);
    // unit u: its place along d, and its quad of the block
    auto unit_of = [&](int u, int& quad, int& place) {
        const int w = u >> 2, i = quotient(w, inv, wide);
        place = w - i * wide;
        quad = q0 + (values ? 4 * i + (u & 3) : i);
    };
    uint4 w[HOLD];
    if (!values) {
#pragma unroll
        for (int i = 0; i < HOLD; i += 2) {
            const int u = first + (i >> 1) * 64 * WAVES;
            int q, ch;
            unit_of(u, q, ch);
            const int t = 4 * q + (u & 3) - off;
            const bool in = u < units && t >= 0 && t < n;
            const uint16_t* p = x0 + t * src.token + ch * 16;
            w[i] = w[i + 1] = make_uint4(0, 0, 0, 0);
            if (in) w[i] = *reinterpret_cast<const uint4*>(p);
            if (in && 2 * ch + 1 < d8) w[i + 1] = *reinterpret_cast<const uint4*>(p + 8);
        }
    } else {
#pragma unroll
        for (int i = 0; i < HOLD; i += 4) {
            const int u = first + (i >> 2) * 64 * WAVES;
            int q, d;
            unit_of(u, q, d);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = 4 * q + j - off;
                w[i + j] = make_uint4(0, 0, 0, 0);
                if (u < units && t >= 0 && t < n)
                    w[i + j] = *reinterpret_cast<const uint4*>(x0 + t * src.token + d * 8);
            }
        }
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
        const uint32_t a = max_pair(w[i].x & 0x7FFF7FFFu, w[i].y & 0x7FFF7FFFu);
        const uint32_t b = max_pair(w[i].z & 0x7FFF7FFFu, w[i].w & 0x7FFF7FFFu);
        m = max_pair(m, max_pair(a, b));
    }
    // largest over the run of `bits`, pairs of 16 bits
    auto run_max = [&](uint32_t v) {
        uint32_t b = (uint32_t)wave_max((float)max(v & 0xFFFFu, v >> 16));
        if constexpr (WAVES > 1) {
            __syncthreads();
            if (lane == 0) shared[wave] = b;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < WAVES; ++i) b = max(b, shared[i]);
        }
        return b;
    };
    constexpr uint32_t inf = DT == kBF16 ? 0x7F80u : 0x7C00u;
    uint32_t top = run_max(m);
    const bool plain = top < inf;
    if (!plain) {  // finite elements only
        m = 0;
#pragma unroll
        for (int i = 0; i < HOLD; ++i) {
            const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t lo = u[j] & 0x7FFFu, hi = u[j] >> 16 & 0x7FFFu;
                m = max(m, lo < inf ? lo : 0u);
                m = max(m, hi < inf ? hi : 0u);
            }
        }
        top = run_max(m);
    }
    float largest = half_to_f32<DT>(top);
    largest = largest < kTinyAmax ? 0.f : largest;
    const float scale = fmaxf(before, largest * (1.f / 127.f));
    const float inverse = scale > 0.f ? 1.f / scale : 0.f;
    const float ratio = scale > 0.f ? before / scale : 0.f;
    const bool again = off > 0 && scale > before;
    if (lane == 0 && wave == 0) *sp = scale;
    if (!values) {
        if (again) recode_keys(base, off, c.d, c.dp, ratio, first, 64 * WAVES);
#pragma unroll
        for (int i = 0; i < HOLD; i += 2) {
            const int u = first + (i >> 1) * 64 * WAVES;
            if (u >= units) break;
            int q, ch;
            unit_of(u, q, ch);
            const int t = 4 * q + (u & 3);
            const uint2 lo = codes8<DT>(w[i], inverse, plain), hi = codes8<DT>(w[i + 1], inverse, plain);
            if (t >= off && t < off + n)
                *reinterpret_cast<uint4*>(base + key_at(t, ch, c.dp)) = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
        return;
    }
    if (again) recode_values(base, q0 >> 2, c.d, c.dp, ratio, first, 64 * WAVES);
#pragma unroll
    for (int i = 0; i < HOLD; i += 4) {
        const int u = first + (i >> 2) * 64 * WAVES;
        if (u >= units) break;
        int q, d;
        unit_of(u, q, d);
        uint32_t row[4][2];
        uint32_t fresh = 0;  // bytes of a word that the run fills
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint2 b = codes8<DT>(w[i + j], inverse, plain);
            row[j][0] = b.x;
            row[j][1] = b.y;
            const int t = 4 * q + j;
            fresh |= t >= off && t < off + n ? 0xFFu << (8 * j) : 0u;
        }
        // words of a group beside the run: of earlier tokens only to be rounded again
        if (fresh == 0 && !(again && 4 * q < off)) continue;
        int8_t* p = base + (q >> 2) * 16 * c.dp + d * 128 + (q & 3) * 4;
        uint32_t word[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // 4 tokens of 4 d -> 4 d of 4 tokens
            const uint32_t a = __builtin_amdgcn_perm(row[1][h], row[0][h], 0x05010400u);
            const uint32_t b = __builtin_amdgcn_perm(row[3][h], row[2][h], 0x05010400u);
            const uint32_t e = __builtin_amdgcn_perm(row[1][h], row[0][h], 0x07030602u);
            const uint32_t f = __builtin_amdgcn_perm(row[3][h], row[2][h], 0x07030602u);
            const uint32_t v[4] = {__builtin_amdgcn_perm(b, a, 0x05040100u),
                                   __builtin_amdgcn_perm(b, a, 0x07060302u),
                                   __builtin_amdgcn_perm(f, e, 0x05040100u),
                                   __builtin_amdgcn_perm(f, e, 0x07060302u)};
#pragma unroll
            for (int j = 0; j < 4; ++j) word[4 * h + j] = v[j];
        }
        uint32_t* o = reinterpret_cast<uint32_t*>(p);
        if (fresh == 0xFFFFFFFFu) {
#pragma unroll
            for (int j = 0; j < 8; ++j) o[4 * j] = word[j];
        } else {
            // bytes before the run, to be rounded again; those after it stay
            const uint32_t old = fresh ? (fresh & (0u - fresh)) - 1u : 0xFFFFFFFFu;
            uint32_t keep[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) keep[j] = o[4 * j];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (again) keep[j] = (recode4(keep[j], ratio) & old) | (keep[j] & ~old);
                o[4 * j] = (word[j] & fresh) | (keep[j] & ~fresh);
            }
        }
    }
}

// Cosines and sines of the workgroup's tokens t0 .. t0 + n - 1 into angles [n][pairs].
__device__ __forceinline__ void form_angles(const Rotation& rot, float2* angles, int64_t t0, int n) {
    const uint32_t inv = inverse_of(rot.pairs);
    for (int i = threadIdx.x; i < n * rot.pairs; i += kAppendWaves * kWave) {
        const int t = quotient(i, inv, rot.pairs);
        float2 a;
        pair_turn(rot, position_at(rot, t0 + t), rot.rates[i - t * rot.pairs], a.x, a.y);
        angles[i] = a;
    }
}

// Elements d0 .. d0 + 15 of a key (those from n on are zeros), the rotated ones among them turned.
template <int DT, bool VEC, bool INTERLEAVED>
__device__ __forceinline__ void load16_turned(const void* p, int64_t key, int d0, int n, int pairs,
                                              const float2* angles, float (&x)[16]) {
    load16<DT, VEC>(p, key + d0, n, x);
    if (d0 >= 2 * pairs) return;
#pragma unroll
    for (int i = 0; i < 16; i += INTERLEAVED ? 2 : 1) {
        const int d = d0 + i;
        if (d >= 2 * pairs) break;
        if constexpr (INTERLEAVED) {
            const float2 a = angles[d >> 1];
            turn_pair(a.x, a.y, x[i], x[i + 1]);
        } else {
            const bool hi = d >= pairs;
            const int pair = hi ? d - pairs : d;
            const float2 a = angles[pair];
            float other = elem<DT>(p, key + (hi ? pair : d + pairs));
            if (hi) turn_pair(a.x, a.y, other, x[i]);
            else turn_pair(a.x, a.y, x[i], other);
        }
    }
}

// A run's scale from its largest element, whose earlier codes are rounded again where it grew.
struct RunScale {
    float inverse;
    // first, step: of the lanes that share the run
    __device__ __forceinline__ RunScale(const KvCache& c, int8_t* base, float* sp, float before, float most,
                                        int off, int first, int step = kWave) {
        most = most < kTinyAmax ? 0.f : most;
        const float scale = fmaxf(before, most * (1.f / 127.f));
        inverse = scale > 0.f ? 1.f / scale : 0.f;
        const float ratio = scale > 0.f ? before / scale : 0.f;
        if (first == 0) *sp = scale;
        if (off > 0 && scale > before) recode_keys(base, off, c.d, c.dp, ratio, first, step);
    }
};

// Eight elements, 16 bytes or 32.
template <int DT> __device__ __forceinline__ void load8(const void* p, int64_t e, float* x) {
    if constexpr (DT == kF32) {
        const float4* w = reinterpret_cast<const float4*>(static_cast<const float*>(p) + e);
        const float4 lo = w[0], hi = w[1];
        x[0] = lo.x; x[1] = lo.y; x[2] = lo.z; x[3] = lo.w;
        x[4] = hi.x; x[5] = hi.y; x[6] = hi.z; x[7] = hi.w;
    } else {
        const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + e);
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = half_to_f32<DT>(v[j] & 0xFFFFu);
            x[2 * j + 1] = half_to_f32<DT>(v[j] >> 16);
        }
    }
}

// Units of a run of keys on the 16-byte grid: 8 pairs of one token, as two chunks of 8 elements, `pairs`
// apart or neighbours; behind them two chunks that are not rotated.
template <bool INTERLEAVED> struct KeyUnits {
    int d8, wide, apart, turned, pairs;
    uint32_t inv;
    __device__ __forceinline__ KeyUnits(int d, int p)
        : d8(d >> 3), wide((d8 + 1) >> 1), apart(INTERLEAVED ? 0 : p >> 3), turned(p >> 2), pairs(p),
          inv(inverse_of(wide)) {}
    // unit u of the quads from q on: its token of the block, and its chunks (the second may be past the
    // head's end)
    __device__ __forceinline__ void place(int u, int q, int& t, int& a, int& b) const {
        const int w = u >> 2, i = quotient(w, inv, wide), at = w - i * wide;
        t = 4 * (q + i) + (u & 3);
        a = at < apart ? at : 2 * at;
        b = at < apart ? at + apart : a + 1;
    }
    // angles: of the unit's token
    __device__ __forceinline__ void turn(float (&x)[16], int a, int b, const float2* angles) const {
        if (a >= turned) return;
        const float2* g = angles + (INTERLEAVED ? 4 * a : 8 * a);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (INTERLEAVED && j >= 4 && b >= turned) break;
            if constexpr (INTERLEAVED) turn_pair(g[j].x, g[j].y, x[2 * j], x[2 * j + 1]);
            else turn_pair(g[j].x, g[j].y, x[j], x[8 + j]);
        }
    }
    __device__ __forceinline__ void store(int8_t* base, int t, int a, int b, int dp, const float (&x)[16],
                                          float inverse, bool plain) const {
        const uint2 lo = codes8(x, inverse, plain), hi = codes8(x + 8, inverse, plain);
        int8_t* pa = base + key_at(t, a >> 1, dp);
        if (!(a & 1) && b == a + 1) {  // a whole place of 16, zeros behind an odd number of chunks
            *reinterpret_cast<uint4*>(pa) = make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
            *reinterpret_cast<uint2*>(pa + 8 * (a & 1)) = lo;
            *reinterpret_cast<uint2*>(base + key_at(t, b >> 1, dp) + 8 * (b & 1)) = hi;
        }
    }
};

// How rotated keys are gone through: element by element, by units, or by units that stay in registers.
enum Keys { kElements, kUnits, kHeldUnits };
constexpr int kHeld = 2;  // units of a lane then

// append_run or append_held of keys that are rotated on the way, one head by each wave of the workgroup
// (those past the last head only help with the angles).  Rotated keys are not rounded before they
// become codes: rounded to 16 bits in between, the largest codes would be a step off in one of five.
// Two passes over the run, one for its maximum, one for its codes, with the angles of as many tokens at
// a time as `room` holds; a run of at most 128 units is held as floats between them.  (Larger runs held
// took 256 registers, two waves a SIMD: a decode step of 64 tokens 8.1 us for 7.0.)  Of one or two heads,
// `share` waves take a run's units by turns.
template <int DT, bool VEC, Keys KEYS, bool INTERLEAVED>
__device__ __forceinline__ void append_turned(const KvCache& c, const KvRows& src, const Rotation& rot,
                                              float2* angles, int room, int head, int share, int part,
                                              uint32_t* shared, int64_t t0, int n, int block, int off,
                                              int lane) {
    const bool on = head < c.heads;
    int8_t* base = c.k + c.at(block, on ? head : 0);
    float* sp = c.scales + c.scale_at(block, on ? head : 0);
    const float before = on && off > 0 ? *sp : 0.f;
    const int64_t e0 = t0 * src.token + head * src.head;
    if constexpr (KEYS == kElements) {
        const int chunks = (c.d + 15) >> 4, pairs = rot.pairs, some = room / pairs;
        float m = 0.f, inverse = 0.f;
        for (int pass = 0; pass < 2; ++pass) {
            for (int c0 = 0; c0 < n; c0 += some) {
                const int part = min(some, n - c0);
                if (pass == 0 || n > some) {
                    __syncthreads();
                    form_angles(rot, angles, t0 + c0, part);
                    __syncthreads();
                }
                if (!on) continue;
                for (int i = lane; i < part * chunks; i += kWave) {
                    const int t = i / chunks, ch = i - t * chunks;
                    float x[16];
                    load16_turned<DT, VEC, INTERLEAVED>(src.p, e0 + (c0 + t) * src.token, ch * 16,
                                                        c.d - ch * 16, pairs, angles + t * pairs, x);
                    if (pass == 0) {
                        m = amax16(m, x);
                        continue;
                    }
                    const uint2 lo = codes8(x, inverse, false), hi = codes8(x + 8, inverse, false);
                    *reinterpret_cast<uint4*>(base + key_at(off + c0 + t, ch, c.dp)) =
                        make_uint4(lo.x, lo.y, hi.x, hi.y);
                }
            }
            if (pass == 0 && on) inverse = RunScale(c, base, sp, before, wave_max(m), off, lane).inverse;
        }
    } else {
        const KeyUnits<INTERLEAVED> k(c.d, rot.pairs);
        const int q0 = off >> 2, q1 = ((off + n - 1) >> 2) + 1;
        if constexpr (KEYS == kHeldUnits) {
            // the same in all lanes: a short run leaves the unrolled loops early
            const int units = __builtin_amdgcn_readfirstlane(on ? (q1 - q0) * k.wide * 4 : 0);
            float x[kHeld][16];
            bool in[kHeld];
            int t[kHeld], a[kHeld], b[kHeld];
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                if (i * 64 >= units) break;
                const int u = lane + i * 64;
                k.place(u, q0, t[i], a[i], b[i]);
                in[i] = u < units && t[i] >= off && t[i] < off + n;
                const int64_t e = e0 + (t[i] - off) * src.token;
#pragma unroll
                for (int j = 0; j < 16; ++j) x[i][j] = 0.f;
                if (in[i]) load8<DT>(src.p, e + 8 * a[i], x[i]);
                if (in[i] && b[i] < k.d8) load8<DT>(src.p, e + 8 * b[i], x[i] + 8);
            }
            __syncthreads();
            form_angles(rot, angles, t0, n);
            __syncthreads();
            uint32_t bits = 0;  // of the largest |element|: NaN and infinities are over all others
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                if (i * 64 >= units) break;
                if (in[i]) k.turn(x[i], a[i], b[i], angles + (t[i] - off) * k.pairs);
#pragma unroll
                for (int j = 0; j < 16; ++j) bits = max(bits, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
            }
            const bool plain = __all(bits < 0x7F800000u);
            float m = __uint_as_float(bits);
            if (!plain) {  // finite elements only
                m = 0.f;
#pragma unroll
                for (int i = 0; i < kHeld; ++i) {
                    if (i * 64 >= units) break;
                    m = amax16(m, x[i]);
                }
            }
            if (!on) return;
            const float inverse = RunScale(c, base, sp, before, wave_max(m), off, lane).inverse;
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                if (i * 64 >= units) break;
                if (in[i]) k.store(base, t[i], a[i], b[i], c.dp, x[i], inverse, plain);
            }
        } else {
            const int some = room / k.pairs >> 2;  // quads whose angles fit
            float m = 0.f, inverse = 0.f;
            bool plain = true;
            for (int pass = 0; pass < 2; ++pass) {
                for (int q = q0; q < q1; q += some) {
                    const int end = min(q + some, q1), lo = max(4 * q, off), hi = min(4 * end, off + n);
                    if (pass == 0 || q1 - q0 > some) {
                        __syncthreads();
                        form_angles(rot, angles, t0 + lo - off, hi - lo);
                        __syncthreads();
                    }
                    if (!on) continue;
                    const int units = (end - q) * k.wide * 4;
#pragma unroll 2
                    for (int u = part * kWave + lane; u < units; u += share * kWave) {
                        int t, a, b;
                        k.place(u, q, t, a, b);
                        if (t < lo || t >= hi) continue;
                        const int64_t e = e0 + (t - off) * src.token;
                        float x[16] = {};
                        load8<DT>(src.p, e + 8 * a, x);
                        if (b < k.d8) load8<DT>(src.p, e + 8 * b, x + 8);
                        k.turn(x, a, b, angles + (t - lo) * k.pairs);
                        if (pass == 1) {
                            k.store(base, t, a, b, c.dp, x, inverse, plain);
                            continue;
                        }
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float v = fabsf(x[j]);
                            plain &= v < INFINITY;
                            m = v < INFINITY ? fmaxf(m, v) : m;
                        }
                    }
                }
                if (pass == 1) break;
                m = wave_max(m);
                plain = __all(plain);
                if (share > 1) {  // the waves of a head
                    const int wave = threadIdx.x >> 6;
                    __syncthreads();
                    if (lane == 0) shared[wave] = __float_as_uint(m) | (plain ? 0u : 0x80000000u);
                    __syncthreads();
                    for (int w = wave - part; w < wave - part + share; ++w) {
                        m = fmaxf(m, fabsf(__uint_as_float(shared[w])));
                        plain &= !(shared[w] >> 31);
                    }
                }
                if (on)
                    inverse = RunScale(c, base, sp, before, m, off, part * kWave + lane, share * kWave).inverse;
            }
        }
    }
}

// Sizes of append_turned_kernel: its workgroups, windows and the angles that LDS has room for.
struct AppendTurned {
    int key_groups, value_groups, window, angles;
    int half_steps;  // queries are taken by 8 bytes, not by 16
    int64_t windows;
};

// Calls write(first token, tokens, block, offset) for each run that begins among the `window` tokens from
// w * window on, by a wave.  Runs end where the slots leave the block or skip.
template <class F>
__device__ __forceinline__ void find_runs(const KvCache& c, const int64_t* __restrict__ slots, int tokens,
                                          int window, int64_t w, int lane, F write) {
    const int64_t end = (int64_t)c.blocks << c.log_block;
    const int block = 1 << c.log_block;
    // lane i has the slot of token base + i - 1: the window's and what may follow it
    const int64_t base = w * window, t = base + lane - 1;
    int64_t slot = -1;
    if (t >= 0 && t < tokens) slot = slots[t];
    const int64_t prev = __shfl_up(slot, 1);
    const bool in = slot >= 0 && slot < end;
    const bool follows = in && lane > 0 && prev == slot - 1 && (slot & (block - 1)) != 0;
    const uint64_t more = __ballot(follows);
    uint64_t heads = __ballot(in && !follows && lane > 0 && lane <= window);
    while (heads) {
        const int i = __builtin_ctzll(heads);
        heads &= heads - 1;
        const int64_t t0 = base + i - 1;
        const int64_t s0 = __shfl(slot, i);
        const int off = (int)(s0 & (block - 1));
        const uint64_t after = i < 63 ? ~(more >> (i + 1)) : ~0ull;
        int n = 1 + __builtin_ctzll(after);
        if (i + n == 64) {  // it may go on past what the lanes hold
            while (n < block - off) {
                const int64_t tn = t0 + n + lane;
                const bool next = n + lane < block - off && tn < tokens && slots[tn] == s0 + n + lane;
                const uint64_t miss = ~__ballot(next);
                n += miss ? __builtin_ctzll(miss) : kWave;
                if (miss) break;
            }
        }
        write(t0, n, (int)(s0 >> c.log_block), off);
    }
}

// A wave (WAVES > 1: a workgroup) writes the runs of a window for one head, keys or values.
template <int DT, bool VEC, int HOLD, int WAVES>
__device__ __forceinline__ void append_unit(const KvCache& c, const KvRows& rows, bool values, int head,
                                            const int64_t* __restrict__ slots, int tokens, int window,
                                            int64_t w, int lane, int wave, uint32_t* shared) {
    find_runs(c, slots, tokens, window, w, lane, [&](int64_t t0, int n, int block, int off) {
        if constexpr (HOLD > 0)
            append_held<DT, HOLD, WAVES>(c, rows, values, head, t0, n, block, off, lane,
                                         WAVES > 1 ? wave : 0, shared);
        else
            append_run<DT, VEC>(c, rows, values, head, t0, n, block, off, lane);
    });
}

// Workgroups start at a few hundred a microsecond at most, so with many units each takes several.
template <int DT, bool VEC, int HOLD, int WAVES>
__global__ __launch_bounds__(kAppendWaves * kWave) void append_kernel(
    KvCache c, KvRows k, KvRows v, const int64_t* __restrict__ slots, int tokens, int window,
    int64_t units) {
    __shared__ uint32_t shared[WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t step = (int64_t)gridDim.x * (WAVES > 1 ? 1 : kAppendWaves);
    const int parts = 2 * c.heads;
    for (int64_t u = WAVES > 1 ? blockIdx.x : (int64_t)blockIdx.x * kAppendWaves + wave; u < units;
         u += step) {
        const int64_t w = u / parts;
        const int part = (int)(u - w * parts);
        append_unit<DT, VEC, HOLD, WAVES>(c, part & 1 ? v : k, part & 1, part >> 1, slots, tokens, window,
                                          w, lane, wave, shared);
    }
}

// Waves of a workgroup that share a head's keys, where there are fewer heads than waves, and the
// workgroups of a window.
__host__ __device__ __forceinline__ int waves_of_head(int heads) { return heads == 1 ? 4 : heads == 2 ? 2 : 1; }
__host__ __device__ __forceinline__ int key_groups(int heads, int share) {
    return (heads * share + kAppendWaves - 1) / kAppendWaves;
}

// Another order of each 8 workgroups, which run on 8 XCDs: where a block is several windows only every
// so many find a run, and in their own order these fell on one XCD or two (16000 tokens of 8 x 128 bf16 in
// blocks of 64, without queries: 149 us, 48 spread).
__device__ __forceinline__ int64_t spread(int64_t i) {
    const int64_t h = i >> 3;
    return i ^ ((h ^ (h >> 3) ^ (h >> 6)) & 7);
}

// append_kernel with rotated keys: workgroups for keys, for values, and behind them for queries.  A
// workgroup of keys takes a window's runs for as many heads as it has waves, whose angles it forms
// once, in LDS (prompts of 23446 tokens, 8 x 80 fp16 half of it rotated: 40 us, 50 where each wave formed
// its own; without a rotation 29).  What bounds it are vector instructions and append_held's chain of a
// load, a maximum and a store, four waves a SIMD, around which queries' workgroups find room: with 16
// heads of them 51 us, 62 in two launches (mixed among the others, so that they start together, slower).
template <int DT, bool VEC, int HOLD, int WAVES, Keys KEYS, bool INTERLEAVED>
__global__ __launch_bounds__(kAppendWaves * kWave) void append_turned_kernel(
    KvCache c, KvRows k, KvRows v, const int64_t* __restrict__ slots, int tokens, AppendTurned p,
    RotaryArgs q) {
    extern __shared__ float2 angles[];
    __shared__ uint32_t shared[kAppendWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int at = blockIdx.x;
    if (at < p.key_groups) {
        const int share = KEYS == kUnits ? waves_of_head(c.heads) : 1, part = wave & (share - 1);
        const int groups = key_groups(c.heads, share);
        const int64_t units = p.windows * groups;
        for (int64_t i = at; i < ((units + 7) & ~7); i += p.key_groups) {
            const int64_t u = spread(i);
            if (u >= units) continue;
            const int64_t w = u / groups;
            const int head = ((int)(u - w * groups) * kAppendWaves + wave) / share;
            find_runs(c, slots, tokens, p.window, w, lane, [&](int64_t t0, int n, int block, int off) {
                append_turned<DT, VEC, KEYS, INTERLEAVED>(c, k, q.rot, angles, p.angles, head, share, part,
                                                           shared, t0, n, block, off, lane);
            });
        }
        return;
    }
    at -= p.key_groups;
    if (at < p.value_groups) {
        constexpr int EACH = WAVES > 1 ? 1 : kAppendWaves;  // units of a workgroup
        const int64_t units = p.windows * c.heads, parts = (units + EACH - 1) / EACH;
        for (int64_t i = at; i < ((parts + 7) & ~7); i += p.value_groups) {
            const int64_t u = spread(i) * EACH + (WAVES > 1 ? 0 : wave);
            if (u >= units) continue;
            const int64_t w = u / c.heads;
            append_unit<DT, VEC, HOLD, WAVES>(c, v, true, (int)(u - w * c.heads), slots, tokens, p.window, w,
                                              lane, wave, shared);
        }
        return;
    }
    constexpr int STEP = DT == kF32 ? 4 : 8;
    if (p.half_steps) rotate_heads<DT, STEP / 2, INTERLEAVED, kHalfStepHeads>(q, at - p.value_groups);
    else rotate_heads<DT, STEP, INTERLEAVED>(q, at - p.value_groups);
}

// ---------------------------------------------------------------- read

// The value of a code: the fp32 product, rounded to DT.
template <int DT> __device__ __forceinline__ void store_value(void* p, int64_t i, int code, float s) {
    float v = (float)code * s;
    keep_f32(v);
    store_from_f32<DT>(p, i, v);
}

constexpr int kReadThreads = 256;
constexpr int kReadUnits = 4;  // per thread

// Eight values from their codes (in the low byte of each of eight words), 16 bytes and more.
template <int DT> __device__ __forceinline__ void store8(void* p, int64_t i, const int (&code)[8], float s) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        v[j] = (float)code[j] * s;
        keep_f32(v[j]);
    }
    if constexpr (DT == kF32) {
        float4* o = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
        o[0] = make_float4(v[0], v[1], v[2], v[3]);
        o[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            w[j] = DT == kF16 ? f32_to_f16_bits(v[2 * j]) | f32_to_f16_bits(v[2 * j + 1]) << 16
                              : bf16_bits_hw(v[2 * j]) | bf16_bits_hw(v[2 * j + 1]) << 16;
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// One block's keys or values per blockIdx.x, a share of its units per blockIdx.y.  The output's
// order (token, head, d) is the units': 8 d of a token's key, or of 4 tokens' values, whose
// codes are 8 words of 4 tokens.  WIDE: d a multiple of 8, else a unit is a single element.  23 us
// for the blocks of 21500 tokens of 8 x 80 fp16 (83 MB read and written, 3.6 TB/s, three quarters of
// a copy's rate): memory, and two divisions and a scale's load ahead of every unit's.
template <int DT, bool WIDE>
__global__ __launch_bounds__(kReadThreads) void read_kernel(KvCache c,
                                                            const int32_t* __restrict__ blocks,
                                                            void* k_out, void* v_out,
                                                            float* scales_out) {
    const int64_t i = blockIdx.x >> 1;
    const int values = blockIdx.x & 1;
    const int b = blocks[i], size = 1 << c.log_block;
    const bool in = b >= 0 && b < c.blocks;
    const int8_t* base = (values ? c.v : c.k) + (in ? c.at(b, 0) : 0);
    const float* scales = c.scales + (in ? c.scale_at(b, 0) : 0) + values;
    void* out = values ? v_out : k_out;
    const int per = WIDE ? c.d >> 3 : c.d;
    const int row = c.heads * per;
    const int units = (WIDE && values ? size >> 2 : size) * row;
    const int64_t head_bytes = c.head_bytes(), o0 = ((i << c.log_block) * c.heads) * c.d;
    const int64_t ot = (int64_t)c.heads * c.d;
    if (blockIdx.y == 0)
        for (int h = threadIdx.x; h < c.heads; h += kReadThreads)
            scales_out[(i * c.heads + h) * 2 + values] = in ? scales[2 * h] : 0.f;
    const int first = blockIdx.y * kReadThreads + threadIdx.x, step = gridDim.y * kReadThreads;
    // (token or quad, head, place in the head) of unit u; lanes go through a group's 4 quads of
    // values first, whose bytes are neighbours
    auto split = [&](int u, int& t, int& h, int& x) {
        const int w = WIDE && values ? u >> 2 : u;
        t = w / row;
        const int e = w - t * row;
        h = e / per;
        x = e - h * per;
        if (WIDE && values) t = 4 * t + (u & 3);
    };
    if (!WIDE || values) {
        for (int u = first; u < units; u += step) {
            int t, h, x;
            split(u, t, h, x);
            const int8_t* p = base + h * head_bytes;
            const float s = in ? scales[2 * h] : 0.f;
            const int64_t o = o0 + h * c.d;
            if constexpr (!WIDE) {
                const int at = values ? (t >> 4) * 16 * c.dp + x * 16 + (t & 15)
                                      : key_at(t, x >> 4, c.dp) + (x & 15);
                store_value<DT>(out, o + t * ot + x, in ? p[at] : 0, s);
            } else {
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    w[j] = in ? *reinterpret_cast<const uint32_t*>(p + (t >> 2) * 16 * c.dp +
                                                                  (x * 8 + j) * 16 + (t & 3) * 4)
                              : 0u;
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    int code[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) code[j] = byte_of(w[j], n);
                    store8<DT>(out, o + (4 * t + n) * ot + x * 8, code, s);
                }
            }
        }
        return;
    }
    for (int u0 = first; u0 < units; u0 += kReadUnits * step) {
        uint2 w[kReadUnits];
        float s[kReadUnits];
        int64_t o[kReadUnits];
#pragma unroll
        for (int i = 0; i < kReadUnits; ++i) {
            int t, h, x;
            split(min(u0 + i * step, units - 1), t, h, x);
            w[i] = make_uint2(0, 0);
            if (in)
                w[i] = *reinterpret_cast<const uint2*>(base + h * head_bytes +
                                                       key_at(t, x >> 1, c.dp) + (x & 1) * 8);
            s[i] = in ? scales[2 * h] : 0.f;
            o[i] = o0 + t * ot + h * c.d + x * 8;
        }
#pragma unroll
        for (int i = 0; i < kReadUnits; ++i) {
            int code[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) code[j] = byte_of(j < 4 ? w[i].x : w[i].y, j & 3);
            if (u0 + i * step < units) store8<DT>(out, o[i], code, s[i]);
        }
    }
}

bool rows_vector(const KvRows& r, int dtype) {
    const int64_t unit = dtype == kF32 ? 4 : 8;
    return ((uintptr_t)r.p & 15) == 0 && r.token % unit == 0 && r.head % unit == 0;
}

}  // namespace

hipError_t launch_kv8_plan(const PlanArgs& a, hipStream_t stream) {
    int64_t grid = ((int64_t)a.tokens + kPlanTokens - 1) / kPlanTokens;
    if (grid < 1) grid = 1;
    plan_kernel<<<(unsigned)grid, kPlanThreads, 0, stream>>>(a);
    return hipGetLastError();
}

namespace {

// How a call's rows are written.
struct AppendPlan {
    bool vec;     // 16 elements by 16 bytes
    bool hold;    // runs stay in registers
    bool shared;  // the workgroup's waves share a run
    int64_t held;
    int window;
    int64_t units;
    int64_t grid;
};

AppendPlan append_plan(const KvCache& c, const KvRows& k, const KvRows& v, int dtype, int tokens) {
    AppendPlan p;
    // Elements that a run's units cover at most: a key's are whole chunks of 16, so a head of 8
    // takes as much room as one of 16; values' units are never more.
    p.held = ((int64_t)c.d + 15) / 16 * 16 << c.log_block;
    p.vec = rows_vector(k, dtype) && rows_vector(v, dtype);
    // Rows that a run is held in registers of: 16-bit ones on a 16-byte grid (append and read of
    // 21500 tokens of 8 x 80: 43 us, 79 where they are read twice).  The others, fp32 among them,
    // are read twice, the second time from the cache.
    p.hold = p.vec && dtype != kF32 && c.d % 8 == 0 && p.held <= 32768;
    p.shared = p.hold && p.held > 8192;
    // A window per token fills the GPU for a decode step, whose tokens all begin runs (append and
    // read of 64 tokens 13 us, 47 with windows of 16); with many tokens most of such waves would
    // find none (21500 tokens 43 us, 189 with a window each).
    p.window = (int64_t)tokens * 2 * c.heads <= 16384 ? 1 : 16;
    p.units = ((int64_t)tokens + p.window - 1) / p.window * 2 * c.heads;
    p.grid = p.shared ? p.units : (p.units + kAppendWaves - 1) / kAppendWaves;
    p.grid = p.grid < kAppendBlocks ? p.grid : kAppendBlocks;
    return p;
}

template <class F> void by_dtype(int dtype, F go) {
    if (dtype == kF32) go(std::integral_constant<int, kF32>{});
    else if (dtype == kF16) go(std::integral_constant<int, kF16>{});
    else go(std::integral_constant<int, kBF16>{});
}

// Calls go(type, rows by 16 bytes, registers held, waves that share a run) for a plan.
template <class F> void by_plan(const AppendPlan& p, int dtype, F go) {
    using One = std::integral_constant<int, 1>;
    by_dtype(dtype, [&](auto dt) {
        if constexpr (decltype(dt)::value != kF32) {
            if (p.shared)
                go(dt, std::true_type{}, std::integral_constant<int, 16>{},
                   std::integral_constant<int, kAppendWaves>{});
            else if (p.hold && p.held > 2048)
                go(dt, std::true_type{}, std::integral_constant<int, 16>{}, One{});
            else if (p.hold)
                go(dt, std::true_type{}, std::integral_constant<int, 4>{}, One{});
            if (p.hold) return;
        }
        if (p.vec) go(dt, std::true_type{}, std::integral_constant<int, 0>{}, One{});
        else go(dt, std::false_type{}, std::integral_constant<int, 0>{}, One{});
    });
}

}  // namespace

hipError_t launch_kv8_append(const KvCache& c, const KvRows& k, const KvRows& v, int dtype,
                             const int64_t* slots, int tokens, hipStream_t stream) {
    const AppendPlan p = append_plan(c, k, v, dtype, tokens);
    by_plan(p, dtype, [&](auto dt, auto vec, auto hold, auto waves) {
        append_kernel<decltype(dt)::value, decltype(vec)::value, decltype(hold)::value,
                      decltype(waves)::value>
            <<<dim3((unsigned)p.grid), kAppendWaves * kWave, 0, stream>>>(c, k, v, slots, tokens,
                                                                          p.window, p.units);
    });
    return hipGetLastError();
}

hipError_t launch_kv8_rotate_append(const KvCache& c, const KvRows& k, const KvRows& v, int dtype,
                                    const int64_t* slots, RotaryArgs q, hipStream_t stream) {
    const int step = q.rot.interleaved ? 4 : 8;  // pairs of whole chunks of 8 elements
    AppendPlan p = append_plan(c, k, v, dtype, q.tokens);
    const bool units = p.vec && c.d % 8 == 0 && q.rot.pairs % step == 0;
    AppendTurned t;
    t.window = p.window > 1 && c.log_block >= 6 ? 32 : p.window;
    t.windows = ((int64_t)q.tokens + t.window - 1) / t.window;
    t.angles = (int)std::min<int64_t>(((int64_t)q.rot.pairs << c.log_block), kAngles);
    // (one head or two make one workgroup a window, whether waves share them or not)
    const int64_t keys = t.windows * key_groups(c.heads, 1);
    const int64_t values = p.shared ? t.windows * c.heads
                                    : (t.windows * c.heads + kAppendWaves - 1) / kAppendWaves;
    t.key_groups = (int)std::min((keys + 7) / 8 * 8, kAppendBlocks);
    t.value_groups = (int)std::min((values + 7) / 8 * 8, kAppendBlocks);
    // Queries go along where they are taken in steps of 16 or 8 bytes, in a small call (64 decode tokens,
    // append and read: 14.0 us along, 15.8 apart) and beside runs that take few registers (prompts of
    // 23446 tokens 51 us, 62 apart), else in a launch of their own, at the rate of a copy.
    int64_t extra = 0;
    t.half_steps = 0;
    if (q.q.heads > 0) {
        const int step = rotary_plan(q, dtype, &extra), most = dtype == kF32 ? 4 : 8;
        t.half_steps = 2 * step == most;
        if (t.half_steps) rotary_plan(q, dtype, &extra, kHalfStepHeads);
        const bool few = p.hold && p.held <= 2048;
        if ((step != most && !t.half_steps) || (p.window > 1 && !few)) {
            extra = 0;
            if (hipError_t e = launch_rotary(q, dtype, stream)) return e;
        }
    }
    const int64_t grid = t.key_groups + t.value_groups + extra;
    if (grid > kMaxGroups256) return hipErrorInvalidValue;
    by_plan(p, dtype, [&](auto dt, auto vec, auto hold, auto waves) {
        constexpr int DT = decltype(dt)::value, HOLD = decltype(hold)::value, WAVES = decltype(waves)::value;
        constexpr bool VEC = decltype(vec)::value;
        auto go = [&](auto inter, auto keys) {
            append_turned_kernel<DT, VEC, HOLD, WAVES, decltype(keys)::value, decltype(inter)::value>
                <<<(unsigned)grid, kAppendWaves * kWave, (size_t)t.angles * sizeof(float2), stream>>>(
                    c, k, v, slots, q.tokens, t, q);
        };
        auto by_layout = [&](auto keys) {
            if (q.rot.interleaved) go(std::true_type{}, keys);
            else go(std::false_type{}, keys);
        };
        if constexpr (VEC) {
            // (the runs of HOLD 4, of at most 2048 elements, have 128 units)
            constexpr Keys KEYS = HOLD == 4 ? kHeldUnits : kUnits;
            if (units) return by_layout(std::integral_constant<Keys, KEYS>{});
        }
        by_layout(std::integral_constant<Keys, kElements>{});
    });
    return hipGetLastError();
}

hipError_t launch_kv8_read(const KvCache& c, const int32_t* blocks, int n, int dtype, void* k_out,
                           void* v_out, float* scales_out, hipStream_t stream) {
    const bool wide = c.d % 8 == 0;
    const int64_t units = ((int64_t)c.heads * (wide ? c.d / 8 : c.d)) << c.log_block;
    int64_t shares = (units + kReadThreads * kReadUnits - 1) / (kReadThreads * kReadUnits);
    // some 2048 workgroups in all
    const int64_t most = 1024 / (n < 1024 ? n : 1024);
    shares = shares < most ? shares : most;
    if ((int64_t)n * 2 > 0x7FFFFFFF) return hipErrorInvalidValue;
    const dim3 g((unsigned)(2 * n), (unsigned)shares), b(kReadThreads);
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (wide) read_kernel<DT, true><<<g, b, 0, stream>>>(c, blocks, k_out, v_out, scales_out);
        else read_kernel<DT, false><<<g, b, 0, stream>>>(c, blocks, k_out, v_out, scales_out);
    };
    by_dtype(dtype, go);
    return hipGetLastError();
}

}  // namespace ojx
