// kv8_cache.hip -- the 8-bit paged key / value cache: block tables and slots of a step (plan),
// new tokens into the cache (append), blocks out of it (read).  Layout: include/ojasx_e8t.h.

#include <hip/hip_runtime.h>

#include <type_traits>

#include "serve.h"

namespace ojx {

namespace {

constexpr int kWave = 64;

// ---------------------------------------------------------------- plan

constexpr int kPlanThreads = 1024;
constexpr int kPlanItems = 4;                            // requests per thread and pass
constexpr int kPlanChunk = kPlanThreads * kPlanItems;    // requests per pass
constexpr int kPlanTokens = kPlanThreads * 4;            // tokens per workgroup

__device__ __forceinline__ int sat32(int64_t v) { return v > 0x7FFFFFFF ? 0x7FFFFFFF : (int)v; }

// Exclusive sum of v over the workgroup; *total: the sum over all of it.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* totals, int64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t s = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int64_t up = __shfl_up(s, o);
        if (lane >= o) s += up;
    }
    if (lane == 63) totals[wave] = s;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / kWave; ++w) {
        const int64_t t = totals[w];
        before += w < wave ? t : 0;
        all += t;
    }
    __syncthreads();
    *total = all;
    return before + s - v;
}

// Every workgroup sums up the requests by itself (a pass over kPlanChunk lengths is a few
// microseconds of latency, less than a second launch) and then maps its own tokens; the first
// one also writes the requests' results.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a) {
    __shared__ int starts[kPlanChunk], held[kPlanChunk], firsts[kPlanChunk];
    __shared__ int64_t totals[kPlanThreads / kWave];
    const int block = 1 << a.log_block;
    const int64_t t0 = (int64_t)blockIdx.x * kPlanTokens, t1 = t0 + kPlanTokens;
    const int nf = *a.num_free < a.capacity ? *a.num_free : a.capacity;
    int64_t q_base = 0, need_base = 0;
    for (int64_t c = 0; c < a.requests; c += kPlanChunk) {
        int64_t now[kPlanItems], old[kPlanItems], q = 0, need = 0, total;
        const int64_t r0 = c + (int64_t)threadIdx.x * kPlanItems;
#pragma unroll
        for (int i = 0; i < kPlanItems; ++i) {
            const bool in = r0 + i < a.requests;
            now[i] = in ? a.new_lens[r0 + i] : 0;
            old[i] = in ? a.seq_lens[r0 + i] : 0;
            now[i] = now[i] > 0 ? now[i] : 0;
            old[i] = old[i] > 0 ? old[i] : 0;
            q += now[i];
        }
        int64_t start = q_base + block_scan(q, totals, &total);
        const int64_t q_next = q_base + total;
#pragma unroll
        for (int i = 0; i < kPlanItems; ++i) {
            // no more tokens than there is room for
            const int64_t room = a.tokens - start;
            const int64_t fit = now[i] < room ? now[i] : (room > 0 ? room : 0);
            const int64_t have = (old[i] + block - 1) >> a.log_block;
            const int64_t want = (old[i] + fit + block - 1) >> a.log_block;
            const int k = threadIdx.x * kPlanItems + i;
            starts[k] = (int)(start < a.tokens ? start : a.tokens);
            held[k] = sat32(old[i]);
            if (blockIdx.x == 0 && r0 + i < a.requests) {
                a.query_starts[r0 + i] = starts[k];
                a.seq_lens_out[r0 + i] = sat32(old[i] + fit);
            }
            start += now[i];
            now[i] = (want < a.width ? want : a.width) - (have < a.width ? have : a.width);
            need += now[i];
        }
        int64_t first = need_base + block_scan(need, totals, &total);
        need_base += total;
#pragma unroll
        for (int i = 0; i < kPlanItems; ++i) {
            firsts[threadIdx.x * kPlanItems + i] = sat32(first);
            first += now[i];
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
        const int64_t left = nf - need_base;
        a.num_free_out[0] = left < -0x7FFFFFFF ? -0x7FFFFFFF : (int)left;
    }
}

// ---------------------------------------------------------------- append

constexpr int kAppendWaves = 4;
constexpr float kTinyAmax = 0x1p-100f;

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

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
// pass over the run for its largest element, one over it (now in the cache) for the codes.
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

// A wave looks for run starts among `window` tokens and writes each run for one head, keys or
// values.  Runs end where the slots leave the block or skip.
template <int DT, bool VEC>
__global__ __launch_bounds__(kAppendWaves * kWave) void append_kernel(
    KvCache c, KvRows k, KvRows v, const int64_t* __restrict__ slots, int tokens, int window,
    int64_t units) {
    const int lane = threadIdx.x & 63;
    const int64_t u = (int64_t)blockIdx.x * kAppendWaves + (threadIdx.x >> 6);
    if (u >= units) return;
    const int parts = 2 * c.heads;
    const int64_t w = u / parts;
    const int part = (int)(u - w * parts), head = part >> 1;
    const int64_t end = (int64_t)c.blocks << c.log_block;
    const int block = 1 << c.log_block;
    const int64_t t = w * window + lane;
    int64_t slot = -1, prev = -1;
    if (lane < window && t < tokens) {
        slot = slots[t];
        if (t > 0) prev = slots[t - 1];
    }
    const bool start = slot >= 0 && slot < end &&
                       (prev != slot - 1 || (slot & (block - 1)) == 0);
    uint64_t heads = __ballot(start);
    while (heads) {
        const int i = __builtin_ctzll(heads);
        heads &= heads - 1;
        const int64_t t0 = w * window + i;
        const int64_t s0 = __shfl(slot, i);
        const int off = (int)(s0 & (block - 1));
        int n = 0;
        for (; n < block - off;) {  // tokens that follow it in the block
            const int64_t tn = t0 + n + lane;
            const bool next = n + lane < block - off && tn < tokens && slots[tn] == s0 + n + lane;
            const uint64_t miss = ~__ballot(next);
            if (miss) {
                n += __builtin_ctzll(miss);
                break;
            }
            n += kWave;
        }
        append_run<DT, VEC>(c, part & 1 ? v : k, part & 1, head, t0, n,
                            (int)(s0 >> c.log_block), off, lane);
    }
}

// ---------------------------------------------------------------- read

// The value of a code: the fp32 product, rounded to DT.
template <int DT> __device__ __forceinline__ void store_value(void* p, int64_t i, int code, float s) {
    float v = (float)code * s;
    keep_f32(v);
    store_from_f32<DT>(p, i, v);
}

constexpr int kReadThreads = 256;

template <int DT>
__global__ __launch_bounds__(kReadThreads) void read_kernel(KvCache c,
                                                            const int32_t* __restrict__ blocks,
                                                            void* k_out, void* v_out,
                                                            float* scales_out) {
    const int parts = 2 * c.heads;
    const int64_t i = blockIdx.x / parts;
    const int part = blockIdx.x % parts, head = part >> 1, values = part & 1;
    const int b = blocks[i], size = 1 << c.log_block;
    const bool in = b >= 0 && b < c.blocks;
    const float s = in ? c.scales[c.scale_at(b, head) + values] : 0.f;
    const int8_t* base = (values ? c.v : c.k) + (in ? c.at(b, head) : 0);
    void* out = values ? v_out : k_out;
    if (threadIdx.x == 0) scales_out[(i * c.heads + head) * 2 + values] = s;
    // output element of (token, d)
    const int64_t o0 = ((i << c.log_block) * c.heads + head) * c.d, ot = (int64_t)c.heads * c.d;
    if (!values) {
        const int chunks = (c.d + 15) >> 4;
        for (int u = threadIdx.x; u < size * chunks; u += kReadThreads) {
            const int t = u / chunks, ch = u - t * chunks;
            uint4 o = make_uint4(0, 0, 0, 0);
            if (in) o = *reinterpret_cast<const uint4*>(base + key_at(t, ch, c.dp));
            const uint32_t w[4] = {o.x, o.y, o.z, o.w};
            for (int j = 0; j < 16 && ch * 16 + j < c.d; ++j)
                store_value<DT>(out, o0 + t * ot + ch * 16 + j, byte_of(w[j >> 2], j & 3), s);
        }
        return;
    }
    for (int u = threadIdx.x; u < (size >> 4) * c.d; u += kReadThreads) {
        const int g = u / c.d, d = u - g * c.d;
        uint4 o = make_uint4(0, 0, 0, 0);
        if (in) o = *reinterpret_cast<const uint4*>(base + (int64_t)g * 16 * c.dp + d * 16);
        const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int j = 0; j < 16; ++j)
            store_value<DT>(out, o0 + (g * 16 + j) * ot + d, byte_of(w[j >> 2], j & 3), s);
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

hipError_t launch_kv8_append(const KvCache& c, const KvRows& k, const KvRows& v, int dtype,
                             const int64_t* slots, int tokens, hipStream_t stream) {
    // A window per token fills the GPU for a decode step, whose tokens all begin runs; with
    // many tokens most of such waves would find none.
    const int window = (int64_t)tokens * 2 * c.heads <= 16384 ? 1 : 16;
    const int64_t units = ((int64_t)tokens + window - 1) / window * 2 * c.heads;
    const int64_t grid = (units + kAppendWaves - 1) / kAppendWaves;
    if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
    const bool vec = rows_vector(k, dtype) && rows_vector(v, dtype);
    const dim3 g((unsigned)grid), b(kAppendWaves * kWave);
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (vec)
            append_kernel<DT, true><<<g, b, 0, stream>>>(c, k, v, slots, tokens, window, units);
        else
            append_kernel<DT, false><<<g, b, 0, stream>>>(c, k, v, slots, tokens, window, units);
    };
    if (dtype == kF32) go(std::integral_constant<int, kF32>{});
    else if (dtype == kF16) go(std::integral_constant<int, kF16>{});
    else go(std::integral_constant<int, kBF16>{});
    return hipGetLastError();
}

hipError_t launch_kv8_read(const KvCache& c, const int32_t* blocks, int n, int dtype, void* k_out,
                           void* v_out, float* scales_out, hipStream_t stream) {
    const int64_t grid = (int64_t)n * 2 * c.heads;
    if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
    const dim3 g((unsigned)grid), b(kReadThreads);
    if (dtype == kF32) read_kernel<kF32><<<g, b, 0, stream>>>(c, blocks, k_out, v_out, scales_out);
    else if (dtype == kF16) read_kernel<kF16><<<g, b, 0, stream>>>(c, blocks, k_out, v_out, scales_out);
    else read_kernel<kBF16><<<g, b, 0, stream>>>(c, blocks, k_out, v_out, scales_out);
    return hipGetLastError();
}

}  // namespace ojx
