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

// Request of token t: the last one that begins at or before it (tokens past the last
// request's end have none: -1).
__device__ __forceinline__ int request_of(const AttnArgs& a, int t) {
    if (!a.query_starts) return t;
    int l = 0, h = a.shape.requests;
    while (h - l > 1) {
        const int m = (l + h) >> 1;
        if (a.query_starts[m] <= t) l = m; else h = m;
    }
    return a.query_starts[l] <= t && t < a.query_starts[l + 1] ? l : -1;
}

// ---------------------------------------------------------------- one row per wave

// Everything in fp32, 64 keys at a time: a lane has a key for the scores and up to four d for
// the values.
template <int DT>
__global__ __launch_bounds__(64) void row_kernel(AttnArgs a) {
    __shared__ float q[256], p[64];
    const KvCache& c = a.cache;
    const int lane = threadIdx.x;
    const int t = blockIdx.x / a.shape.heads, head = blockIdx.x % a.shape.heads;
    const int r = request_of(a, t);
    if (r < 0) return;
    const int q0 = a.query_starts ? a.query_starts[r] : t;
    const int q1 = a.query_starts ? a.query_starts[r + 1] : t + 1;
    if (t - q0 >= a.shape.max_query) return;
    const int len = min(a.seq_lens[r], a.shape.max_seq);
    // keys [lo, hi)
    const int hi = min(a.seq_lens[r] - (q1 - q0) + (t - q0) + 1, len);
    const int lo = a.shape.window && hi > a.shape.window ? hi - a.shape.window : 0;
    const int kvh = head / (a.shape.heads / a.shape.kv_heads);
    bool bad = false;
    for (int d = lane; d < c.dp; d += 64) {
        const float x = d < c.d ? load_as_f32<DT>(a.q.p, t * a.q.token + head * a.q.head + d) : 0.f;
        bad |= !(fabsf(x) < INFINITY);
        q[d] = x * (a.scale * kLog2e);
    }
    bad = __any(bad);
    __syncthreads();
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    bool some = false;
    const int32_t* row = a.tables + r * a.table_ld;
    const int block = 1 << c.log_block;
    for (int j0 = lo / 64 * 64; j0 < hi; j0 += 64) {
        const int j = j0 + lane;
        float s = -INFINITY, vs = 0.f;
        int b = -1;
        if (j >= lo && j < hi) b = row[j >> c.log_block];
        if (b >= 0 && b < c.blocks) {
            const int tok = j & (block - 1);
            const int8_t* k = c.k + c.at(b, kvh) + (tok >> 4) * 16 * c.dp +
                              ((tok & 15) >> 2) * 256 + (tok & 3) * 16;
            float dot = 0.f;
            for (int ch = 0; ch < c.dp >> 4; ++ch) {
                const uint4 o = *reinterpret_cast<const uint4*>(k + (ch >> 2) * 1024 + (ch & 3) * 64);
                const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    dot = __builtin_fmaf((float)(int8_t)(w[i >> 2] >> (8 * (i & 3))), q[ch * 16 + i],
                                         dot);
            }
            s = dot * c.scales[c.scale_at(b, kvh)];
            vs = c.scales[c.scale_at(b, kvh) + 1];
        }
        some |= __any(b >= 0 && b < c.blocks);
        float top = s;
#pragma unroll
        for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float next = fmaxf(m, top);
        const float keep = next == -INFINITY ? 1.f : exp2f(m - next);
        float w = next == -INFINITY ? 0.f : exp2f(s - next);
        m = next;
        p[lane] = w * vs;
#pragma unroll
        for (int o = 32; o; o >>= 1) w += __shfl_xor(w, o);
        l = l * keep + w;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= keep;
        for (int g = 0; g < 4; ++g) {
            // the 16 tokens share a block; those outside [lo, hi) have none
            const uint64_t seen = __ballot(b >= 0 && b < c.blocks) >> (16 * g) & 0xFFFFu;
            if (!seen) continue;
            const int from = __shfl(b, 16 * g + __builtin_ctzll(seen));
            const int tok = (j0 + 16 * g) & (block - 1);
            const int8_t* v = c.v + c.at(from, kvh) + (tok >> 4) * 16 * c.dp;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = lane + 64 * i;
                if (d >= c.d) continue;
                const uint4 o = *reinterpret_cast<const uint4*>(v + d * 16);
                const uint32_t w4[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                for (int n = 0; n < 16; ++n)
                    acc[i] = __builtin_fmaf(p[16 * g + n],
                                            (float)(int8_t)(w4[n >> 2] >> (8 * (n & 3))), acc[i]);
            }
        }
        __syncthreads();
    }
    const int64_t o0 = ((int64_t)t * a.shape.heads + head) * c.d;
    const float nan = __uint_as_float(0x7FC00000u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + 64 * i;
        if (d < c.d)
            store_from_f32<DT>(a.out, o0 + d, some ? (bad ? nan : acc[i] / l) : 0.f);
    }
    if (lane == 0 && a.lse)
        a.lse[(int64_t)t * a.shape.heads + head] =
            some ? (bad ? nan : (m + log2f(l)) * kLn2) : -INFINITY;
}

}  // namespace

size_t kv8_attention_bytes(const AttnShape& s) { return 0; }

hipError_t launch_kv8_attention(const AttnArgs& a, void* ws, size_t ws_bytes, hipStream_t stream) {
    const int64_t rows = (int64_t)a.shape.tokens * a.shape.heads;
    if (rows > 0x7FFFFFFF) return hipErrorInvalidValue;
    const dim3 g((unsigned)rows), b(64);
    if (a.shape.dtype == kF32) row_kernel<kF32><<<g, b, 0, stream>>>(a);
    else if (a.shape.dtype == kF16) row_kernel<kF16><<<g, b, 0, stream>>>(a);
    else row_kernel<kBF16><<<g, b, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace ojx
