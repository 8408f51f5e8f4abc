// token_logprobs.hip -- log probabilities of given tokens with the entropy of their
// distributions and the most likely alternatives, and the gradient of the logits.
//
// For a row x of logits with m = max x, s = sum exp(x - m), u = sum (x - m) exp(x - m):
//   lse = m + log s,  log p_j = (x_j - m) - log s,  H = -sum p log p = log s - u / s.
// m and log s are kept apart: in rows of large magnitude (masks of the type's lowest value)
// their sum has no bits left for log s.

#include <hip/hip_runtime.h>

#include <type_traits>

#include "serve.h"

namespace ojx {

namespace {

constexpr int kThreads = 256;

// fp32 bits in rising order as unsigned, -0 as +0, NaN above everything.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// A logit with its place: larger keys come first among the alternatives.
__device__ __forceinline__ uint64_t key_of(float x, int j) {
    return (uint64_t)ordered(x) << 32 | (0xFFFFFFFFu - (uint32_t)j);
}

template <class T, class F> __device__ T block_reduce(T v, T* shared, F f) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = f(v, __shfl_xor(v, o));
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = shared[0];
    for (int w = 1; w < kThreads / 64; ++w) v = f(v, shared[w]);
    __syncthreads();
    return v;
}

// One workgroup per row, one pass for the maximum, one for the sums, one per alternative.
template <int DT>
__global__ __launch_bounds__(kThreads) void row_kernel(LogprobArgs a) {
    __shared__ float sf[kThreads / 64];
    __shared__ uint64_t sk[kThreads / 64];
    const int row = blockIdx.x, v = a.vocab;
    const int64_t x0 = row * a.ld;
    auto add = [](float p, float q) { return p + q; };
    auto most = [](float p, float q) { return fmaxf(p, q); };
    float m = -INFINITY, odd = 0.f;
    for (int j = threadIdx.x; j < v; j += kThreads) {
        const float x = load_as_f32<DT>(a.x, x0 + j);
        if (!(x < INFINITY)) odd = 1.f;  // NaN or +inf
        m = fmaxf(m, x);
    }
    m = block_reduce(m, sf, most);
    odd = block_reduce(odd, sf, most);
    const bool none = m == -INFINITY;  // nothing but -inf
    float s = 0.f, u = 0.f;
    if (!none)
        for (int j = threadIdx.x; j < v; j += kThreads) {
            const float d = load_as_f32<DT>(a.x, x0 + j) - m;
            const float e = expf(d);
            s += e;
            if (e > 0.f) u += d * e;
        }
    s = block_reduce(s, sf, add);
    u = block_reduce(u, sf, add);
    const float nan = __uint_as_float(0x7FC00000u);
    const bool bad = odd > 0.f;
    const float ls = none ? 0.f : logf(s);
    // the log probability of a logit
    auto log_p = [&](float x) { return bad ? nan : x == -INFINITY ? x : (x - m) - ls; };
    if (threadIdx.x == 0) {
        const int64_t id = a.ids[row];
        const bool in = id >= 0 && id < v;
        const float x = in ? load_as_f32<DT>(a.x, x0 + id) : 0.f;
        a.lse[row] = bad ? nan : m + ls;
        a.stats[2 * (int64_t)row] = bad ? nan : m;
        a.stats[2 * (int64_t)row + 1] = ls;
        a.logprob[row] = in ? log_p(x) : 0.f;
        a.entropy[row] = bad ? nan : none ? 0.f : ls - u / s;
    }
    uint64_t last = ~0ull;
    for (int i = 0; i < a.top; ++i) {
        uint64_t best = 0;
        for (int j = threadIdx.x; j < v; j += kThreads) {
            const uint64_t k = key_of(load_as_f32<DT>(a.x, x0 + j), j);
            if (k < last && k > best) best = k;
        }
        last = block_reduce(best, sk, [](uint64_t p, uint64_t q) { return p > q ? p : q; });
        if (threadIdx.x == 0) {
            const float x = unordered((uint32_t)(last >> 32));
            const int64_t o = (int64_t)row * a.top + i;
            a.top_ids[o] = 0xFFFFFFFFu - (uint32_t)last;
            a.top_lp[o] = log_p(x);
        }
    }
}

// One workgroup per row: p for every logit, then the tokens that a gradient names.
template <int DT>
__global__ __launch_bounds__(kThreads) void grad_kernel(LogprobGradArgs a) {
    const int row = blockIdx.x, v = a.vocab;
    const int64_t x0 = row * a.ld, g0 = (int64_t)row * v;
    const int64_t id = a.ids[row];
    const bool in = id >= 0 && id < v;
    const float g_id = in && a.g_lp ? a.g_lp[row] : 0.f;
    const float g_h = a.g_h ? a.g_h[row] : 0.f;
    const float m = a.stats[2 * (int64_t)row], ls = a.stats[2 * (int64_t)row + 1];
    const float h = a.entropy[row];
    float g_all = g_id - (a.g_lse ? a.g_lse[row] : 0.f);
    for (int i = 0; i < a.top; ++i) g_all += a.g_top[(int64_t)row * a.top + i];
    auto grad = [&](int64_t j) {
        const float x = load_as_f32<DT>(a.x, x0 + j);
        const float lp = (x - m) - ls;
        const float p = x == -INFINITY ? 0.f : expf(lp);
        return -p * (g_all + (p > 0.f ? g_h * (lp + h) : 0.f));
    };
    for (int j = threadIdx.x; j < v; j += kThreads) store_from_f32<DT>(a.gx, g0 + j, grad(j));
    __syncthreads();
    // Named tokens, each once: with its own gradient and those of equal names.
    for (int i = threadIdx.x; i <= a.top; i += kThreads) {
        const int64_t j = i < a.top ? a.top_ids[(int64_t)row * a.top + i] : id;
        if (j < 0 || j >= v) continue;
        float g = in && j == id ? g_id : 0.f;
        for (int n = 0; n < a.top; ++n)
            if (a.top_ids[(int64_t)row * a.top + n] == j) g += a.g_top[(int64_t)row * a.top + n];
        store_from_f32<DT>(a.gx, g0 + j, grad(j) + g);
    }
}

template <class F> void by_dtype(int dtype, F f) {
    if (dtype == kF32) f(std::integral_constant<int, kF32>{});
    else if (dtype == kF16) f(std::integral_constant<int, kF16>{});
    else f(std::integral_constant<int, kBF16>{});
}

}  // namespace

size_t token_logprobs_bytes(int rows, int vocab, int top, int dtype) { return 0; }

hipError_t launch_token_logprobs(const LogprobArgs& a, void* ws, size_t ws_bytes,
                                 hipStream_t stream) {
    by_dtype(a.dtype, [&](auto dt) {
        row_kernel<decltype(dt)::value><<<a.rows, kThreads, 0, stream>>>(a);
    });
    return hipGetLastError();
}

hipError_t launch_token_logprobs_bwd(const LogprobGradArgs& a, hipStream_t stream) {
    by_dtype(a.dtype, [&](auto dt) {
        grad_kernel<decltype(dt)::value><<<a.rows, kThreads, 0, stream>>>(a);
    });
    return hipGetLastError();
}

}  // namespace ojx
