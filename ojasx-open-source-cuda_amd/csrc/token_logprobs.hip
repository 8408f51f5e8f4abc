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
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Largest |logit| that the one pass over a row takes as a reference (struct Sums): its rounding in
// binary units is an exponent's error, up to 2^3 here (half of the spacing at 1.44e8).  2^(2^3) is
// harmless in a sum; at 3e9 it would be 2^128, an infinity.
constexpr float kPlainMax = 1e8f;

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

// ---------------------------------------------------------------- rows out of the ordinary

// A row with NaN or infinities, or whose largest logit is beyond +-kPlainMax (all of it masked
// by a large negative value, say): one workgroup, one pass for the maximum, one for the sums,
// one per alternative (77 such rows of 50021 fp32 with 20: 683 us, 17 for ordinary ones).
template <int DT>
__device__ __forceinline__ void odd_row(const LogprobArgs& a, int row, float* sf, uint64_t* sk) {
    const int v = a.vocab;
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
        a.lse[row] = bad ? nan : m + ls;
        a.stats[2 * (int64_t)row] = bad ? nan : m;
        a.stats[2 * (int64_t)row + 1] = ls;
        a.logprob[row] = in ? log_p(load_as_f32<DT>(a.x, x0 + id)) : 0.f;
        a.entropy[row] = bad ? nan : none ? 0.f : ls - u / s;
    }
    uint64_t last = ~0ull;  // which is also the key of NaN at token 0: the first pass takes any
    for (int i = 0; i < a.top; ++i) {
        uint64_t best = 0;
        for (int j = threadIdx.x; j < v; j += kThreads) {
            const uint64_t k = key_of(load_as_f32<DT>(a.x, x0 + j), j);
            if ((i == 0 || k < last) && k > best) best = k;
        }
        last = block_reduce(best, sk, [](uint64_t p, uint64_t q) { return p > q ? p : q; });
        if (threadIdx.x == 0) {
            const int64_t o = (int64_t)row * a.top + i;
            a.top_ids[o] = 0xFFFFFFFFu - (uint32_t)last;
            a.top_lp[o] = log_p(unordered((uint32_t)(last >> 32)));
        }
    }
}

// ---------------------------------------------------------------- one pass over a row

// Sums of some of a row's logits in binary units: r a reference near the largest of them times
// log2(e), s = sum 2^t and u = sum t 2^t over t = x log2(e) - r.  r is only a reference: its own
// rounding is in every t alike and leaves the results, as long as it is small enough for the sums
// to hold 2^rounding (kPlainMax: lanes of larger masks only have none).  m is the largest logit
// itself.
struct Sums {
    float r, s, u, m;
};

// The larger of two, NaN if either is (v_maximum3_f32).
__device__ __forceinline__ float or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// t below which 2^t is zero: keeps t 2^t from becoming -inf * 0 at masked logits.
__device__ __forceinline__ float term(float x, float base) {
    return fmaxf(__builtin_fmaf(x, kLog2e, -base), -200.f);
}

__device__ __forceinline__ void rescale(Sums& a, float base) {
    const float d = fmaxf(a.r - base, -200.f), f = __builtin_amdgcn_exp2f(d);
    a.u = f * __builtin_fmaf(d, a.s, a.u);
    a.s *= f;
}

__device__ __forceinline__ Sums merge(Sums a, Sums b) {
    const float r = fmaxf(a.r, b.r), base = r == -INFINITY ? 0.f : r;
    rescale(a, base);
    rescale(b, base);
    return Sums{r, a.s + b.s, a.u + b.u, or_nan(a.m, b.m)};
}

__device__ __forceinline__ Sums merge_wave(Sums a) {
    const bool bad = __any(a.m != a.m);
    const float r = wave_max(a.r);
    rescale(a, r == -INFINITY ? 0.f : r);
    const float m = wave_max(a.m);
    return Sums{r, wave_sum(a.s), wave_sum(a.u), bad ? __uint_as_float(0x7FC00000u) : m};
}

__device__ __forceinline__ bool ordinary(const Sums& a) {
    return a.m > -kPlainMax && a.m < kPlainMax;  // not NaN
}

// The k best keys that a wave has seen, the i-th in lane i.
struct Best {
    uint64_t key;   // 0: none yet
    float least;    // the k-th one's logit; -inf while there are fewer
};

__device__ __forceinline__ uint64_t read_lane(uint64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
    return (uint64_t)hi << 32 | lo;
}

__device__ __forceinline__ void insert(Best& b, uint64_t key, int k, int lane) {
    if (key <= read_lane(b.key, k - 1)) return;
    const int at = __popcll(__ballot(b.key > key));
    const uint64_t up = __shfl_up(b.key, 1);
    b.key = lane < at ? b.key : lane == at ? key : up;
}

// A wave's candidates on their way into its best k.
constexpr int kPool = 256;
struct Pool {
    uint64_t keys[kPool];
    uint64_t sorted[64];
    float maxima[64];
};

// The k-th largest of the lanes' values: the least of those that fewer than k exceed.
__device__ __forceinline__ float kth_of_lanes(float v, int k, int lane, Pool& pool) {
    pool.maxima[lane] = v;
    __builtin_amdgcn_wave_barrier();
    int above = 0;
#pragma unroll
    for (int j = 0; j < 64; j += 4) {
        const float4 f = *reinterpret_cast<const float4*>(pool.maxima + j);
        above += f.x > v;
        above += f.y > v;
        above += f.z > v;
        above += f.w > v;
    }
    return -wave_max(above < k ? -v : -INFINITY);
}

// Takes the first n of the pool into the best k: up to four one by one, about 200 cycles each, more
// by their ranks among all of them and the k (4096 rows of 32000 with 5 alternatives: 72 us, 79 by
// ranks alone).
__device__ __forceinline__ void settle(Best& b, Pool& pool, int n, int k, int lane) {
    __builtin_amdgcn_wave_barrier();
    if (n <= 4) {
        for (int i = 0; i < n; ++i) insert(b, read_lane(pool.keys[i], 0), k, lane);
    } else {
        const int all = n + k;  // the best so far behind the new
        if (lane < k) pool.keys[n + lane] = b.key;
        if (lane < k) pool.sorted[lane] = 0;
        __builtin_amdgcn_wave_barrier();
        for (int i0 = 0; i0 < all; i0 += 64) {
            const uint64_t mine = i0 + lane < all ? pool.keys[i0 + lane] : 0;
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < all; ++j) rank += pool.keys[j] > mine;
            if (mine != 0 && rank < k) pool.sorted[rank] = mine;
        }
        __builtin_amdgcn_wave_barrier();
        b.key = lane < k ? pool.sorted[lane] : 0;
        __builtin_amdgcn_wave_barrier();
    }
    const uint64_t last = read_lane(b.key, k - 1);
    b.least = last != 0 ? unordered((uint32_t)(last >> 32)) : -INFINITY;
}

constexpr int kLaneLogits = 32;                  // logits of a lane in one batch
constexpr int kBatch = 64 * kLaneLogits;         // of a wave
constexpr int kGroups = kThreads / 64;
constexpr int kMaxRowSplits = 64;
// Lanes whose maximum is the bound of a batch's candidates, from which on their places are bounded
// too: fewer hold at most one pool of equal logits.
constexpr int kTied = kPool / kLaneLogits;

template <int DT> struct Batch {
    static constexpr int kVec = DT == kF32 ? 4 : 8;  // logits of 16 bytes
    static constexpr int kVecs = kLaneLogits / kVec;
    uint4 w[kVecs];

    // logit i of the lane in the row, for batch b of a row that begins `shift` logits after an
    // address that is a multiple of 16 bytes
    static __device__ __forceinline__ int index(int b, int i, int lane, int shift) {
        return ((b * kVecs + i / kVec) * 64 + lane) * kVec + i % kVec - shift;
    }

    // Vectors that reach over an end of the row are put together from its logits and -inf.
    __device__ __forceinline__ void load(const void* x, int64_t x0, int v, int b, int lane,
                                         int shift) {
        // a batch within the row: the same for all lanes, and nothing to check
        if (b * kBatch >= shift && (int64_t)(b + 1) * kBatch - shift <= v) {
            const char* p = static_cast<const char*>(x) +
                            (x0 + index(b, 0, lane, shift)) * (16 / kVec);
#pragma unroll
            for (int n = 0; n < kVecs; ++n) w[n] = *reinterpret_cast<const uint4*>(p + n * 1024);
            return;
        }
#pragma unroll
        for (int n = 0; n < kVecs; ++n) {
            const int j = index(b, n * kVec, lane, shift);
            if (j >= 0 && j + kVec <= v) {
                if constexpr (DT == kF32)
                    w[n] = *reinterpret_cast<const uint4*>(static_cast<const float*>(x) + x0 + j);
                else
                    w[n] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + x0 + j);
            } else {
                uint32_t u[4];
                constexpr uint32_t low = DT == kF32 ? 0xFF800000u : DT == kF16 ? 0xFC00u : 0xFF80u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (DT == kF32) {
                        const bool in = j + i >= 0 && j + i < v;
                        u[i] = in ? static_cast<const uint32_t*>(x)[x0 + j + i] : low;
                    } else {
                        const uint16_t* h = static_cast<const uint16_t*>(x) + x0;
                        const int p = j + 2 * i;
                        const uint32_t lo = p >= 0 && p < v ? h[p] : low;
                        const uint32_t hi = p + 1 >= 0 && p + 1 < v ? h[p + 1] : low;
                        u[i] = lo | hi << 16;
                    }
                }
                w[n] = make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
    }

    // Logits read from here on are converted anew: kept as floats they would cost a register each.
    __device__ __forceinline__ void drop_floats() {
        if constexpr (DT != kF32)
#pragma unroll
            for (int n = 0; n < kVecs; ++n)
                asm("" : "+v"(w[n].x), "+v"(w[n].y), "+v"(w[n].z), "+v"(w[n].w));
    }

    __device__ __forceinline__ float get(int i) const {
        const uint4& q = w[i / kVec];
        const int n = i % kVec;
        const uint32_t u[4] = {q.x, q.y, q.z, q.w};
        if constexpr (DT == kF32) return __uint_as_float(u[n]);
        else if constexpr (DT == kF16) return f16_bits_to_f32(n & 1 ? u[n >> 1] >> 16 : u[n >> 1] & 0xFFFFu);
        else return __uint_as_float(n & 1 ? u[n >> 1] & 0xFFFF0000u : u[n >> 1] << 16);
    }
};

// The least float over x (of -inf: the lowest finite one).
__device__ __forceinline__ float above(float x) { return unordered(ordered(x) + 1); }

// Puts the lanes' keys (0: none) behind the pool's first n, which are taken first where they leave
// no room.  Returns the number then there; `settled` tells of the best k's change.
__device__ __forceinline__ int push(Best& b, Pool& pool, int n, bool on, uint64_t key, int k, int lane,
                                    bool& settled) {
    const uint64_t c = __ballot(on);
    settled = n + __popcll(c) + k > kPool;
    if (settled) {
        settle(b, pool, n, k, lane);
        n = 0;
    }
    const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(c >> 32),
                                                 __builtin_amdgcn_mbcnt_lo((uint32_t)c, 0));
    if (on) pool.keys[at] = key;
    return n + __popcll(c);
}

// Takes a batch's candidates into the wave's best k: logits of at least `lo`.  Batches come by
// rising token, so a later logit that only equals the k-th one loses; within a batch it may not.
// Where many lanes have a candidate (all at first), the k-th largest of the lanes' maxima is a
// bound under which none can stay: about k candidates are left whatever the row's order.  Logits
// that equal this bound in many lanes (a row of one value, a mask of the type's lowest one) are
// bounded by their places alike.  -inf is no candidate (finish adds what a row lacks), nor is the
// padding beyond the row's ends.
template <int DT>
__device__ __forceinline__ void take(Best& best, Batch<DT>& x, float lane_max, int b, int k,
                                     int lane, int shift, Pool& pool) {
    const bool may = lane_max > best.least;
    const uint64_t lanes = __ballot(may);
    if (!lanes) return;
    float lo = above(best.least);
    int n = 0;
    bool settled;
    const int many = __popcll(lanes);
    if (many >= k && (many > k + 12 || best.least == -INFINITY)) {
        const float cut = kth_of_lanes(may ? lane_max : -INFINITY, k, lane, pool);
        lo = fmaxf(lo, cut);
        if (__popcll(__ballot(lane_max == cut)) > kTied) {
            lo = above(cut);
            constexpr int kVec = Batch<DT>::kVec;
            uint32_t equal = 0;
#pragma unroll
            for (int i = 0; i < kLaneLogits; ++i) {
                // one after the other: all conversions at once would cost a wave of occupancy
                if constexpr (DT != kF32)
                    asm volatile("" : "+v"(equal), "+v"((&x.w[i / kVec].x)[i % kVec * 4 / kVec]));
                equal |= x.get(i) == cut ? 1u << i : 0u;
            }
            // a lane's logits come by rising token, kVec together
            auto place = [&](int i) { return (i / kVec * 64 + lane) * kVec + i % kVec; };
            __builtin_amdgcn_wave_barrier();
            const int last = (int)-kth_of_lanes(
                equal ? -(float)place(__builtin_ctz(equal)) : -(float)kBatch, k, lane, pool);
            __builtin_amdgcn_wave_barrier();
            for (;;) {
                const int i = __builtin_ctz(equal | 1u << 31);
                const bool on = equal && place(i) <= last;
                if (!__any(on)) break;
                n = push(best, pool, n, on, key_of(cut, b * kBatch + place(i) - shift), k, lane, settled);
                equal &= equal - 1;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kLaneLogits; ++i) {
        const float f = x.get(i);
        if (!__any(f >= lo)) continue;
        n = push(best, pool, n, f >= lo, key_of(f, Batch<DT>::index(b, i, lane, shift)), k, lane, settled);
        if (settled) lo = fmaxf(lo, best.least);
    }
    if (n) settle(best, pool, n, k, lane);
}

// A row's given token: read ahead of its use.
struct Asked {
    int64_t id;
    bool in;
    float x;
};
template <int DT> __device__ __forceinline__ Asked asked_of(const LogprobArgs& a, int row) {
    Asked t;
    t.id = a.ids[row];
    t.in = t.id >= 0 && t.id < a.vocab;
    t.x = t.in ? load_as_f32<DT>(a.x, row * a.ld + t.id) : 0.f;
    return t;
}

// A row's results from its sums and n keys in LDS (behind a barrier), its best among them.
template <int DT>
__device__ __forceinline__ void finish(const LogprobArgs& a, int row, const Sums& t, const Asked& asked,
                                       const uint64_t* keys, int n, float* sf, uint64_t* sk) {
    if (!ordinary(t)) return odd_row<DT>(a, row, sf, sk);
    const float l2 = log2f(t.s);
    const float ls = (l2 - __builtin_fmaf(t.m, kLog2e, -t.r)) * kLn2;
    auto log_p = [&](float x) { return x == -INFINITY ? x : (x - t.m) - ls; };
    if (threadIdx.x == 0) {
        a.lse[row] = t.m + ls;
        a.stats[2 * (int64_t)row] = t.m;
        a.stats[2 * (int64_t)row + 1] = ls;
        a.logprob[row] = asked.in ? log_p(asked.x) : 0.f;
        a.entropy[row] = (l2 - t.u / t.s) * kLn2;
    }
    if (n == 0) return;
    // a key's rank is its place
    bool lacks = false;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t k = keys[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += keys[j] > k;
        if (rank >= a.top) continue;
        if (k != 0) {
            const int64_t o = (int64_t)row * a.top + rank;
            a.top_ids[o] = 0xFFFFFFFFu - (uint32_t)k;
            a.top_lp[o] = log_p(unordered((uint32_t)(k >> 32)));
        } else {
            lacks = true;
        }
    }
    if (!__syncthreads_or(lacks)) return;
    // Fewer logits than alternatives: masked ones follow, by rising token.
    int have = 0;
    for (int j = 0; j < n; ++j) have += keys[j] != 0;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int j0 = 0; j0 < a.vocab && have < a.top; j0 += kThreads) {
        const int j = j0 + threadIdx.x;
        const bool masked = j < a.vocab && load_as_f32<DT>(a.x, row * a.ld + j) == -INFINITY;
        const uint64_t those = __ballot(masked);
        if (lane == 0) sk[wave] = __popcll(those);
        __syncthreads();
        int rank = have + __popcll(those & ((1ull << lane) - 1));
        for (int w = 0; w < kGroups; ++w) {
            if (w < wave) rank += (int)sk[w];
            have += (int)sk[w];
        }
        if (masked && rank < a.top) {
            const int64_t o = (int64_t)row * a.top + rank;
            a.top_ids[o] = j;
            a.top_lp[o] = -INFINITY;
        }
        __syncthreads();
    }
}

// Partial results of a row's splits: sums, then k keys each.
struct Parts {
    Sums* sums;      // [rows][splits]
    uint64_t* keys;  // [rows][splits][top]
    int splits;
};

// A workgroup reads a row, or with splits > 1 a part of it, once: every wave keeps its sums and
// its best k.  Without alternatives memory bounds it (2048 rows of 128256 bf16, 525 MB: 125 us,
// 4.2 TB/s), with them vector instructions (4096 rows of 32000 fp16 with 5: 72 us, 3.6 TB/s: 17 for
// every logit, of which the conversion, maximum, exponential and sums are 8; the others convert it
// again and look for candidates in every batch that has one).
template <int DT, bool TOP>
__global__ __launch_bounds__(kThreads) void pass_kernel(LogprobArgs a, Parts p) {
    __shared__ Sums sums[kGroups];
    __shared__ Pool pool[TOP ? kGroups : 1];
    __shared__ uint64_t keys[TOP ? kGroups * kTopMax : 1];
    __shared__ float sf[kGroups];
    __shared__ uint64_t sk[kGroups];
    using B = Batch<DT>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits;
    const int64_t x0 = row * a.ld;
    const int size = DT == kF32 ? 4 : 2;
    const int shift = (int)((((uintptr_t)a.x + x0 * size) & 15) / size);
    const int batches = (int)(((int64_t)a.vocab + shift + kBatch - 1) / kBatch);
    const int per = (batches + p.splits - 1) / p.splits;
    const int end = min(batches, (split + 1) * per);
    Sums t{-INFINITY, 0.f, 0.f, -INFINITY};
    Best best{0, -INFINITY};
    B x;
    int b = split * per + wave;
    for (; b < end; b += kGroups) {
        x.load(a.x, x0, a.vocab, b, lane, shift);
        float m = x.get(0);
#pragma unroll
        for (int i = 1; i < kLaneLogits; ++i) m = or_nan(m, x.get(i));
        const float r = fmaxf(t.r, m < -kPlainMax ? -INFINITY : m * kLog2e);
        const float base = r == -INFINITY ? 0.f : r;
        rescale(t, base);
        t.r = r;
        t.m = or_nan(t.m, m);  // NaN would be lost in term()
#pragma unroll
        for (int i = 0; i < kLaneLogits; ++i) {
            const float d = term(x.get(i), base), e = __builtin_amdgcn_exp2f(d);
            t.s += e;
            t.u = __builtin_fmaf(d, e, t.u);
        }
        if constexpr (TOP) x.drop_floats();
        if constexpr (TOP) take<DT>(best, x, m, b, a.top, lane, shift, pool[wave]);
    }
    t = merge_wave(t);
    if (lane == 0) sums[wave] = t;
    if (TOP && lane < a.top) keys[wave * a.top + lane] = best.key;
    __syncthreads();
    t = merge(merge(sums[0], sums[1]), merge(sums[2], sums[3]));
    if (p.splits == 1)
        return finish<DT>(a, row, t, asked_of<DT>(a, row), keys, TOP ? kGroups * a.top : 0, sf, sk);
    const int64_t at = (int64_t)row * p.splits + split;
    if (threadIdx.x == 0) p.sums[at] = t;
    if constexpr (TOP) {
        // the waves' lists in order, for the next kernel
        for (int i = threadIdx.x; i < kGroups * a.top; i += kThreads) {
            const uint64_t k = keys[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < kGroups * a.top; ++j) rank += keys[j] > k || (keys[j] == k && j < i);
            if (rank < a.top) p.keys[at * a.top + rank] = k;
        }
    }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void join_kernel(LogprobArgs a, Parts p) {
    __shared__ uint64_t keys[kGroups * kTopMax];
    __shared__ float sf[kGroups];
    __shared__ uint64_t sk[kGroups];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.x;
    const Asked asked = asked_of<DT>(a, row);
    const int n = p.splits * a.top;
    const uint64_t* from = p.keys + (int64_t)row * n;
    const bool few = n <= kGroups * kTopMax;
    if (few && (int)threadIdx.x < n) keys[threadIdx.x] = from[threadIdx.x];
    Sums t{-INFINITY, 0.f, 0.f, -INFINITY};
    if (lane < p.splits) t = p.sums[(int64_t)row * p.splits + lane];
    t = merge_wave(t);
    if (!few) {
        // every split's list is in order; the first is the wave's to begin with
        const uint64_t* list = from + wave * a.top + lane;
        Best b{wave < p.splits && lane < a.top ? *list : 0, 0.f};
        for (int s = wave + kGroups; s < p.splits; s += kGroups) {
            list += kGroups * a.top;
            const uint64_t k = lane < a.top ? *list : 0;
            uint64_t c = __ballot(k > read_lane(b.key, a.top - 1));
            while (c) {
                const int i = __builtin_ctzll(c);
                c &= c - 1;
                insert(b, read_lane(k, i), a.top, lane);
            }
        }
        if (lane < a.top) keys[wave * a.top + lane] = b.key;
    }
    __syncthreads();
    finish<DT>(a, row, t, asked, keys, few ? n : kGroups * a.top, sf, sk);
}

// ---------------------------------------------------------------- gradient

constexpr int kGradLogits = 8 * kThreads;  // of a workgroup's step, 16 bytes a thread and more

// A workgroup writes the gradient of a part of a row, then goes over the tokens that a gradient
// names and that lie in its part.  Memory bounds it: 2048 rows of 128256 bf16 (1050 MB) in 187 us,
// 5.6 TB/s.
template <int DT>
__global__ __launch_bounds__(kThreads) void grad_kernel(LogprobGradArgs a, int splits, int per) {
    constexpr int VE = Batch<DT>::kVec;
    const int row = blockIdx.x / splits, split = blockIdx.x - row * splits, v = a.vocab;
    const int64_t x0 = row * a.ld, g0 = (int64_t)row * v;
    const int size = DT == kF32 ? 4 : 2;
    const int shift = (int)((((uintptr_t)a.x + x0 * size) & 15) / size);
    const bool same = shift == (int)((((uintptr_t)a.gx + g0 * size) & 15) / size);
    const int64_t id = a.ids[row];
    const bool in = id >= 0 && id < v;
    const float g_id = in && a.g_lp ? a.g_lp[row] : 0.f;
    const float g_h = a.g_h ? a.g_h[row] : 0.f;
    const float m = a.stats[2 * (int64_t)row], ls = a.stats[2 * (int64_t)row + 1];
    const float h = a.entropy[row];
    float g_all = g_id - (a.g_lse ? a.g_lse[row] : 0.f);
    for (int i = 0; i < a.top; ++i) g_all += a.g_top[(int64_t)row * a.top + i];
    // -p (g_all + g_h (log p + h)); the log probability bounded as in term(), where p is 0; a
    // row with NaN has it in the factor
    const float c0 = m == m ? -__builtin_fmaf(g_h, h, g_all) : m, c1 = -g_h;
    const bool none = m == -INFINITY;
    auto grad = [&](float x) {
        const float lp = none ? -200.f : fmaxf((x - m) - ls, -200.f);
        const float p = __builtin_amdgcn_exp2f(lp * kLog2e);
        return p * __builtin_fmaf(c1, lp, c0);
    };
    // the part: logits [j0, j1) on the row's 16-byte grid
    const int64_t j0 = (int64_t)split * per - shift, j1 = j0 + per;
    for (int64_t j = j0 + (int64_t)threadIdx.x * VE; j < j1 && j < v; j += kThreads * VE) {
        if (same && j >= 0 && j + VE <= v) {
            if constexpr (DT == kF32) {
                const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(a.x) + x0 + j);
                *reinterpret_cast<float4*>(static_cast<float*>(a.gx) + g0 + j) =
                    make_float4(grad(x.x), grad(x.y), grad(x.z), grad(x.w));
            } else {
                const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + x0 + j);
                const uint32_t u[4] = {q.x, q.y, q.z, q.w};
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float lo, hi;
                    if constexpr (DT == kF16) {
                        lo = f16_bits_to_f32(u[i] & 0xFFFFu);
                        hi = f16_bits_to_f32(u[i] >> 16);
                        o[i] = f32_to_f16_bits(grad(lo)) | f32_to_f16_bits(grad(hi)) << 16;
                    } else {
                        lo = __uint_as_float(u[i] << 16);
                        hi = __uint_as_float(u[i] & 0xFFFF0000u);
                        o[i] = bf16_bits_hw(grad(lo)) | bf16_bits_hw(grad(hi)) << 16;
                    }
                }
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.gx) + g0 + j) =
                    make_uint4(o[0], o[1], o[2], o[3]);
            }
        } else {
            for (int i = 0; i < VE; ++i)
                if (j + i >= 0 && j + i < v)
                    store_from_f32<DT>(a.gx, g0 + j + i, grad(load_as_f32<DT>(a.x, x0 + j + i)));
        }
    }
    __syncthreads();
    // Named tokens: each once for all its names, with its own gradient added.
    for (int i = threadIdx.x; i <= a.top; i += kThreads) {
        const int64_t j = i < a.top ? a.top_ids[(int64_t)row * a.top + i] : id;
        if (j < 0 || j >= v || j < j0 || j >= j1) continue;
        float g = in && j == id ? g_id : 0.f;
        for (int n = 0; n < a.top; ++n)
            if (a.top_ids[(int64_t)row * a.top + n] == j) g += a.g_top[(int64_t)row * a.top + n];
        store_from_f32<DT>(a.gx, g0 + j, grad(load_as_f32<DT>(a.x, x0 + j)) + g);
    }
}

template <class F> void by_dtype(int dtype, F f) {
    if (dtype == kF32) f(std::integral_constant<int, kF32>{});
    else if (dtype == kF16) f(std::integral_constant<int, kF16>{});
    else f(std::integral_constant<int, kBF16>{});
}

// Splits of a row: until the workgroups fill the GPU twice, none under a batch per wave (77 rows of
// 50021: 17 us, 19.4 with a quarter of them; 4096 rows of 32000: 72 us unsplit, 90 in two).
int row_splits(int rows, int vocab) {
    const int64_t most = ((int64_t)vocab + kBatch * kGroups - 1) / (kBatch * kGroups);
    int64_t n = rows > 0 ? 2048 / rows : 1;
    if (n > most) n = most;
    if (n > kMaxRowSplits) n = kMaxRowSplits;
    return n < 1 ? 1 : (int)n;
}

size_t parts_bytes(int rows, int splits, int top) {
    return splits > 1 ? (size_t)rows * splits * (sizeof(Sums) + top * sizeof(uint64_t)) : 0;
}

}  // namespace

size_t token_logprobs_bytes(int rows, int vocab, int top, int dtype) {
    return parts_bytes(rows, row_splits(rows, vocab), top);
}

hipError_t launch_token_logprobs(const LogprobArgs& a, void* ws, size_t ws_bytes,
                                 hipStream_t stream) {
    Parts p{};
    p.splits = row_splits(a.rows, a.vocab);
    if (p.splits > 1) {
        const size_t per = (size_t)a.rows * (sizeof(Sums) + a.top * sizeof(uint64_t));
        const size_t fit = ws ? ws_bytes / per : 0;
        if ((size_t)p.splits > fit) p.splits = fit < 2 ? 1 : (int)fit;
    }
    p.sums = static_cast<Sums*>(ws);
    p.keys = reinterpret_cast<uint64_t*>(p.sums + (size_t)a.rows * p.splits);
    const int64_t grid = (int64_t)a.rows * p.splits;
    if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
    by_dtype(a.dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (a.top > 0) pass_kernel<DT, true><<<(unsigned)grid, kThreads, 0, stream>>>(a, p);
        else pass_kernel<DT, false><<<(unsigned)grid, kThreads, 0, stream>>>(a, p);
        if (p.splits > 1) join_kernel<DT><<<a.rows, kThreads, 0, stream>>>(a, p);
    });
    return hipGetLastError();
}

hipError_t launch_token_logprobs_bwd(const LogprobGradArgs& a, hipStream_t stream) {
    int64_t splits = a.rows > 0 ? 4096 / a.rows : 1;
    const int64_t most = ((int64_t)a.vocab + kGradLogits - 1) / kGradLogits;
    splits = splits < 1 ? 1 : splits > most ? most : splits;
    // parts of whole steps; the row's shift may need one more logit's step
    int64_t per = ((int64_t)a.vocab + 8 + splits - 1) / splits;
    per = (per + kGradLogits - 1) / kGradLogits * kGradLogits;
    splits = ((int64_t)a.vocab + 8 + per - 1) / per;
    const int64_t grid = a.rows * splits;
    if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
    by_dtype(a.dtype, [&](auto dt) {
        grad_kernel<decltype(dt)::value>
            <<<(unsigned)grid, kThreads, 0, stream>>>(a, (int)splits, (int)per);
    });
    return hipGetLastError();
}

}  // namespace ojx
