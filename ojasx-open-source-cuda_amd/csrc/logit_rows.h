// logit_rows.h -- a pass of a wave over a part of a row of logits that keeps its k largest: shared by
// token log probabilities (token_logprobs.hip) and the selection of beams (beam_select.hip).
#pragma once

#include <hip/hip_runtime.h>

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

// The larger of two, NaN if either is (v_maximum3_f32).
__device__ __forceinline__ float or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// t below which 2^t is zero: keeps t 2^t from becoming -inf * 0 at masked logits.
__device__ __forceinline__ float term(float x, float base) {
    return fmaxf(__builtin_fmaf(x, kLog2e, -base), -200.f);
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

}  // namespace

}  // namespace ojx
