// rotary_heads.h -- the heads of a token rotated by a thread: the body of rotary_kernel (rotary.hip)
// and of the workgroups that rotate queries beside a cache's append (kv8_cache.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "serve.h"

namespace ojx {

constexpr int kRotaryThreads = 256;
// Heads of a thread, which share its angles: with one the angles cost more than the memory they wait
// for (8192 tokens of 32 + 8 heads of 128 bf16, 168 MB: 40 us, 31.8 with two, 33.2 with four), with more
// a small call has too few threads (64 tokens: 3.7 us, 3.8, 4.2; eight 5.2).
constexpr int kRotaryHeads = 2;

template <int BYTES> struct Words;
template <> struct Words<16> { using T = uint4; };
template <> struct Words<8> { using T = uint2; };
template <> struct Words<4> { using T = uint32_t; };
template <> struct Words<2> { using T = uint16_t; };

// V neighbouring elements as they lie in memory.
template <int DT, int V> struct Piece {
    using E = typename Elem<DT>::T;
    using W = typename Words<V * sizeof(E)>::T;
    W w;
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        w = *reinterpret_cast<const W*>(static_cast<const E*>(p) + i);
    }
    __device__ __forceinline__ void store(void* p, int64_t i) const {
        *reinterpret_cast<W*>(static_cast<E*>(p) + i) = w;
    }
    __device__ __forceinline__ void get(float (&x)[V]) const {
        E e[V];
        __builtin_memcpy(e, &w, sizeof(w));
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if constexpr (DT == kF32) x[i] = e[i];
            else x[i] = DT == kF16 ? f16_bits_to_f32(e[i]) : bf16_bits_to_f32(e[i]);
        }
    }
    __device__ __forceinline__ void set(const float (&x)[V]) {
        E e[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            // fp16 is rounded from the fp32 result in every unrolled copy alike: left alone, some of them
            // are fused to one rounding, and a head's bits hang on its number
            float f = x[i];
            if constexpr (DT == kF16) keep_f32(f);
            if constexpr (DT == kF32) e[i] = f;
            else e[i] = (uint16_t)(DT == kF16 ? f32_to_f16_bits(f) : bf16_bits_hw(f));
        }
        __builtin_memcpy(&w, e, sizeof(w));
    }
};

// A thread has 2 V elements of a head (V pairs, or as many that are copied) and forms their cosines
// and sines once for HEADS heads of its token, queries and keys alike.  Memory bounds it, at
// 5.3 TB/s for large calls (read and written; a large copy reaches 5.2), the latency of a launch, a
// load, the angles and a store for small ones.
template <int DT, int V, bool INTERLEAVED, int HEADS = kRotaryHeads>
__device__ __forceinline__ void rotate_heads(const RotaryArgs& a, uint32_t workgroup) {
    // (token, group of heads, chunk) of the thread: a division of 64 bits for the workgroup alone
    const uint32_t unit_count = (uint32_t)a.groups * a.chunks;
    const uint64_t base = (uint64_t)workgroup * kRotaryThreads;
    const uint64_t t0 = base >> 32 ? base / unit_count : (uint32_t)base / unit_count;
    const uint32_t local = (uint32_t)(base - t0 * unit_count) + threadIdx.x;
    const uint32_t over = local / unit_count, unit = local - over * unit_count;
    const int64_t token = (int64_t)t0 + over;
    if (token >= (int64_t)a.batches * a.tokens) return;
    const int group = unit / (uint32_t)a.chunks, chunk = unit - group * a.chunks;
    const int64_t b = a.batches == 1 ? 0 : (uint32_t)token / (uint32_t)a.tokens;
    const int64_t t = token - b * a.tokens;

    const int pairs = a.rot.pairs;
    const bool copy = chunk * V >= pairs;
    const int lo = INTERLEAVED || copy ? 2 * V * chunk : V * chunk;
    int hi = INTERLEAVED || copy ? lo + V : lo + pairs;
    if (V == 1 && copy) hi = min(hi, a.d - 1);  // the last one of an odd head, twice
    const int h0 = group * HEADS, heads = a.q.heads + a.k.heads;
    const int64_t qx = b * a.q.x_batch + t * a.q.x_token, qy = b * a.q.y_batch + t * a.q.y_token;
    const int64_t kx = b * a.k.x_batch + t * a.k.x_token, ky = b * a.k.y_batch + t * a.k.y_token;
    // on their way while the angles are formed
    Piece<DT, V> p[HEADS], r[HEADS];
#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
        const int h = min(h0 + j, heads - 1);
        const bool key = h >= a.q.heads;
        const void* x = key ? a.k.x : a.q.x;
        const int64_t e = key ? kx + (h - a.q.heads) * a.k.x_head : qx + h * a.q.x_head;
        p[j].load(x, e + lo);
        r[j].load(x, e + hi);
    }
    float c[V], s[V];
    if (!copy) {
        const uint64_t position = position_at(a.rot, b * a.position_batch + t * a.position_token);
#pragma unroll
        for (int i = 0; i < V; ++i) pair_turn(a.rot, position, a.rot.rates[chunk * V + i], c[i], s[i]);
    }
#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
        const int h = h0 + j;
        if (h >= heads) break;
        if (!copy) {
            float u[V], v[V];
            p[j].get(u);
            r[j].get(v);
            if constexpr (INTERLEAVED) {
                float e[2 * V];
#pragma unroll
                for (int i = 0; i < V; ++i) e[i] = u[i], e[V + i] = v[i];
#pragma unroll
                for (int i = 0; i < V; ++i) turn_pair(c[i], s[i], e[2 * i], e[2 * i + 1]);
#pragma unroll
                for (int i = 0; i < V; ++i) u[i] = e[i], v[i] = e[V + i];
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) turn_pair(c[i], s[i], u[i], v[i]);
            }
            p[j].set(u);
            r[j].set(v);
        }
        const bool key = h >= a.q.heads;
        void* y = key ? a.k.y : a.q.y;
        const int64_t e = key ? ky + (h - a.q.heads) * a.k.y_head : qy + h * a.q.y_head;
        p[j].store(y, e + lo);
        r[j].store(y, e + hi);
    }
}

// The largest step, up to 16 bytes, that divides pairs, copied elements, strides and addresses, and
// the launch's sizes for it.  An odd head size leaves one element to copy: it is taken by single
// elements, two of them a chunk.  Returns the step; *grid: workgroups.
int rotary_plan(RotaryArgs& a, int dtype, int64_t* grid, int heads_of_thread = kRotaryHeads);

}  // namespace ojx
