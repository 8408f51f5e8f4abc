// serve.h -- arguments and launchers of the 8-bit paged cache (kv8_cache.hip), its attention
// (kv8_attention.hip) and token log probabilities (token_logprobs.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "e8t_device.h"

namespace ojx {

// ---------------------------------------------------------------- sums over lanes

// v of the lane N places round in its row of 16.
template <int N> __device__ __forceinline__ float row_turn(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v),
                                                                 0x120 + N, 0xF, 0xF, true));
}

// a, b = the lower and the upper lane's v of each pair (l, l + 16) or (l, l + 32), in both lanes:
// v_permlane*_swap exchanges the odd rows (the upper half) of its first operand with the even
// rows (the lower half) of its second.  Its wait after a vector write stands with it.
__device__ __forceinline__ void pair16(float v, float& a, float& b) {
    a = b = v;
    asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ void pair32(float v, float& a, float& b) {
    a = b = v;
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}

// Over the lanes n, n + 16, n + 32, n + 48.
__device__ __forceinline__ float col_max(float v) {
    float a, b;
    pair16(v, a, b);
    pair32(fmaxf(a, b), a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float col_sum(float v) {
    float a, b;
    pair16(v, a, b);
    pair32(a + b, a, b);
    return a + b;
}

// Over the wave, in every lane.
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, row_turn<8>(v));
    v = fmaxf(v, row_turn<4>(v));
    v = fmaxf(v, row_turn<2>(v));
    return col_max(fmaxf(v, row_turn<1>(v)));
}
__device__ __forceinline__ float wave_sum(float v) {
    v += row_turn<8>(v);
    v += row_turn<4>(v);
    v += row_turn<2>(v);
    return col_sum(v + row_turn<1>(v));
}

// e8t_capi.cpp: the calling thread's error message, the arch check and a launch's status
int api_failf(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int api_check_device();
int api_done(hipError_t e, const char* what);

constexpr int64_t kKvMaxHeads = 4096;
constexpr int64_t kTopMax = 64;

// A cache; its layout is in include/ojasx_e8t.h.
struct KvCache {
    int8_t* k;
    int8_t* v;
    float* scales;
    int blocks;
    int heads;
    int log_block;
    int d;
    int dp;  // d rounded up to a multiple of 64

    // bytes of one head of a block
    __host__ __device__ int64_t head_bytes() const { return (int64_t)dp << log_block; }
    // byte offset of (block, head)
    __host__ __device__ int64_t at(int block, int head) const {
        return ((int64_t)block * heads + head) * head_bytes();
    }
    __host__ __device__ int64_t scale_at(int block, int head) const {
        return ((int64_t)block * heads + head) * 2;
    }
};

// [token][head][d] elements with strides between tokens and heads, d contiguous.
struct KvRows {
    const void* p;
    int64_t token;
    int64_t head;
};

struct PlanArgs {
    const int32_t* seq_lens;
    const int32_t* new_lens;
    int32_t* tables;
    const int32_t* free_blocks;
    const int32_t* num_free;
    int64_t* slots;
    int32_t* positions;
    int32_t* request_ids;
    int32_t* query_starts;
    int32_t* seq_lens_out;
    int32_t* num_free_out;
    int64_t table_ld;
    int requests;
    int width;
    int capacity;
    int log_block;
    int tokens;
};

struct AttnShape {
    int tokens;
    int requests;
    int heads;
    int kv_heads;
    int d;
    int window;  // 0: none
    int max_query;
    int max_seq;
    int dtype;
};

struct AttnArgs {
    KvCache cache;
    KvRows q;
    const int32_t* tables;
    int64_t table_ld;
    const int32_t* seq_lens;
    const int32_t* query_starts;  // null: one token a request
    void* out;
    float* lse;
    float scale;
    int width;
    AttnShape shape;
};

struct LogprobArgs {
    const void* x;
    int64_t ld;
    int rows;
    int vocab;
    int dtype;
    int top;
    const int64_t* ids;
    float* logprob;
    float* entropy;
    float* lse;
    float* stats;
    float* top_lp;
    int64_t* top_ids;
};

struct LogprobGradArgs {
    const void* x;
    int64_t ld;
    int rows;
    int vocab;
    int dtype;
    int top;
    const int64_t* ids;
    const float* entropy;
    const float* stats;
    const int64_t* top_ids;
    const float* g_lp;
    const float* g_h;
    const float* g_lse;
    const float* g_top;
    void* gx;
};

hipError_t launch_kv8_plan(const PlanArgs& a, hipStream_t stream);
hipError_t launch_kv8_append(const KvCache& c, const KvRows& k, const KvRows& v, int dtype,
                             const int64_t* slots, int tokens, hipStream_t stream);
hipError_t launch_kv8_read(const KvCache& c, const int32_t* blocks, int n, int dtype, void* k_out,
                           void* v_out, float* scales_out, hipStream_t stream);
size_t kv8_attention_bytes(const AttnShape& s);
hipError_t launch_kv8_attention(const AttnArgs& a, void* ws, size_t ws_bytes, hipStream_t stream);
size_t token_logprobs_bytes(int rows, int vocab, int top, int dtype);
hipError_t launch_token_logprobs(const LogprobArgs& a, void* ws, size_t ws_bytes,
                                 hipStream_t stream);
hipError_t launch_token_logprobs_bwd(const LogprobGradArgs& a, hipStream_t stream);

}  // namespace ojx
