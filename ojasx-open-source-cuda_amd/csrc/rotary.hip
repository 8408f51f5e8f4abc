// rotary.hip -- positions rotated into queries and keys, and the gradient (the rotation back).
//
//   y_lo = g (x_lo cos a - x_hi sin a),  y_hi = g (x_hi cos a + x_lo sin a),  a = position * rate,
// for the pairs of a head's first elements; the others are copied.  rotary.h has the angles.

#include <hip/hip_runtime.h>

#include <type_traits>

#include "rotary_heads.h"

namespace ojx {

namespace {

template <int DT, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a) {
    rotate_heads<DT, V, INTERLEAVED>(a, blockIdx.x);
}

// Whether V elements are a step of every address in rows.
bool fits(const RotaryRows& r, int v, int size) {
    const int64_t strides = r.x_batch | r.x_token | r.x_head | r.y_batch | r.y_token | r.y_head;
    return r.heads == 0 || ((strides & (v - 1)) == 0 &&
                            (((uintptr_t)r.x | (uintptr_t)r.y) & (uintptr_t)(v * size - 1)) == 0);
}

}  // namespace

int rotary_plan(RotaryArgs& a, int dtype, int64_t* grid, int heads_of_thread) {
    const int size = dtype == kF32 ? 4 : 2, heads = a.q.heads + a.k.heads;
    const int pairs = a.rot.pairs, rest = a.d - 2 * pairs;
    int v = 16 / size;
    while (v > 1 && (pairs % v != 0 || rest % (2 * v) != 0 || !fits(a.q, v, size) || !fits(a.k, v, size)))
        v >>= 1;
    a.chunks = (a.d + 2 * v - 1) / (2 * v);
    a.groups = (heads + heads_of_thread - 1) / heads_of_thread;
    const int64_t units = (int64_t)a.batches * a.tokens * a.groups * a.chunks;
    *grid = (units + kRotaryThreads - 1) / kRotaryThreads;
    return v;
}

bool rotary_fits(RotaryArgs a, int dtype) {
    int64_t grid;
    rotary_plan(a, dtype, &grid);
    return grid <= kMaxGroups256;
}

hipError_t launch_rotary(RotaryArgs a, int dtype, hipStream_t stream) {
    int64_t grid;
    const int v = rotary_plan(a, dtype, &grid);
    if (grid == 0) return hipSuccess;
    if (grid > kMaxGroups256) return hipErrorInvalidValue;
    auto go = [&](auto dt, auto step) {
        constexpr int DT = decltype(dt)::value, V = decltype(step)::value;
        if (a.rot.interleaved)
            rotary_kernel<DT, V, true><<<(unsigned)grid, kRotaryThreads, 0, stream>>>(a);
        else
            rotary_kernel<DT, V, false><<<(unsigned)grid, kRotaryThreads, 0, stream>>>(a);
    };
    auto by_step = [&](auto dt) {
        if (v == 8) {
            if constexpr (decltype(dt)::value != kF32) go(dt, std::integral_constant<int, 8>{});
        } else if (v == 4) {
            go(dt, std::integral_constant<int, 4>{});
        } else if (v == 2) {
            go(dt, std::integral_constant<int, 2>{});
        } else {
            go(dt, std::integral_constant<int, 1>{});
        }
    };
    if (dtype == kF32) by_step(std::integral_constant<int, kF32>{});
    else if (dtype == kF16) by_step(std::integral_constant<int, kF16>{});
    else by_step(std::integral_constant<int, kBF16>{});
    return hipGetLastError();
}

}  // namespace ojx
