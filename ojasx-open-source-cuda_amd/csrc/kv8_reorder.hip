// kv8_reorder.hip -- requests of the paged cache that go on from others: block tables, lengths and
// the stack of free blocks after beams were chosen (reorder), and the copies of begun blocks
// (copy_blocks).  Rules: include/ojasx_e8t.h.

#include <hip/hip_runtime.h>

#include "serve.h"

namespace ojx {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kNone = 0x7FFFFFFF;

// What a call works on: the first child of every old row, and a bit for each block that a row with
// children (live) or one without (dead) holds.
struct Marks {
    int32_t* first;
    uint32_t* live;
    uint32_t* dead;
};

__device__ __forceinline__ int parent_of(const ReorderArgs& a, int64_t child) {
    const int64_t p = a.parents[child];
    return p >= 0 && p < a.rows ? (int)p : -1;
}

__device__ __forceinline__ int length_of(const ReorderArgs& a, int row) {
    return row < 0 ? 0 : max(a.seq_lens[row], 0);
}

// Table entries of a row of `len` tokens.
__device__ __forceinline__ int used_of(const ReorderArgs& a, int len) {
    const int64_t n = ((int64_t)len + (1 << a.log_block) - 1) >> a.log_block;
    return (int)(n < a.width ? n : a.width);
}

// Column of a child's begun block that is to be its own, or -1: the first child keeps the parent's.
__device__ __forceinline__ int copied_column(const ReorderArgs& a, const int32_t* first, int64_t child,
                                             int parent, int len) {
    const int64_t at = len >> a.log_block;
    if (parent < 0 || (len & ((1 << a.log_block) - 1)) == 0 || at >= a.width || first[parent] == child)
        return -1;
    const int block = a.tables[parent * a.table_ld + at];
    return block >= 0 && block < a.blocks ? (int)at : -1;
}

__device__ __forceinline__ void mark_row(const ReorderArgs& a, const Marks& m, int row, int lane,
                                         int step) {
    const int used = used_of(a, length_of(a, row));
    uint32_t* bits = m.first[row] != kNone ? m.live : m.dead;
    const int32_t* t = a.tables + row * a.table_ld;
    for (int j = lane; j < used; j += step) {
        const int b = t[j];
        if (b < 0 || b >= a.blocks) continue;
        // many rows share a block: a bit that is seen set needs no second time
        if (!(bits[b >> 5] >> (b & 31) & 1)) atomicOr(bits + (b >> 5), 1u << (b & 31));
    }
}

// A new row's entries and length; the entry that copied_column names is write_stack's.
__device__ __forceinline__ void write_row(const ReorderArgs& a, const int32_t* first, int64_t child,
                                          int lane, int step) {
    const int p = parent_of(a, child), len = length_of(a, p), used = p < 0 ? 0 : used_of(a, len);
    const int skip = copied_column(a, first, child, p, len);
    const int32_t* from = a.tables + (p < 0 ? 0 : p) * a.table_ld;
    int32_t* to = a.tables_out + child * a.width;
    for (int j = lane; j < a.width; j += step)
        if (j != skip) to[j] = j < used ? from[j] : -1;
    if (lane == 0) a.seq_lens_out[child] = len;
}

// Exclusive sum over the workgroup.
__device__ __forceinline__ int block_scan(int v, int* totals, int* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(s, o);
        s += lane >= o ? up : 0;
    }
    if (lane == 63) totals[wave] = s;
    __syncthreads();
    int before = s - v, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        before += w < wave ? totals[w] : 0;
        all += totals[w];
    }
    __syncthreads();
    *total = all;
    return before;
}

// The new stack: what is on the old one, then the freed blocks by rising number, less what children
// take from its top for begun blocks of their own, by rising child.  One workgroup.
__device__ __forceinline__ void write_stack(const ReorderArgs& a, const Marks& m, int* totals) {
    int top = max(min(min(*a.num_free, a.capacity), a.blocks), 0);
    const int kept = top;
    for (int i = threadIdx.x; i < kept; i += kThreads) a.free_out[i] = a.free_blocks[i];
    const int words = (a.blocks + 31) >> 5;
    for (int w0 = 0; w0 < words; w0 += kThreads) {
        const int w = w0 + threadIdx.x;
        uint32_t f = w < words ? m.dead[w] & ~m.live[w] : 0;
        int total, at = top + block_scan(__popc(f), totals, &total);
        for (; f; f &= f - 1, ++at)
            if (at < a.blocks) a.free_out[at] = w * 32 + __builtin_ctz(f);
        top += total;
    }
    top = min(top, a.blocks);
    __syncthreads();
    for (int64_t c0 = 0; c0 < a.children; c0 += kThreads) {
        const int64_t child = c0 + threadIdx.x;
        int p = -1, column = -1, total;
        if (child < a.children) {
            p = parent_of(a, child);
            column = copied_column(a, m.first, child, p, length_of(a, p));
        }
        const int take = top - 1 - block_scan(column >= 0, totals, &total);
        if (child < a.children) {
            int source = -1, target = -1;
            if (column >= 0) {
                source = a.tables[p * a.table_ld + column];
                target = take >= 0 ? a.free_out[take] : -1;
                a.tables_out[child * a.width + column] = target;
            }
            a.sources[child] = source;
            a.targets[child] = target;
        }
        top -= total;
    }
    __syncthreads();
    for (int i = max(top, 0) + threadIdx.x; i < a.blocks; i += kThreads) a.free_out[i] = -1;
    if (threadIdx.x == 0) *a.num_free_out = top;
}

__device__ __forceinline__ void clear(const ReorderArgs& a, const Marks& m) {
    for (int i = threadIdx.x; i < a.rows; i += kThreads) m.first[i] = kNone;
    const int words = (a.blocks + 31) >> 5;
    for (int i = threadIdx.x; i < words; i += kThreads) m.live[i] = m.dead[i] = 0;
    __threadfence();  // the atomics below are done in L2
    __syncthreads();
    for (int64_t c = threadIdx.x; c < a.children; c += kThreads) {
        const int p = parent_of(a, c);
        if (p >= 0) atomicMin(m.first + p, (int)c);  // the least, in whatever order
    }
}

// All of a small call in one workgroup, whose marks are in LDS.
__global__ __launch_bounds__(kThreads) void reorder_kernel(ReorderArgs a) {
    extern __shared__ int32_t lds[];
    __shared__ int totals[kWaves];
    const int words = (a.blocks + 31) >> 5, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Marks m{lds, reinterpret_cast<uint32_t*>(lds) + a.rows,
                  reinterpret_cast<uint32_t*>(lds) + a.rows + words};
    clear(a, m);
    __syncthreads();
    for (int r = wave; r < a.rows; r += kWaves) mark_row(a, m, r, lane, 64);
    for (int64_t c = wave; c < a.children; c += kWaves) write_row(a, m.first, c, lane, 64);
    __syncthreads();
    write_stack(a, m, totals);
}

// A large call, in three launches.
__global__ __launch_bounds__(kThreads) void reorder_clear_kernel(ReorderArgs a, Marks m) { clear(a, m); }

__global__ __launch_bounds__(256) void reorder_mark_kernel(ReorderArgs a, Marks m) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row < a.rows) mark_row(a, m, row, blockIdx.y * 64 + (threadIdx.x & 63), 64 * gridDim.y);
}

// The first workgroup writes the stack, the others rows.
__global__ __launch_bounds__(kThreads) void reorder_write_kernel(ReorderArgs a, Marks m) {
    __shared__ int totals[kWaves];
    if (blockIdx.x == 0) return write_stack(a, m, totals);
    const int64_t child = (int64_t)(blockIdx.x - 1) * kWaves + (threadIdx.x >> 6);
    if (child < a.children) write_row(a, m.first, child, threadIdx.x & 63, 64);
}

// ---------------------------------------------------------------- copies

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int kPiece = 4;  // 16-byte words of a lane in a wave's piece of a block

// Every wave goes through all copies that are asked for, 64 rows at a time, and takes each
// waves-th piece of them.
__global__ __launch_bounds__(256) void copy_kernel(CopyArgs a) {
    const int lane = threadIdx.x & 63;
    const uint32_t waves = gridDim.x * 4;
    const uint32_t mine = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t before = 0;  // pieces of earlier rows, modulo the waves
    for (int64_t r0 = 0; r0 < a.rows; r0 += 64) {
        int from = -1, to = -1;
        if (r0 + lane < a.rows) from = a.sources[r0 + lane], to = a.targets[r0 + lane];
        const bool on = from >= 0 && from < a.blocks && to >= 0 && to < a.blocks && from != to;
        const uint64_t rows = __ballot(on);
        const int rank = __popcll(rows & ((1ull << lane) - 1));
        const int64_t pieces = (int64_t)__popcll(rows) * a.layers * a.pieces;
        for (int64_t i = (mine + waves - before) % waves; i < pieces; i += waves) {
            // pieces of a layer's block first, then layers, then rows
            const int64_t block = i / a.pieces;
            const int piece = (int)(i - block * a.pieces);
            const int row = (int)(block / a.layers), layer = (int)(block - (int64_t)row * a.layers);
            const int at = __builtin_ctzll(__ballot(on && rank == row));
            const int64_t f = __shfl(from, at), t = __shfl(to, at);
            const int half = a.pieces >> 1;
            int8_t* codes = piece < half ? a.k[layer] : a.v[layer];
            const u32x4* x = reinterpret_cast<const u32x4*>(codes + f * a.bytes);
            u32x4* y = reinterpret_cast<u32x4*>(codes + t * a.bytes);
            // a block's bytes are whole kilobytes; words past them are its last ones again
            const int64_t w0 = (int64_t)(piece < half ? piece : piece - half) * 64 * kPiece + lane;
            const int64_t end = (a.bytes >> 4) - 64 + lane;
            u32x4 w[kPiece];
#pragma unroll
            for (int j = 0; j < kPiece; ++j) w[j] = x[min(w0 + j * 64, end)];
#pragma unroll
            for (int j = 0; j < kPiece; ++j) y[min(w0 + j * 64, end)] = w[j];
            if (piece == 0)
                for (int j = lane; j < a.scales; j += 64)
                    a.s[layer][t * a.scales + j] = a.s[layer][f * a.scales + j];
        }
        before = (uint32_t)((before + (uint64_t)pieces) % waves);
    }
}

// LDS of a call in one workgroup.
int64_t small_bytes(const ReorderArgs& a) { return (int64_t)a.rows * 4 + ((int64_t)a.blocks + 31) / 32 * 8; }

// One workgroup while its loads and stores of all rows cost less than two more launches.
bool small_call(const ReorderArgs& a) {
    return small_bytes(a) <= 60 * 1024 && ((int64_t)a.rows + a.children) * a.width <= 32768;
}

}  // namespace

size_t kv8_reorder_bytes(const ReorderArgs& a) { return small_call(a) ? 0 : (size_t)small_bytes(a); }

hipError_t launch_kv8_reorder(const ReorderArgs& a, void* ws, hipStream_t stream) {
    if (small_call(a)) {
        reorder_kernel<<<1, kThreads, (size_t)small_bytes(a), stream>>>(a);
        return hipGetLastError();
    }
    Marks m;
    m.first = static_cast<int32_t*>(ws);
    m.live = reinterpret_cast<uint32_t*>(m.first + a.rows);
    m.dead = m.live + (a.blocks + 31) / 32;
    reorder_clear_kernel<<<1, kThreads, 0, stream>>>(a, m);
    if (a.rows > 0) {
        // long tables of few rows by several waves each
        int64_t split = a.rows < 1024 ? 1024 / a.rows : 1;
        const int64_t most = ((int64_t)a.width + 255) / 256;
        split = split < most ? split : most;
        reorder_mark_kernel<<<dim3((unsigned)((a.rows + 3) / 4), (unsigned)(split < 1 ? 1 : split)), 256, 0,
                              stream>>>(a, m);
    }
    reorder_write_kernel<<<(unsigned)(1 + ((int64_t)a.children + kWaves - 1) / kWaves), kThreads, 0,
                           stream>>>(a, m);
    return hipGetLastError();
}

hipError_t launch_kv8_copy(CopyArgs a, hipStream_t stream) {
    a.pieces = 2 * (int)((a.bytes + 64 * kPiece * 16 - 1) / (64 * kPiece * 16));
    // all of them asked for, at most; a wave goes on with the next of its pieces
    const int64_t pieces = (int64_t)a.rows * a.layers * a.pieces;
    const int64_t grid = (pieces + 3) / 4;
    copy_kernel<<<(unsigned)(grid < 2048 ? grid : 2048), 256, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace ojx
