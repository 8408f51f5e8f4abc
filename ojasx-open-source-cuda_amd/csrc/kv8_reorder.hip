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

// Of a large call: the first child of every old row, and a byte for each block that a row with
// children (live) or one without (dead) holds.
struct Marks {
    int32_t* first;
    uint8_t* live;
    uint8_t* dead;
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

// Column of a child's begun block if it is to have one of its own (the first child keeps the
// parent's), or -1; *block: the parent's.
template <class First>
__device__ __forceinline__ int copied_column(const ReorderArgs& a, int parent, int len, First is_first,
                                             int* block) {
    const int64_t at = len >> a.log_block;
    *block = -1;
    if (parent < 0 || (len & ((1 << a.log_block) - 1)) == 0 || at >= a.width) return -1;
    const int b = a.tables[parent * a.table_ld + at];
    if (b < 0 || b >= a.blocks || is_first()) return -1;
    *block = b;
    return (int)at;
}

// A new row's entries and length, by a wave; the entry that copied_column names is write_stack's.
template <class First>
__device__ __forceinline__ void write_row(const ReorderArgs& a, int64_t child, int lane, First is_first) {
    const int p = parent_of(a, child), len = length_of(a, p), used = p < 0 ? 0 : used_of(a, len);
    int block;
    const int skip = copied_column(a, p, len, [&] { return is_first(p); }, &block);
    const int32_t* from = a.tables + (p < 0 ? 0 : p) * a.table_ld;
    int32_t* to = a.tables_out + child * a.width;
    for (int j = lane; j < a.width; j += 64)
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

// A child's begun block that is to be copied: its column and its number, or -1.
struct Copy {
    int column, block;
};

template <class First>
__device__ __forceinline__ Copy copy_of(const ReorderArgs& a, int64_t child, First is_first) {
    Copy c{-1, -1};
    if (child < a.children) {
        const int p = parent_of(a, child);
        c.column = copied_column(a, p, length_of(a, p), [&] { return is_first(p, child); }, &c.block);
    }
    return c;
}

// Size of the old stack.
__device__ __forceinline__ int old_top(const ReorderArgs& a) {
    return max(min(min(*a.num_free, a.capacity), a.blocks), 0);
}

// The new stack: what is on the old one, then the freed blocks by rising number, less what children
// take from its top for begun blocks of their own, by rising child.  One workgroup.  freed(w): those
// of the blocks 32 w .. 32 w + 31.
template <class Freed, class First>
__device__ __forceinline__ void write_stack(const ReorderArgs& a, int* totals, Freed freed, First is_first) {
    int top = old_top(a);
    for (int i = threadIdx.x; i < top; i += kThreads) a.free_out[i] = a.free_blocks[i];
    const int words = (a.blocks + 31) >> 5;
    for (int w0 = 0; w0 < words; w0 += kThreads) {
        const int w = w0 + threadIdx.x;
        uint32_t f = w < words ? freed(w) : 0;
        int total, at = top + block_scan(__popc(f), totals, &total);
        for (; f; f &= f - 1, ++at)
            if (at < a.blocks) a.free_out[at] = w * 32 + __builtin_ctz(f);
        top += total;
    }
    top = min(top, a.blocks);
    __syncthreads();
    for (int64_t c0 = 0; c0 < a.children; c0 += kThreads) {
        const int64_t child = c0 + threadIdx.x;
        const Copy copy = copy_of(a, child, is_first);
        int total;
        const int take = top - 1 - block_scan(copy.column >= 0, totals, &total);
        if (child < a.children) {
            int target = -1;
            if (copy.column >= 0) {
                if (take >= 0) target = a.free_out[take];
                a.tables_out[child * a.width + copy.column] = target;
            }
            a.sources[child] = copy.block;
            a.targets[child] = target;
        }
        top -= total;
    }
    __syncthreads();
    for (int i = max(top, 0) + threadIdx.x; i < a.blocks; i += kThreads) a.free_out[i] = -1;
    if (threadIdx.x == 0) *a.num_free_out = top;
}

__device__ __forceinline__ void first_children(const ReorderArgs& a, int32_t* first) {
    for (int64_t c = threadIdx.x; c < a.children; c += kThreads) {
        const int p = parent_of(a, c);
        if (p >= 0) atomicMin(first + p, (int)c);  // the least, in whatever order
    }
}

constexpr int kRowsAhead = 8;  // rows of a wave whose loads are under way together

// Bytes of a call's blocks in LDS.
__host__ __device__ __forceinline__ int lds_room(const ReorderArgs& a) { return (a.blocks + 32) / 32 * 32; }


// A bit for each of 32 bytes that are 0 or 1.
__device__ __forceinline__ uint32_t bits_of(const uint8_t* bytes) {
    const uint4* w = reinterpret_cast<const uint4*>(bytes);
    const uint4 lo = w[0], hi = w[1];
    const uint32_t u[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) bits |= ((u[i] * 0x10204080u) >> 28) << (4 * i);
    return bits;
}

// A barrier for what is in LDS: stores to memory go on.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

constexpr int kOneChildren = 1;  // of a thread, in a call in one launch

// A call in one launch.  The first workgroup finds the blocks that are free again, by two bytes for each
// in LDS, and writes the stack; the others write rows, and look for themselves whether a child is its
// parent's first one.
//
// One workgroup that runs once is bound by what it waits for: loads that follow each other, and its own
// instructions, which come from memory too (16 rows with 2 KB more of unrolled code 1 us longer).  16
// rows of 16 blocks 4.9 us, 512 rows with 23000 entries of 2282 blocks 9.5; with a bit a block in place
// of a byte, set by atomics, 14, and in three launches with those bits in memory, where a prompt's
// blocks are held by many rows and lie in few lines, 22.5.
__global__ __launch_bounds__(kThreads) void reorder_kernel(ReorderArgs a) {
    extern __shared__ int32_t lds[];
    __shared__ int totals[kWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (blockIdx.x > 0) {
        const int64_t child = (int64_t)(blockIdx.x - 1) * kWaves + wave;
        if (child >= a.children) return;
        return write_row(a, child, lane, [&](int p) {
            for (int64_t end = child; end > 0; end -= 64 * kRowsAhead) {  // siblings are often near
                bool same = false;
#pragma unroll
                for (int i = 0; i < kRowsAhead; ++i) {
                    const int64_t c = end - 1 - lane - 64 * i;
                    same |= a.parents[max(c, (int64_t)0)] == p && c >= 0;
                }
                if (__any(same)) return false;
            }
            return true;
        });
    }
    // live and dead: a byte for each block, and one for entries that are none
    const int room = lds_room(a), words = room / 32;
    uint8_t *live = reinterpret_cast<uint8_t*>(lds), *dead = live + room;
    int32_t *first = lds + room / 2, *used = first + a.rows, *fresh = used + a.rows;
    // The thread's children, and the copies that they may need: three loads that follow each other, each
    // under way while something else is waited for.
    const int c0 = threadIdx.x * kOneChildren;
    int parent[kOneChildren], len[kOneChildren], block[kOneChildren], column[kOneChildren];
#pragma unroll
    for (int i = 0; i < kOneChildren; ++i) parent[i] = c0 + i < a.children ? parent_of(a, c0 + i) : -1;
    const int kept = old_top(a);
    for (int i = threadIdx.x; i < a.rows; i += kThreads) {
        first[i] = kNone;
        used[i] = used_of(a, length_of(a, i));
    }
    for (int i = threadIdx.x; i < room / 2; i += kThreads) lds[i] = 0;
    lds_barrier();
#pragma unroll
    for (int i = 0; i < kOneChildren; ++i) {
        len[i] = length_of(a, parent[i]);
        if (parent[i] >= 0) atomicMin(first + parent[i], c0 + i);  // the least, in whatever order
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < kOneChildren; ++i)
        column[i] = copied_column(a, parent[i], len[i], [&] { return first[parent[i]] == c0 + i; }, &block[i]);
    for (int r0 = wave; r0 < a.rows; r0 += kWaves * kRowsAhead) {
        // without a branch: of rows and columns that there are not, the last ones again, to no block
        int n[kRowsAhead], most = 0;
        uint8_t* held[kRowsAhead];
        const int32_t* from[kRowsAhead];
#pragma unroll
        for (int i = 0; i < kRowsAhead; ++i) {
            const int r = min(r0 + kWaves * i, a.rows - 1);
            n[i] = used[r];
            most = max(most, n[i]);
            held[i] = first[r] != kNone ? live : dead;
            from[i] = a.tables + r * a.table_ld;
        }
        for (int j = lane; j < most; j += 64) {
            uint32_t b[kRowsAhead];
#pragma unroll
            for (int i = 0; i < kRowsAhead; ++i) b[i] = from[i][min(j, a.width - 1)];
#pragma unroll
            for (int i = 0; i < kRowsAhead; ++i)
                held[i][j < n[i] ? min(b[i], (uint32_t)a.blocks) : (uint32_t)a.blocks] = 1;
        }
    }
    lds_barrier();
    // freed blocks before the thread's 32, and copies before its children
    uint32_t free_bits = 0;
    if ((int)threadIdx.x < words) {
        // the byte past the last block is of none
        const int w = threadIdx.x, in = a.blocks - 32 * w;
        free_bits = bits_of(dead + 32 * w) & ~bits_of(live + 32 * w) & (in < 32 ? (1u << in) - 1 : ~0u);
    }
    int copies = 0;
#pragma unroll
    for (int i = 0; i < kOneChildren; ++i) copies += column[i] >= 0;
    const int mine = __popc(free_bits) << 16 | copies;  // both sums are under 2^16
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(sum, o);
        sum += lane >= o ? up : 0;
    }
    if (lane == 63) totals[wave] = sum;
    lds_barrier();
    int before = sum - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        before += w < wave ? totals[w] : 0;
        all += totals[w];
    }
    const int freed = (uint32_t)all >> 16, taken = all & 0xFFFF;
    const int top = min(kept + freed, a.blocks), left = top - taken;
    // the stack's new part, and what of it is taken again: the top is fresh[0]
    for (int at = kept + (int)((uint32_t)before >> 16); free_bits; free_bits &= free_bits - 1, ++at) {
        const int b = 32 * threadIdx.x + __builtin_ctz(free_bits);
        if (at < left) a.free_out[at] = b;
        else if (top - 1 - at >= 0 && top - 1 - at < taken) fresh[top - 1 - at] = b;
    }
    lds_barrier();
    int rank = before & 0xFFFF;
#pragma unroll
    for (int i = 0; i < kOneChildren; ++i) {
        if (c0 + i >= a.children) break;
        int target = -1;
        if (column[i] >= 0) {
            const int at = top - 1 - rank++;
            target = at >= kept ? fresh[top - 1 - at] : at >= 0 ? a.free_blocks[at] : -1;
            a.tables_out[(int64_t)(c0 + i) * a.width + column[i]] = target;
        }
        a.sources[c0 + i] = block[i];
        a.targets[c0 + i] = target;
    }
    for (int i = threadIdx.x; i < min(kept, left); i += kThreads) a.free_out[i] = a.free_blocks[i];
    for (int i = max(left, 0) + threadIdx.x; i < a.blocks; i += kThreads) a.free_out[i] = -1;
    if (threadIdx.x == 0) *a.num_free_out = left;
}

// A large call, in three launches.
__global__ __launch_bounds__(kThreads) void reorder_clear_kernel(ReorderArgs a, Marks m) {
    if (blockIdx.x > 0) {
        // live and dead lie side by side, in whole words
        uint32_t* words = reinterpret_cast<uint32_t*>(m.live);
        const int64_t count = ((int64_t)a.blocks + 31) / 32 * 16;
        for (int64_t i = (int64_t)(blockIdx.x - 1) * kThreads + threadIdx.x; i < count;
             i += (int64_t)(gridDim.x - 1) * kThreads)
            words[i] = 0;
        return;
    }
    for (int i = threadIdx.x; i < a.rows; i += kThreads) m.first[i] = kNone;
    __threadfence();  // the minima are formed in L2
    __syncthreads();
    first_children(a, m.first);
}

__global__ __launch_bounds__(256) void reorder_mark_kernel(ReorderArgs a, Marks m) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.rows) return;
    const int used = used_of(a, length_of(a, row));
    uint8_t* held = m.first[row] != kNone ? m.live : m.dead;
    const int32_t* t = a.tables + row * a.table_ld;
    for (int j = blockIdx.y * 64 + (threadIdx.x & 63); j < used; j += 64 * gridDim.y) {
        const int b = t[j];
        if (b >= 0 && b < a.blocks) held[b] = 1;
    }
}

// The first workgroup writes the stack, the others rows.
__global__ __launch_bounds__(kThreads) void reorder_write_kernel(ReorderArgs a, Marks m) {
    __shared__ int totals[kWaves];
    auto is_first = [&](int p, int64_t child) { return m.first[p] == child; };
    if (blockIdx.x == 0)
        return write_stack(
            a, totals,
            [&](int64_t w) { return bits_of(m.dead + 32 * w) & ~bits_of(m.live + 32 * w); }, is_first);
    const int64_t child = (int64_t)(blockIdx.x - 1) * kWaves + (threadIdx.x >> 6);
    if (child < a.children)
        write_row(a, child, threadIdx.x & 63, [&](int p) { return is_first(p, child); });
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
    int next_from = -1, next_to = -1;
    if (lane < a.rows) next_from = a.sources[lane], next_to = a.targets[lane];
    for (int64_t r0 = 0; r0 < a.rows; r0 += 64) {
        const int from = next_from, to = next_to;
        next_from = next_to = -1;
        if (r0 + 64 + lane < a.rows)
            next_from = a.sources[r0 + 64 + lane], next_to = a.targets[r0 + 64 + lane];
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

// LDS of a call in one launch.
int64_t lds_bytes(const ReorderArgs& a) {
    return (int64_t)a.rows * 8 + 2 * (int64_t)lds_room(a) + (int64_t)a.children * 4;
}

// One launch while the blocks' bytes fit LDS, one workgroup goes through the entries in the time of two
// more launches, and looking for siblings is short.
bool one_launch(const ReorderArgs& a) {
    return lds_bytes(a) <= 60 * 1024 && lds_room(a) <= 32 * kThreads &&
           (int64_t)a.rows * a.width <= 65536 && a.children <= kThreads * kOneChildren;
}

int64_t mark_bytes(const ReorderArgs& a) { return ((int64_t)a.blocks + 31) / 32 * 32; }

}  // namespace

size_t kv8_reorder_bytes(const ReorderArgs& a) {
    return one_launch(a) ? 0 : (size_t)(2 * mark_bytes(a) + (int64_t)a.rows * 4);
}

hipError_t launch_kv8_reorder(const ReorderArgs& a, void* ws, hipStream_t stream) {
    const unsigned writers = (unsigned)(1 + ((int64_t)a.children + kWaves - 1) / kWaves);
    if (one_launch(a)) {
        reorder_kernel<<<writers, kThreads, (size_t)lds_bytes(a), stream>>>(a);
        return hipGetLastError();
    }
    Marks m;
    m.live = static_cast<uint8_t*>(ws);
    m.dead = m.live + mark_bytes(a);
    m.first = reinterpret_cast<int32_t*>(m.dead + mark_bytes(a));
    const int64_t clearing = (2 * mark_bytes(a) + 65535) / 65536;
    reorder_clear_kernel<<<(unsigned)(1 + (clearing < 256 ? clearing : 256)), kThreads, 0, stream>>>(a, m);
    if (a.rows > 0) {
        // long tables of few rows by several waves each
        int64_t split = a.rows < 1024 ? 1024 / a.rows : 1;
        const int64_t most = ((int64_t)a.width + 255) / 256;
        split = split < most ? split : most;
        const dim3 grid((unsigned)(((int64_t)a.rows + 3) / 4), (unsigned)(split < 1 ? 1 : split));
        reorder_mark_kernel<<<grid, 256, 0, stream>>>(a, m);
    }
    reorder_write_kernel<<<writers, kThreads, 0, stream>>>(a, m);
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
