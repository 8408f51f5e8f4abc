// beam_select.hip -- the best continuations of groups of beams: for each group the largest of
//   value(b, t) = score_b + (x_bt - m_b) - log s_b,   m_b = max x_b,   s_b = sum exp(x_b - m_b),
// over its beams b and all tokens t of the vocabulary, equal values by rising beam, of one
// beam by falling logit, then by rising token.
//
// Two launches.  The first reads every beam's logits once: sums, and the largest few of each part of
// a row (logit_rows.h).  The second joins a group: at most `num` logits of a beam can be among the
// group's best.

#include <hip/hip_runtime.h>

#include <type_traits>

#include "logit_rows.h"

namespace ojx {

namespace {

// Of a part of a row: s = sum 2^(x log2(e) - r) with r a whole number near the largest exponent, so
// that sums of different r join without a rounding.
struct BeamSum {
    double s;
    float r, m;
};

struct BeamParts {
    BeamSum* sums;   // [rows][splits]
    uint64_t* keys;  // [rows][splits][num], falling, 0 behind the last
    int splits;
};

// Whether a beam's logits matter: not those of a finished one, nor where no finite score leaves them.
__device__ __forceinline__ bool reads_logits(const BeamArgs& a, int64_t row) {
    const float score = a.scores[row];
    return !(a.done && a.done[row]) && score < INFINITY && score > -INFINITY;
}

__device__ __forceinline__ double scaled(double s, float r, float to) {
    return ldexp(s, (int)fmaxf(r - to, -2000.f));
}

constexpr int kSlots = 16;        // maxima that a lane keeps of the batches it has seen
constexpr int kCandidates = 192;  // that a wave has room for

// A workgroup reads a row or a part of it once; rows that do not matter not at all.  Four partial
// sums of 8 terms a batch are held in 32 bits, everything beyond in 64: whole numbers (which beam)
// hang on these sums, and the join has to settle in 64 bits what they leave open.
//
// Nothing is selected on the way, a lane only keeps its batches' maxima.  Of 64 shares of the part,
// the num-th largest maximum is not over num logits at least, and few more than num are over it: the
// batches of the few lanes that have one are read again.  Where there are too many (a row of few
// values, a short one), the part is gone through once more batch by batch.
//
// 512 rows of 128256 bf16 (131 MB) take 39 us, 3.4 TB/s: about 5 us until all workgroups run and have
// their first logits, and 6 for what follows a row's last one, around a stream at 4.9 TB/s (selecting
// on the way, batch by batch, 51 us; the next batch's loads ahead, no change).
template <int DT>
__global__ __launch_bounds__(kThreads) void beam_pass_kernel(BeamArgs a, BeamParts p) {
    __shared__ union {
        struct {
            float maxima[kSlots * kThreads];
            uint64_t keys[kGroups][kCandidates];
        } few;
        struct {
            Pool pool[kGroups];
            uint64_t keys[kGroups * kTopMax];
        } many;
    } mem;
    __shared__ BeamSum sums[kGroups];
    __shared__ float lanes[kThreads], columns[kGroups][64];
    __shared__ int counts[kGroups];
    using B = Batch<DT>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x / (unsigned)p.splits;
    const int split = blockIdx.x - (unsigned)row * p.splits;
    if (!reads_logits(a, row)) return;
    const int64_t x0 = row * a.ld;
    const int size = DT == kF32 ? 4 : 2;
    const int shift = (int)((((uintptr_t)a.x + x0 * size) & 15) / size);
    const int batches = (int)(((int64_t)a.vocab + shift + kBatch - 1) / kBatch);
    const int per = (batches + p.splits - 1) / p.splits;
    const int first = split * per + wave, end = min(batches, (split + 1) * per);
    // batches of this wave that share a slot
    const int share = (per + kGroups * kSlots - 1) / (kGroups * kSlots);
    double sum = 0;
    float ref = -INFINITY, most = -INFINITY, slot = -INFINITY;
    B x;
    int s_at = 0, s_left = share, held = -1;
    for (int b = first; b < end; b += kGroups) {
        x.load(a.x, x0, a.vocab, b, lane, shift);
        held = b;
        float m = x.get(0);
#pragma unroll
        for (int i = 1; i < kLaneLogits; ++i) m = or_nan(m, x.get(i));
        const float r = fmaxf(ref, m < -kPlainMax ? -INFINITY : ceilf(m * kLog2e));
        const float base = r == -INFINITY ? 0.f : r;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kLaneLogits; ++i)
            s[i & 3] += __builtin_amdgcn_exp2f(__builtin_fmaf(x.get(i), kLog2e, -base));
        sum = scaled(sum, ref, base) + (((double)s[0] + s[1]) + ((double)s[2] + s[3]));
        ref = r;
        most = or_nan(most, m);
        slot = fmaxf(slot, m);
        if (--s_left == 0 || b + kGroups >= end) {
            mem.few.maxima[s_at * kThreads + threadIdx.x] = slot;
            ++s_at, s_left = share, slot = -INFINITY;
        }
    }
    lanes[threadIdx.x] = most;
    // over the wave
    const bool bad = __any(most != most);
    {
        const float r = wave_max(ref), base = r == -INFINITY ? 0.f : r;
        double t = scaled(sum, ref, base);
#pragma unroll
        for (int o = 32; o; o >>= 1) t += __shfl_xor(t, o);
        const float m = wave_max(most);
        if (lane == 0) sums[wave] = BeamSum{t, r, bad ? __uint_as_float(0x7FC00000u) : m};
    }
    __syncthreads();
    const int64_t at = row * p.splits + split;
    if (threadIdx.x == 0) {
        BeamSum t = sums[0];
        for (int w = 1; w < kGroups; ++w) {
            const float to = fmaxf(t.r, sums[w].r), from = to == -INFINITY ? 0.f : to;
            t = BeamSum{scaled(t.s, t.r, from) + scaled(sums[w].s, sums[w].r, from), to,
                        or_nan(t.m, sums[w].m)};
        }
        p.sums[at] = t;
    }
    // the num-th largest of the shares' maxima: the least of those that fewer exceed
    const float share_max = fmaxf(fmaxf(lanes[lane], lanes[lane + 64]),
                                  fmaxf(lanes[lane + 128], lanes[lane + 192]));
    columns[wave][lane] = share_max;
    __builtin_amdgcn_wave_barrier();
    int over = 0;
#pragma unroll
    for (int j = 0; j < 64; j += 4) {
        const float4 f = *reinterpret_cast<const float4*>(columns[wave] + j);
        over += f.x > share_max;
        over += f.y > share_max;
        over += f.z > share_max;
        over += f.w > share_max;
    }
    const float bound = -wave_max(over < a.num ? -share_max : -INFINITY);
    int n = 0;
    if (bound > -INFINITY) {
        for (int s = 0; s < s_at; ++s) {
            const bool mine = mem.few.maxima[s * kThreads + threadIdx.x] >= bound;
            if (!__any(mine)) continue;
            for (int i = 0; i < share; ++i) {
                const int b = first + (s * share + i) * kGroups;
                if (b >= end) break;
                if (mine && b != held) {
                    x.load(a.x, x0, a.vocab, b, lane, shift);
                    held = b;
                }
#pragma unroll
                for (int j = 0; j < kLaneLogits; ++j) {
                    const float f = x.get(j);
                    const uint64_t those = __ballot(mine && f >= bound);
                    if (!those) continue;
                    const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(those >> 32),
                                                                 __builtin_amdgcn_mbcnt_lo((uint32_t)those, 0));
                    if (mine && f >= bound && at < kCandidates)
                        mem.few.keys[wave][at] = key_of(f, B::index(b, j, lane, shift));
                    n += __popcll(those);
                }
            }
        }
    }
    if (lane == 0) counts[wave] = n;
    __syncthreads();
    bool fits = bound > -INFINITY;
    for (int w = 0; w < kGroups; ++w) fits &= counts[w] <= kCandidates;
    if (!fits) {
        Best best{0, -INFINITY};
        for (int b = first; b < end; b += kGroups) {
            x.load(a.x, x0, a.vocab, b, lane, shift);
            float m = x.get(0);
#pragma unroll
            for (int i = 1; i < kLaneLogits; ++i) m = or_nan(m, x.get(i));
            x.drop_floats();
            take<DT>(best, x, m, b, a.num, lane, shift, mem.many.pool[wave]);
        }
        if (lane < a.num) mem.many.keys[wave * a.num + lane] = best.key;
        __syncthreads();
        for (int i = threadIdx.x; i < kGroups * a.num; i += kThreads) {
            const uint64_t k = mem.many.keys[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < kGroups * a.num; ++j)
                rank += mem.many.keys[j] > k || (mem.many.keys[j] == k && j < i);
            if (rank < a.num) p.keys[at * a.num + rank] = k;
        }
        return;
    }
    // at least num of them, all different
    for (int i = lane; i < n; i += 64) {
        const uint64_t k = mem.few.keys[wave][i];
        int rank = 0;
        for (int w = 0; w < kGroups; ++w) {
            const int m = counts[w];
#pragma unroll 4
            for (int j = 0; j < m; ++j) rank += mem.few.keys[w][j] > k;
        }
        if (rank < a.num) p.keys[at * a.num + rank] = k;
    }
}

constexpr int kJoinThreads = 512;
constexpr int kJoinWaves = kJoinThreads / 64;
constexpr int kJoinBytes = 60 * 1024;  // of LDS for a row's lists and the group's candidates
// Two values of different beams that are closer than this are compared again with sums in 64 bits.
// What a beam's sum in the first pass is off by at most, of itself, in units of 2^-20:
//   0.125  its exponentials, 2^-23 each;
//   0.70   their exponents' rounding, half a step: 2^-20 ln 2 from 16 to 32 binary places under the lane's
//          largest so far, less above; a lane's 2^22 terms (of 2^30 logits) that are further under weigh
//          2^-10 together;
//   0.30   the constant's error, 2^-26.1 of the terms' mean distance from the largest, which is under
//          ln 2^30;
//   0.44   sums of 8 in 32 bits, 7 * 2^-24.
// Together 1.57, under 2^-19; two beams' may lean apart.  Two calls of 60 of 64 x 8 beams had such a
// pair (which takes a workgroup some 80 us).
constexpr double kNear = 0x1p-18;

// fp64 bits in rising order as unsigned; NaN above everything.
__device__ __forceinline__ uint64_t ordered64(double v) {
    if (v != v) return ~0ull;
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double unordered64(uint64_t k) {
    if (k == ~0ull) return __longlong_as_double(0x7FF8000000000000ll);
    return __longlong_as_double((int64_t)(k >> 63 ? k & ~(1ull << 63) : ~k));
}

// Whether the order of two values, u the larger, may be another with sums in 64 bits: beside a large
// score each is rounded by half a step of its own too, up to 2^-53 of it, before and after: 2^-51 of
// it together, and this is twice as much.
__device__ __forceinline__ bool near(double u, double v) { return u - v < kNear + 0x1p-50 * fabs(u); }

// A beam in the join.
struct Beam {
    double ls;   // log of the sum of exp(x - m)
    float m, score;
    int count;   // candidates
    bool exact;  // ls is a sum in 64 bits, or none is needed
    bool need;   // such a sum is asked for
};

// One workgroup a group.
template <int DT>
__global__ __launch_bounds__(kJoinThreads) void beam_join_kernel(BeamArgs a, BeamParts p) {
    extern __shared__ uint64_t lds[];
    __shared__ Beam beams[kBeamMax];
    __shared__ uint64_t top_value[kTopMax];
    __shared__ int top_beam[kTopMax], top_token[kTopMax];
    __shared__ double part[kJoinWaves];
    __shared__ int listed;
    __shared__ unsigned long long close;  // beams near the last place
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = p.splits * a.num, all = a.beams * a.num;
    uint64_t* list = lds + wave * n;
    uint64_t* value = lds + kJoinWaves * n;                        // [beams][num], falling
    int* token = reinterpret_cast<int*>(value + all);              // [beams][num]
    const int64_t row0 = (int64_t)blockIdx.x * a.beams;

    for (int b = wave; b < a.beams; b += kJoinWaves) {
        const int64_t row = row0 + b;
        const float score = a.scores[row];
        const bool ended = a.done && a.done[row];
        // (of a row that does not matter these are not written, nor used)
        BeamSum s{0.0, -INFINITY, -INFINITY};
        if (lane < p.splits) s = p.sums[row * p.splits + lane];
        for (int i = lane; i < n; i += 64) list[i] = p.keys[row * n + i];
        Beam t{0.0, 0.f, score, 0, true, false};
        bool nan = !(score < INFINITY);
        if (!ended && score < INFINITY && score > -INFINITY) {
            const float r = wave_max(s.r), base = r == -INFINITY ? 0.f : r;
            double sum = scaled(s.s, s.r, base);
#pragma unroll
            for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
            nan = __any(s.m != s.m);
            t.m = wave_max(s.m);
            nan |= t.m == INFINITY;
            if (!nan && t.m > -INFINITY) {
                // the pass's own log2(e), so that what it is off by cancels at m
                t.ls = log(sum) - ((double)t.m * (double)kLog2e - (double)r) * 0.6931471805599453;
                t.exact = false;
                t.need = !(t.m > -kPlainMax && t.m < kPlainMax);
                __builtin_amdgcn_wave_barrier();
                // Parts' lists fall: of all but the last part, which may be short, the (num / parts)-th
                // keys are a bound that num keys reach; what is under it goes.
                int m = n;
                if (p.splits > 2) {
                    const int parts = p.splits - 1, at = (a.num + parts - 1) / parts - 1;
                    uint64_t least = lane < parts ? list[lane * a.num + at] : ~0ull;
#pragma unroll
                    for (int o = 32; o; o >>= 1) {
                        const uint64_t other = __shfl_xor(least, o);
                        least = least < other ? least : other;
                    }
                    m = 0;
                    for (int i0 = 0; i0 < n; i0 += 64) {
                        const uint64_t mine = i0 + lane < n ? list[i0 + lane] : 0;
                        const bool in = mine != 0 && mine >= least;
                        const uint64_t those = __ballot(in);
                        __builtin_amdgcn_wave_barrier();
                        if (in) list[m + __popcll(those & ((1ull << lane) - 1))] = mine;
                        __builtin_amdgcn_wave_barrier();
                        m += __popcll(those);
                    }
                }
                for (int i0 = 0; i0 < m; i0 += 64) {
                    const uint64_t mine = i0 + lane < m ? list[i0 + lane] : 0;
                    int rank = 0;
#pragma unroll 8
                    for (int j = 0; j < m; ++j) rank += list[j] > mine;
                    const bool in = mine != 0 && rank < a.num;
                    if (in) {
                        const float x = unordered((uint32_t)(mine >> 32));
                        value[b * a.num + rank] = ordered64(score + (((double)x - t.m) - t.ls));
                        token[b * a.num + rank] = (int)(0xFFFFFFFFu - (uint32_t)mine);
                    }
                    t.count += __popcll(__ballot(in));
                }
                __builtin_amdgcn_wave_barrier();
            }
        } else if (ended && !nan && score > -INFINITY) {
            t.count = 1;
            if (lane == 0) value[b * a.num] = ordered64(score), token[b * a.num] = (int)a.pad;
        }
        if (nan) {  // every token
            t.count = min(a.num, a.vocab);
            if (lane < t.count) value[b * a.num + lane] = ~0ull, token[b * a.num + lane] = lane;
        }
        if (lane == 0) beams[b] = t;
    }
    __syncthreads();

    int total = lane < a.beams ? beams[lane].count : 0;
#pragma unroll
    for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
    bool needed = __any(lane < a.beams && beams[lane].need);
    for (;;) {
        // sums in 64 bits of the beams that need one, over tokens in the same order for each beam:
        // equal rows have equal sums
        for (int b = 0; needed && b < a.beams; ++b) {
            if (!beams[b].need) continue;
            const int64_t x0 = (row0 + b) * a.ld;
            const double m = beams[b].m;
            double s = 0;
#pragma unroll 4
            for (int j = threadIdx.x; j < a.vocab; j += kJoinThreads)
                s += exp((double)load_as_f32<DT>(a.x, x0 + j) - m);
#pragma unroll
            for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
            if (lane == 0) part[wave] = s;
            __syncthreads();
            s = 0;
            for (int w = 0; w < kJoinWaves; ++w) s += part[w];
            const double ls = log(s);
            for (int i = threadIdx.x; i < beams[b].count; i += kJoinThreads) {
                const float x = load_as_f32<DT>(a.x, x0 + token[b * a.num + i]);
                value[b * a.num + i] = ordered64(beams[b].score + (((double)x - m) - ls));
            }
            __syncthreads();
            if (threadIdx.x == 0) beams[b].ls = ls, beams[b].exact = true, beams[b].need = false;
            __syncthreads();
        }
        // Of many candidates those under a bound have no place: the least of the (q + 1)-th values of
        // beams that have so many, for the first q where these are num in all.  The others are listed
        // (where the parts' lists were), in any order.
        int count = all;
        int* alive = reinterpret_cast<int*>(lds);
        if (all > kJoinThreads) {
            uint64_t bound = 0;
            const int mine = lane < a.beams ? beams[lane].count : 0;
            for (int q = 0; q < a.num; ++q) {
                const uint64_t those = __ballot(mine > q);
                if (__popcll(those) * (q + 1) < a.num) continue;
                bound = mine > q ? value[lane * a.num + q] : ~0ull;
#pragma unroll
                for (int o = 32; o; o >>= 1) {
                    const uint64_t other = __shfl_xor(bound, o);
                    bound = bound < other ? bound : other;
                }
                break;
            }
            if (threadIdx.x == 0) listed = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < all; i += kJoinThreads) {
                const int b = i / a.num;
                if (i - b * a.num >= beams[b].count || value[i] < bound) continue;
                const int at = atomicAdd(&listed, 1);
                if (at < kJoinWaves * n * 2) alive[at] = i;
            }
            __syncthreads();
            if (listed <= kJoinWaves * n * 2) count = listed;
        }
        if (threadIdx.x == 0) close = 0;  // (the last round's has been seen by all)
        // lanes for a candidate: a power of two of at most a wave, none without a beam to look through
        int team = 1;
        while (team < 64 && 2 * team * count <= kJoinThreads && team < a.beams) team *= 2;
        // a candidate's rank: those before it in its beam, and in the others' lists, which the lanes
        // of a team share out
        for (int at = (int)threadIdx.x / team; at < count; at += kJoinThreads / team) {
            const int i = count < all ? alive[at] : at;
            const int b = i / a.num, place = i - b * a.num;
            if (place >= beams[b].count) continue;
            const uint64_t v = value[i];
            int rank = 0;
            for (int o = threadIdx.x & (team - 1); o < a.beams; o += team) {
                if (o == b) continue;
                // of an earlier beam equal ones come first
                const uint64_t least = v + (o < b ? 0 : 1);
                int lo = 0, hi = v == ~0ull && o > b ? 0 : beams[o].count;
                while (lo < hi) {
                    const int m = (lo + hi) >> 1;
                    if (value[o * a.num + m] >= least) lo = m + 1;
                    else hi = m;
                }
                rank += lo;
            }
            for (int o = team >> 1; o; o >>= 1) rank += __shfl_xor(rank, o);
            rank += place;
            if (rank < a.num && (threadIdx.x & (team - 1)) == 0) {
                top_value[rank] = v;
                top_beam[rank] = b;
                top_token[rank] = token[i];
            }
        }
        __syncthreads();
        // Neighbours of different beams that are near, and beams that are near the last place in it or
        // not: among the former, ranks tell which candidates are next to each other, but those behind the
        // last place have none.
        const int last = min(total, a.num) - 1;
        bool again = false;
        if ((int)threadIdx.x < last) {
            const int i = threadIdx.x, b = top_beam[i], c = top_beam[i + 1];
            if (b != c && !(beams[b].exact && beams[c].exact) &&
                near(unordered64(top_value[i]), unordered64(top_value[i + 1]))) {
                again = true;
                // (lanes that find the same beam write the same)
                if (!beams[b].exact) beams[b].need = true;
                if (!beams[c].exact) beams[c].need = true;
            }
        }
        if (total > a.num) {
            const double border = unordered64(top_value[a.num - 1]);
            for (int i = threadIdx.x; i < all; i += kJoinThreads) {
                const int b = i / a.num;
                if (i - b * a.num >= beams[b].count) continue;
                const double v = unordered64(value[i]);
                if (v > border ? near(v, border) : near(border, v)) atomicOr(&close, 1ull << b);
            }
            __syncthreads();
            const uint64_t those = close;
            if ((int)threadIdx.x < a.beams && __popcll(those) > 1 && (those >> threadIdx.x & 1) &&
                !beams[threadIdx.x].exact)
                again = beams[threadIdx.x].need = true;
        }
        // (the same in all lanes, which the compiler has to know: they go round together)
        needed = __builtin_amdgcn_readfirstlane(__syncthreads_or(again));
        if (!needed) break;
    }

    const int64_t o0 = (int64_t)blockIdx.x * a.num;
    if ((int)threadIdx.x < min(total, a.num)) {
        const int i = threadIdx.x;
        a.out_scores[o0 + i] = (float)unordered64(top_value[i]);
        a.out_parents[o0 + i] = row0 + top_beam[i];
        a.out_tokens[o0 + i] = top_token[i];
    }
    // Fewer than asked for: impossible ones follow, by rising beam and token.  Those possible are all
    // in the lists, so the first `num` others are among the group's first total + num.
    if (total < a.num && wave == 0) {
        int have = total;
        for (int64_t f0 = 0; have < a.num; f0 += 64) {
            const int64_t f = f0 + lane, b = f / a.vocab;
            const int t = (int)(f - b * a.vocab);
            bool free = b < a.beams;
            if (free)
                for (int i = 0; i < beams[b].count; ++i) free &= token[b * a.num + i] != t;
            const uint64_t those = __ballot(free);
            const int rank = have + __popcll(those & ((1ull << lane) - 1));
            if (free && rank < a.num) {
                a.out_scores[o0 + rank] = -INFINITY;
                a.out_parents[o0 + rank] = row0 + b;
                a.out_tokens[o0 + rank] = t;
            }
            have += __popcll(those);
        }
    }
}

size_t join_bytes(int splits, int beams, int num) {
    return (size_t)kJoinWaves * splits * num * 8 + (size_t)beams * num * 12;
}

// Parts of a row: until there are four workgroups for each CU, which run at once, none under a batch
// for each wave, and as many as the join has room for (512 rows of 128256 whole 48.4 us, in two 46.3;
// 4 rows of 32000 whole 17.2, in two 15.4, in four 13.5).
int beam_splits(const BeamArgs& a) {
    const int64_t rows = (int64_t)a.groups * a.beams;
    const int64_t most = ((int64_t)a.vocab + kBatch * kGroups - 1) / (kBatch * kGroups);
    int64_t n = rows > 0 ? 1024 / rows : 1;
    if (n > most) n = most;
    if (n > kMaxRowSplits) n = kMaxRowSplits;
    while (n > 1 && join_bytes((int)n, a.beams, a.num) > kJoinBytes) --n;
    return n < 1 ? 1 : (int)n;
}

size_t part_bytes(const BeamArgs& a) {
    return (size_t)a.groups * a.beams * (sizeof(BeamSum) + a.num * sizeof(uint64_t));
}

}  // namespace

size_t beam_select_bytes(const BeamArgs& a) { return part_bytes(a) * beam_splits(a); }
size_t beam_select_least_bytes(const BeamArgs& a) { return part_bytes(a); }

hipError_t launch_beam_select(const BeamArgs& a, void* ws, size_t ws_bytes, hipStream_t stream) {
    BeamParts p{};
    p.splits = beam_splits(a);
    const size_t fit = ws_bytes / part_bytes(a);
    if (fit < 1) return hipErrorInvalidValue;
    if ((size_t)p.splits > fit) p.splits = (int)fit;
    const int64_t rows = (int64_t)a.groups * a.beams, grid = rows * p.splits;
    if (grid > kMaxGroups256 || a.groups > kMaxGroups512) return hipErrorInvalidValue;
    p.sums = static_cast<BeamSum*>(ws);
    p.keys = reinterpret_cast<uint64_t*>(p.sums + (size_t)rows * p.splits);
    hipError_t pass = hipSuccess;
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        beam_pass_kernel<DT><<<(unsigned)grid, kThreads, 0, stream>>>(a, p);
        // the join reads logits at the tokens that the pass found: never without it
        if ((pass = hipGetLastError()) != hipSuccess) return;
        beam_join_kernel<DT><<<(unsigned)a.groups, kJoinThreads, join_bytes(p.splits, a.beams, a.num),
                               stream>>>(a, p);
    };
    if (a.dtype == kF32) go(std::integral_constant<int, kF32>{});
    else if (a.dtype == kF16) go(std::integral_constant<int, kF16>{});
    else go(std::integral_constant<int, kBF16>{});
    return pass != hipSuccess ? pass : hipGetLastError();
}

}  // namespace ojx
