// beam.hip -- the best continuations of groups of beams: log-softmax of each
// beam's logits, selection over beams and vocabulary.
//
// Candidate (b, t) of a group has the score s_b + x_bt - log sum_u exp x_bu; an
// ended beam has one, (b, eos) with s_b.  The k best of a group: within a beam by
// logit, then the lower token, between beams by score in 64 bits, then the lower
// beam.  (Logits that differ may have equal scores: 0 and 1e-20.)
//
// One pass over the logits.  A wave holds a tile of 2048 of a row's in registers:
// their maximum, the sum of exponentials against it (published, a pair a tile),
// and what of them is among the wave's k best so far.  A tile whose largest is
// no better than the k-th best has nothing.  Else a border is searched, by
// bisection with ballots, that at least k of the lanes' maxima reach and few
// more; the values that reach it and the k-th best so far go to the wave's list
// in LDS, in which each finds its rank by comparing itself with all.  A key is the
// logit's order-preserving bits over the complement of its token, unique, so ties
// cost nothing.  Tiles and sums are the same whatever the number of workgroups a
// row has, which follows the number of rows: waves get one tile more at a time
// once there are more than 16 a CU.
//
// The last workgroup of a group to arrive (ticket) merges: a wave a beam weighs the
// tiles' sums by f32 exponentials of their largest logits, adds them in order and in
// 64 bits, and takes the k best of the waves' lists in the same way as of a tile;
// then each of the beams' candidates counts those that come before it, in 64-bit
// scores.  Results are a function of the group's rows alone.
//
// What bounds it, us a call of 151936 tokens (bytes at the 5.1 TB/s of a large
// copy in brackets): 1 x 5 beams 9.8-10.0 (0.6) and 16 x 5 with 10 candidates
// 18.9-19.2 (9.5): a chain of launch 1.5, a tile 2.5-3 (loads 0.5, maximum and sum 0.6, border
// 0.4, list 1), stores and ticket 2, the merge 4-5 (two trips to memory, list, ranks),
// and behind it, for 16 x 5, the loads; 64 x 4 with 40 ended 30.0-30.6 (25.7): the loads, 4.3 TB/s.
// Measured against this: workgroups of 4 waves 12.5 / 23.0 / 31.7; keys ranked one
// after the other by readlane 10.6 / 21.1 / 30.5; the next tile's loads ahead of a
// tile (4 waves a SIMD instead of 6) 10.0 / 21.0 / 32.1; loads past the caches 9.8 /
// 19.5 / 30.0; 8 or 24 tiles a CU and turn instead of 16: 24.4 and 22.3 for 16 x 5.
#include "beam.hpp"

namespace qasr {

namespace {

constexpr int kThreads = kBeamWaves * 64;
// A lane's logits of a tile; a vector, as a choice between elements of an array
// is one between addresses and puts it into memory.
typedef float Tile __attribute__((ext_vector_type(kBeamValues)));
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -__builtin_inff();

__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(float x, int token) { return (uint64_t)order_of(x) << 32 | ~(uint32_t)token; }
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o ^ ((int32_t)o < 0 ? 0x80000000u : 0xffffffffu));
}
// The least finite value whose ordered bits reach `border`.
__device__ __forceinline__ float value_of(uint32_t border) {
    return logit_of((uint64_t)max(border, order_of(-3.4028234663852886e38f)) << 32);
}
__device__ __forceinline__ int token_of(uint64_t key) { return (int)~(uint32_t)key; }

__device__ __forceinline__ void store_dev64(uint64_t* p, uint64_t v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t load_dev64(const uint64_t* p) {
    return __hip_atomic_load(const_cast<uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// A scalar load of what no workgroup writes before all have read it.
template <class T>
__device__ __forceinline__ T scalar(const T* p) {
    return *(const __attribute__((address_space(4))) T*)p;
}

__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, dpp<kDppXor1>(x));
    x = fmaxf(x, dpp<kDppXor2>(x));
    x = fmaxf(x, dpp<kDppHalfMirror>(x));
    x = fmaxf(x, dpp<kDppMirror>(x));
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float wave_sum(float x) {
    x = row_sum16(x);
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A border that at least k of the lanes' values reach, by their ordered bits, of
// which `top` are the largest, and few more than k, unless several are equal to
// the k-th; 0 if fewer than k are not 0.
constexpr int kSpare = 3;  // (ranking some values more is cheaper than to go on; 8: the same within 0.2 us)
__device__ __forceinline__ uint32_t border_of(uint32_t mine, uint32_t top, int k) {
    uint32_t lo = 0, hi = top + 1;  // at least k reach lo, fewer hi (none has all bits set)
    int n = __popcll(__ballot(mine != 0));
    if (n < k) return 0;
    // (The k-th is mostly near: from further below the top each time.)
    for (uint32_t d = 1u << 20; d != 0 && d < top; d <<= 2) {  // 2^20 .. 2^30, then 0
        const int m = __popcll(__ballot(mine >= top - d));
        if (m >= k) {
            lo = top - d;
            n = m;
            break;
        }
        hi = top - d;
    }
    while (n > k + kSpare && hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        const int m = __popcll(__ballot(mine >= mid));
        if (m >= k) {
            lo = mid;
            n = m;
        } else {
            hi = mid;
        }
    }
    return max(lo, 1u);
}

// A beam that offers nothing: its score is -inf, +inf or NaN.
__device__ __forceinline__ bool dead(float score) { return !(fabsf(score) < __builtin_inff()); }

// LDS accesses of this wave in order.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A wave's k best keys so far, best first, in its list in LDS, and behind them
// what may be among them.
constexpr int kPending = 64;
constexpr int kList = kBeamMaxK + kPending;
struct Best {
    uint64_t kth = 0;  // 0 while there are fewer
    int held = 0, pending = 0;
};
// Each key's rank is the number of better ones: every lane compares its own (or
// two) with all, which it reads two at a time.  Keys are unique.
__device__ __forceinline__ void rank_list(Best& b, int k, int lane, uint64_t* list) {
    typedef unsigned long long Two __attribute__((ext_vector_type(2)));
    const int total = b.held + b.pending;
    if (lane == 0) list[total] = 0;
    wave_sync();
    const uint64_t x = list[lane], y = total > 64 ? list[min(lane + 64, kList)] : 0;
    int rank = 0, rank_y = 0;
#pragma unroll 4
    for (int j = 0; j < total; j += 2) {
        const Two z = *(const Two*)(list + j);
        rank += (z[0] > x) + (z[1] > x);
        if (total > 64) rank_y += (z[0] > y) + (z[1] > y);
    }
    wave_sync();
    if (lane < total && rank < k) list[rank] = x;
    if (lane + 64 < total && rank_y < k) list[rank_y] = y;
    b.held = min(total, k);
    b.pending = 0;
    wave_sync();
    b.kth = b.held == k ? list[k - 1] : 0;
}
// Takes a key of each lane (0: none) into the list.
__device__ __forceinline__ void take(Best& b, uint64_t key, int k, int lane, uint64_t* list) {
    uint64_t some = __ballot(key > b.kth);
    if (b.pending + __popcll(some) > kPending) {
        rank_list(b, k, lane, list);
        some = __ballot(key > b.kth);
    }
    if (key > b.kth) list[b.held + b.pending + __popcll(some & ((1ull << lane) - 1))] = key;
    b.pending += __popcll(some);
}

// A tile's values, of which this lane's largest is `top`, the wave's M.  Token of
// v[i]: first + 256 (i / 4) + i % 4.
__device__ __forceinline__ void take_tile(Best& b, const Tile& v, float top, float M, int first, int k, int lane, uint64_t* list) {
    // At least k of the row reach the border, a value.
    uint32_t border = max((uint32_t)(b.kth >> 32), 1u);
    const uint32_t mine = top == kNone ? 0 : order_of(top + 0.0f);
    if (__popcll(__ballot(mine >= border)) > k + kSpare) border = max(border, border_of(mine, order_of(M + 0.0f), k));
    const float least = value_of(border);
    uint32_t mask = 0;
#pragma unroll
    for (int i = kBeamValues - 1; i >= 0; --i) mask = 2 * mask + (v[i] >= least);
    while (__ballot(mask != 0)) {  // a value of each lane at a time, the lower token first
        const int i = mask ? __builtin_ctz(mask) : 0;
        Tile x = v;  // v[i]: a bit of i a step
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = i & 1 ? x[2 * j + 1] : x[2 * j];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = i & 2 ? x[2 * j + 1] : x[2 * j];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = i & 4 ? x[2 * j + 1] : x[2 * j];
#pragma unroll
        for (int j = 0; j < 2; ++j) x[j] = i & 8 ? x[2 * j + 1] : x[2 * j];
        const float y = (i & 16 ? x[1] : x[0]) + 0.0f;  // -0 is 0
        take(b, mask ? key_of(y, first + 256 * (i >> 2) + (i & 3)) : 0, k, lane, list);
        mask &= mask - 1;
    }
    if (b.pending) rank_list(b, k, lane, list);
}

struct Shared {
    alignas(16) uint64_t list[kBeamWaves][kList + 2];
    int last;
};

// Row sums and lists of the group's beams, a wave a beam; then the beams'
// candidates against each other.  score, ended: of beam `lane`.
constexpr int kBatch = 8;  // keys of a lane at a time
typedef unsigned long long Keys __attribute__((ext_vector_type(kBatch)));
__device__ __forceinline__ void merge(const BeamArgs& a, int group, int lists, float score, bool ended, Shared& sh,
                                      double* s_score) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), k = a.k;
    const int tiles = (a.vocab + kBeamTile - 1) / kBeamTile, n = a.width * k;
    int *s_token = (int*)(s_score + n), *s_rank = s_token + n;
    const uint64_t endeds = __ballot(ended);
    for (int b = wave; b < a.width; b += kBeamWaves) {
        const int row = group * a.width + b;
        const float s_b = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(score), b));
        double mine = kNone;  // candidate `lane`
        int token = a.eos;
        if (!dead(s_b) && (endeds >> b & 1)) {
            mine = lane == 0 ? (double)s_b : mine;
        } else if (!dead(s_b)) {
            const uint64_t* keys = a.keys + (int64_t)row * lists * k;
            const uint64_t* sums = a.sums + (int64_t)row * tiles;
            Best best;
            Keys x;
            auto load = [&](int i0) {
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    const int i = i0 + 64 * j + lane;
                    x[j] = i < lists * k ? load_dev64(keys + i) : 0;
                }
            };
            load(0);
            float top = kNone;
            bool broken = false;
            double sum = 0.0;
            for (int t0 = 0; t0 < tiles; t0 += 128) {  // (one turn for up to 262144 tokens)
                float m[2], s[2];
                const float before = top;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int t = t0 + 64 * i + lane;
                    const uint64_t y = t < tiles ? load_dev64(sums + t) : (uint64_t)__float_as_uint(kNone);
                    m[i] = __uint_as_float((uint32_t)y);
                    s[i] = __uint_as_float((uint32_t)(y >> 32));
                    broken |= s[i] != s[i];
                    top = fmaxf(top, m[i]);
                }
                top = wave_max(top);
                const float base = top == kNone ? 0.0f : top;
                sum *= before == kNone ? 0.0f : fast_exp2((before - base) * kLog2e);
#pragma unroll
                for (int i = 0; i < 2; ++i) sum += (double)(s[i] * fast_exp2((m[i] - base) * kLog2e));
            }
            broken = __ballot(broken);
            if (!broken && top != kNone) {
#pragma unroll
                for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
                const double lse = (double)top + log(sum);
                for (int i0 = 0;;) {  // (one turn for up to 512 keys)
                    uint64_t most = 0;
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) most = max(most, (uint64_t)x[j]);
                    const uint32_t border = border_of((uint32_t)(most >> 32), order_of(top + 0.0f), k);
                    uint32_t mask = 0;
#pragma unroll
                    for (int j = kBatch - 1; j >= 0; --j) mask = 2 * mask + (x[j] != 0 && (uint32_t)(x[j] >> 32) >= border);
                    while (__ballot(mask != 0)) {
                        const int j = mask ? __builtin_ctz(mask) : 0;
                        const uint64_t y0 = j & 1 ? x[1] : x[0], y1 = j & 1 ? x[3] : x[2], y2 = j & 1 ? x[5] : x[4], y3 = j & 1 ? x[7] : x[6];
                        const uint64_t z0 = j & 2 ? y1 : y0, z1 = j & 2 ? y3 : y2;
                        take(best, mask ? (j & 4 ? z1 : z0) : 0, k, lane, sh.list[wave]);
                        mask &= mask - 1;
                    }
                    i0 += 64 * kBatch;
                    if (i0 >= lists * k) break;
                    load(i0);
                }
                if (best.pending) rank_list(best, k, lane, sh.list[wave]);
                if (lane < best.held) {
                    const uint64_t key = sh.list[wave][lane];
                    mine = (double)s_b + ((double)logit_of(key) - lse);
                    token = token_of(key);
                }
            }
        }
        if (lane < k) {
            s_score[b * k + lane] = mine;
            s_token[b * k + lane] = token;
            s_rank[b * k + lane] = 0;
        }
    }
    __syncthreads();
    // Each candidate's rank: how many come before it; those that are none are the
    // last.  64 candidates a wave, against a part of them all.
    const int chunks = (n + 63) / 64, shares = max(1, kBeamWaves / chunks);
    for (int u = wave; u < chunks * shares; u += kBeamWaves) {
        const int chunk = u / shares, share = u - chunk * shares, i = chunk * 64 + lane;
        const double x = s_score[min(i, n - 1)];
        int rank = 0;
#pragma unroll 8
        for (int j = share * n / shares; j < (share + 1) * n / shares; ++j) {
            const double y = s_score[j];
            rank += y > x || (y == x && j < i);
        }
        if (i < n) atomicAdd(s_rank + i, rank);
    }
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
        const int rank = s_rank[i];
        if (rank >= k) continue;
        const double x = s_score[i];
        const bool none = x == (double)kNone;
        const int at = group * k + rank, b = i / k, token = s_token[i];
        a.parent[at] = none ? -1 : group * a.width + b;
        a.token[at] = none ? -1 : token;
        a.out_scores[at] = (float)x;
        if (a.out_done) a.out_done[at] = !none && ((endeds >> b & 1) || (a.eos >= 0 && token == a.eos));
    }
}

__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(6, 8))) void beam_select_kernel(BeamArgs a, int parts) {
    __shared__ Shared sh;
    extern __shared__ double s_score[];  // [width][k], and as many tokens and ranks
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), k = a.k;
    const int row = __builtin_amdgcn_readfirstlane(blockIdx.x / parts), part = blockIdx.x - row * parts;
    const int group = __builtin_amdgcn_readfirstlane(row / a.width);
    // Of the group, a beam a lane, for the merge: read before any output is written.
    const int beam = group * a.width + min(lane, a.width - 1);
    const float score = a.scores[beam];
    const bool ended = a.done && a.done[beam];
    if (!dead(scalar(a.scores + row)) && !(a.done && scalar(a.done + row))) {
        // (A row need not start at a 16-byte border: its loads only ask for one of 4.)
        typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
        const float* x = a.logits + row * a.stride;
        const int tiles = (a.vocab + kBeamTile - 1) / kBeamTile;
        Best best;
        auto load = [&](Tile& v, int t) {
            const int first = t * kBeamTile + lane * 4;
            if ((t + 1) * kBeamTile <= a.vocab) {
#pragma unroll
                for (int i = 0; i < kBeamValues / 4; ++i) {
                    const float4u y = *(const float4u*)(x + first + 256 * i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[4 * i + e] = y[e];
                }
            } else {
#pragma unroll
                for (int i = 0; i < kBeamValues; ++i) {
                    const int at = first + 256 * (i >> 2) + (i & 3);
                    v[i] = at < a.vocab ? x[at] : kNone;
                }
            }
        };
        const int step = parts * kBeamWaves;
        for (int t = part * kBeamWaves + wave; t < tiles; t += step) {
            Tile v;
            load(v, t);
            float top = kNone;
#pragma unroll
            for (int i = 0; i < kBeamValues; ++i) top = fmaxf(top, v[i]);
            const float M = wave_max(top), base = M == kNone ? 0.0f : M;
            float4v s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kBeamValues; ++i) s[i & 3] += fast_exp2((v[i] - base) * kLog2e);
            // (NaN if a value is NaN, or +inf, which is the maximum then.)
            const float sum = wave_sum((s[0] + s[1]) + (s[2] + s[3]));
            if (lane == 0)
                store_dev64(a.sums + (int64_t)row * tiles + t, (uint64_t)__float_as_uint(sum) << 32 | __float_as_uint(M));
            if (!(sum == sum) || M == kNone || (best.kth != 0 && M <= logit_of(best.kth))) continue;  // (of equal ones the earlier tile's)
            take_tile(best, v, top, M, t * kBeamTile + lane * 4, k, lane, sh.list[wave]);
        }
        uint64_t* keys = a.keys + (((int64_t)row * parts + part) * kBeamWaves + wave) * k;
        if (lane < k) store_dev64(keys + lane, lane < best.held ? sh.list[wave][lane] : 0);
    }
    stores_done_barrier();
    uint32_t* arrived = a.arrived + group * kBeamCounterStep;
    if (tid == 0) sh.last = ticket_add(arrived) == (uint32_t)(a.width * parts - 1);
    __syncthreads();
    if (!sh.last) return;
    merge(a, group, parts * kBeamWaves, score, ended, sh, s_score);
    if (tid == 0) ticket_reset(arrived);
}

}  // namespace

hipError_t launch_beam_select(const BeamArgs& a, int cus, hipStream_t stream) {
    if (a.groups < 1 || a.groups > kBeamMaxGroups || a.width < 1 || a.width > kBeamMaxWidth || a.k < 1 ||
        a.k > kBeamMaxK || a.vocab < 1 || a.vocab > kBeamMaxVocab)
        return hipErrorInvalidValue;
    const int rows = a.groups * a.width, parts = beam_parts(rows, a.vocab, cus);
    hipLaunchKernelGGL(beam_select_kernel, dim3((unsigned)(rows * parts)), dim3(kThreads), (size_t)a.width * a.k * 16,
                       stream, a, parts);
    return hipGetLastError();
}

}  // namespace qasr
