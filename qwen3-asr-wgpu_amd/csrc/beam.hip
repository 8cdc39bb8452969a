// beam.hip -- the best continuations of groups of beams: log-softmax of each
// beam's logits, selection over beams and vocabulary.
//
// Candidate (b, t) of a group has the score s_b + x_bt - log sum_u exp x_bu; an
// ended beam has one, (b, eos) with s_b.  The k best of a group, ties to the
// lower beam, then to the lower token.
//
// One pass over the logits.  A workgroup holds a piece of a row in registers
// (512 threads of 8 values, two 16-byte loads each): its maximum, the sum of
// exponentials against it, and its k best.  For these every wave finds the k-th
// largest of its 64 lanes' maxima, by bisection of the keys' bits with ballots;
// at least k values of the row are as large as the largest of the waves' finds,
// so only those that are, mostly little more than k, go to LDS and are ranked
// there by comparing each with all.  A key is the logit's order-preserving bits
// over the complement of its token, unique, so that ties cost nothing and the
// list is never longer than waves * k * values.
//
// The last workgroup of a group to arrive (ticket) merges: a wave a beam takes
// the pieces' sums, in 64 bits and in order, and out of its sorted pieces' lists
// the k best in the same way, by the k-th largest of the lists' heads; then each
// of the beams' sorted candidates finds its rank by a bisection in the other
// beams' lists, in 64-bit scores.  Everything is a function of the row alone up
// to there: results do not depend on the batch, or on who comes last.
//
// Bound by the logits' bytes for many rows, by launch, one load, the ballots and
// the merge's two round trips for few.
#include "beam.hpp"

namespace qasr {

namespace {

constexpr int kWaves = kBeamThreads / 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -__builtin_inff();

__device__ __forceinline__ uint64_t key_of(float x, int token) {
    const uint32_t u = __float_as_uint(x);
    const uint32_t o = u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
    return (uint64_t)o << 32 | ~(uint32_t)token;
}
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o ^ ((int32_t)o < 0 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int token_of(uint64_t key) { return (int)~(uint32_t)key; }

__device__ __forceinline__ void store_dev64(uint64_t* p, uint64_t v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t load_dev64(const uint64_t* p) {
    return __hip_atomic_load(const_cast<uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The k-th largest of the lanes' keys, or 0 if fewer than k are not 0.
__device__ __forceinline__ uint64_t kth_of_lanes(uint64_t key, int k) {
    uint64_t t = 0;
    for (int b = 63; b >= 0; --b) {
        const uint64_t cand = t | 1ull << b;
        const int n = __popcll(__ballot(key >= cand));
        if (n >= k) {
            t = cand;
            if (n == k) break;  // as good a border as the k-th itself
        }
    }
    return t;
}

// A beam that offers nothing: its score is -inf, +inf or NaN.
__device__ __forceinline__ bool dead(float score) { return !(fabsf(score) < __builtin_inff()); }

struct Shared {
    uint64_t border[kWaves];
    float top[kWaves];
    float sum[kWaves];
    int count[kWaves];
    int last;
    int offers[kBeamMaxWidth];
};
// And by the call's sizes: a list, of what reaches the border in a piece or, a
// part for each wave, in the pieces' lists; the beams' candidates, best first.
__host__ __device__ constexpr int list_entries(int values, int k) { return kWaves * k * (values > k ? values : k); }
struct Lists {
    uint64_t* list;
    double* score;
    int* token;
};

// LDS writes of this wave before its reads behind.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ void merge(const BeamArgs& a, int group, int splits, Shared& sh, const Lists& ls) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = a.k;
    uint64_t* list = ls.list + wave * k * k;
    for (int b = wave; b < a.width; b += kWaves) {
        const int row = group * a.width + b;
        const float score = a.scores[row];
        const bool ended = a.done && a.done[row];
        int offers = 0;
        if (!dead(score) && ended) {
            offers = 1;
            if (lane == 0) {
                ls.score[b * k] = score;
                ls.token[b * k] = a.eos;
            }
        } else if (!dead(score)) {
            const uint64_t* keys = a.keys + (int64_t)row * splits * k;
            const float* sums = a.sums + (int64_t)row * splits * 2;
            const bool on = lane < splits;
            const uint64_t head = on ? load_dev64(keys + lane * k) : 0;
            const uint64_t ms = on ? load_dev64((const uint64_t*)sums + lane) : 0;
            const float m = on ? __uint_as_float((uint32_t)ms) : kNone, s = __uint_as_float((uint32_t)(ms >> 32));
            const bool broken = __ballot(on && s != s);
            float top = m;
#pragma unroll
            for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
            double sum = on && m != kNone ? (double)s * exp((double)m - (double)top) : 0.0;
#pragma unroll
            for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
            if (!broken && top != kNone) {
                const double lse = (double)top + log(sum);
                const uint64_t border = kth_of_lanes(head, k);
                // At most k lists have such heads.
                if (lane == 0) sh.count[wave] = 0;
                wave_sync();
                for (int i = lane; i < splits * k; i += 64) {
                    const uint64_t key = load_dev64(keys + i);
                    if (key != 0 && key >= border) list[atomicAdd(&sh.count[wave], 1)] = key;
                }
                wave_sync();
                const int n = sh.count[wave];
                for (int i = lane; i < n; i += 64) {
                    const uint64_t key = list[i];
                    int rank = 0;
                    for (int j = 0; j < n; ++j) rank += list[j] > key;
                    if (rank < k) {
                        ls.score[b * k + rank] = (double)score + ((double)logit_of(key) - lse);
                        ls.token[b * k + rank] = token_of(key);
                    }
                }
                offers = min(n, k);
            }
        }
        if (lane == 0) sh.offers[b] = offers;
    }
    __syncthreads();
    int all = 0;
    for (int b = 0; b < a.width; ++b) all += sh.offers[b];
    for (int i = tid; i < a.width * k; i += kBeamThreads) {
        const int b = i / k, j = i - b * k;
        if (j >= sh.offers[b]) continue;
        const double score = ls.score[i];
        int rank = j;  // and how many of the other beams' come before it
        for (int c = 0; c < a.width && rank < k; ++c) {
            if (c == b) continue;
            int lo = 0, hi = sh.offers[c];
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                const double x = ls.score[c * k + mid];
                if (x > score || (x == score && c < b))
                    lo = mid + 1;
                else
                    hi = mid;
            }
            rank += lo;
        }
        if (rank >= k) continue;
        const int row = group * a.width + b, token = ls.token[i];
        const bool ended = (a.done && a.done[row]) || (a.eos >= 0 && token == a.eos);
        ls.list[2 * rank] = (uint64_t)(uint32_t)token << 32 | (uint32_t)(row << 1 | (int)ended);
        ls.list[2 * rank + 1] = __float_as_uint((float)score);
    }
    __syncthreads();  // what may be replaced in place has been read
    if (tid < k) {
        const int at = group * k + tid;
        const bool some = tid < all;
        const uint64_t x = ls.list[2 * tid];
        a.parent[at] = some ? (int)((uint32_t)x >> 1) : -1;
        a.token[at] = some ? (int)(x >> 32) : -1;
        a.out_scores[at] = some ? __uint_as_float((uint32_t)ls.list[2 * tid + 1]) : kNone;
        if (a.out_done) a.out_done[at] = some ? (int)(x & 1) : 0;
    }
}

template <int VALUES>
__global__ __launch_bounds__(kBeamThreads) __attribute__((amdgpu_waves_per_eu(6, 6))) void beam_select_kernel(BeamArgs a, int splits) {
    __shared__ Shared sh;
    extern __shared__ uint64_t s_lists[];
    Lists ls;
    ls.list = s_lists;
    ls.score = (double*)(s_lists + list_entries(VALUES, a.k));
    ls.token = (int*)(ls.score + a.width * a.k);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = a.k;
    const int row = blockIdx.x / splits, split = blockIdx.x - row * splits, group = row / a.width;
    const float score = a.scores[row];
    if (!dead(score) && !(a.done && a.done[row])) {
        // (A row need not start at a 16-byte border: its loads only ask for one of 4.)
        typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
        const float* x = a.logits + row * a.stride;
        const int first = split * (kBeamThreads * VALUES) + tid * 4;
        float v[VALUES];
#pragma unroll
        for (int i = 0; i < VALUES / 4; ++i) {
            const int t = first + i * kBeamThreads * 4;
            if (t + 4 <= a.vocab) {
                const float4u y = *(const float4u*)(x + t);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * i + e] = y[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * i + e] = t + e < a.vocab ? x[t + e] : kNone;
            }
        }
        float top = kNone;
        bool broken = false;
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            v[i] += 0.0f;  // -0 is 0
            broken |= !(v[i] < __builtin_inff());
            top = fmaxf(top, v[i]);
        }
        int best = -1;  // the first of the largest
#pragma unroll
        for (int i = VALUES - 1; i >= 0; --i) best = v[i] == top ? i : best;
        auto token = [&](int i) { return first + (i >> 2) * kBeamThreads * 4 + (i & 3); };
        const uint64_t mine = top == kNone || broken ? 0 : key_of(top, token(best));
        uint64_t border = kth_of_lanes(mine, k);
        float wave_top = top;
#pragma unroll
        for (int d = 32; d; d >>= 1) wave_top = fmaxf(wave_top, __shfl_xor(wave_top, d));
        broken = __ballot(broken);
        if (lane == 0) {
            sh.border[wave] = border;
            sh.top[wave] = broken ? __builtin_nanf("") : wave_top;
        }
        if (tid == 0) sh.count[0] = 0;
        __syncthreads();
        float M = kNone;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            border = max(border, sh.border[w]);
            M = fmaxf(M, sh.top[w]);
            broken |= sh.top[w] != sh.top[w];
        }
        // Sums of exponentials against the workgroup's maximum.
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const float base = M == kNone ? 0.0f : M;
        const float least = logit_of(border);
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            s[i & 3] += fast_exp2((v[i] - base) * kLog2e);
            if (v[i] >= least || border == 0) {
                const uint64_t key = key_of(v[i], token(i));
                if (v[i] != kNone && !broken && key >= border) ls.list[atomicAdd(&sh.count[0], 1)] = key;
            }
        }
        float sum = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
        for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
        if (lane == 0) sh.sum[wave] = sum;
        __syncthreads();
        uint64_t* keys = a.keys + ((int64_t)row * splits + split) * k;
        const int n = sh.count[0];
        for (int i = tid; i < n; i += kBeamThreads) {
            const uint64_t key = ls.list[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += ls.list[j] > key;
            if (rank < k) store_dev64(keys + rank, key);
        }
        if (tid >= n && tid < k) store_dev64(keys + tid, 0);
        if (tid == 0) {
            float total = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) total += sh.sum[w];
            if (broken) total = __builtin_nanf("");
            store_dev64((uint64_t*)a.sums + (int64_t)row * splits + split,
                        (uint64_t)__float_as_uint(total) << 32 | __float_as_uint(M));
        }
    }
    stores_done_barrier();
    uint32_t* arrived = a.arrived + group * kBeamCounterStep;
    if (tid == 0) sh.last = ticket_add(arrived) == (uint32_t)(a.width * splits - 1);
    __syncthreads();
    if (!sh.last) return;
    merge(a, group, splits, sh, ls);
    if (tid == 0) ticket_reset(arrived);
}

template <int VALUES>
hipError_t launch(const BeamArgs& a, hipStream_t stream) {
    const int splits = beam_splits(a.vocab);
    const size_t lds = (size_t)list_entries(VALUES, a.k) * 8 + (size_t)a.width * a.k * 12;
    const int64_t wgs = (int64_t)a.groups * a.width * splits;
    hipLaunchKernelGGL(beam_select_kernel<VALUES>, dim3((unsigned)wgs), dim3(kBeamThreads), lds, stream, a, splits);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_beam_select(const BeamArgs& a, hipStream_t stream) {
    if (a.groups < 1 || a.groups > kBeamMaxGroups || a.width < 1 || a.width > kBeamMaxWidth || a.k < 1 ||
        a.k > kBeamMaxK || a.vocab < 1 || a.vocab > kBeamMaxVocab)
        return hipErrorInvalidValue;
    switch (beam_values(a.vocab)) {
        case 8: return launch<8>(a, stream);
        case 16: return launch<16>(a, stream);
        default: return launch<32>(a, stream);
    }
}

}  // namespace qasr
