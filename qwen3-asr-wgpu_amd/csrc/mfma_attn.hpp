// mfma_attn.hpp -- the MFMA attention step shared by the prefill kernel
// (prefill_attn.hip) and the paged kernel (paged_attn.hip): operand layouts in
// LDS, S^T = K Q^T, the online softmax of one query column per lane, and
// O^T += V^T P^T, on v_mfma_f32_32x32x16_f16.
#pragma once

#include "common.hpp"

namespace qasr {

constexpr float kNegInf = -__builtin_inff();
constexpr float kRescaleSlack = 8.0f;  // log2 of the largest p before the max moves

typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_short4v;

__device__ __forceinline__ float16v mfma32(const half8v& a, const half8v& b, const float16v& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Lanes l and l^32 hold the two key halves of one query column.  One
// v_permlane32_swap gives every lane both values (no LDS round trip).
__device__ __forceinline__ float halves_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// K tile: row r (key) is 256 contiguous bytes; its 16-byte chunk c (dims
// 8c..8c+7) sits at slot c ^ swz16(r).  swz16 permutes 0..15 over every 16
// consecutive rows, so the K operand read (16 consecutive rows, one chunk)
// hits 16 different slots.
__device__ __forceinline__ int swz16(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }

// 4 halves of V^T: ds_read_b64_tr_b16 transposes 16-bit elements within each
// 16-lane group (result lane 4m+e, element k <- source lane 4k+m, element e).
__device__ __forceinline__ half4v read_tr(const f16* p) {
    return __builtin_bit_cast(half4v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4v*)p));
}

// Per-wave state.
struct Wave {
    half8v qb[8];     // Q^T B operand, k-step ks: dims 16*ks + 8*g .. +8 of query n
    float16v o[4];    // O^T: o[db][i] = dim db*32 + 8*(i/4) + 4*g + i%4 of query n
    float m;          // running max the exponents are taken against
    float l;          // running row sum
    int kaddr[8];     // K operand of k-step ks, rows 0..31 of the half tile (halves)
    int vbase;        // V^T operand source address, slab 0, key 0 (halves)
    int g, qpos;
    float scale_log2;
};

// Scores of a step over NB * 32 keys: S^T from K rows kt[0..32 NB - 1], keys
// kb*32 + (8*(i/4) + 4*g + i%4) x query n, accumulated over dims.
template <int NB>
__device__ __forceinline__ void step_scores(const Wave& w, const f16* kt, float16v (&s)[NB]) {
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) s[kb] = (float16v){};
#pragma unroll
    for (int ks = 0; ks < 8; ++ks)
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) {
            const half8v ka = *(const half8v*)&kt[kb * 32 * kHeadDim + w.kaddr[ks]];
            s[kb] = mfma32(ka, w.qb[ks], s[kb]);
        }
    // Operand reads run at most two k-steps ahead of the MFMAs (bounded
    // register lifetime; 8 NB reads + 8 NB MFMAs).
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * NB, 0);
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, NB, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, NB, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 2 * NB, 0);
}

// The softmax of those scores (first key k0): row max, the running-max
// update, P^T (f16, B-operand layout) and its row sum.  MASK: some key is
// past some row's position.
template <bool MASK, int NB>
__device__ __forceinline__ void step_softmax(Wave& w, float16v (&s)[NB], int k0, half8v (&pb)[2 * NB]) {
    float mx = kNegInf;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (MASK) {
                const int key = k0 + kb * 32 + 8 * (i >> 2) + 4 * w.g + (i & 3);
                s[kb][i] = key > w.qpos ? kNegInf : s[kb][i];
            }
            mx = fmaxf(mx, s[kb][i]);
        }
    mx = halves_max(mx) * w.scale_log2;
    // Move the running max when a row max passed it by more than the slack.
    {
        const bool up = mx > w.m + kRescaleSlack;
        if (__ballot(up)) {
            const float mn = up ? mx : w.m;
            const float alpha = w.m == kNegInf ? 0.0f : fast_exp2(w.m - mn);
#pragma unroll
            for (int db = 0; db < 4; ++db) w.o[db] *= alpha;
            w.l *= alpha;
            w.m = mn;
        }
    }
    const float mu = w.m == kNegInf ? 0.0f : w.m;
    // P^T = 2^(s*scale_log2 - m), k-step w4 covering keys 16*w4 + 4*g +
    // {0..3, 8..11}; the row sum from the same f16 values (v_dot2, f32 sum).
#pragma unroll
    for (int w4 = 0; w4 < 2 * NB; ++w4)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            pb[w4][j] = (f16)softmax_w_raw(s[w4 >> 1][8 * (w4 & 1) + j], w.scale_log2, mu);
    const half2v ones2 = {(f16)1.0f, (f16)1.0f};
    float ps = 0.0f;
#pragma unroll
    for (int w4 = 0; w4 < 2 * NB; ++w4)
#pragma unroll
        for (int q2 = 0; q2 < 4; ++q2) {
            const half2v pr = {pb[w4][2 * q2], pb[w4][2 * q2 + 1]};
            ps = __builtin_amdgcn_fdot2(pr, ones2, ps, false);
        }
    w.l += halves_sum(ps);
}

// First half of a step: both.
template <bool MASK, int NB>
__device__ __forceinline__ void step_s(Wave& w, const f16* kt, int k0, half8v (&pb)[2 * NB]) {
    float16v s[NB];
    step_scores<NB>(w, kt, s);
    step_softmax<MASK, NB>(w, s, k0, pb);
}

// Second half: O^T += V^T P^T with V rows vt[0..32 NB - 1] of a tile of ROWS
// rows (slab stride ROWS*32 halves).
template <int ROWS, int NB>
__device__ __forceinline__ void step_pv(Wave& w, const f16* vt, const half8v (&pb)[2 * NB]) {
#pragma unroll
    for (int w4 = 0; w4 < 2 * NB; ++w4)
#pragma unroll
        for (int db = 0; db < 4; ++db) {
            const f16* vp = vt + w.vbase + db * (ROWS * 32) + w4 * 16 * 32;
            const half4v lo = read_tr(vp);
            const half4v hi = read_tr(vp + 8 * 32);
            const half8v va = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            w.o[db] = mfma32(va, pb[w4], w.o[db]);
        }
    // Two transposing reads per MFMA, at most two MFMAs ahead.
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < 8 * NB - 2; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
}

// Operand addresses of a lane: K operand of k-step ks: row n, chunk 2*ks + g;
// V^T operand: source lane 16*q4 + 4*k + m reads row 4*(q4>>1) + k, dims
// 16*(q4&1) + 4*m .. +3.
__device__ __forceinline__ void operand_addrs(Wave& w, int lane) {
    const int n = lane & 31, g = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) w.kaddr[ks] = n * kHeadDim + (((2 * ks + g) ^ swz16(n)) * 8);
    const int q4 = lane >> 4;
    w.vbase = (4 * (q4 >> 1) + ((lane >> 2) & 3)) * 32 + 16 * (q4 & 1) + 4 * (lane & 3);
}

}  // namespace qasr
