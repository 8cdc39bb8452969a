// mfma_attn.hpp -- what the MFMA attention kernels over slots (prefill_attn.hip)
// and over pages (paged_attn.hip) share: the v_mfma_f32_32x32x16_f16 product,
// operand layouts in LDS and their addresses, lane swaps, and a wave's state.
// Each has its own tile loop: the paged one runs its operand reads ahead of the
// MFMAs in an order of its own and hides groups of keys.
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
