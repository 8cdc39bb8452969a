// paged_append8.hip -- stage (a) into e4m3 pages: qk-norm + RoPE of a step's
// rows (norm_rope.hpp, the bits of the f16 pools' stage (a)), K and V stored in
// 8 bits with one power of two for each 16-row block of a head.
//
// A block's unit is 2^k, the smallest from 2^-15 on of which the largest finite
// value in it is at most 448 (e4m3's largest); an element is e4m3(x / 2^k), to
// the nearest, ties to even, of the f16 value x that an f16 pool would hold.
// Steps of e4m3 below 2^-9 would be finer than f16 itself, hence 2^-15; and at
// 2^8, which the largest f16 numbers need, magnitudes end at 240 instead of 448,
// as 256 * 2^8 is no f16 number.  So every stored value stands for an f16 number.
// e4m3 has no infinities: what is not finite is stored as NaN.
//
// New rows join the rows that their block holds already: the unit is then the
// larger of the block's and the one that the new rows need, and where it grows
// the earlier rows are rounded again.  Halving an e4m3 number is exact down to
// 2^-6 units, so what a row stands for depends on how the rows came only in
// values 2^-14 times the largest of the block and less.
//
// A run: rows of a step that follow each other in one block.  A workgroup
// takes the runs that start in 16 rows of the step, for one kv head and its two q
// heads, at most 16 rows of whole runs at a time: a thread of 256 holds 8 dims and
// their rotation partners of a row, of one of the q heads and of K or V, so that
// cos and sin are read once for both.  The sums of squares are serial (one lane a
// head and row, as the reference adds), the largest values meet in LDS.  Units are
// powers of two so that a growing unit costs the earlier rows nothing, and the
// conversions are instructions.
//
// What bounds it, us a layer of 16 q and 8 kv heads: 1 row 4.4, the chain: launch,
// places, cos / sin and the blocks' units, the sums, three barriers (stage (a) into
// f16 pages, without units, 3.1); 16 and 64 single rows 5.1 and 5.4 (6.5 and 6.8 where
// every run is looked at for rows to be rounded again, not those found by a
// ballot); 5185 rows of 16 prompts 20.0 (74 MB, 14.6 at the
// rate of a large copy): 118 registers, 4 workgroups a CU.  Q and K or V in
// separate threads with their own cos and sin and all of a head read ahead of its
// sum took 179, 2 workgroups: 27.7 and 4.7.  5 a CU spill (32); loads of the rows
// past the caches 21.6.
#include "norm_rope.hpp"
#include "paged.hpp"

namespace qasr {

namespace {

constexpr int kThreads = 256;
constexpr int kRun = 16;   // rows of a block
constexpr int kWindow = 2 * kRun;  // rows that runs starting in 16 rows can reach, and one
constexpr int kPad = kHeadDim + 8;
constexpr uint32_t kMinUnit = 127 - 15;  // exponent bytes

// The exponent byte of the unit for a largest magnitude (f16 bits, finite).
__device__ __forceinline__ uint32_t unit_of(uint32_t top) {
    return max(kMinUnit, (top >> 10) + (127 - 15 - 8) + ((top & 0x3ff) > 0x300));
}
// Largest finite magnitude of 8 values, as f16 bits.
__device__ __forceinline__ uint32_t top_of(const H8& x) {
    const uint32_t w[4] = {x.u.x, x.u.y, x.u.z, x.u.w};
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = w[i] & 0x7fff, b = (w[i] >> 16) & 0x7fff;
        top = max(top, max(a < 0x7c00 ? a : 0, b < 0x7c00 ? b : 0));
    }
    return top;
}
// 8 f16 values in e4m3, in units of `unit`.
__device__ __forceinline__ uint2 narrow8(const H8& x, float unit) {
    typedef short short2v __attribute__((ext_vector_type(2)));
    const f16 most = (f16)(240.0f * 256.0f);
    uint32_t r[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        short2v y = {0, 0};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const half2v v = x.h2[2 * i + k];
            half2v c = __builtin_elementwise_max(__builtin_elementwise_min(v, (half2v){most, most}), (half2v){-most, -most});
            c -= v - v;  // NaN if v is not finite (and -0 keeps its sign)
            y = k ? __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(y, c, unit, true)
                  : __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(y, c, unit, false);
        }
        r[i] = __builtin_bit_cast(uint32_t, y);
    }
    return make_uint2(r[0], r[1]);
}
__device__ __forceinline__ H8 widen8(uint2 x, float unit) {
    H8 y;
    y.h2[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x.x, unit, false);
    y.h2[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x.x, unit, true);
    y.h2[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x.y, unit, false);
    y.h2[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x.y, unit, true);
    return y;
}
template <int Ctrl>
__device__ __forceinline__ uint32_t other(uint32_t x) {
    return __float_as_uint(dpp<Ctrl>(__uint_as_float(x)));
}
__device__ __forceinline__ float unit_value(uint32_t byte) { return __uint_as_float(byte << 23); }

__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(4))) void paged_append8_kernel(PagedAppend8Args a) {
    __shared__ __attribute__((aligned(16))) f16 s_raw[3 * kRun * kPad];
    __shared__ __attribute__((aligned(16))) f16 s_gain[2 * kHeadDim];  // of Q, of K
    __shared__ float s_inv[3 * kRun];
    __shared__ int s_slot[kWindow], s_pos[kWindow];
    __shared__ uint32_t s_starts;  // rows of the window at which a run starts
    __shared__ uint32_t s_top[2][kRun];
    __shared__ uint32_t s_old[2][kRun];  // run starts: the block's byte, if it has earlier rows

    const int tid = threadIdx.x, chunk = blockIdx.x / a.nkvh, kvh = blockIdx.x - chunk * a.nkvh;
    const int first = chunk * kRun, rows = min(kWindow, a.rows - first);
    // A thread: 8 dims and their partners of row `ar` of a pass, of Q's head `half`
    // of the two and of K (0) or V (1).
    const int w = tid & 7, d = 8 * w, half = (tid >> 3) & 1, ar = tid >> 4;
    const int nh = a.nqh + 2 * a.nkvh;
    const f16* q_src = a.qkv + ((int64_t)first * nh + 2 * kvh + half) * kHeadDim + d;
    const f16* k_src = a.qkv + ((int64_t)first * nh + a.nqh + half * a.nkvh + kvh) * kHeadDim + d;
    H8 q[2], k[2];
    auto load_row = [&](int row) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            q[i].u = *(const uint4*)(q_src + (int64_t)row * nh * kHeadDim + i * (kHeadDim / 2));
            k[i].u = *(const uint4*)(k_src + (int64_t)row * nh * kHeadDim + i * (kHeadDim / 2));
        }
    };
    // (The step's first row starts a run: rows of small steps need not wait for
    // their places.)
    if (chunk == 0) load_row(min(ar, rows - 1));
    if (tid >= kThreads - 32) {  // (not the wave of the serial sums)
        const int i = tid & 15;
        *(uint4*)&s_gain[8 * (tid & 31)] = *(const uint4*)((tid & 16 ? a.k_gain : a.q_gain) + 8 * i);
    }
    // The window's rows: a slot of -1 where there is nothing to store.  A row
    // goes on with the run of the row before it if it lies behind it in its block.
    if (tid < 64) {
        const int r = first + min(tid, rows - 1);
        int pos = a.pos[r], slot = a.slot[r], before = r > 0 ? a.slot[r - 1] : -1;
        const bool placed = (uint32_t)pos < (uint32_t)a.rope_rows;
        const bool stored = placed && (uint32_t)slot < (uint32_t)a.slots;
        const bool on = stored && before >= 0 && slot == before + 1 && (slot & (kRun - 1)) != 0 && r > 0 &&
                        (uint32_t)a.pos[max(r - 1, 0)] < (uint32_t)a.rope_rows;
        const uint64_t starts = __ballot(!on && tid < rows);
        if (tid < kWindow) {
            s_slot[tid] = stored ? slot : -1;
            s_pos[tid] = placed ? pos : -1;
        }
        if (tid == 0) s_starts = (uint32_t)starts;
    }
    __syncthreads();
    const uint32_t starts = __builtin_amdgcn_readfirstlane(s_starts);
    auto run_of = [&](int r) { return 31 - __builtin_clz(starts & ((2u << r) - 1)); };  // of a row behind a start
    auto start_from = [&](int r) {  // the first start at or behind r, or the rows' end
        const uint32_t x = r < 32 ? starts >> r : 0;
        return x ? r + __builtin_ctz(x) : rows;
    };
    const int end = start_from(kRun);  // runs that start behind are the next workgroup's
    for (int p0 = start_from(0), p1; p0 < min(kRun, rows); p0 = p1) {
        p1 = p0 + kRun < end ? run_of(p0 + kRun) : end;  // whole runs, 16 rows at most
        const bool on = p0 + ar < p1;
        const int row = min(p0 + ar, p1 - 1);
        if (chunk != 0 || p0 != 0) load_row(row);
        const int pos = max(s_pos[row], 0), slot = s_slot[row], start = run_of(row), start_slot = s_slot[start];
        H8 c[2], sn[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            c[i].u = *(const uint4*)(a.cos_tab + (int64_t)pos * kHeadDim + d + i * (kHeadDim / 2));
            sn[i].u = *(const uint4*)(a.sin_tab + (int64_t)pos * kHeadDim + d + i * (kHeadDim / 2));
        }
        // Block of the run: its byte, and its first row's place.
        const int page = max(start_slot, 0) >> a.page_shift, in_page = max(start_slot, 0) & ((1 << a.page_shift) - 1);
        uint8_t* unit_at = a.scales + (int64_t)page * a.page_scales + half * a.kv_scales + kvh * a.head_scales + (in_page >> 4);
        uint8_t* block = a.base + (int64_t)page * a.page_stride + half * a.kv_stride + kvh * a.head_stride +
                         (int64_t)(in_page & ~(kRun - 1)) * kHeadDim;
        uint32_t old = *unit_at;
        const int held = start_slot >= 0 ? start_slot & (kRun - 1) : 0;  // rows that the block has
        old = held ? old : 0;
        if (on) {
            f16* at = &s_raw[(2 * ar + half) * kPad + d];
            *(uint4*)at = q[0].u;
            *(uint4*)(at + kHeadDim / 2) = q[1].u;
        }
        if (on && !half) {
            f16* at = &s_raw[(2 * kRun + ar) * kPad + d];
            *(uint4*)at = k[0].u;
            *(uint4*)(at + kHeadDim / 2) = k[1].u;
        }
        if (tid < 2 * kRun) s_top[tid >> 4][tid & 15] = 0;
        __syncthreads();
        {
            const int n = p1 - p0;
            if (tid < 3 * kRun && (tid < 2 * kRun ? tid >> 1 : tid - 2 * kRun) < n)
                s_inv[tid] = head_inv_rms_lean(&s_raw[tid * kPad], a.eps);
        }
        __syncthreads();
        {
            H8 o[2], gain[2];
            auto from = [&](H8 (&x)[2], const f16* p) {
                x[0].u = *(const uint4*)p;
                x[1].u = *(const uint4*)(p + kHeadDim / 2);
            };
            from(q, &s_raw[(2 * ar + half) * kPad + d]);
            from(gain, s_gain + d);
            rope16(q, gain, c, sn, s_inv[2 * ar + half], o);
            if (on && s_pos[row] >= 0) {
                f16* dst = a.q_out + ((int64_t)(first + row) * a.nqh + 2 * kvh + half) * kHeadDim + d;
                *(uint4*)dst = o[0].u;
                *(uint4*)(dst + kHeadDim / 2) = o[1].u;
            }
            from(gain, s_gain + kHeadDim + d);
            rope16(k, gain, c, sn, s_inv[2 * kRun + ar], o);
            if (!half) {
                k[0] = o[0];
                k[1] = o[1];
            }
        }
        uint32_t top = max(top_of(k[0]), top_of(k[1]));  // of the row's: of 8 lanes
        top = max(top, other<kDppXor1>(top));
        top = max(top, other<kDppXor2>(top));
        top = max(top, other<kDppHalfMirror>(top));
        if (on && slot >= 0 && w == 0) atomicMax(&s_top[half][start - p0], top);
        if (on && start == row && w == 0) s_old[half][ar] = slot >= 0 ? old | held << 8 : 0;
        __syncthreads();
        const uint32_t need = unit_of(s_top[half][start - p0]), unit = max(old, need);
        if (on && slot >= 0) {
            uint8_t* dst = block + (slot & (kRun - 1)) * kHeadDim + d;
            *(uint2*)dst = narrow8(k[0], unit_value(unit));
            *(uint2*)(dst + kHeadDim / 2) = narrow8(k[1], unit_value(unit));
            if (start == row && w == 0) *unit_at = (uint8_t)unit;
        }
        // Earlier rows of blocks whose unit grew, a row for 8 lanes.  Bit j, 16 + j: the run that starts at p0 + j, its K, V.
        const uint32_t tops = s_top[(tid >> 4) & 1][tid & 15], olds = s_old[(tid >> 4) & 1][tid & 15];
        const uint32_t grew = (uint32_t)__ballot((tid & 63) < 2 * kRun && p0 + (tid & 15) < p1 &&
                                                 (starts >> (p0 + (tid & 15)) & 1) && (olds >> 8) != 0 &&
                                                 (olds & 0xff) < unit_of(tops));
        for (uint32_t todo = (grew | grew >> 16) & 0xffff; todo; todo &= todo - 1) {
            const int j = __builtin_ctz(todo);
            const uint32_t was = s_old[half][j];
            if (!(grew >> (16 * half + j) & 1) || ar >= (int)(was >> 8)) continue;
            const float from = unit_value(was & 0xff), to = unit_value(unit_of(s_top[half][j]));
            const int s = s_slot[p0 + j], pg = s >> a.page_shift, ip = s & ((1 << a.page_shift) - 1);
            uint8_t* at = a.base + (int64_t)pg * a.page_stride + half * a.kv_stride + kvh * a.head_stride +
                          (int64_t)((ip & ~(kRun - 1)) + ar) * kHeadDim + d;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint2* x = (uint2*)(at + i * (kHeadDim / 2));
                *x = narrow8(widen8(*x, from), to);
            }
        }
        __syncthreads();  // the LDS is used again
    }
}

}  // namespace

hipError_t launch_paged_append8(const PagedAppend8Args& a, hipStream_t stream) {
    if (a.rows <= 0) return hipSuccess;
    if (a.nqh != kRep * a.nkvh) return hipErrorInvalidValue;
    const int64_t wgs = (int64_t)((a.rows + kRun - 1) / kRun) * a.nkvh;
    hipLaunchKernelGGL(paged_append8_kernel, dim3((unsigned)wgs), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace qasr
