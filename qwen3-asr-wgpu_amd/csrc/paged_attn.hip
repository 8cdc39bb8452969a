// paged_attn.hip -- attention of each request's new rows over its pages.
//
// Row r at position p of a request attends keys 0..p of it: softmax(q.k_t /
// sqrt(128)) . v, keys whose page lies outside the pool left out; a row that
// sees no key is zero.  A call takes any mix of single rows and chunks: the
// work lists (paged_plan.hip) are on the GPU, the workgroups walk them; a
// launch for narrow items and, where a step can have some, one for wide ones.
//
// Work item = (row block and key range of a request), for one kv head: with 8
// kv heads workgroup i runs kv head i mod 8 on XCD i mod 8, and the row blocks
// of a kv head share its keys in that XCD's L2.  Both q heads of a kv head are
// columns of one matrix product, so each key read serves both: S^T = K Q^T, the
// softmax of a column in the registers of its lanes, O^T += V^T P^T.
//  - narrow items, up to 16 rows, 4 waves: every 128-key tile is cut into the
//    waves' slices of 32 keys.  A wave copies its own slice into its own LDS
//    (16 KB), so the loop has no barrier; K of the next tile is requested when
//    the scores are done with this one, V when its product is.  The waves'
//    states combine through LDS at the end.  68 KB of LDS: two workgroups a CU,
//    one's softmax and latencies run under the other's products and copies.
//    Blocks of up to 8 rows (decode) run on products of 16 columns.
//  - wide items, up to 64 rows, 8 waves: 4 waves of 16 rows (32 columns) take
//    the first 64 keys of a 128-key tile and 4 the others; a tile is copied by
//    all into one of two buffers while the other is worked on, one barrier a
//    tile, 135 KB of LDS.  Each key is read once for 64 rows.
//
// What bounds it.  Decode: bytes, and below some 100 MB the chain of one item:
// a tile takes a wave 0.87 us (16 columns; 0.96 with 32) however early its copy
// was asked for (two tiles in flight a wave: no gain), launch, item and first
// tile 3.5 us, the end 1.3 us.  us a layer of 16 q and 8 kv heads (ranges: over
// runs, warm and cold inputs):
//   1 row of 512 keys 7.9-8.1, of 8192 (33.6 MB) 14.0-14.7, 16 rows of 400-2400
//   23.6-24.3 (93.8 MB, 3.9 TB/s; a large copy reaches 5.2).
// Chunks: MFMA and VALU work, which share the issue slots of a SIMD (two waves
// overlap about half of the smaller part), at a clock that falls to 1.9 GHz:
//   2 x 2048 rows at 4096 182-200 (172 GFLOP, 0.86-0.95 PFLOP/s; a large f16 product
//   reaches 1.1-1.3), 512 at 7680 52-55 (0.60-0.64), 8 chunks of 7-45 rows at
//   200-1700 17-20.7, 24 single rows of 100-2400 with 4 chunks of 100-450 rows
//   44.5-45.2.
// Also measured: 64-row items of 4 waves 223 us for the first of these, the
// key groups half a tile apart 223; narrow items of 8 waves 5.7 against 4.8 us
// for a single row's loop; 64-row blocks for every chunk 85 us for the last
// step.
//
// Copies are 1 KB global -> LDS instructions of 4 K rows or 16 V rows of 32
// dims: with pages of at least 16 rows each stays in one page, whose address
// is a scalar and whose lane offsets are constants of the kernel.  Rows past
// the last key are read from the last key: what a page holds behind it may be
// anything.
//
// A key range that is split publishes its unnormalised output, max and sum
// per (row, q head) with device-scope stores; the last of a row block to
// arrive (ticket) merges them in range order, so the bits do not depend on
// who that is.

#include <algorithm>

#include "mfma_attn.hpp"
#include "paged.hpp"

namespace qasr {

namespace {

constexpr int kSlice = 32;                          // keys of a wave's slice of a narrow tile
constexpr int kNarrowWaves = kNarrowTile / kSlice;  // 4
constexpr int kWideWaves = kWideTile / 16;          // 8

template <int NW>
struct Shared {
    f16 buf[NW * 2 * kSlice * kHeadDim];  // 16 KB a wave: a slice of K and V, or two wide tiles
    float ml[NW][2][64];
    int last, next;
};
static_assert(sizeof(Shared<kWideWaves>::buf) == 2 * 2 * kWideTile * kHeadDim * sizeof(f16), "two wide tiles of K and V");

// The thread's index, opaque to the compiler: what is derived from it then
// lives in one place of the item loop instead of in registers all through it
// (74 of them spilled).
__device__ __forceinline__ int thread_id() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

__device__ __forceinline__ void store_dev2(float* p, float a, float b) {
    const uint64_t v = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_dev2(const float* p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<uint64_t*>(const_cast<float*>(p)), __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// What a workgroup knows of its item.
struct Item {
    int row0, rows, planned, pos0, kend, tile0, tile1, splits, split, rec, block, kvh;
    int page0, last_page;  // first page of the range, last of the row block's keys (table places)
    const int32_t* table;  // the request's pages
    const f16* base;       // the kv head's K in page 0
};

// Copies of one 16-key group, 1 KB an instruction (lane l's 16 bytes to m0 +
// 16 l): K instruction j reads rows 4 j .. +4 with their 16-byte chunks
// permuted (swz16: lane l's chunk is (l % 16) ^ (4 (l / 16) | j)), V
// instruction j dims 32 j .. +32 of the 16 rows, `slab` bytes on in the LDS.
// The group's address is scalar, a lane's offsets are registers of the kernel,
// so a copy is an instruction and its LDS address (which m0 needs a cycle to
// take).  Waited for by count.
struct Offsets {
    uint32_t k[4], v[4];
};
__device__ __forceinline__ void copy4(const f16* base, const uint32_t (&voff)[4], uint32_t lds, uint32_t step) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff[j]), "s"(base), "{m0}"(lds + j * step)
                     : "memory");
}
// Row r of the group reads row min(r + add, last): 0 and 15, but in the group
// of the last key or past it.  `v_from_k`: bytes from a page's K to its V.
__device__ __forceinline__ Offsets group_offsets(int lane, int add, int last, uint32_t v_from_k) {
    Offsets o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int r = lane >> 4;
        o.k[j] = min(4 * j + r + add, last) * 256 + (((lane & 15) ^ (r << 2) ^ j) * 16);
        o.v[j] = v_from_k + min((lane >> 2) + add, last) * 256 + j * 64 + (lane & 3) * 16;
    }
    return o;
}

// The range's pages, a lane each: lane l of the first registers is page page0
// + lo + l of the table, of the second the 64 after them.  The work item
// brings the first 48 ids (lanes 16 .. 63, lo = -16), so that the first copies
// wait for one load; longer ranges read on from the table.  An id outside the
// pool sets its lane's bit in `bad`, which hides its keys, and reads the zero
// page: page 0, say, is another request's, whose infinities times a weight of 0
// would be NaN here.
struct PageRun {
    int id;
    uint64_t bad;
};
struct Pages {
    PageRun cur, nxt;
    int lo;
};
__device__ __forceinline__ int load_pages(const Item& it, int rel) {
    return it.last_page - it.page0 >= rel ? it.table[min(it.page0 + rel + (thread_id() & 63), it.last_page)] : 0;
}
__device__ __forceinline__ PageRun check_pages(const PagedAttnArgs& a, int id) {
    const bool bad = (uint32_t)id >= (uint32_t)a.pages;
    return {bad ? a.zero_page : id, __ballot(bad)};
}
__device__ __forceinline__ int page_rel(const PagedAttnArgs& a, const Item& it, int key) {
    return (min(key, it.kend - 1) >> a.page_shift) - it.page0;
}
// Before the pages from `key` on are asked for: on to the next 64.
__device__ __forceinline__ void advance_pages(const PagedAttnArgs& a, const Item& it, Pages& p, int key) {
    if (__builtin_expect(page_rel(a, it, key) - p.lo >= 64, 0)) {
        p.cur = p.nxt;
        p.lo += 64;
        p.nxt = check_pages(a, load_pages(it, p.lo + 64));
    }
}
// Address of K of the 16-key group of `key` (past the end: of the last key).
__device__ __forceinline__ const f16* group_base(const PagedAttnArgs& a, const Item& it, const Pages& p, int key) {
    const int k = min(key, it.kend - 1), r = (k >> a.page_shift) - it.page0 - p.lo;
    const int id = __builtin_amdgcn_readlane(r < 64 ? p.cur.id : p.nxt.id, r & 63);
    const uint64_t page = (uint64_t)(uint32_t)id * (uint32_t)a.page_stride;  // a page is < 2^21 elements
    return it.base + page + ((k & ((1 << a.page_shift) - 1)) & ~15) * kHeadDim;
}
// Bit j: the page of keys key + 16 j .. +16 lies outside the pool.
template <int N>
__device__ __forceinline__ uint32_t hidden_groups(const PagedAttnArgs& a, const Item& it, const Pages& p, int key) {
    uint32_t bits = 0;
    if (__builtin_expect((p.cur.bad | p.nxt.bad) != 0, 0)) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int r = page_rel(a, it, key + 16 * j) - p.lo;
            bits |= (uint32_t)((r < 64 ? p.cur.bad : p.nxt.bad) >> (r & 63) & 1) << j;
        }
    }
    return bits;
}
// K and V of the 16-key group of `key` into kd (1 KB a step) and vd (`slab` a
// step).
__device__ __forceinline__ void copy_group(const PagedAttnArgs& a, const Item& it, const f16* base, const Offsets& whole,
                                           int key, bool v, uint32_t lds, uint32_t step) {
    if (key + 16 <= it.kend) {
        copy4(base, v ? whole.v : whole.k, lds, step);
    } else {
        const int gkey = min(key, (it.kend - 1) & ~15);
        const Offsets o = group_offsets(thread_id() & 63, key - gkey, it.kend - 1 - gkey, (uint32_t)a.kv_stride * 2);
        copy4(base, v ? o.v : o.k, lds, step);
    }
}

// ---- results --------------------------------------------------------------

// The published state of a (row block, kv head, range): for each pair of dims
// the values of all columns next to each other, 2 floats a column, so that a
// store instruction of an MFMA accumulator (a column a lane) writes whole
// lines; then (max, sum) of every column.  Columns: q head h of row r is 32
// (r / 16) + h * (rows of that 16) + r % 16.
__device__ __forceinline__ int column(const Item& it, int r, int h) {
    return (r >> 4) * 32 + h * min(16, it.rows - (r & ~15)) + (r & 15);
}
__device__ __forceinline__ float* range_o(const PagedAttnArgs& a, const Item& it, int range) {
    return a.ws_o + ((int64_t)it.rec * a.nkvh + (it.kvh * it.splits + range) * it.rows) * (kRep * kHeadDim);
}
__device__ __forceinline__ float* range_ml(const PagedAttnArgs& a, const Item& it, int range) {
    return a.ws_ml + ((int64_t)it.rec * a.nkvh + (it.kvh * it.splits + range) * it.rows) * (kRep * 2);
}

// A thread's pairs of dims of a column, kFlight / SP at a time with all their
// ranges (up to SP) in flight together; more than SP ranges in groups.
template <int THREADS, int SP>
__device__ __forceinline__ void merge_pairs(const float* src, int cols, int splits, const float* wt, const float* sums,
                                            uint32_t* res, int pad) {
    constexpr int kFlight = 16, kUnits = kFlight / SP;
    const int units = cols * (kHeadDim / 2);
    for (int u0 = thread_id(); u0 < units; u0 += THREADS * kUnits) {
        float o[kUnits][2];
#pragma unroll
        for (int k = 0; k < kUnits; ++k) o[k][0] = o[k][1] = 0.0f;
        for (int i0 = 0; i0 < splits; i0 += SP) {
            float2 x[kUnits][SP];
#pragma unroll
            for (int k = 0; k < kUnits; ++k)
#pragma unroll
                for (int i = 0; i < SP; ++i)
                    x[k][i] = load_dev2(src + (min(i0 + i, splits - 1) * units + min(u0 + k * THREADS, units - 1)) * 2);
#pragma unroll
            for (int k = 0; k < kUnits; ++k) {
                const int c = min(u0 + k * THREADS, units - 1) % cols;
#pragma unroll
                for (int i = 0; i < SP; ++i) {
                    const bool on = i0 + i < splits;
                    const float w = wt[c * splits + min(i0 + i, splits - 1)];
                    o[k][0] = on ? fmaf(x[k][i].x, w, o[k][0]) : o[k][0];
                    o[k][1] = on ? fmaf(x[k][i].y, w, o[k][1]) : o[k][1];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const int u = u0 + k * THREADS, p = u / cols, c = u - p * cols;
            if (u < units) {
                const float inv = sums[c * splits];  // 0: no key weighs anything, whatever o is
                const half2v y = {(f16)(inv == 0.0f ? 0.0f : o[k][0] * inv), (f16)(inv == 0.0f ? 0.0f : o[k][1] * inv)};
                res[c * pad + p] = __builtin_bit_cast(uint32_t, y);
            }
        }
    }
}

// Merge of the published ranges of a row block.  The (max, sum) of every
// column and range turn into weights 2^(m_i - M) in LDS; then the threads take
// pairs of dims of a column, sums in range order.  Results pass through LDS, as
// the columns lie in the outputs 4 KB apart.  Many ranges' weights are made
// by as many lanes (one row of 8192 keys, 17 ranges: 16.4 -> 14.8 us), few
// ranges' by a thread a column, whose code is shorter to fetch (8 chunks of 2 or
// 3 ranges: 17.4 against 18.3 us).
template <int NW>
__device__ __forceinline__ void merge_splits(const PagedAttnArgs& a, const Item& it, Shared<NW>& sh) {
    constexpr int kThreads = NW * 64, kPairs = kHeadDim / 2, kPad = kPairs + 4;
    const int tid = thread_id();
    const int cols = it.rows * kRep, splits = it.splits;
    const float* src = range_o(a, it, 0);
    const float* ml = range_ml(a, it, 0);
    uint32_t* res = reinterpret_cast<uint32_t*>(sh.buf);          // [cols][kPad] pairs of f16
    float* wt = reinterpret_cast<float*>(res + cols * kPad);      // [cols][splits]
    float* sums = wt + cols * splits;
    if (splits > 8) {  // a column for 32 lanes, a range a lane
        static_assert(kPagedMaxSplits == 32, "a range a lane");
        const int i = tid & 31;
        const bool on = i < splits;
#pragma unroll 1
        for (int c = tid >> 5; c < cols; c += kThreads / 32) {
            const float2 x = load_dev2(ml + ((on ? i : 0) * cols + c) * 2);
            const float m = on ? x.x : kNegInf;
            float M = m;
#pragma unroll
            for (int d = 16; d; d >>= 1) M = fmaxf(M, __shfl_xor(M, d));
            const float w = m == kNegInf ? 0.0f : fast_exp2(m - M);
            float l = on ? x.y * w : 0.0f;
#pragma unroll
            for (int d = 16; d; d >>= 1) l += __shfl_xor(l, d);
            if (on) wt[c * splits + i] = w;
            if (i == 0) sums[c * splits] = l == 0.0f ? 0.0f : 1.0f / l;
        }
    } else {
        for (int e = tid; e < cols * splits; e += kThreads) {
            const int i = e / cols, c = e - i * cols;
            const float2 x = load_dev2(ml + e * 2);
            wt[c * splits + i] = x.x;
            sums[c * splits + i] = x.y;
        }
        __syncthreads();
        for (int c = tid; c < cols; c += kThreads) {
            float M = kNegInf, l = 0.0f;
            for (int i = 0; i < splits; ++i) M = fmaxf(M, wt[c * splits + i]);
            for (int i = 0; i < splits; ++i) {
                const float m = wt[c * splits + i], w = m == kNegInf ? 0.0f : fast_exp2(m - M);
                wt[c * splits + i] = w;
                l = fmaf(sums[c * splits + i], w, l);
            }
            sums[c * splits] = l == 0.0f ? 0.0f : 1.0f / l;
        }
    }
    __syncthreads();
    if (splits <= 2)
        merge_pairs<kThreads, 2>(src, cols, splits, wt, sums, res, kPad);
    else if (splits <= 4)
        merge_pairs<kThreads, 4>(src, cols, splits, wt, sums, res, kPad);
    else if (splits <= 8)
        merge_pairs<kThreads, 8>(src, cols, splits, wt, sums, res, kPad);
    else
        merge_pairs<kThreads, 16>(src, cols, splits, wt, sums, res, kPad);
    __syncthreads();
    for (int u = tid; u < cols * (kHeadDim / 8); u += kThreads) {  // 16 bytes a thread, a column 16 threads
        const int r = u >> 5, h = (u >> 4) & 1, p = u & 15;
        const uint4 y = *reinterpret_cast<const uint4*>(res + column(it, r, h) * kPad + 4 * p);
        *(uint4*)(a.out + ((int64_t)(it.row0 + r) * a.nkvh + it.kvh) * (kRep * kHeadDim) + h * kHeadDim + 8 * p) = y;
    }
}

// After this range's state is stored: the last range of the row block to
// arrive merges them.  Called by every thread of the workgroup.
template <int NW>
__device__ __forceinline__ void arrive(const PagedAttnArgs& a, const Item& it, Shared<NW>& sh) {
    stores_done_barrier();
    uint32_t* ctr = a.counters + ((int64_t)it.block * a.nkvh + it.kvh) * kPagedCounterStep;
    if (threadIdx.x == 0) sh.last = ticket_add(ctr) == (uint32_t)(it.splits - 1);
    __syncthreads();
    if (!sh.last) return;
    merge_splits(a, it, sh);
    if (threadIdx.x == 0) ticket_reset(ctr);
}

// Accumulator elements 4 q0 .. +4 NQ of column (r, h): dims db*32 + 8*(q0 +
// q) + 4*g + x; stored as outputs, or as the range's state.
template <int NQ>
__device__ __forceinline__ void put_block(const PagedAttnArgs& a, const Item& it, const float* o, float l, int db,
                                          int q0, int g, int r, int h) {
    if (it.splits == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        f16* dst = a.out + ((int64_t)(it.row0 + r) * a.nkvh + it.kvh) * (kRep * kHeadDim) + h * kHeadDim + db * 32;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            half4v y;
#pragma unroll
            for (int x = 0; x < 4; ++x) y[x] = (f16)(o[4 * q + x] * inv);
            *(half4v*)(dst + 8 * (q0 + q) + 4 * g) = y;
        }
    } else {
        const int step = it.rows * kRep * 2;  // floats of a pair of dims
        float* dst = range_o(a, it, it.split) + (db * 16 + 4 * q0 + 2 * g) * step + column(it, r, h) * 2;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            store_dev2(dst + 4 * q * step, o[4 * q], o[4 * q + 1]);
            store_dev2(dst + (4 * q + 1) * step, o[4 * q + 2], o[4 * q + 3]);
        }
    }
}

// NaN if some element is not finite and has to be computed again: not if the
// weights' sum is NaN, which all dims of the column are then anyway.
template <int N>
__device__ __forceinline__ float not_finite(const float* o, float l) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) t = fmaf(o[i], 0.0f, t);
    return l == l ? t : 0.0f;
}

// One column's output dims again, in f32 and key by key, by one wave: for
// states that are not finite.  The MFMA product weighs a hidden key with 0,
// and 0 * inf is NaN: here hidden keys are left out, so infinities and NaN
// reach only the rows that see them.  Lane l < 32 returns dim 32 db + l of row
// r, q head h; `sum`: the sum of the weights, which are taken against these
// scores' own maximum (-inf: they are 0), as the sums of the MFMA round
// otherwise.
__device__ __forceinline__ float exact_dims(const PagedAttnArgs& a, const Item& it, int key0, int key1, int r, int h,
                                            int db, int lane, float& sum) {
    const int pos = it.pos0 + r, end = min(key1, pos + 1);
    const f16* q = a.q + ((int64_t)(it.row0 + r) * a.nkvh + it.kvh) * (kRep * kHeadDim) + h * kHeadDim;
    // This lane's key of the 64 from k0 on: its row, whether it is seen, and its
    // score.
    auto score = [&](int k0, uint64_t& row, bool& seen) {
        const int key = k0 + lane;
        const int id = it.table[min(key, it.kend - 1) >> a.page_shift];
        seen = key < end && (uint32_t)id < (uint32_t)a.pages;
        row = (uint64_t)(uint32_t)(seen ? id : 0) * (uint32_t)a.page_stride +
              (key & ((1 << a.page_shift) - 1)) * kHeadDim;
        float s = 0.0f;
        for (int d = 0; d < kHeadDim; d += 8) {
            H8 x, y;
            x.u = *(const uint4*)(it.base + row + d);
            y.u = *(const uint4*)(q + d);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(h2f(x.e[e]), h2f(y.e[e]), s);
        }
        return s * a.scale_log2;
    };
    uint64_t row;
    bool seen;
    float M = kNegInf, l = 0.0f, o = 0.0f;
    for (int k0 = key0; k0 < end; k0 += 64) {
        const float s = score(k0, row, seen);
        M = fmaxf(M, seen ? s : kNegInf);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) M = fmaxf(M, __shfl_xor(M, d));
    for (int k0 = key0; k0 < end; k0 += 64) {
        const float s = score(k0, row, seen);
        const float p = M == kNegInf ? 0.0f : softmax_w_scaled(s, M);  // (-inf) - (-inf): weighs nothing
        l += seen ? p : 0.0f;
        uint64_t todo = __ballot(seen);
        while (todo) {
            const int j = __builtin_ctzll(todo);
            todo &= todo - 1;
            const uint64_t at = (uint64_t)__shfl((int)(uint32_t)(row >> 32), j) << 32 |
                                (uint32_t)__shfl((int)(uint32_t)row, j);
            o = fmaf(__shfl(p, j), h2f(it.base[at + a.kv_stride + 32 * db + (lane & 31)]), o);
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
    sum = l;
    return o;
}
// Puts the columns of a wave whose dim block db (32 dims) is not finite.
// every lane: its column's sum; valid columns only.  The sum that the state has
// is of weights against another maximum, rounded to f16 (weights()): the dims
// are divided by their own sum, and a range's state holds them times the
// state's sum over theirs.
__device__ __forceinline__ void put_exact(const PagedAttnArgs& a, const Item& it, int key0, int key1, float L, int db,
                                          int r, int h, bool valid, uint32_t cols) {
    const int lane = thread_id() & 63;
    uint64_t todo = __ballot(valid) & cols;  // a lane a column: those of g = 0
    while (todo) {
        const int j = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int rj = __shfl(r, j), hj = __shfl(h, j);
        const float l = __shfl(L, j);
        float sum;
        float o = exact_dims(a, it, key0, key1, rj, hj, db, lane, sum);
        if (lane >= 32) continue;
        if (it.splits == 1) {
            o = l == 0.0f ? 0.0f : o / sum;
            a.out[((int64_t)(it.row0 + rj) * a.nkvh + it.kvh) * (kRep * kHeadDim) + hj * kHeadDim + db * 32 + lane] = f2h(o);
        } else {
            o = l == 0.0f ? o : o * (l / sum);
            store_dev(range_o(a, it, it.split) + (db * 16 + (lane >> 1)) * it.rows * kRep * 2 +
                          column(it, rj, hj) * 2 + (lane & 1),
                      o);
        }
    }
}

// The draw of a workgroup's next item, asked for when the keys of this one are
// done and needed when its results are stored.  Asked for when an
// item starts, the last items go to workgroups that are busy for long: 4 chunks
// of 100-450 rows 25.7 against 21.6 us, 2 with 8 single rows 38.3 against 30.7.
struct Draw {
    uint32_t* counter;
    bool more;       // items than workgroups
    uint32_t drawn;  // thread 0
};
__device__ __forceinline__ void draw(Draw& d) {
    if (d.more && threadIdx.x == 0) d.drawn = ticket_add(d.counter);
}

// ---- the two kinds of item ------------------------------------------------

// This lane's query column (row rin of the block, q head h): its Q^T operand
// straight from memory, its position and the empty softmax state.
__device__ __forceinline__ void init_wave(Wave& w, const PagedAttnArgs& a, const Item& it, int rin, int h, int lane) {
    const int r = min(rin, it.rows - 1);  // columns past the block repeat its last row
    const f16* q = a.q + ((int64_t)(it.row0 + r) * a.nkvh + it.kvh) * (kRep * kHeadDim) + h * kHeadDim + 8 * (lane >> 5);
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) w.qb[ks] = *(const half8v*)(q + 16 * ks);
    w.g = lane >> 5;
    w.qpos = it.pos0 + r;
    w.scale_log2 = a.scale_log2;
#pragma unroll
    for (int db = 0; db < 4; ++db) w.o[db] = (float16v){};
    w.m = kNegInf;
    w.l = 0.0f;
    operand_addrs(w, lane);
}
// Every load and copy so far has landed, Q among them.  The registers are
// named here, once: else the compiler, which does not count the copies, waits
// for Q inside the tile loop, and so for every copy in flight.
__device__ __forceinline__ void wait_q(Wave& w) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) asm volatile("" : "+v"(w.qb[ks]));
}

// Marks what the fast path hardly ever takes: the compiler then lays it out
// away from it.  A launch starts with a cold instruction cache, so that short
// items cost about what their code's lines cost to fetch.
__device__ __forceinline__ bool rarely(bool x) { return __builtin_expect(x, 0); }

// Scores of keys past the row's position out of the way: element i of block
// kb is key k0 + 32 kb + 4 g + 8 (i / 4) + i % 4.
template <int NB>
__device__ __forceinline__ void mask_scores(const Wave& w, float16v (&s)[NB], int k0) {
    const int last = w.qpos - k0 - 4 * w.g;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = 32 * kb + 8 * (i >> 2) + (i & 3) > last ? kNegInf : s[kb][i];
}
// And of the 16-key groups whose bit is set in `hidden`.
template <int NB>
__device__ __forceinline__ void hide_scores(float16v (&s)[NB], uint32_t hidden) {
#pragma unroll
    for (int j = 0; j < 2 * NB; ++j)
        if (hidden >> j & 1)
#pragma unroll
            for (int i = 0; i < 8; ++i) s[j >> 1][8 * (j & 1) + i] = kNegInf;
}

// The running maximum moves when a score passes it by more than the slack.  A
// weight is then 2^(s * e.scale - e.base).  The scale is fused into the
// subtraction, which leaves the rounding of the scaled maximum in it: next to
// nothing, but 1 and more for maxima past 2^24, and the weights would pass f16.
// Scores that large are scaled and reduced here, one rounding after the other.
constexpr float kLargeScore = 1 << 20;
struct Exponent {
    float scale, base;
};
template <int NB>
__device__ __forceinline__ Exponent move_max(Wave& w, float16v (&s)[NB]) {
    float mx = kNegInf;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
    mx = halves_max(mx) * w.scale_log2;
    const bool up = mx > w.m + kRescaleSlack;
    Exponent e{w.scale_log2, w.m};
    if (__ballot(up || !(fabsf(mx) < kLargeScore))) {
        if (rarely(__ballot(up && w.m != kNegInf))) {  // not at the first keys
            const float alpha = !up ? 1.0f : w.m == kNegInf ? 0.0f : fast_exp2(w.m - mx);
#pragma unroll
            for (int db = 0; db < 4; ++db) w.o[db] *= alpha;
            w.l *= alpha;
        }
        w.m = up ? mx : w.m;
        e.base = w.m;
        if (rarely(__ballot(fabsf(mx) >= kLargeScore && mx != kNegInf))) {
#pragma clang fp contract(off)
            const float base = w.m == kNegInf ? 0.0f : w.m;
#pragma unroll
            for (int kb = 0; kb < NB; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[kb][i] = s[kb][i] * w.scale_log2 - base;
            e = {1.0f, 0.0f};
        }
    }
    e.base = e.base == kNegInf ? 0.0f : e.base;
    return e;
}

// The weights of a step's scores, as P^T (B-operand layout), and their row sum.
// They are rounded to f16, as in the slot pool's prefill: the product takes f16,
// and two of them for each weight (Few) would be half as many MFMAs again where
// MFMAs bound the time.  The sum is of the rounded values, so that a rounding
// shifts weight between keys and does not scale the row: an output moves by at
// most 2^-11 of the values' mean distance from it.  Four sums of v_fma_mix_f32, which runs
// beside another wave's MFMAs; v_dot2_f32_f16 does not (MFMA and VALU work of
// two waves a SIMD: no overlap with it, about half of the smaller part
// without).
template <int NB>
__device__ __forceinline__ void weights(Wave& w, const float16v (&s)[NB], const Exponent& e, half8v (&pb)[2 * NB]) {
    float ps[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w4 = 0; w4 < 2 * NB; ++w4) {
        union {
            half8v h;
            uint32_t u[4];
        } p;
#pragma unroll
        for (int j = 0; j < 8; ++j) p.h[j] = (f16)softmax_w_raw(s[w4 >> 1][8 * (w4 & 1) + j], e.scale, e.base);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            asm("v_fma_mix_f32 %0, 1.0, %1, %0 op_sel_hi:[0,1,0]" : "+v"(ps[j]) : "v"(p.u[j]));
            asm("v_fma_mix_f32 %0, 1.0, %1, %0 op_sel:[0,1,0] op_sel_hi:[0,1,0]" : "+v"(ps[j]) : "v"(p.u[j]));
        }
        pb[w4] = p.h;
    }
    w.l += halves_sum((ps[0] + ps[1]) + (ps[2] + ps[3]));
}

#define WAIT_VM(n) asm volatile("s_waitcnt vmcnt(" #n ")" ::: "memory")

// The matrix products of a step.  Operand reads run kAhead products ahead of
// their MFMA: reads and MFMAs stay in this order (vector and scalar work may
// move between them), else each MFMA waits out its own read's latency.
constexpr int kAhead = 3;
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0x406); }  // VALU, SALU, exp may cross

// S^T of K rows kt[0 .. 32 NB - 1], keys kb*32 + (8*(i/4) + 4*g + i%4) x query
// n.
template <int NB>
__device__ __forceinline__ void scores(const Wave& w, const f16* kt, float16v (&s)[NB]) {
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) s[kb] = (float16v){};
    half8v ka[8 * NB];
    auto read = [&](int x) { ka[x] = *(const half8v*)&kt[(x % NB) * 32 * kHeadDim + w.kaddr[x / NB]]; };
#pragma unroll
    for (int x = 0; x < kAhead; ++x) read(x);
    keep_order();
#pragma unroll
    for (int x = 0; x < 8 * NB; ++x) {
        if (x + kAhead < 8 * NB) read(x + kAhead);
        keep_order();
        s[x % NB] = mfma32(ka[x], w.qb[x / NB], s[x % NB]);
        keep_order();
    }
}

// O^T += V^T P^T with V rows vt[0 .. 32 NB - 1] of a tile of ROWS rows.
template <int ROWS, int NB>
__device__ __forceinline__ void product(Wave& w, const f16* vt, const half8v (&pb)[2 * NB]) {
    half4v lo[8 * NB], hi[8 * NB];
    auto read = [&](int x) {
        const f16* vp = vt + w.vbase + (x & 3) * (ROWS * 32) + (x >> 2) * 16 * 32;
        lo[x] = read_tr(vp);
        hi[x] = read_tr(vp + 8 * 32);
    };
#pragma unroll
    for (int x = 0; x < kAhead; ++x) read(x);
    keep_order();
#pragma unroll
    for (int x = 0; x < 8 * NB; ++x) {
        if (x + kAhead < 8 * NB) read(x + kAhead);
        keep_order();
        const half8v va = __builtin_shufflevector(lo[x], hi[x], 0, 1, 2, 3, 4, 5, 6, 7);
        w.o[x & 3] = mfma32(va, pb[x >> 2], w.o[x & 3]);
        keep_order();
    }
}

// The state of column lane & 31 that the waves j0, j0 + dj, .. (N of them)
// left in LDS: dims' elements e0 .. e0 + NE, each wave's weighed by 2^(m_j -
// M), in wave order.  Wave j's elements lie at buf + j * 16 KB: element e of
// lane l at (e / 4) * 256 + 4 l + e % 4.
template <int N, int NE, int NW>
__device__ __forceinline__ void combine(const Shared<NW>& sh, int j0, int dj, int e0, int lane, float (&o)[NE], float& M,
                                        float& L) {
    float4 x[N][NE / 4];
    float mj[N], lj[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        mj[j] = sh.ml[j0 + j * dj][0][lane];
        lj[j] = sh.ml[j0 + j * dj][1][lane];
        const float4* src = reinterpret_cast<const float4*>(sh.buf) + (j0 + j * dj) * 1024 + e0 * 16 + lane;
#pragma unroll
        for (int q = 0; q < NE / 4; ++q) x[j][q] = src[q * 64];
    }
    keep_order();  // every read is on its way before the first is waited for
    M = mj[0];
#pragma unroll
    for (int j = 1; j < N; ++j) M = fmaxf(M, mj[j]);
    L = 0.0f;
#pragma unroll
    for (int e = 0; e < NE; ++e) o[e] = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float aj = mj[j] == kNegInf ? 0.0f : fast_exp2(mj[j] - M);
        L = fmaf(lj[j], aj, L);
#pragma unroll
        for (int q = 0; q < NE / 4; ++q) {
            o[4 * q] = fmaf(x[j][q].x, aj, o[4 * q]);
            o[4 * q + 1] = fmaf(x[j][q].y, aj, o[4 * q + 1]);
            o[4 * q + 2] = fmaf(x[j][q].z, aj, o[4 * q + 2]);
            o[4 * q + 3] = fmaf(x[j][q].w, aj, o[4 * q + 3]);
        }
    }
}
// A wave leaves its state for combine(): 16 accumulator elements of NDB dim
// blocks from db0 on.
template <int NDB, int NW>
__device__ __forceinline__ void leave(Shared<NW>& sh, const Wave& w, int wave, int db0, int lane) {
    float4* dst = reinterpret_cast<float4*>(sh.buf) + wave * 1024 + lane;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float16v& o = w.o[db0 + db];
            dst[((db0 + db) * 4 + q) * 64] = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
        }
}

// Narrow items of up to 8 rows: their 16 columns on v_mfma_f32_16x16x32_f16,
// whose products take half the time, with half the scores a lane.  us a layer
// on 32 columns against 16 (f16 weights on both): 1 row of 512 keys 8.4 / 7.7, of 8192 14.8 / 14.4, 16 rows
// of 400-2400 24.7 / 24.1.
//
// Their weights are held to 22 bits, as the slot pool's decode step holds them
// in f32: a weight is a sum of two f16 numbers, hi and its remainder lo, each
// with a product of its own.  (One f16 number moves an output by up to 2^-11 of
// the values' spread, about as much again as its own rounding.)  Exponents are
// taken against the running maximum less 7, so that the largest weight is 2^7
// to 2^15 and lo holds down to 2^-32 of it; f16 ends at 65504.  us a layer with
// one product and with two: 1 row of 512 keys 7.6 / 7.9, of 8192 14.4 / 14.6, 16
// rows of 400-2400 24.2 / 24.3.
constexpr int kFewRows = 8;
constexpr float kFewBase = 7.0f;
static_assert(kFewBase + kRescaleSlack < 16.0f, "weights fit f16");
struct Few {
    static constexpr int kRows = kFewRows;
    half8v qb[4];  // Q^T of k-step ks: dims 32*ks + 8*g .. +8 of query n
    float4v o[8];  // O^T: o[db][i] = dim db*16 + 4*g + i of query n
    float m, l;    // the running maximum less kFewBase, and the sum of weights
    int kaddr[4];  // K operand of k-step ks, rows 0..15 (halves)
    int vbase;
    int g, qpos;  // g: the lane's quarter
    float scale_log2;
};
__device__ __forceinline__ float quarters_max(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return halves_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quarters_sum(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return halves_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}
__device__ __forceinline__ float4v mfma16(const half8v& a, const half8v& b, const float4v& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void init_wave(Few& w, const PagedAttnArgs& a, const Item& it, int rin, int h, int lane) {
    const int r = min(rin, it.rows - 1), n = lane & 15;
    w.g = lane >> 4;
    const f16* q = a.q + ((int64_t)(it.row0 + r) * a.nkvh + it.kvh) * (kRep * kHeadDim) + h * kHeadDim + 8 * w.g;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
        w.qb[ks] = *(const half8v*)(q + 32 * ks);
        w.kaddr[ks] = n * kHeadDim + (((4 * ks + w.g) ^ swz16(n)) * 8);
    }
    w.vbase = (4 * w.g + (n >> 2)) * 32 + 4 * (n & 3);
    w.qpos = it.pos0 + r;
    w.scale_log2 = a.scale_log2;
#pragma unroll
    for (int db = 0; db < 8; ++db) w.o[db] = (float4v){};
    w.m = kNegInf;
    w.l = 0.0f;
}
__device__ __forceinline__ void wait_q(Few& w) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) asm volatile("" : "+v"(w.qb[ks]));
}
// P^T of a slice: S^T of keys 16 kb + 4 g + i, masked, the running maximum,
// the weights (B operand: its k 8 g + j is key 16 (j / 4) + 4 g + j % 4), hi and
// lo, and their sum.
__device__ __forceinline__ void slice_scores(const Few& w, const f16* kt, float4v (&s)[2]) {
    half8v ka[8];
    auto read = [&](int x) { ka[x] = *(const half8v*)&kt[(x & 1) * 16 * kHeadDim + w.kaddr[x >> 1]]; };
    s[0] = s[1] = (float4v){};
#pragma unroll
    for (int x = 0; x < 4; ++x) read(x);
    keep_order();
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        if (x + 4 < 8) read(x + 4);
        keep_order();
        s[x & 1] = mfma16(ka[x], w.qb[x >> 1], s[x & 1]);
        keep_order();
    }
}
__device__ __forceinline__ void slice_weights(Few& w, float4v (&s)[2], int k0, bool mask, uint32_t hidden, half8v (&pb)[2]) {
#pragma clang fp contract(off)
    if (mask) {
        const int last = w.qpos - k0 - 4 * w.g;
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j >> 2][j & 3] = 16 * (j >> 2) + (j & 3) > last ? kNegInf : s[j >> 2][j & 3];
    }
    if (rarely(hidden)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j >> 2][j & 3] = hidden >> (j >> 2) & 1 ? kNegInf : s[j >> 2][j & 3];
    }
    // (Scaled first: a largest score minus itself is 0 then.  A fused multiply
    // and subtract leaves the rounding of the maximum, which past 2^24 is 1 and
    // more, and the weights would pass f16.)
    float mx = kNegInf;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        s[j >> 2][j & 3] *= w.scale_log2;
        mx = fmaxf(mx, s[j >> 2][j & 3]);
    }
    mx = quarters_max(mx) - kFewBase;
    const bool up = mx > w.m + kRescaleSlack;
    if (__ballot(up)) {
        if (rarely(__ballot(up && w.m != kNegInf))) {
            const float alpha = !up ? 1.0f : w.m == kNegInf ? 0.0f : fast_exp2(w.m - mx);
#pragma unroll
            for (int db = 0; db < 8; ++db) w.o[db] *= alpha;
            w.l *= alpha;
        }
        w.m = up ? mx : w.m;
    }
    const float mu = w.m == kNegInf ? 0.0f : w.m;
    float ps[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float p = softmax_w_scaled(s[j >> 2][j & 3], mu);
        pb[0][j] = (f16)p;
        pb[1][j] = (f16)(p - (float)pb[0][j]);
        ps[j & 1] += p;
    }
    w.l += quarters_sum(ps[0] + ps[1]);
}
__device__ __forceinline__ void slice_product(Few& w, const f16* vt, const half8v (&pb)[2]) {
    half4v lo[8], hi[8];  // keys 0..15 and 16..31
    auto add = [&](int x, int part) {
        w.o[x] = mfma16(__builtin_shufflevector(lo[x], hi[x], 0, 1, 2, 3, 4, 5, 6, 7), pb[part], w.o[x]);
        keep_order();
    };
    auto read = [&](int x) {
        const f16* vp = vt + w.vbase + (x >> 1) * (kSlice * 32) + (x & 1) * 16;
        lo[x] = read_tr(vp);
        hi[x] = read_tr(vp + 16 * 32);
    };
#pragma unroll
    for (int x = 0; x < 4; ++x) read(x);
    keep_order();
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        if (x + 4 < 8) read(x + 4);
        keep_order();
        add(x, 0);
        if (x >= 2) add(x - 2, 1);  // not right behind the product it adds to
    }
    add(6, 1);
    add(7, 1);
}
template <int NW>
__device__ __forceinline__ void leave_all(Shared<NW>& sh, const Few& w, int wave, int lane) {
    float4* dst = reinterpret_cast<float4*>(sh.buf) + wave * 1024 + lane;
#pragma unroll
    for (int db = 0; db < 8; ++db) dst[db * 64] = make_float4(w.o[db][0], w.o[db][1], w.o[db][2], w.o[db][3]);
}
__device__ __forceinline__ void put_dims(const PagedAttnArgs& a, const Item& it, const float (&o)[8], float l, int wave,
                                         int g, int r, int h) {
    put_block<1>(a, it, o, l, wave, g >> 1, g & 1, r, h);
    put_block<1>(a, it, o + 4, l, wave, 2 + (g >> 1), g & 1, r, h);
}

// And of up to 16 rows.
struct Many : Wave {
    static constexpr int kRows = kNarrowRows;
};
__device__ __forceinline__ void slice_scores(const Many& w, const f16* kt, float16v (&s)[1]) { scores<1>(w, kt, s); }
__device__ __forceinline__ void slice_weights(Many& w, float16v (&s)[1], int k0, bool mask, uint32_t hidden, half8v (&pb)[2]) {
    if (mask) mask_scores<1>(w, s, k0);
    if (rarely(hidden)) hide_scores<1>(s, hidden);
    const Exponent e = move_max<1>(w, s);
    weights<1>(w, s, e, pb);
}
__device__ __forceinline__ void slice_product(Many& w, const f16* vt, const half8v (&pb)[2]) { product<kSlice, 1>(w, vt, pb); }
template <int NW>
__device__ __forceinline__ void leave_all(Shared<NW>& sh, const Many& w, int wave, int lane) { leave<4>(sh, w, wave, 0, lane); }
__device__ __forceinline__ void put_dims(const PagedAttnArgs& a, const Item& it, const float (&o)[16], float l, int wave,
                                         int g, int r, int h) {
    put_block<4>(a, it, o, l, wave, 0, g, r, h);
}

template <class W, class S, int NS, int NP>
__device__ __forceinline__ void run_narrow(const PagedAttnArgs& a, const Item& it, Pages pg, Shared<kNarrowWaves>& sh, Draw& next) {
    const int tid = thread_id(), lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr int kCols = kRep * W::kRows, kElems = kCols / 2;
    const int n = lane & (kCols - 1), h = n / W::kRows, rin = n % W::kRows;
    f16* kbuf = sh.buf + wave * (2 * kSlice * kHeadDim);
    f16* vbuf = kbuf + kSlice * kHeadDim;
    const Offsets whole = group_offsets(lane, 0, 15, (uint32_t)a.kv_stride * 2);

    // Copies of the slice of tile t: its K or its V.
    auto copy_slice = [&](int t, bool v) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int key = t * kNarrowTile + wave * kSlice + 16 * p;
            const uint32_t lds = v ? lds_addr(vbuf) + p * 1024 : lds_addr(kbuf) + p * 4096;
            copy_group(a, it, group_base(a, it, pg, key), whole, key, v, lds, v ? kSlice * 64 : 1024);
        }
    };
    W w;
    init_wave(w, a, it, rin, h, lane);
    if (it.tile0 < it.tile1) {
        copy_slice(it.tile0, false);
        copy_slice(it.tile0, true);
    }
    wait_q(w);
    for (int t = it.tile0; t < it.tile1; ++t) {
        const int k0 = t * kNarrowTile + wave * kSlice;
        const bool more = t + 1 < it.tile1;
        const uint32_t hidden = hidden_groups<2>(a, it, pg, k0);
        if (more) advance_pages(a, it, pg, k0 + kNarrowTile);
        if (k0 >= it.kend) {  // a wave's slice of the last tile: nothing to see
            WAIT_VM(0);
            break;
        }
        WAIT_VM(8);  // K landed, V in flight
        S s[NS];
        half8v pb[NP];
        slice_scores(w, kbuf, s);
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            copy_slice(t + 1, false);
        }
        slice_weights(w, s, k0, k0 + kSlice - 1 > it.pos0, hidden, pb);
        if (more)
            WAIT_VM(8);
        else
            WAIT_VM(0);
        slice_product(w, vbuf, pb);
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            copy_slice(t + 1, true);
        }
    }

    draw(next);
    // The waves' states combine: wave w finishes dim block w, out of each
    // wave's own (now free) slice buffer.
    const bool valid = rin < it.rows;
    if (valid) {
        leave_all(sh, w, wave, lane);
        sh.ml[wave][0][lane] = w.m;
        sh.ml[wave][1][lane] = w.l;
    }
    __syncthreads();
    float o[kElems], M = 0.0f, L = 0.0f, t = 0.0f;
    if (valid) {
        combine<kNarrowWaves, kElems>(sh, 0, 1, kElems * wave, lane, o, M, L);
        t = not_finite<kElems>(o, L);
    }
    if (rarely(__ballot(t != t)))
        put_exact(a, it, it.tile0 * kNarrowTile, min(it.tile1 * kNarrowTile, it.kend), L, wave, rin, h, valid,
                  kCols == 32 ? ~0u : 0xffffu);
    else if (valid)
        put_dims(a, it, o, L, wave, w.g, rin, h);
    if (it.splits > 1 && valid && wave == 0 && w.g == 0) store_dev2(range_ml(a, it, it.split) + column(it, rin, h) * 2, M, L);
}

__device__ __forceinline__ void run_item(const PagedAttnArgs& a, const Item& it, Pages pg, Shared<kNarrowWaves>& sh, Draw& next) {
    if (it.planned <= kFewRows)
        run_narrow<Few, float4v, 2, 2>(a, it, pg, sh, next);
    else
        run_narrow<Many, float16v, 1, 2>(a, it, pg, sh, next);
    if (it.splits > 1) arrive(a, it, sh);
}

__device__ __forceinline__ void run_item(const PagedAttnArgs& a, const Item& it, Pages pg, Shared<kWideWaves>& sh, Draw& next) {
    const int tid = thread_id(), lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rw = wave & 3, kg = wave >> 2;  // 16 rows; 64 keys of every tile
    const int n = lane & 31, h = n >> 4, rin = rw * 16 + (n & 15);
    constexpr int kTile = kWideTile * kHeadDim, kGroup = kWideTile / 2;
    const Offsets whole = group_offsets(lane, 0, 15, (uint32_t)a.kv_stride * 2);

    // This wave's 16 keys of tile t into buffer t & 1: K, then V in slabs.
    auto copy_tile = [&](int t) {
        const int key = t * kWideTile + wave * 16;
        const f16* base = group_base(a, it, pg, key);
        const uint32_t lds = lds_addr(sh.buf) + (t & 1) * (4 * kTile);
        copy_group(a, it, base, whole, key, false, lds + wave * 4096, 1024);
        copy_group(a, it, base, whole, key, true, lds + 2 * kTile + wave * 1024, kWideTile * 64);
    };
    Wave w;
    init_wave(w, a, it, rin, h, lane);
    if (it.tile0 < it.tile1) copy_tile(it.tile0);
    const int first_pos = it.pos0 + rw * 16;
    const int last_pos = it.pos0 + min(rw * 16 + 15, it.rows - 1);
    const bool live = rw * 16 < it.rows;
    wait_q(w);
    for (int t = it.tile0; t < it.tile1; ++t) {
        WAIT_VM(0);
        __syncthreads();  // tile t is here, and the other buffer is read
        const int k0 = t * kWideTile + kg * kGroup;
        const uint32_t hidden = hidden_groups<4>(a, it, pg, k0);
        if (t + 1 < it.tile1) {
            advance_pages(a, it, pg, (t + 1) * kWideTile);
            copy_tile(t + 1);
        }
        if (!live || k0 > last_pos) continue;
        const f16* kt = sh.buf + (t & 1) * 2 * kTile + kg * kGroup * kHeadDim;
        float16v s[2];
        half8v pb[4];
        scores<2>(w, kt, s);
        if (k0 + kGroup - 1 > first_pos) mask_scores<2>(w, s, k0);
        if (rarely(hidden)) hide_scores<2>(s, hidden);
        const Exponent e = move_max<2>(w, s);
        weights<2>(w, s, e, pb);
        product<kWideTile, 2>(w, sh.buf + (t & 1) * 2 * kTile + kTile + kg * kGroup * 32, pb);
    }
    draw(next);
    __syncthreads();  // the buffers are read
    // The two key groups of a row wave combine: each leaves its state and
    // finishes two dim blocks.
    const bool valid = rin < it.rows;
    leave<4>(sh, w, wave, 0, lane);
    sh.ml[wave][0][lane] = w.m;
    sh.ml[wave][1][lane] = w.l;
    __syncthreads();
    float o[16], M, L;
#pragma unroll 1
    for (int db = 2 * kg; db < 2 * kg + 2; ++db) {
        combine<2, 16>(sh, rw, 4, db * 16, lane, o, M, L);
        const float t = not_finite<16>(o, L);
        if (rarely(__ballot(valid && t != t)))
            put_exact(a, it, it.tile0 * kWideTile, min(it.tile1 * kWideTile, it.kend), L, db, rin, h, valid, ~0u);
        else if (valid)
            put_block<4>(a, it, o, L, db, 0, w.g, rin, h);
    }
    if (it.splits > 1 && valid && kg == 0 && w.g == 0) store_dev2(range_ml(a, it, it.split) + column(it, rin, h) * 2, M, L);
    if (it.splits > 1) arrive(a, it, sh);
}

// Each kv head has a list of the items; its workgroups (every nkvh-th of the
// launch) start with one each and, where there are more items, draw the next
// from the head's counter, so that a workgroup of short items takes more of
// them.  The last workgroup to leave puts the counters back to zero.
template <int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_attn_kernel(
    PagedAttnArgs a) {
    __shared__ __attribute__((aligned(1024))) Shared<NW> sh;
    constexpr bool kWide = NW == kWideWaves;
    const PagedItem* list = kWide ? a.wide : a.narrow;
    const int last_item = (kWide ? a.max_wide : a.max_narrow) - 1;
    uint32_t* drawn = a.drawn + kWide * kPagedDrawWords;
    // (The division is done in vector registers.)
    int i = __builtin_amdgcn_readfirstlane(blockIdx.x / a.nkvh);
    const int kvh = __builtin_amdgcn_readfirstlane(blockIdx.x - i * a.nkvh);
    // Every lane reads a word of the item's record.
    auto load_item = [&](int k) {
        return reinterpret_cast<const int*>(list + min(k, last_item))[thread_id() & 63];
    };
    int words = load_item(i);
    const int items = a.n_items[kWide], share = __builtin_amdgcn_readfirstlane(gridDim.x / a.nkvh);
    const int peers = share + (kvh < (int)gridDim.x - share * a.nkvh);  // workgroups of this kv head
    Draw draw_next{drawn + kvh * kPagedCounterStep, items > share, 0};
    while (i < items) {
        auto word = [&](int k) { return __builtin_amdgcn_readlane(words, k); };
        Item it;
        it.kvh = kvh;
        const int shape = word(3);
        it.row0 = word(1);
        it.planned = shape & 0xff;
        it.rows = min(it.planned, a.rows - it.row0);  // rows past the caller's q are left out
        it.pos0 = word(2);
        it.kend = it.pos0 + it.rows;
        it.tile0 = word(4);
        it.tile1 = word(5);
        it.splits = (shape >> 8) & 0xff;
        it.split = (shape >> 16) & 0xff;
        it.rec = word(6);
        it.block = word(7);
        it.page0 = word(8);
        it.last_page = (it.kend - 1) >> a.page_shift;
        it.table = a.table + (int64_t)word(0) * a.stride;
        it.base = a.base + it.kvh * a.head_stride;
        if (it.rows > 0) {
            Pages pg;
            pg.cur = check_pages(a, words);
            pg.cur.bad &= ~0ull << kPagedItemHead;  // the header's lanes are no pages
            pg.lo = -kPagedItemHead;
            pg.nxt = {0, 0};
            if (it.last_page - it.page0 >= kPagedItemPages) pg.nxt = check_pages(a, load_pages(it, kPagedItemPages));
            run_item(a, it, pg, sh, draw_next);
        } else {
            draw(draw_next);
        }
        if (!draw_next.more) break;
        if (threadIdx.x == 0) sh.next = peers + (int)draw_next.drawn;
        __syncthreads();  // the next item reuses the LDS
        i = __builtin_amdgcn_readfirstlane(sh.next);
        words = load_item(i);
        __syncthreads();
    }
    uint32_t* gone = drawn + kPagedDrawWords - kPagedCounterStep;
    if (draw_next.more && threadIdx.x == 0 && ticket_add(gone) == gridDim.x - 1) {
        for (int k = 0; k < a.nkvh; ++k) ticket_reset(drawn + k * kPagedCounterStep);
        ticket_reset(gone);
    }
}

}  // namespace

hipError_t launch_paged_attn(const PagedAttnArgs& a, int cus, hipStream_t stream) {
    if (a.rows <= 0) return hipSuccess;
    if (a.max_wide > 0) {
        const int64_t wgs = std::min<int64_t>((int64_t)a.max_wide * a.nkvh, cus);
        hipLaunchKernelGGL(paged_attn_kernel<kWideWaves>, dim3((unsigned)wgs), dim3(kWideWaves * 64), 0, stream, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    const int64_t wgs = std::min<int64_t>((int64_t)a.max_narrow * a.nkvh, 2 * (int64_t)cus);
    hipLaunchKernelGGL(paged_attn_kernel<kNarrowWaves>, dim3((unsigned)wgs), dim3(kNarrowWaves * 64), 0, stream, a);
    return hipGetLastError();
}

}  // namespace qasr
