// paged_attn.hip -- attention of each request's new rows over its pages.
//
// Row r at position p of a request attends keys 0..p of it: softmax(q.k_t /
// sqrt(128)) . v, keys whose page lies outside the pool left out; a row that
// sees no key is zero.  One launch takes any mix of single rows and chunks:
// the work list (paged_plan.hip) is on the GPU, the workgroups walk it.
//
// Work item = (row block and key range of a request, kv head), kv head minor:
// with 8 kv heads workgroup i runs kv head i mod 8 on XCD i mod 8, and the
// row blocks of a kv head share its keys in that XCD's L2.  A workgroup is 4
// waves; a wave's 32 MFMA columns are 16 rows x the 2 q heads of the kv head
// (mfma_attn.hpp), so both heads use each key read.
//  - narrow items, up to 16 rows: every 128-key tile is cut into the waves'
//    slices of 32 keys.  A wave copies its own slice into its own LDS (16
//    KB), so the loop has no barrier; K of the next tile is requested when
//    the scores are done with this one, V when its product is.  The waves'
//    states combine through LDS at the end.
//  - wide items, up to 64 rows: wave w takes rows 16 w .. +16 against whole
//    64-key tiles, copied by all waves into two 32 KB buffers in turn, one
//    barrier a tile.
// Both fit 66 KB of LDS and 256 registers: two workgroups a CU, so one's
// softmax and latencies run under the other's MFMAs and copies.
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

constexpr int kThreads = 256;
constexpr int kSlice = 32;                        // keys of a wave's slice of a narrow tile
constexpr int kBufHalves = 4 * 2 * kSlice * kHeadDim;  // 64 KB
static_assert(kBufHalves == 2 * 2 * kWideTile * kHeadDim, "two wide tiles of K and V");

// One copy instruction: lane l's 16 bytes from base + voff to lds + 16 l.
// Waited for by count; the address registers are scalar and constant.
__device__ __forceinline__ void copy16(const f16* base, uint32_t voff, uint32_t lds) {
    asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "{m0}"(lds) : "memory");
}

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
    int row0, rows, pos0, kend, tile0, tile1, splits, split, rec, block, kvh;
    const int32_t* table;  // the request's pages
};

// The copies of one 16-key group at `base`: K instruction j reads rows 4 j ..
// +4 with their 16-byte chunks permuted (swz16: lane l's chunk is (l % 16) ^ (4
// (l / 16) | j)), V instruction j dims 32 j .. +32 of the 16 rows.  A lane's
// offsets are two registers of the kernel: what j adds is a scalar, and for K
// an exclusive or of j.
struct Offsets {
    uint32_t k, v;
};
__device__ __forceinline__ Offsets group_offsets(int lane) {
    const int r = lane >> 4;
    return {(uint32_t)(r * 256 + (((lane & 15) ^ (r << 2)) * 16)), (uint32_t)((lane >> 2) * 256 + (lane & 3) * 16)};
}
__device__ __forceinline__ void copy_k(const f16* base, Offsets o, uint32_t lds) {
    asm volatile("" : "+v"(o.k), "+s"(lds));  // made here, not kept for the whole kernel
#pragma unroll
    for (int j = 0; j < 4; ++j) copy16(base + j * 4 * kHeadDim, o.k ^ (16 * j), lds + j * 1024);
}
__device__ __forceinline__ void copy_v(const f16* base, const Offsets& o, uint32_t lds, uint32_t slab) {
    asm volatile("" : "+s"(lds));
#pragma unroll
    for (int j = 0; j < 4; ++j) copy16(base + j * 32, o.v, lds + j * slab);
}
// The same for the group of the last key, or past it (`base`: the last
// group): row r reads row min(r + add, last).
__device__ __forceinline__ void copy_k_tail(const f16* base, int add, int last, uint32_t lds) {
    asm volatile("" : "+s"(lds));
    const int lane = thread_id() & 63;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int r = lane >> 4;
        copy16(base, min(4 * j + r + add, last) * 256 + (((lane & 15) ^ (r << 2) ^ j) * 16), lds + j * 1024);
    }
}
__device__ __forceinline__ void copy_v_tail(const f16* base, int add, int last, uint32_t lds, uint32_t slab) {
    asm volatile("" : "+s"(lds));
    const int lane = thread_id() & 63;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        copy16(base + j * 32, min((lane >> 2) + add, last) * 256 + (lane & 3) * 16, lds + j * slab);
}

// Page ids of 64 key groups, a lane each: of the 16-key group (k0 + 16 *
// stride_groups ...), see the callers.  Keys past the end read the last
// key's page.  `bad`: lanes whose page lies outside the pool; their id is
// made 0, which is readable.
struct Pages {
    int id;
    uint64_t bad;
};
__device__ __forceinline__ Pages load_pages(const PagedAttnArgs& a, const Item& it, int key) {
    Pages p;
    p.id = it.table[min(key, it.kend - 1) >> a.page_shift];
    return p;
}
__device__ __forceinline__ void check_pages(const PagedAttnArgs& a, Pages& p) {
    const bool bad = (uint32_t)p.id >= (uint32_t)a.pages;
    p.bad = __ballot(bad);
    p.id = bad ? 0 : p.id;
}

// Address of K of the 16-key group that holds `key`, in page id.
__device__ __forceinline__ const f16* group_base(const PagedAttnArgs& a, int kvh, int id, int key) {
    return a.base + id * a.page_stride + kvh * a.head_stride +
           ((key & ((1 << a.page_shift) - 1)) & ~15) * kHeadDim;
}

// ---- results --------------------------------------------------------------

// Merge of the published ranges of a row block: 32 lanes a (row, q head)
// column, 4 dims a lane.  Weights 2^(m_i - M), sums in range order.
__device__ __forceinline__ void merge_splits(const PagedAttnArgs& a, const Item& it) {
    const int tid = thread_id(), lane = tid & 31, sub = tid >> 5;
    for (int c = sub; c < it.rows * kRep; c += kThreads / 32) {
        const int r = c >> 1, h = c & 1;
        const int64_t rec = ((int64_t)(it.rec + r) * a.nkvh + it.kvh) * kRep + h;
        const int64_t step = (int64_t)it.rows * a.nkvh * kRep;  // records of a range
        float m = kNegInf, l = 0.0f;
        if (lane < it.splits) {
            const float2 ml = load_dev2(a.ws_ml + (rec + lane * step) * 2);
            m = ml.x;
            l = ml.y;
        }
        float M = m;
#pragma unroll
        for (int d = 16; d; d >>= 1) M = fmaxf(M, __shfl_xor(M, d, 32));
        const float w = m == kNegInf ? 0.0f : fast_exp2(m - M);
        l *= w;
#pragma unroll
        for (int d = 16; d; d >>= 1) l += __shfl_xor(l, d, 32);
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float* src = a.ws_o + rec * kHeadDim + 4 * lane;
        for (int i0 = 0; i0 < it.splits; i0 += 8) {
            float2 x[8][2];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float* p = src + min(i0 + u, it.splits - 1) * step * kHeadDim;
                x[u][0] = load_dev2(p);
                x[u][1] = load_dev2(p + 2);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                if (i0 + u < it.splits) {
                    const float wi = __shfl(w, i0 + u, 32);
                    // A range without a visible key has weight 0 and zeros;
                    // one with infinities keeps them.
                    acc.x = fmaf(x[u][0].x, wi, acc.x);
                    acc.y = fmaf(x[u][0].y, wi, acc.y);
                    acc.z = fmaf(x[u][1].x, wi, acc.z);
                    acc.w = fmaf(x[u][1].y, wi, acc.w);
                }
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        half4v o = {(f16)(acc.x * inv), (f16)(acc.y * inv), (f16)(acc.z * inv), (f16)(acc.w * inv)};
        *(half4v*)(a.out + ((int64_t)(it.row0 + r) * a.nkvh + it.kvh) * (kRep * kHeadDim) + h * kHeadDim +
                   4 * lane) = o;
    }
}

// After this range's records are stored: the last range of the row block to
// arrive merges them.  Called by every thread of the workgroup.
__device__ __forceinline__ void arrive(const PagedAttnArgs& a, const Item& it, int& s_last) {
    stores_done_barrier();
    uint32_t* ctr = a.counters + (int64_t)it.block * a.nkvh + it.kvh;
    if (threadIdx.x == 0) s_last = ticket_add(ctr) == (uint32_t)(it.splits - 1);
    __syncthreads();
    if (!s_last) return;
    merge_splits(a, it);
    if (threadIdx.x == 0) ticket_reset(ctr);
}

// Record (range, row, kv head, q head) of this item.
__device__ __forceinline__ int64_t record(const PagedAttnArgs& a, const Item& it, int r, int h) {
    return ((int64_t)(it.rec + it.split * it.rows + r) * a.nkvh + it.kvh) * kRep + h;
}

// 16 accumulator elements of column (r, h), dims db*32 + 8*q4 + 4*g + x:
// stored as outputs, or as the range's record.
__device__ __forceinline__ void put_block(const PagedAttnArgs& a, const Item& it, const float16v& o, float l, int db,
                                          int g, int r, int h) {
    if (it.splits == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        f16* dst = a.out + ((int64_t)(it.row0 + r) * a.nkvh + it.kvh) * (kRep * kHeadDim) + h * kHeadDim + db * 32;
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            half4v y;
#pragma unroll
            for (int x = 0; x < 4; ++x) y[x] = (f16)(o[4 * q4 + x] * inv);
            *(half4v*)(dst + 8 * q4 + 4 * g) = y;
        }
    } else {
        float* dst = a.ws_o + record(a, it, r, h) * kHeadDim + db * 32;
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            store_dev2(dst + 8 * q4 + 4 * g, o[4 * q4], o[4 * q4 + 1]);
            store_dev2(dst + 8 * q4 + 4 * g + 2, o[4 * q4 + 2], o[4 * q4 + 3]);
        }
    }
}

// NaN if some element is not finite.
__device__ __forceinline__ float not_finite(const float16v& o) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t = fmaf(o[i], 0.0f, t);
    return t;
}

// The item again, one (row, q head) column a wave at a time, in f32 and key by
// key: for items whose fast result is not finite.  The MFMA product weighs a
// hidden key with 0, and 0 * inf is NaN: here hidden keys are left out, so
// infinities and NaN reach only the rows that see them.
__device__ __forceinline__ void exact_item(const PagedAttnArgs& a, const Item& it, int key0, int key1) {
    const int tid = thread_id(), lane = tid & 63, wave = tid >> 6;
    for (int c = wave; c < it.rows * kRep; c += kThreads / 64) {
        const int r = c >> 1, h = c & 1, pos = it.pos0 + r;
        const int64_t col = ((int64_t)(it.row0 + r) * a.nkvh + it.kvh) * (kRep * kHeadDim) + h * kHeadDim;
        const f16* q = a.q + col;
        float m = kNegInf, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
        for (int k0 = key0; k0 < min(key1, pos + 1); k0 += 64) {
            const int key = k0 + lane;
            const int id = it.table[min(key, it.kend - 1) >> a.page_shift];
            const bool seen = key < key1 && key <= pos && (uint32_t)id < (uint32_t)a.pages;
            const f16* kp = a.base + (seen ? id : 0) * a.page_stride + it.kvh * a.head_stride +
                            (key & ((1 << a.page_shift) - 1)) * kHeadDim;
            float s = 0.0f;
            for (int d = 0; d < kHeadDim; d += 8) {
                H8 x, y;
                x.u = *(const uint4*)(kp + d);
                y.u = *(const uint4*)(q + d);
#pragma unroll
                for (int e = 0; e < 8; ++e) s = fmaf(h2f(x.e[e]), h2f(y.e[e]), s);
            }
            s = seen ? s * a.scale_log2 : kNegInf;
            float top = s;
#pragma unroll
            for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
            const float mn = fmaxf(m, top);
            const float mu = mn == kNegInf ? 0.0f : mn;
            const float alpha = m == kNegInf ? 0.0f : fast_exp2(m - mu);
            const float p = seen ? fast_exp2(s - mu) : 0.0f;
            m = mn;
            float ps = p;
#pragma unroll
            for (int d = 32; d; d >>= 1) ps += __shfl_xor(ps, d);
            l = l * alpha + ps;
            o0 *= alpha;
            o1 *= alpha;
            uint64_t todo = __ballot(seen);
            while (todo) {
                const int j = __builtin_ctzll(todo);
                todo &= todo - 1;
                const f16* vp = a.base + (int64_t)__shfl(id, j) * a.page_stride + it.kvh * a.head_stride +
                                a.kv_stride + ((k0 + j) & ((1 << a.page_shift) - 1)) * kHeadDim + 2 * lane;
                const float pj = __shfl(p, j);
                o0 = fmaf(pj, h2f(vp[0]), o0);
                o1 = fmaf(pj, h2f(vp[1]), o1);
            }
        }
        if (it.splits == 1) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            a.out[col + 2 * lane] = f2h(o0 * inv);
            a.out[col + 2 * lane + 1] = f2h(o1 * inv);
        } else {
            const int64_t rec = record(a, it, r, h);
            store_dev2(a.ws_o + rec * kHeadDim + 2 * lane, o0, o1);
            if (lane == 0) store_dev2(a.ws_ml + rec * 2, m, l);
        }
    }
}

// ---- the two kinds of item ------------------------------------------------

struct Shared {
    f16 buf[kBufHalves];
    float ml[4][2][64];
    int last;
};

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

#define WAIT_VM(n) asm volatile("s_waitcnt vmcnt(" #n ")" ::: "memory")

__device__ __forceinline__ void narrow_item(const PagedAttnArgs& a, const Item& it, Shared& sh) {
    const int tid = thread_id(), lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = n >> 4, rin = n & 15;
    f16* kbuf = sh.buf + wave * (2 * kSlice * kHeadDim);
    f16* vbuf = kbuf + kSlice * kHeadDim;

    // Lane l of a Pages: group l & 1 of this wave's slice of tile tp + l / 2.
    int tp = it.tile0;
    const int lane_key = (lane >> 1) * kNarrowTile + wave * kSlice + 16 * (lane & 1);
    Pages pg = load_pages(a, it, tp * kNarrowTile + lane_key);
    Pages next = load_pages(a, it, (tp + 32) * kNarrowTile + lane_key);
    Wave w;
    init_wave(w, a, it, rin, h, lane);
    const Offsets whole = group_offsets(lane);
    check_pages(a, pg);

    // Copies of group p (0, 1) of the slice of tile t: its K or its V.
    auto copy_group = [&](int t, int p, bool v) {
        const int key = t * kNarrowTile + wave * kSlice + 16 * p;
        const int id = __builtin_amdgcn_readlane(pg.id, 2 * (t - tp) + p);
        const int gkey = min(key, (it.kend - 1) & ~15);
        const f16* base = group_base(a, it.kvh, id, gkey) + (v ? a.kv_stride : 0);
        const uint32_t lds = v ? lds_addr(vbuf) + p * 1024 : lds_addr(kbuf) + p * 4096;
        if (key + 16 <= it.kend) {
            if (v)
                copy_v(base, whole, lds, kSlice * 64);
            else
                copy_k(base, whole, lds);
        } else if (v) {
            copy_v_tail(base, key - gkey, it.kend - 1 - gkey, lds, kSlice * 64);
        } else {
            copy_k_tail(base, key - gkey, it.kend - 1 - gkey, lds);
        }
    };
    auto copy_slice = [&](int t, bool v) {
        copy_group(t, 0, v);
        copy_group(t, 1, v);
    };
    const int last_pos = it.pos0 + it.rows - 1;  // == kend - 1
    if (it.tile0 < it.tile1) {
        copy_slice(it.tile0, false);
        copy_slice(it.tile0, true);
    }
    for (int t = it.tile0; t < it.tile1; ++t) {
        const int k0 = t * kNarrowTile + wave * kSlice;
        const bool more = t + 1 < it.tile1;
        const uint32_t bad = (uint32_t)(pg.bad >> (2 * (t - tp))) & 3;
        if (more && t + 1 - tp == 32) {
            tp += 32;
            pg = next;
            check_pages(a, pg);
            next = load_pages(a, it, (tp + 32) * kNarrowTile + lane_key);
        }
        if (k0 > last_pos) {  // only a wave's slice of the last tile: nothing to see
            WAIT_VM(0);
            break;
        }
        WAIT_VM(8);  // K landed, V in flight
        float16v s[1];
        half8v pb[2];
        step_scores<1>(w, kbuf, s);
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            copy_slice(t + 1, false);
        }
        if (k0 + kSlice - 1 <= it.pos0 && !bad)
            step_softmax<false, 1>(w, s, k0, 0u, pb);
        else
            step_softmax<true, 1>(w, s, k0, bad, pb);
        if (more)
            WAIT_VM(8);
        else
            WAIT_VM(0);
        step_pv<kSlice, 1>(w, vbuf, pb);
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            copy_slice(t + 1, true);
        }
    }

    // The four waves' states combine: wave w finishes dim block w, the other
    // blocks pass through each wave's own (now free) slice buffer.
    float* mine = reinterpret_cast<float*>(kbuf);
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) mine[db * 1024 + i * 64 + lane] = w.o[db][i];
    sh.ml[wave][0][lane] = w.m;
    sh.ml[wave][1][lane] = w.l;
    __syncthreads();
    float M = kNegInf, L = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) M = fmaxf(M, sh.ml[j][0][lane]);
    float16v o = (float16v){};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float mj = sh.ml[j][0][lane];
        const float aj = mj == kNegInf ? 0.0f : fast_exp2(mj - M);
        L = fmaf(sh.ml[j][1][lane], aj, L);
        const float* src = reinterpret_cast<const float*>(sh.buf) + j * 4096 + wave * 1024;
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = fmaf(src[i * 64 + lane], aj, o[i]);
    }
    const bool valid = rin < it.rows;
    const float t = not_finite(o);
    if (__syncthreads_or(valid && (t != t || L != L))) {
        exact_item(a, it, it.tile0 * kNarrowTile, min(it.tile1 * kNarrowTile, it.kend));
    } else if (valid) {
        put_block(a, it, o, L, wave, w.g, rin, h);
        if (it.splits > 1 && wave == 0 && w.g == 0) store_dev2(a.ws_ml + record(a, it, rin, h) * 2, M, L);
    }
    if (it.splits > 1) arrive(a, it, sh.last);
}

__device__ __forceinline__ void wide_item(const PagedAttnArgs& a, const Item& it, Shared& sh) {
    const int tid = thread_id(), lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = n >> 4, rin = wave * 16 + (n & 15);
    constexpr int kTile = kWideTile * kHeadDim;

    // Lane l of a Pages: group l & 3 of tile tp + l / 4.
    int tp = it.tile0;
    const int lane_key = lane * 16;
    Pages pg = load_pages(a, it, tp * kWideTile + lane_key);
    Pages next = load_pages(a, it, (tp + 16) * kWideTile + lane_key);
    Wave w;
    init_wave(w, a, it, rin, h, lane);
    const Offsets whole = group_offsets(lane);
    check_pages(a, pg);

    // This wave's 16 keys of tile t into buffer b: K 16 KB, V 4 slabs.
    auto copy_tile = [&](int t, int b) {
        const int key = t * kWideTile + wave * 16;
        const int id = __builtin_amdgcn_readlane(pg.id, 4 * (t - tp) + wave);
        const int gkey = min(key, (it.kend - 1) & ~15);
        const f16* base = group_base(a, it.kvh, id, gkey);
        const uint32_t kd = lds_addr(sh.buf + b * 2 * kTile) + wave * 4096;
        const uint32_t vd = lds_addr(sh.buf + b * 2 * kTile + kTile) + wave * 1024;
        if (key + 16 <= it.kend) {
            copy_k(base, whole, kd);
            copy_v(base + a.kv_stride, whole, vd, kWideTile * 64);
        } else {
            copy_k_tail(base, key - gkey, it.kend - 1 - gkey, kd);
            copy_v_tail(base + a.kv_stride, key - gkey, it.kend - 1 - gkey, vd, kWideTile * 64);
        }
    };
    const int first_pos = it.pos0 + wave * 16;
    const int last_pos = it.pos0 + min(wave * 16 + 15, it.rows - 1);
    const bool live = wave * 16 < it.rows;
    if (it.tile0 < it.tile1) copy_tile(it.tile0, 0);
    auto run = [&](int t, int b) {
        WAIT_VM(0);
        __syncthreads();  // tile t is here, and the other buffer is read
        const uint32_t bad = (uint32_t)(pg.bad >> (4 * (t - tp))) & 15;
        if (t + 1 < it.tile1) {
            if (t + 1 - tp == 16) {
                tp += 16;
                pg = next;
                check_pages(a, pg);
                next = load_pages(a, it, (tp + 16) * kWideTile + lane_key);
            }
            copy_tile(t + 1, b ^ 1);
        }
        const int k0 = t * kWideTile;
        if (!live || k0 > last_pos) return;
        const f16* kt = sh.buf + b * 2 * kTile;
        float16v s[2];
        half8v pb[4];
        step_scores<2>(w, kt, s);
        if (k0 + kWideTile - 1 <= first_pos && !bad)
            step_softmax<false, 2>(w, s, k0, 0u, pb);
        else
            step_softmax<true, 2>(w, s, k0, bad, pb);
        step_pv<kWideTile, 2>(w, kt + kTile, pb);
    };
    for (int t = it.tile0; t < it.tile1; t += 2) {
        run(t, 0);
        if (t + 1 < it.tile1) run(t + 1, 1);
    }
    const bool valid = rin < it.rows;
    float t = 0.0f;
#pragma unroll
    for (int db = 0; db < 4; ++db) t += not_finite(w.o[db]);
    if (__syncthreads_or(valid && (t != t || w.l != w.l))) {
        exact_item(a, it, it.tile0 * kWideTile, min(it.tile1 * kWideTile, it.kend));
    } else if (valid) {
#pragma unroll
        for (int db = 0; db < 4; ++db) put_block(a, it, w.o[db], w.l, db, w.g, rin, h);
        if (it.splits > 1 && w.g == 0) store_dev2(a.ws_ml + record(a, it, rin, h) * 2, w.m, w.l);
    }
    if (it.splits > 1) arrive(a, it, sh.last);
}

__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_attn_kernel(
    PagedAttnArgs a) {
    __shared__ __attribute__((aligned(1024))) Shared sh;
    const int items = a.n_items[0] * a.nkvh;
    for (int i = blockIdx.x; i < items; i += gridDim.x) {
        const PagedItem p = a.items[i / a.nkvh];
        Item it;
        it.kvh = i % a.nkvh;
        it.row0 = p.row0;
        it.rows = min(p.shape & 0xff, a.rows - p.row0);  // rows past the caller's q are left out
        it.pos0 = p.pos0;
        it.kend = p.pos0 + it.rows;
        it.tile0 = p.tile0;
        it.tile1 = p.tile1;
        it.splits = (p.shape >> 8) & 0xff;
        it.split = (p.shape >> 16) & 0xff;
        it.rec = p.rec;
        it.block = p.block;
        it.table = a.table + (int64_t)p.req * a.stride;
        if (it.rows <= 0) continue;
        if (p.shape >> 24)
            wide_item(a, it, sh);
        else
            narrow_item(a, it, sh);
        __syncthreads();  // the next item reuses the LDS
    }
}

}  // namespace

hipError_t launch_paged_attn(const PagedAttnArgs& a, int64_t max_items, int cus, hipStream_t stream) {
    if (a.rows <= 0) return hipSuccess;
    const int64_t wgs = std::min<int64_t>(max_items * a.nkvh, 2 * (int64_t)cus);
    hipLaunchKernelGGL(paged_attn_kernel, dim3((unsigned)wgs), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace qasr
