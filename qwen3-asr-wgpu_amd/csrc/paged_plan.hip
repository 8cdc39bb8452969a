// paged_plan.hip -- one step of a paged KV cache, planned on the GPU from the
// requests' lengths: block tables, row maps and the attention work list.
//
// With new_i = max(rows_i, 0), P rows a page and need_i = ceil((len_i +
// new_i) / P) - ceil(len_i / P), everything is a prefix sum over requests:
// row_start = sum new, the first free page of request i = sum need (taken
// from the ring in request order, so the tables do not depend on timing),
// the first work item = sum blocks * splits.  A request is refused when its
// inclusive sum of needs passes the free count; the sums only grow, so the
// placed requests take one contiguous run of the ring.
//
// Nothing here is bandwidth: a step moves some tens of KB and costs a chain
// of memory round trips (lengths, the table entry of a torn page, ring
// entries) and barriers.  One launch therefore does it all: every workgroup
// repeats the scans of all requests (one request a thread) and then expands
// its share of rows, fresh pages and work items, finding each one's request
// by a binary search of the prefix sums in LDS.  What may alias an input
// (lengths and the cursor, updated in place by a replayed graph) is written
// by the workgroup that arrives last, when every other has read it.
// us a launch: 16 single rows 7.3, 256 requests of 220 single rows and 20 chunks,
// 16 of them ended, 15.8-17; with three scans and items by the row blocks'
// workgroups 43.  A given table is checked by each request's own thread, entry
// by entry: 2048 new rows of one request on pages of 256 rows 6.1, of 16 14.2.
// Pages go back in the last workgroup alone, a workgroup's threads of them at a
// time.

#include "paged.hpp"

namespace qasr {

namespace {

constexpr int kFew = 256;  // requests up to which a workgroup is 4 waves, not 16

enum : int32_t { kOk = 0, kInvalid = 1, kRange = 2, kNoPage = 3 };  // QASR_OK, _EINVAL, _ERANGE, _ENOMEM

// Six sums below 2^31.
struct Sums {
    uint64_t v[3];
};
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) { return (uint64_t)hi << 32 | lo; }
__device__ __forceinline__ int lo32(uint64_t x) { return (int)(uint32_t)x; }
__device__ __forceinline__ int hi32(uint64_t x) { return (int)(x >> 32); }

// Exclusive prefix sums over the workgroup's threads, and the totals.
template <int THREADS, int N>
__device__ __forceinline__ void block_scan(uint64_t (&v)[N], uint64_t (&total)[N], uint64_t (*s_wave)[THREADS / 64]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t own[N];
#pragma unroll
    for (int i = 0; i < N; ++i) own[i] = v[i];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint64_t up = __shfl_up(v[i], d);
            if (lane >= d) v[i] += up;
        }
    if (lane == 63)
#pragma unroll
        for (int i = 0; i < N; ++i) s_wave[i][wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        uint64_t before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) {
            const uint64_t x = s_wave[i][w];
            before += w < wave ? x : 0;
            all += x;
        }
        v[i] += before - own[i];
        total[i] = all;
    }
    __syncthreads();
}

// The last request whose prefix sum is at most x (s[0] = 0 <= x).
template <int THREADS>
__device__ __forceinline__ int find(const int* s, int n, int x) {
    int i = 0;
#pragma unroll
    for (int d = THREADS / 2; d; d >>= 1)
        if (i + d < n && s[i + d] <= x) i += d;
    return i;
}

template <int kThreads>
__global__ __launch_bounds__(kThreads) void paged_plan_kernel(PagedPlanArgs a) {
    __shared__ uint64_t s_wave[3][kThreads / 64];
    __shared__ int s_row[kThreads], s_len[kThreads], s_new[kThreads], s_page[kThreads];
    __shared__ int s_narrow[kThreads], s_wide[kThreads], s_rec[kThreads], s_block[kThreads], s_gone[kThreads];
    __shared__ int s_last;

    const int tid = threadIdx.x, ps = 1 << a.page_shift, sh = a.page_shift;
    const bool mine = tid < a.nreq;
    int len = 0, rows = 0, head = 0, free = 0;
    if (mine) {
        len = a.len[tid];
        rows = a.rows[tid];
    }
    if (a.ring) {
        head = a.cursor[0];
        free = a.cursor[1];
        if (head < 0 || head >= a.pages || free < 0 || free > a.pages) head = free = 0;
    }
    int* trow = a.table + (int64_t)(mine ? tid : 0) * a.stride;

    // What a request asks for, and the sums of rows and fresh pages.
    // Saturated, so that no sum of 1024 requests passes 2^31.
    const int want = mine ? min(max(rows, 0), a.max_rows + 1) : 0;
    int status = kOk;
    if (mine && (len < 0 || len > a.max_seq || rows < -1)) status = kInvalid;
    const int held = status ? 0 : (len + ps - 1) >> sh;
    const int full = status ? 0 : (len + want + ps - 1) >> sh;
    if (!status && mine && rows != 0)
        if (len + want > a.max_seq || max(held, full) > a.stride) status = kRange;
    if (!status && rows > 0) {
        // The page that the first new row shares with cached ones, and
        // without a ring every page of the new rows, must be in the pool.
        const int j1 = a.ring ? held : full;
        for (int j = len >> sh; j < j1; ++j)
            if ((uint32_t)trow[j] >= (uint32_t)a.pages) status = kInvalid;
    }
    // (Once the rows pass max_rows they do for every later request, so whose
    // pages those count makes no difference.)
    const int need = !status && rows > 0 && a.ring ? full - held : 0;
    uint64_t v1[1] = {pack2(want, need)}, t1[1];
    block_scan<kThreads, 1>(v1, t1, s_wave);
    const int row0 = lo32(v1[0]), nrows = lo32(t1[0]), page0 = hi32(v1[0]);
    if (!status && rows > 0 && row0 + want > a.max_rows) status = kRange;
    if (!status && need > 0 && page0 + need > free) status = kNoPage;
    const bool placed = mine && !status && rows > 0;
    const bool gone = mine && !status && rows == -1;

    PagedShape shape{0, 0, 0};
    if (placed) shape = paged_shape(len, want);
    const int my_items = shape.blocks * shape.splits;
    Sums v{{pack2(shape.wide ? 0 : my_items, shape.wide ? my_items : 0),
            pack2(shape.splits > 1 ? want * shape.splits : 0, shape.blocks), pack2(gone ? held : 0, placed ? need : 0)}};
    Sums t;
    block_scan<kThreads, 3>(v.v, t.v, s_wave);
    s_row[tid] = row0;
    s_len[tid] = len;
    s_new[tid] = placed ? want : 0;
    s_page[tid] = page0;
    s_narrow[tid] = lo32(v.v[0]);
    s_wide[tid] = hi32(v.v[0]);
    s_rec[tid] = lo32(v.v[1]);
    s_block[tid] = hi32(v.v[1]);
    s_gone[tid] = lo32(v.v[2]);
    const int narrow = lo32(t.v[0]), wide = hi32(t.v[0]), back = lo32(t.v[2]), taken = hi32(t.v[2]);
    if (blockIdx.x == 0) {
        if (mine) {
            a.status[tid] = status;
            a.row_start[tid] = row0;
        }
        if (tid == 0) {
            a.row_start[a.nreq] = nrows;
            a.n_items[0] = narrow;
            a.n_items[1] = wide;
        }
    }
    // Every load of what may alias an output has returned (the sums need
    // them); the last workgroup to come here writes those outputs at the end.
    uint32_t came = 0;
    if (tid == 0 && gridDim.x > 1) came = ticket_add(a.arrived);
    __syncthreads();

    const int n = a.nreq, step = gridDim.x * kThreads, first = blockIdx.x * kThreads + tid;
    // Page at place j of request i's table: the table's, or a fresh one.
    auto page_at = [&](int i, int j) {
        const int had = (s_len[i] + ps - 1) >> sh;
        if (j < had || !a.ring) return a.table[(int64_t)i * a.stride + j];
        int k = head + s_page[i] + j - had;  // < 2 pages: at most `free` taken
        k -= k >= a.pages ? a.pages : 0;
        return a.ring[k];
    };
    // Row maps.
    for (int r = first; r < a.max_rows; r += step) {
        int pos = -1, slot = -1;
        if (r < nrows) {
            const int i = find<kThreads>(s_row, n, r), at = r - s_row[i];
            if (at < s_new[i]) {
                pos = s_len[i] + at;
                const int page = page_at(i, pos >> sh);
                slot = (uint32_t)page < (uint32_t)a.pages ? (page << sh) + (pos & (ps - 1)) : -1;
            }
        }
        a.row_pos[r] = pos;
        a.row_slot[r] = slot;
    }
    // Fresh table entries.
    for (int k = first; k < taken; k += step) {
        const int i = find<kThreads>(s_page, n, k);
        int w = head + k;
        w -= w >= a.pages ? a.pages : 0;
        a.table[(int64_t)i * a.stride + ((s_len[i] + ps - 1) >> sh) + k - s_page[i]] = a.ring[w];
    }
    // Work items, a wave each, a word a lane.
    const int lane = tid & 63;
    for (int k = first >> 6; k < narrow + wide; k += step >> 6) {
        const int k0 = k < narrow ? 0 : narrow;
        const int* sums = k < narrow ? s_narrow : s_wide;
        PagedItem* out = (k < narrow ? a.narrow : a.wide) + k - k0;
        const int i = find<kThreads>(sums, n, k - k0), l = s_len[i], m = s_new[i];
        const PagedShape p = paged_shape(l, m);
        const int e = k - k0 - sums[i], split = e % p.splits, b = p.blocks - 1 - e / p.splits;  // the longest first
        const int rb = p.wide ? kWideRows : kNarrowRows, tile = p.wide ? kWideTile : kNarrowTile;
        const int br = min(rb, m - b * rb), end = l + b * rb + br;
        const int tiles = (end + tile - 1) / tile;
        const int tile0 = (int)((int64_t)tiles * split / p.splits), tile1 = (int)((int64_t)tiles * (split + 1) / p.splits);
        const int page0 = tile0 * tile >> sh;
        int word = 0;
        switch (lane) {
            case 0: word = i; break;
            case 1: word = s_row[i] + b * rb; break;
            case 2: word = l + b * rb; break;
            case 3: word = br | p.splits << 8 | split << 16; break;
            case 4: word = tile0; break;
            case 5: word = tile1; break;
            case 6: word = s_rec[i] + b * rb * p.splits; break;
            case 7: word = s_block[i] + b; break;
            case 8: word = page0; break;
            default:
                if (lane >= kPagedItemHead) word = page_at(i, min(page0 + lane - kPagedItemHead, (end - 1) >> sh));
        }
        reinterpret_cast<int*>(out)[lane] = word;
    }
    if (tid == 0) {
        s_last = came == gridDim.x - 1;
        if (s_last && gridDim.x > 1) ticket_reset(a.arrived);
    }
    __syncthreads();
    if (!s_last) return;
    if (mine) a.lens_out[tid] = gone ? 0 : placed ? len + want : len;
    if (!a.ring) return;
    // Pages of ended requests to the end of the ring, in request and table
    // order, entries outside the pool left out.
    int pushed = 0;
    for (int k0 = 0; k0 < back; k0 += kThreads) {
        const int k = k0 + tid;
        int page = -1;
        if (k < back) {
            const int i = find<kThreads>(s_gone, n, k);
            page = a.table[(int64_t)i * a.stride + k - s_gone[i]];
        }
        const bool ok = (uint32_t)page < (uint32_t)a.pages;
        uint64_t v3[1] = {ok ? 1u : 0u}, t3[1];
        block_scan<kThreads, 1>(v3, t3, s_wave);
        const int at = pushed + lo32(v3[0]);
        if (ok && free + at < a.pages) {  // more than the pool holds: a page given back twice
            int w = head + free + at;
            w -= w >= a.pages ? a.pages : 0;
            a.ring[w] = page;
        }
        pushed += lo32(t3[0]);
    }
    if (tid == 0) {
        int h = head + taken;
        h -= h >= a.pages ? a.pages : 0;
        a.cursor_out[0] = h;
        a.cursor_out[1] = min(free + pushed, a.pages) - taken;
    }
}

}  // namespace

hipError_t launch_paged_plan(const PagedPlanArgs& a, hipStream_t stream) {
    if (a.nreq < 1 || a.nreq > kPagedMaxRequests || a.max_rows < 1) return hipErrorInvalidValue;
    // A workgroup for every THREADS rows and for the work items of every few
    // requests.  us a launch with 4 waves a workgroup, against 16 waves: 16 single
    // rows 7.3 to 8.0, 256 mixed requests 15.7 to 18.
    if (a.nreq <= kFew) {
        const int wgs = a.max_rows / kFew + (a.nreq + 1) / 2;
        hipLaunchKernelGGL(paged_plan_kernel<kFew>, dim3(wgs < 128 ? wgs : 128), dim3(kFew), 0, stream, a);
    } else {
        const int wgs = a.max_rows / kPagedMaxRequests + (a.nreq + 7) / 8;
        hipLaunchKernelGGL(paged_plan_kernel<kPagedMaxRequests>, dim3(wgs < 128 ? wgs : 128),
                           dim3(kPagedMaxRequests), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace qasr
