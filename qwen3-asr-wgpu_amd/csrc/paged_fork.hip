// paged_fork.hip -- the requests of a step go on as their parents do: what
// beams need after a selection, and whoever samples one prompt several times.
//
// Request i takes its parent's length and pages.  A full page is held by as many
// requests as go on from its holder, one more or fewer in `shared` for each; a
// page that none holds any more goes back to the ring.  An unfinished last page
// will be written: one of those that go on from its holder (itself, else the
// first) keeps it, if no request outside holds it too, the others get copies of
// its rows on fresh pages.
//
// Two launches.  The first, a workgroup with a request a thread, finds who goes
// on from whom, ranks the copies (their fresh pages are the ring's next ones, in
// request order) and decides whether the call is carried out at all.  In the
// second, one part of the workgroups copies rows of K and V of all layers, 16
// bytes a thread, the other part rewrites the table, 2 columns each: a page
// lies at the same place in all tables that list it, so a workgroup meets every
// holder that the call has of its pages, and rows of the table can be replaced
// by others of the same columns in place.  Counts change by atomics, whose
// order leaves no trace: exactly the last holder finds the count below zero, and
// the pages given back are put in the order of their columns, then of the first
// request that listed them, before the last workgroup to arrive moves them to
// the ring.
//
// What bounds it, us a call: two launches, the second behind the first, and in each
// dependent trips to memory (row and table; count, ticket, pages given back, ring).
// 1 x 5 beams of 523 rows on pages of 16 (28 layers): 3.7 and 7.2 in a profile,
// 9.4-10.1 a call in a replayed graph, 10.7-11.2 eagerly, where the host takes as
// long.  16 x 5 of 400-1500 rows 12.2-12.8 either way (18 MB read and written).  16
// columns a workgroup, each request's facts read again at each use: 24.9; 4 columns
// 15.9.  Where copies are large they are all: 851 MB in 172-175, 4.9 TB/s (a large copy
// reaches 5.1).
#include "paged_fork.hpp"

namespace qasr {

namespace {

constexpr int kThreads = 256;
enum : int32_t { kOk = 0, kInvalid = 1, kNoPage = 3 };  // QASR_OK, _EINVAL, _ENOMEM

__device__ __forceinline__ int wrap(int x, int pages) { return x >= pages ? x - pages : x; }

// One workgroup, a request a thread.
__global__ __launch_bounds__(kPagedMaxRequests) void fork_rows_kernel(ForkArgs a) {
    __shared__ int s_len[kPagedMaxRequests], s_last[kPagedMaxRequests];  // unfinished page: its id, -1: none
    __shared__ int s_sons[kPagedMaxRequests], s_heir[kPagedMaxRequests];
    __shared__ int s_wave[kPagedMaxRequests / 64];
    __shared__ uint8_t s_alone[kPagedMaxRequests];

    const int i = threadIdx.x, lane = i & 63, ps = 1 << a.page_shift;
    const bool mine = i < a.nreq;
    int parent = -1, len = 0, head = 0, free = 0;
    if (mine) {
        parent = a.parent[i];
        len = a.len[i];
    }
    head = a.cursor[0];
    free = a.cursor[1];
    // A cursor that is none: no page is free, and pages given back have no place,
    // so a call that wants no copy is refused too.
    const bool lost = head < 0 || head >= a.pages || free < 0 || free > a.pages;
    if (lost) head = free = 0;
    const bool bad = mine && (parent < -1 || parent >= a.nreq || len < 0 ||
                              ((int64_t)len + ps - 1) >> a.page_shift > a.stride);
    const bool refused = __syncthreads_or(bad);
    if (refused) {  // nothing is done
        if (mine) a.status[i] = bad ? kInvalid : kOk;
        if (i == 0) a.w->ok = 0;
        return;
    }
    const int whole = len >> a.page_shift, rest = len & (ps - 1);
    s_sons[i] = 0;
    s_heir[i] = kPagedMaxRequests;
    int last = mine && rest ? a.table[(int64_t)i * a.stride + whole] : -1;
    last = (uint32_t)last < (uint32_t)a.pages ? last : -1;
    s_len[i] = len;
    s_last[i] = last;
    const bool alone = last >= 0 && a.shared[last] <= 0;
    s_alone[i] = alone;
    __syncthreads();
    if (parent >= 0) {
        atomicAdd(&s_sons[parent], 1);
        atomicMin(&s_heir[parent], parent == i ? -1 : i);
    }
    __syncthreads();
    bool copy = false;
    if (parent >= 0 && s_last[parent] >= 0) {
        const int heir = s_heir[parent] < 0 ? parent : s_heir[parent];
        copy = !(heir == i && s_alone[parent]);
    }
    // Copies of the requests before this one.
    const uint64_t votes = __ballot(copy);
    if (lane == 0) s_wave[i >> 6] = __popcll(votes);
    __syncthreads();
    int rank = __popcll(votes & ((1ull << lane) - 1)), copies = 0;
    for (int w = 0; w < (int)blockDim.x / 64; ++w) {
        rank += w < i >> 6 ? s_wave[w] : 0;
        copies += s_wave[w];
    }
    const bool ok = copies <= free && !lost;
    if (mine) {
        a.status[i] = ok ? kOk : copies == 0 ? kInvalid : copy ? kNoPage : kOk;
        ForkRow r;
        r.parent = parent;
        r.used = whole + (rest != 0);  // (len + ps - 1 passes 2^31 for the longest)
        r.whole = whole;
        r.more = s_sons[i] - 1;
        r.more_last = (s_sons[i] > 0 && alone ? 1 : 0) - 1;
        r.copy = copy;
        r.fresh = copy && ok ? a.ring[wrap(head + rank, a.pages)] : -1;
        r.unused = 0;
        a.rows[i] = r;
        if (copy && ok) {
            const bool there = (uint32_t)r.fresh < (uint32_t)a.pages;
            a.copies[rank] = {s_last[parent], there ? r.fresh : 0, there ? s_len[parent] & (ps - 1) : 0, 0};
        }
        if (ok) a.len[i] = parent >= 0 ? s_len[parent] : 0;  // (every length was read)
    }
    if (i == 0) {
        a.w->ok = ok;
        a.w->copies = copies;
        a.w->head = head;
        a.w->free = free;
    }
}

// Rows of K and V, 16 bytes a thread: unit (copy, part of 1024 of them).  Past the
// caches, as nothing here reads them again: 16 x 5 beams on f16 pages of 256 rows
// (851 MB read and written) 283 -> 175 us, on e4m3 pages of 64 (88 MB) 36 -> 25.
constexpr int kCopyVectors = 1024;
typedef unsigned int Vector __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void copy_pages(const ForkArgs& a, int first, int step, int parts) {
    const int units = a.w->copies * parts;
    for (int u = first; u < units; u += step) {
        const int c = u / parts, part = u - c * parts;
        const ForkCopy p = a.copies[c];
        const int n = p.rows * (a.row_bytes / 16);  // vectors of a head
        const int64_t head_bytes = (int64_t)a.row_bytes << a.page_shift;
        const int all = n * a.heads * a.layers;
        Vector x[kCopyVectors / kThreads];
        int64_t to[kCopyVectors / kThreads];
#pragma unroll
        for (int k = 0; k < kCopyVectors / kThreads; ++k) {
            const int v = part * kCopyVectors + k * kThreads + (int)threadIdx.x;
            to[k] = -1;
            if (v < all) {
                const int h = v / n, at = v - h * n, layer = h / a.heads, head = h - layer * a.heads;
                const int64_t in = layer * a.layer_bytes + head * head_bytes + at * 16ll;
                x[k] = __builtin_nontemporal_load((const Vector*)(a.base + in + p.from * a.page_bytes));
                to[k] = in + p.to * a.page_bytes;
            }
        }
#pragma unroll
        for (int k = 0; k < kCopyVectors / kThreads; ++k)
            if (to[k] >= 0) __builtin_nontemporal_store(x[k], (Vector*)(a.base + to[k]));
        if (part == 0 && a.scales && p.rows) {  // units of the copied rows' blocks
            const int blocks = (1 << a.page_shift) / kPagedScaleRows, held = (p.rows + kPagedScaleRows - 1) / kPagedScaleRows;
            for (int s = threadIdx.x; s < a.layers * a.page_scales; s += kThreads) {
                const int layer = s / a.page_scales, at = s - layer * a.page_scales;
                if (at % blocks < held) {
                    uint8_t* q = a.scales + layer * a.layer_scales + at;
                    q[p.to * (int64_t)a.page_scales] = q[p.from * (int64_t)a.page_scales];
                }
            }
        }
    }
}

// kForkColumns columns of the table.
__device__ __forceinline__ void rewrite_columns(const ForkArgs& a, int block, int blocks, int* s_page) {
    // s_page, s_more: [nreq][kForkColumns] pages listed now, -1: none that counts,
    // and how many holders more (or, below zero, one less) they get.
    constexpr int C = kForkColumns, kWords = kPagedMaxRequests / 32;
    __shared__ uint32_t s_gone[C][kWords];  // requests whose page of the column nobody holds any more
    __shared__ uint32_t s_many[C][kWords];  // whose page's count changes
    __shared__ int s_first[C + 1];
    __shared__ int s_upto[kThreads], s_wave[kThreads / 64];
    __shared__ int s_arrived;
    const int tid = threadIdx.x, n = a.nreq * C, k0 = block * C, words = (a.nreq + 31) / 32;
    int* s_more = s_page + n;
    for (int x = tid; x < C * kWords; x += kThreads) s_gone[x / kWords][x % kWords] = s_many[x / kWords][x % kWords] = 0;
    const int ok = a.w->ok;
    for (int x = tid; x < n; x += kThreads) {
        const int j = x / C, k = k0 + x % C;
        const ForkRow r = a.rows[j];  // (of an earlier call if this one is not carried out)
        int page = a.table[(int64_t)j * a.stride + min(k, a.stride - 1)];
        page = k < r.used ? page : -1;
        s_page[x] = page;
        s_more[x] = (uint32_t)page >= (uint32_t)a.pages ? 0 : k < r.whole ? r.more : r.more_last;
    }
    if (!ok) return;
    __syncthreads();
    // Holders.  Whose page has no other loses its last one; counts of pages with
    // several, and of those that get more, change behind the barrier.
    auto set = [&](uint32_t (*bits)[kWords], int j, int c) { atomicOr(&bits[c][j >> 5], 1u << (j & 31)); };
    for (int x = tid; x < n; x += kThreads) {
        const int more = s_more[x];
        if (more < 0 && a.shared[s_page[x]] <= 0)
            set(s_gone, x / C, x % C);
        else if (more)
            set(s_many, x / C, x % C);
    }
    __syncthreads();
    for (int x = tid; x < n; x += kThreads) {
        if (!(s_many[x % C][x / C >> 5] >> (x / C & 31) & 1)) continue;
        const int more = s_more[x];
        int* count = a.shared + s_page[x];
        const int was = __hip_atomic_fetch_add(count, more, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (more < 0 && was == 0) {  // the last holder
            __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            int j = x % C;  // the first request that lists it
            while (j < x && s_page[j] != s_page[x]) j += C;
            set(s_gone, j / C, x % C);
        }
    }
    __syncthreads();
    // Their pages by column, then by request.
    if (tid < C) {
        int sum = 0;
        for (int w = 0; w < words; ++w) sum += __popc(s_gone[tid][w]);
        s_first[tid + 1] = sum;
    }
    __syncthreads();
    if (tid == 0) {
        s_first[0] = 0;
        for (int c = 0; c < C; ++c) s_first[c + 1] += s_first[c];
    }
    __syncthreads();
    int* gone = a.gone + (int64_t)block * a.nreq * C;
    for (int x = tid; x < n; x += kThreads) {
        const int j = x / C, c = x % C;
        if (!(s_gone[c][j >> 5] >> (j & 31) & 1)) continue;
        int at = s_first[c] + __popc(s_gone[c][j >> 5] & ((1u << (j & 31)) - 1));
        for (int w = 0; w < j >> 5; ++w) at += __popc(s_gone[c][w]);
        __hip_atomic_store(gone + at, s_page[x], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (tid == 0)
        __hip_atomic_store(a.n_gone + block, s_first[C], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // New rows of the table.
    for (int x = tid; x < n; x += kThreads) {
        const ForkRow r = a.rows[x / C];
        if (r.parent < 0 || (r.parent == x / C && !r.copy)) continue;
        const ForkRow& p = a.rows[r.parent];
        const int k = k0 + x % C;
        if (k >= p.used) continue;
        a.table[(int64_t)(x / C) * a.stride + k] = r.copy && k == p.whole ? r.fresh : s_page[r.parent * C + x % C];
    }
    // The last workgroup moves all that is gone to the ring's end.
    stores_done_barrier();
    if (tid == 0) s_arrived = ticket_add(&a.w->arrived) == (uint32_t)(blocks - 1);
    __syncthreads();
    if (!s_arrived) return;
    const int head = a.w->head, free = a.w->free, copies = a.w->copies;
    int pushed = 0;
    for (int b0 = 0; b0 < blocks; b0 += kThreads) {  // (one turn for tables of up to 1024 pages)
        const int m = b0 + tid < blocks ? __hip_atomic_load(a.n_gone + b0 + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
        // How many the blocks up to each have, then a page a thread: its block is
        // the first that has more up to it than come before the page.
        int upto = m;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int y = __shfl_up(upto, d);
            upto += (tid & 63) >= d ? y : 0;
        }
        __syncthreads();
        if ((tid & 63) == 63) s_wave[tid >> 6] = upto;
        __syncthreads();
        for (int w = 0; w < tid >> 6; ++w) upto += s_wave[w];
        s_upto[tid] = upto;
        __syncthreads();
        const int all = s_upto[kThreads - 1];
        for (int x = tid; x < all && free + pushed + x < a.pages; x += kThreads) {  // (a page given back twice)
            int b = 0;
#pragma unroll
            for (int d = kThreads / 2; d; d /= 2) b += s_upto[b + d - 1] <= x ? d : 0;
            const int at = x - (b ? s_upto[b - 1] : 0);
            a.ring[wrap(head + free + pushed + x, a.pages)] = __hip_atomic_load(
                a.gone + (int64_t)(b0 + b) * a.nreq * C + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        pushed = min(pushed + all, a.pages);  // (that many are not stored any more; a sum of all passes 2^31 some time)
    }
    if (tid == 0) {
        a.cursor[0] = wrap(head + copies, a.pages);
        a.cursor[1] = min(free + pushed, a.pages) - copies;
        ticket_reset(&a.w->arrived);
    }
}

__global__ __launch_bounds__(kThreads) void fork_pages_kernel(ForkArgs a, int blocks, int parts) {
    extern __shared__ int s_page[];
    if ((int)blockIdx.x < blocks)
        rewrite_columns(a, blockIdx.x, blocks, s_page);
    else if (a.w->ok)
        copy_pages(a, blockIdx.x - blocks, gridDim.x - blocks, parts);
}

}  // namespace

hipError_t launch_paged_fork(const ForkArgs& a, int cus, hipStream_t stream) {
    if (a.nreq < 1 || a.nreq > kPagedMaxRequests || a.stride < 1) return hipErrorInvalidValue;
    hipLaunchKernelGGL(fork_rows_kernel, dim3(1), dim3((a.nreq + 63) / 64 * 64), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int blocks = (a.stride + kForkColumns - 1) / kForkColumns;
    const int64_t most = (int64_t)((1 << a.page_shift) - 1) * (a.row_bytes / 16) * a.heads * a.layers;  // vectors of a copy
    const int parts = (int)((most + kCopyVectors - 1) / kCopyVectors);
    const int64_t units = (int64_t)parts * a.nreq;
    const int64_t copiers = units < 8 * cus ? units : 8 * cus;
    hipLaunchKernelGGL(fork_pages_kernel, dim3((unsigned)(blocks + copiers)), dim3(kThreads),
                       (size_t)a.nreq * kForkColumns * 8, stream, a, blocks, parts);
    return hipGetLastError();
}

}  // namespace qasr
