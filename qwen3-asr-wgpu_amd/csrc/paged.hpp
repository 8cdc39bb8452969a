// paged.hpp -- the paged KV cache's structs and launchers, shared by its C ABI
// (paged_abi.hip) and kernels (paged_plan.hip, paged_attn.hip, norm_rope.hip).
//
// A pool is pages of 2^page_shift rows; element (layer, page, kv, head, row,
// d) is at base + layer*layer_stride + page*page_stride + kv*kv_stride +
// head*head_stride + row*kHeadDim + d, so a (page, K or V, head) is one
// contiguous block.  A request's position p lives in row p % rows of page
// table[p / rows].
#pragma once

#include "kernels.hpp"

namespace qasr {

constexpr int kPagedMaxRequests = 1024;  // one thread of the plan kernel each
constexpr int kPagedMinShift = 4;        // pages of 16 rows: one copy instruction stays in a page
constexpr int kPagedMaxShift = 8;

// Attention work items.  A request's new rows are cut into row blocks of
// kNarrowRows rows (whose waves share the keys) or kWideRows rows (whose waves
// share the rows too), a row block's key tiles into `splits` ranges of equal
// length.  Both follow from the request's own rows and length (paged_shape), so
// a request's bits do not depend on its batch mates.
constexpr int kNarrowRows = 16, kNarrowTile = 128;
constexpr int kWideRows = 64, kWideTile = 128;
constexpr int kPagedMaxSplits = 32;     // row blocks x splits of a split request
constexpr int kPagedRangeKeys = 512;
constexpr int64_t kWideWork = 5 << 18;  // rows x mean keys from which on row blocks are wide

struct PagedShape {
    int32_t wide;    // row blocks of kWideRows rows
    int32_t blocks;  // row blocks
    int32_t splits;  // key ranges of each
};

// Wide row blocks read each key once for 64 rows, narrow ones for 16, but
// narrow ones are four times as many, start sooner and combine for less: us a
// layer, narrow against wide, 128 rows at 4000 22.4 / 30.6, 1000 at 0 18 / 23.5,
// 256 at 4000 29 / 32, 512 at 2000 28.8 / 28.1, 2048 at 0 43 / 38.6, 1024 at
// 4000 65 / 55.5, 512 at 7680 74 / 51.  Ranges: one row at 1024, 2048, 8192 keys
// 9.2, 9.6, 17.2 in ranges of 256 keys, 10.9, 11.3, 15.9 of 512, 12.9, 15.5, 19.4
// of 1024; 16 rows at 2000 keys each 32.9, 29.6, 29.5.
__host__ __device__ inline PagedShape paged_shape(int len, int rows) {
    PagedShape s;
    s.wide = (int64_t)rows * (len + rows / 2) >= kWideWork;
    const int rb = s.wide ? kWideRows : kNarrowRows;
    s.blocks = (rows + rb - 1) / rb;
    const int first = len + (rows < rb ? rows : rb);  // keys of the first row block
    const int most = s.blocks < kPagedMaxSplits ? kPagedMaxSplits / s.blocks : 1;
    const int want = (first + kPagedRangeKeys - 1) / kPagedRangeKeys;
    s.splits = want < most ? want : most;
    return s;
}
// Whether a step of up to `rows` rows and tables of `keys` keys can have wide
// row blocks.
inline bool paged_wide(int64_t rows, int64_t keys) {
    const int64_t m = rows < keys ? rows : keys;
    return m * (keys - m / 2) >= kWideWork;
}

constexpr int kPagedItemHead = 16, kPagedItemPages = 48;
struct PagedItem {  // one row block and key range, for every kv head: 64 words, one a lane
    int32_t req;
    int32_t row0;   // first row, in the step's rows
    int32_t pos0;   // its position
    int32_t shape;  // rows | splits << 8 | split << 16
    int32_t tile0, tile1;  // key tiles (kNarrowTile or kWideTile keys)
    int32_t rec;    // split state: records of the row blocks before it
    int32_t block;  // arrival counter of the row block
    int32_t page0;  // place in the table of the range's first page
    int32_t unused[kPagedItemHead - 9];
    int32_t page[kPagedItemPages];  // ids from page0 on, as far as the row block's keys reach
};
static_assert(sizeof(PagedItem) == 64 * 4, "a word a lane");

// Capacities for max_requests requests and max_rows rows together.  A
// request has at most max(kPagedMaxSplits, blocks) items and, split, rows *
// splits records: at most kPagedMaxSplits a row and kPagedMaxSplits *
// kWideRows in all.
inline int64_t paged_max_blocks(int64_t requests, int64_t rows) { return requests + rows / kNarrowRows; }
inline int64_t paged_max_items(int64_t requests, int64_t rows, int64_t rows_a_block) {
    return requests * kPagedMaxSplits + requests + rows / rows_a_block;
}
inline int64_t paged_max_records(int64_t requests, int64_t rows) {
    const int64_t a = rows * kPagedMaxSplits, b = requests * kPagedMaxSplits * kWideRows;
    return a < b ? a : b;
}

// The plan kernel's arguments (device pointers unless said otherwise).
struct PagedPlanArgs {
    const int32_t* len;   // [nreq]
    const int32_t* rows;  // [nreq]
    int32_t* table;       // [nreq][stride]
    int32_t* ring;        // [pages], or NULL: the table holds every page already
    const int32_t* cursor;
    int32_t nreq, stride, pages, page_shift, max_seq, max_rows;
    int32_t* status;      // [nreq]
    int32_t* lens_out;    // [nreq]
    int32_t* row_start;   // [nreq + 1]
    int32_t* row_pos;     // [max_rows]
    int32_t* row_slot;    // [max_rows]
    int32_t* cursor_out;  // [2]
    int32_t* n_items;     // [2]: narrow, wide
    PagedItem *narrow, *wide;
    uint32_t* arrived;    // workgroup ticket, zero at rest
};
hipError_t launch_paged_plan(const PagedPlanArgs& a, hipStream_t stream);

// Stage (a) into pages: row r goes to row slot[r] % rows of page slot[r] /
// rows at position pos[r].
struct RowMap {
    const int32_t* pos;
    const int32_t* slot;
    int32_t slots;  // pages * rows of a page
    int32_t page_shift;
    int32_t rope_rows;
    int32_t nqh;
    float eps;
};
hipError_t launch_paged_append(const CacheGeom& g, int layer, const RowMap& P, int rows,
                               const f16* qkv, const f16* q_gain, const f16* k_gain,
                               const f16* cos_tab, const f16* sin_tab, f16* q_out,
                               hipStream_t stream);

// Attention.  Split state, `records` rows of it (a row of a range): nqh * 128
// unnormalised f32 outputs and nqh (max, sum) pairs each, laid out per (row
// block, kv head, range) (paged_attn.hip); one arrival counter per (row block,
// kv head), zero at rest, each in a line of its own.
constexpr int kPagedCounterStep = 32;  // words
constexpr int kPagedDrawWords = 17 * kPagedCounterStep;  // 16 kv heads and one, a line each
struct PagedAttnArgs {
    const f16* q;    // [rows][nqh*128], roped
    f16* out;        // [rows][nqh*128]
    const f16* base; // the layer's pages
    int64_t page_stride, kv_stride, head_stride;
    const int32_t* table;
    int32_t stride, pages, page_shift, nkvh, rows;
    float scale_log2;
    const int32_t* n_items;
    const PagedItem *narrow, *wide;
    int32_t max_narrow, max_wide;  // 0: none can come
    float* ws_o;
    float* ws_ml;
    uint32_t* counters;
    uint32_t* drawn;  // [2][kPagedDrawWords], zero at rest: items drawn per kv head, workgroups gone
};
hipError_t launch_paged_attn(const PagedAttnArgs& a, int cus, hipStream_t stream);

}  // namespace qasr
