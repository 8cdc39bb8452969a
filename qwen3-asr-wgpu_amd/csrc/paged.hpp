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
// kNarrowRows rows (whose four waves share the keys) or kWideRows rows (whose
// four waves share the rows); a row block's key tiles into `splits` ranges of
// equal length.  Both follow from the request's own rows and length
// (paged_shape), so a request's bits do not depend on its batch mates.
constexpr int kNarrowRows = 16, kNarrowTile = 128;
constexpr int kWideRows = 64, kWideTile = 64;
constexpr int kPagedMaxSplits = 32;  // row blocks x splits of a split request

struct PagedShape {
    int32_t wide;    // row blocks of kWideRows rows
    int32_t blocks;  // row blocks
    int32_t splits;  // key ranges of each
};

__host__ __device__ inline PagedShape paged_shape(int len, int rows) {
    PagedShape s;
    s.wide = rows > 2 * kNarrowRows;
    const int rb = s.wide ? kWideRows : kNarrowRows;
    s.blocks = (rows + rb - 1) / rb;
    // At least 256 keys a range, counted for the first row block.
    const int first = len + (rows < rb ? rows : rb);
    const int most = s.blocks < kPagedMaxSplits ? kPagedMaxSplits / s.blocks : 1;
    const int want = (first + 255) / 256;
    s.splits = want < most ? want : most;
    return s;
}

struct PagedItem {  // one row block and key range, for every kv head
    int32_t req;
    int32_t row0;   // first row, in the step's rows
    int32_t pos0;   // its position
    int32_t shape;  // rows | splits << 8 | split << 16 | wide << 24
    int32_t tile0, tile1;  // key tiles (kNarrowTile or kWideTile keys)
    int32_t rec;    // split partials: record of (split 0, row 0)
    int32_t block;  // arrival counter of the row block
};

// Capacities for max_requests requests and max_rows rows together.  A
// request has at most max(kPagedMaxSplits, blocks) items and, split, rows *
// splits records: at most kPagedMaxSplits a row and kPagedMaxSplits *
// kWideRows in all.
inline int64_t paged_max_blocks(int64_t requests, int64_t rows) { return requests + rows / kNarrowRows; }
inline int64_t paged_max_items(int64_t requests, int64_t rows) {
    return requests * kPagedMaxSplits + paged_max_blocks(requests, rows);
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
    int32_t* n_items;     // [1]
    PagedItem* items;
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

// Attention.  Split partials: record r of (kv head, q head of it) holds 128
// unnormalised f32 outputs at ws_o[((r * nkvh + kvh) * 2 + h) * 128] and
// (max, sum) at ws_ml[((r * nkvh + kvh) * 2 + h) * 2]; one arrival counter per
// (row block, kv head), zero at rest.
struct PagedAttnArgs {
    const f16* q;    // [rows][nqh*128], roped
    f16* out;        // [rows][nqh*128]
    const f16* base; // the layer's pages
    int64_t page_stride, kv_stride, head_stride;
    const int32_t* table;
    int32_t stride, pages, page_shift, nkvh, rows;
    float scale_log2;
    const int32_t* n_items;
    const PagedItem* items;
    float* ws_o;
    float* ws_ml;
    uint32_t* counters;
};
hipError_t launch_paged_attn(const PagedAttnArgs& a, int64_t max_items, int cus, hipStream_t stream);

}  // namespace qasr
