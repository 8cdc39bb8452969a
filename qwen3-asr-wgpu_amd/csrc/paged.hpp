// paged.hpp -- the paged KV cache's structs and launchers, shared by its C ABI
// (paged_abi.hip) and kernels (paged_plan.hip, paged_attn.hip, norm_rope.hip).
//
// A pool is pages of 2^page_shift rows; element (layer, page, kv, head, row,
// d) is at base + layer*layer_stride + page*page_stride + kv*kv_stride +
// head*head_stride + row*kHeadDim + d, so a (page, K or V, head) is one
// contiguous block.  A request's position p lives in row p % rows of page
// table[p / rows].  Behind the last layer lies one page of zeros, which stands
// for table entries outside the pool.
// e4m3 pools hold bytes in the same places, and a byte for each 16 rows of a
// (layer, page, kv, head), the exponent of an f32 power of two: [layer][page]
// [2][nkvh][rows / 16], the zero page's behind the last layer's.
#pragma once

#include "kernels.hpp"

namespace qasr {

constexpr int kPagedMaxRequests = 1024;  // one thread of the plan kernel each
constexpr int kPagedMinShift = 4;        // pages of 16 rows: one copy instruction stays in a page
constexpr int kPagedMaxShift = 8;
constexpr int kPagedScaleRows = 16;  // e4m3: rows of a scale

// Attention work items.  A request's new rows are cut into row blocks of
// kNarrowRows rows (whose waves share the keys) or kWideRows rows (whose waves
// share the rows too), a row block's key tiles into `splits` ranges of equal
// length.  Both follow from the request's own rows and length (paged_shape), so
// a request's bits do not depend on its batch mates.
constexpr int kNarrowRows = 16, kNarrowTile = 128;
constexpr int kWideRows = 64, kWideTile = 128;
constexpr int kPagedMaxSplits = 32;     // row blocks x ranges of a split request
constexpr int kPagedManyBlocks = 16;    // but of one of more narrow row blocks than this
constexpr int kPagedMaxItems = 64;      // (those)
constexpr int kPagedRangeKeys = 512, kPagedManyRangeKeys = 2048;
constexpr int64_t kWideWork = 1 << 21;  // rows x mean keys from which on row blocks are wide

struct PagedShape {
    int32_t wide;    // row blocks of kWideRows rows
    int32_t blocks;  // row blocks
    int32_t splits;  // key ranges of each
};

// Wide row blocks read each key once for 64 rows, narrow ones for 16, but
// narrow ones are four times as many, start sooner and combine for less: us a
// layer, narrow against wide (each without a launch for the other kind), 1000
// rows at 0 17.2 / 24.1, 512 at 2000 26.9 / 28.4, 1024 at 1000 27.2 / 31.9, 4
// requests of 256 at 6000 108 / 125, 2048 at 0 40.9 / 39.8, 512 at 4000 43.4 /
// 36.7, 1024 at 4000 64 / 57, 3000 at 0 71 / 58.  A launch that finds no wide
// items takes 4.6 us on its own and adds 1.4-2 to a layer of a graph.
// Ranges, up to 16 row blocks: one row at 512, 8192 keys in ranges of 256 keys
// 8.3, 13.4, of 512 7.9, 14.0; 16 rows of 400-2400 27.4, 24.1; 8 chunks of 7-45
// rows 22.7, 17.1.  Of more row blocks, 300 rows at 5000 not split 49, in 3 ranges 33; 4 requests of 300 rows
// at 1200 not split 38, in ranges of 512 53: longer ranges, of 2048 keys.
__host__ __device__ inline PagedShape paged_shape(int len, int rows) {
    PagedShape s;
    s.wide = (int64_t)rows * (len + rows / 2) >= kWideWork;
    const int rb = s.wide ? kWideRows : kNarrowRows;
    s.blocks = (rows + rb - 1) / rb;
    const int first = len + (rows < rb ? rows : rb);  // keys of the first row block
    const bool many = !s.wide && s.blocks > kPagedManyBlocks;
    const int cap = many ? kPagedMaxItems : kPagedMaxSplits, range = many ? kPagedManyRangeKeys : kPagedRangeKeys;
    const int most = s.blocks < cap ? cap / s.blocks : 1;
    const int want = (first + range - 1) / range;
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
// request has at most max(kPagedMaxItems, blocks) items and, split, rows *
// splits records: at most kPagedMaxSplits a row, no more than a context of
// max_seq positions has ranges, and kPagedMaxSplits * kWideRows in all.
static_assert(kPagedMaxItems * kNarrowRows <= kPagedMaxSplits * kWideRows && kPagedMaxItems >= kPagedMaxSplits &&
                  kPagedMaxItems / (kPagedManyBlocks + 1) <= kPagedMaxSplits,
              "splits and records of a request");
inline int64_t paged_max_blocks(int64_t requests, int64_t rows) { return requests + rows / kNarrowRows; }
inline int64_t paged_max_items(int64_t requests, int64_t rows, int64_t rows_a_block) {
    return requests * kPagedMaxItems + requests + rows / rows_a_block;
}
static_assert(kPagedRangeKeys <= kPagedManyRangeKeys, "the shorter range bounds the splits");
inline int64_t paged_max_records(int64_t requests, int64_t rows, int64_t max_seq) {
    const int64_t ranges = (max_seq + kPagedRangeKeys - 1) / kPagedRangeKeys;
    if (ranges <= 1) return 0;  // nothing is split
    const int64_t a = rows * (ranges < kPagedMaxSplits ? ranges : kPagedMaxSplits);
    const int64_t b = requests * kPagedMaxSplits * kWideRows;
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

// And into e4m3 pages (paged_append8.hip): the layer's pages and scale bytes.
struct PagedAppend8Args {
    const f16 *qkv, *q_gain, *k_gain, *cos_tab, *sin_tab;
    f16* q_out;
    const int32_t* pos;
    const int32_t* slot;
    int32_t rows, slots, page_shift, rope_rows, nqh, nkvh;
    float eps;
    uint8_t* base;
    int64_t page_stride, kv_stride, head_stride;
    uint8_t* scales;  // exponents of f32 powers of two, one for 16 rows of a head
    int32_t page_scales, kv_scales, head_scales;
};
hipError_t launch_paged_append8(const PagedAppend8Args& a, hipStream_t stream);

// Attention.  Split state, `records` rows of it (a row of a range): nqh * 128
// unnormalised f32 outputs and nqh (max, sum) pairs each, laid out per (row
// block, kv head, range) (paged_attn.hip); one arrival counter per (row block,
// kv head), zero at rest, each in a line of its own.
constexpr int kPagedCounterStep = 32;  // words
constexpr int kPagedDrawWords = 17 * kPagedCounterStep;  // 16 kv heads and one, a line each
struct PagedAttnArgs {
    const f16* q;    // [rows][nqh*128], roped
    f16* out;        // [rows][nqh*128]
    const void* base; // the layer's pages
    int64_t page_stride, kv_stride, head_stride;
    const int32_t* table;
    int32_t stride, pages, page_shift, nkvh, rows;
    int32_t zero_page;  // page of zeros behind the pool, counted from `base`
    float scale_log2;
    const int32_t* n_items;
    const PagedItem *narrow, *wide;
    int32_t max_narrow, max_wide;  // 0: none can come
    float* ws_o;
    float* ws_ml;
    uint32_t* counters;
    uint32_t* drawn;  // [2][kPagedDrawWords], zero at rest: items drawn per kv head, workgroups gone
    const uint8_t* scales;  // e4m3: the layer's scale bytes; NULL: f16
    int32_t page_scales, kv_scales, head_scales;  // their strides
};
hipError_t launch_paged_attn(const PagedAttnArgs& a, int cus, hipStream_t stream);

}  // namespace qasr
