// paged_abi.hip -- C ABI of the paged KV cache (include/qasr_attn.h): page
// pools, step plans, argument checks and dispatch.
//
// The reference's caches are one buffer per slot (decoder.rs:1270-1271,
// 2453-2457): nothing here has a counterpart in it.

#include <algorithm>
#include <limits>
#include <new>

#include "abi_internal.hpp"
#include "paged.hpp"

using qasr::f16;
using qasr_abi::DeviceScope;
using qasr_abi::fail;
using qasr_abi::hip_fail;

struct qasr_pages {
    qasr_ctx* ctx;
    int device;
    int32_t pages;
    int32_t shift;  // log2 of a page's rows
    f16* base = nullptr;  // the layers' pages, then the zero page
    size_t bytes = 0;     // without the zero page
};

struct qasr_paged_plan {
    qasr_ctx* ctx;
    int device;
    qasr_pages* pool;
    int32_t max_requests;
    int32_t max_rows;
    int32_t max_narrow, max_wide;  // work items
    char* mem = nullptr;  // everything below, one allocation
    size_t bytes = 0;
    int32_t *status, *lens, *row_start, *row_pos, *row_slot, *cursor, *n_items;
    qasr::PagedItem *narrow, *wide;
    uint32_t *arrived, *drawn, *counters;
    float *ws_o, *ws_ml;
    // The last build, for the checks of the calls that follow it.
    int32_t nreq = 0;
    int32_t stride = 0;
};

namespace {

qasr::CacheGeom page_geom(const qasr_pages* p) {
    const qasr_attn_cfg& c = p->ctx->cfg;
    qasr::CacheGeom g;
    g.base = p->base;
    g.head_stride = (int64_t)qasr::kHeadDim << p->shift;
    g.kv_stride = g.head_stride * c.num_key_value_heads;
    g.slot_stride = 2 * g.kv_stride;  // page
    g.layer_stride = g.slot_stride * p->pages;
    g.nkvh = c.num_key_value_heads;
    g.cap = 1 << p->shift;
    return g;
}

int check_plan(qasr_ctx* ctx, qasr_paged_plan* plan) {
    if (!ctx || !plan) return fail(QASR_EINVAL, "null context or plan");
    if (plan->ctx != ctx) return fail(QASR_EINVAL, "plan belongs to another context");
    return QASR_OK;
}

int check_layer_rows(qasr_ctx* ctx, qasr_paged_plan* plan, int layer, int rows) {
    const int rc = check_plan(ctx, plan);
    if (rc) return rc;
    if (layer < 0 || layer >= ctx->cfg.num_hidden_layers)
        return fail(QASR_EINVAL, "layer %d outside [0, %d)", layer, ctx->cfg.num_hidden_layers);
    if (rows < 0) return fail(QASR_EINVAL, "negative rows");
    if (rows > plan->max_rows) return fail(QASR_ERANGE, "%d rows, the plan holds %d", rows, plan->max_rows);
    if (!plan->nreq) return fail(QASR_ESTATE, "plan not built (qasr_paged_plan_build)");
    return QASR_OK;
}

// Rows in and out: 16-byte loads and stores, and workgroups that read `in`
// after others have written `out`.
int check_arrays(const void* in, int64_t in_bytes, const void* out, int64_t out_bytes) {
    const uintptr_t i = (uintptr_t)in, o = (uintptr_t)out;
    if ((i | o) & 15) return fail(QASR_EINVAL, "rows must be 16-byte aligned");
    if (i < o + out_bytes && o < i + in_bytes) return fail(QASR_EINVAL, "the output overlaps the input");
    return QASR_OK;
}

// What a build's workgroups all read, none of them may write before the last
// has read it: they would plan different requests, and one count work items
// that another never wrote.  Only the plan's lens and cursor are written by the
// workgroup that arrives last.  Fresh table entries are written, and pages given
// back to the ring, where no one reads them: only with a ring.
struct Range {
    uintptr_t at;
    int64_t bytes;
    bool meets(const Range& o) const {
        return at && o.at && bytes > 0 && o.bytes > 0 && at < o.at + o.bytes && o.at < at + bytes;
    }
};
int check_build_arrays(const qasr_paged_plan* p, int nreq, const int32_t* len, const int32_t* rows, const int32_t* table,
                       int stride, const int32_t* ring, const int32_t* cursor) {
    if (((uintptr_t)len | (uintptr_t)rows | (uintptr_t)table | (uintptr_t)ring | (uintptr_t)cursor) & 3)
        return fail(QASR_EINVAL, "an array of 32-bit numbers is not 4-byte aligned");
    const Range own{(uintptr_t)p->mem, (int64_t)p->bytes}, t{(uintptr_t)table, (int64_t)nreq * stride * 4},
        g{(uintptr_t)ring, (int64_t)p->pool->pages * 4}, l{(uintptr_t)len, (int64_t)nreq * 4},
        r{(uintptr_t)rows, (int64_t)nreq * 4}, c{(uintptr_t)cursor, 8};
    if (t.meets(own) || g.meets(own) || r.meets(own) || (len != p->lens && l.meets(own)) ||
        (cursor != p->cursor && c.meets(own)))
        return fail(QASR_EINVAL, "an array lies in the plan's own (only its lens and cursor may)");
    if (!ring) return QASR_OK;
    if (t.meets(g) || t.meets(l) || t.meets(r) || t.meets(c) || g.meets(l) || g.meets(r) || g.meets(c))
        return fail(QASR_EINVAL, "the table or the ring overlaps another array");
    return QASR_OK;
}

}  // namespace

extern "C" {

int qasr_pages_create(qasr_ctx* ctx, int pages, int page_rows, qasr_pages** out) {
    if (!ctx || !out) return fail(QASR_EINVAL, "null argument");
    *out = nullptr;
    int shift = qasr::kPagedMinShift;
    while (shift < qasr::kPagedMaxShift && (1 << shift) != page_rows) ++shift;
    if ((1 << shift) != page_rows)
        return fail(QASR_EINVAL, "page_rows %d is not a power of two from %d to %d", page_rows,
                    1 << qasr::kPagedMinShift, 1 << qasr::kPagedMaxShift);
    if (pages <= 0) return fail(QASR_EINVAL, "pages must be > 0");
    if ((int64_t)pages << shift > std::numeric_limits<int32_t>::max())
        return fail(QASR_EINVAL, "%d pages of %d rows pass 2^31 rows", pages, page_rows);
    if ((int64_t)pages * ctx->cfg.num_hidden_layers > std::numeric_limits<int32_t>::max())
        return fail(QASR_ENOMEM, "%d pages of %d layers: more than a card holds", pages, ctx->cfg.num_hidden_layers);
    qasr_pages* p = new (std::nothrow) qasr_pages();
    if (!p) return fail(QASR_ENOMEM, "out of host memory");
    p->ctx = ctx;
    p->device = ctx->device;
    p->pages = pages;
    p->shift = shift;
    p->bytes = (size_t)page_geom(p).layer_stride * ctx->cfg.num_hidden_layers * sizeof(f16);
    const size_t all = p->bytes + (size_t)page_geom(p).slot_stride * sizeof(f16);
    DeviceScope ds(ctx->device);
    hipError_t e = ds.err;
    if (e == hipSuccess) e = hipMalloc(&p->base, all);
    if (e == hipSuccess) e = hipMemset(p->base, 0, all);
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        if (p->base) (void)hipFree(p->base);
        delete p;
        (void)hipGetLastError();  // the next launch must not report it
        return hip_fail(e, "page pool allocation");
    }
    *out = p;
    return QASR_OK;
}

void qasr_pages_destroy(qasr_pages* p) {
    if (!p) return;
    DeviceScope ds(p->device);
    (void)hipDeviceSynchronize();
    if (p->base) (void)hipFree(p->base);
    delete p;
}

int qasr_pages_get_info(const qasr_pages* p, qasr_pages_info* out) {
    if (!p || !out) return fail(QASR_EINVAL, "null argument");
    const qasr::CacheGeom g = page_geom(p);
    out->base_dev = p->base;
    out->pages = p->pages;
    out->page_rows = 1 << p->shift;
    out->layers = p->ctx->cfg.num_hidden_layers;
    out->nkvh = g.nkvh;
    out->head_dim = qasr::kHeadDim;
    out->layer_stride = g.layer_stride;
    out->page_stride = g.slot_stride;
    out->kv_stride = g.kv_stride;
    out->head_stride = g.head_stride;
    out->bytes = p->bytes;
    return QASR_OK;
}

int qasr_paged_plan_create(qasr_ctx* ctx, qasr_pages* pool, int max_requests, int max_rows, qasr_paged_plan** out) {
    if (!ctx || !pool || !out) return fail(QASR_EINVAL, "null argument");
    *out = nullptr;
    if (pool->ctx != ctx) return fail(QASR_EINVAL, "page pool belongs to another context");
    if (max_requests < 1 || max_requests > qasr::kPagedMaxRequests)
        return fail(QASR_EINVAL, "max_requests %d outside [1, %d]", max_requests, qasr::kPagedMaxRequests);
    if (max_rows < 1 || max_rows > QASR_PAGED_MAX_ROWS)
        return fail(QASR_EINVAL, "max_rows %d outside [1, %d]", max_rows, QASR_PAGED_MAX_ROWS);
    qasr_paged_plan* p = new (std::nothrow) qasr_paged_plan();
    if (!p) return fail(QASR_ENOMEM, "out of host memory");
    const int nkvh = ctx->cfg.num_key_value_heads;
    p->ctx = ctx;
    p->device = ctx->device;
    p->pool = pool;
    p->max_requests = max_requests;
    p->max_rows = max_rows;
    p->max_narrow = (int32_t)qasr::paged_max_items(max_requests, max_rows, qasr::kNarrowRows);
    p->max_wide = (int32_t)qasr::paged_max_items(max_requests, max_rows, qasr::kWideRows);
    const int64_t blocks = qasr::paged_max_blocks(max_requests, max_rows) * nkvh;
    const int64_t recs = qasr::paged_max_records(max_requests, max_rows, ctx->cfg.max_seq) * nkvh * qasr::kRep;
    // One allocation, each part from a multiple of 256 bytes; the parts up to
    // `clear` start at zero (counters, and a plan that was never built has no
    // items).
    size_t at = 0, clear = 0;
    auto part = [&](size_t n) {
        const size_t a = at;
        at += (n + 255) / 256 * 256;
        return a;
    };
    const size_t o_ni = part(8), o_arr = part(4), o_dr = part(2 * 4 * qasr::kPagedDrawWords), o_ctr = part(blocks * 4 * qasr::kPagedCounterStep), o_cur = part(8);
    const size_t o_st = part(4 * (size_t)max_requests), o_len = part(4 * (size_t)max_requests);
    const size_t o_rs = part(4 * (size_t)(max_requests + 1));
    const size_t o_rp = part(4 * (size_t)max_rows), o_sl = part(4 * (size_t)max_rows);
    clear = at;
    const size_t o_it = part(sizeof(qasr::PagedItem) * (size_t)p->max_narrow);
    const size_t o_wi = part(sizeof(qasr::PagedItem) * (size_t)p->max_wide);
    const size_t o_o = part(recs * qasr::kHeadDim * 4), o_ml = part(recs * 8);
    p->bytes = at;
    DeviceScope ds(ctx->device);
    hipError_t e = ds.err;
    if (e == hipSuccess) e = hipMalloc(&p->mem, p->bytes);
    if (e == hipSuccess) e = hipMemset(p->mem, 0, clear);
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        if (p->mem) (void)hipFree(p->mem);
        delete p;
        (void)hipGetLastError();  // the next launch must not report it
        return hip_fail(e, "paged plan allocation");
    }
    p->n_items = (int32_t*)(p->mem + o_ni);
    p->arrived = (uint32_t*)(p->mem + o_arr);
    p->drawn = (uint32_t*)(p->mem + o_dr);
    p->counters = (uint32_t*)(p->mem + o_ctr);
    p->cursor = (int32_t*)(p->mem + o_cur);
    p->status = (int32_t*)(p->mem + o_st);
    p->lens = (int32_t*)(p->mem + o_len);
    p->row_start = (int32_t*)(p->mem + o_rs);
    p->row_pos = (int32_t*)(p->mem + o_rp);
    p->row_slot = (int32_t*)(p->mem + o_sl);
    p->narrow = (qasr::PagedItem*)(p->mem + o_it);
    p->wide = (qasr::PagedItem*)(p->mem + o_wi);
    p->ws_o = (float*)(p->mem + o_o);
    p->ws_ml = (float*)(p->mem + o_ml);
    *out = p;
    return QASR_OK;
}

void qasr_paged_plan_destroy(qasr_paged_plan* p) {
    if (!p) return;
    DeviceScope ds(p->device);
    (void)hipDeviceSynchronize();
    if (p->mem) (void)hipFree(p->mem);
    delete p;
}

int qasr_paged_plan_get_info(const qasr_paged_plan* p, qasr_paged_plan_info* out) {
    if (!p || !out) return fail(QASR_EINVAL, "null argument");
    out->max_requests = p->max_requests;
    out->max_rows = p->max_rows;
    out->status_dev = p->status;
    out->lens_dev = p->lens;
    out->row_start_dev = p->row_start;
    out->row_pos_dev = p->row_pos;
    out->row_slot_dev = p->row_slot;
    out->cursor_dev = p->cursor;
    out->bytes = p->bytes;
    return QASR_OK;
}

int qasr_paged_plan_build(qasr_ctx* ctx, qasr_paged_plan* plan, int nreq, const int32_t* len_dev,
                          const int32_t* rows_dev, int32_t* table_dev, int table_stride,
                          int32_t* ring_dev, const int32_t* cursor_dev, void* stream) {
    const int rc = check_plan(ctx, plan);
    if (rc) return rc;
    if (nreq < 1) return fail(QASR_EINVAL, "nreq must be > 0");
    if (nreq > plan->max_requests)
        return fail(QASR_ERANGE, "%d requests, the plan holds %d", nreq, plan->max_requests);
    if (table_stride < 1) return fail(QASR_EINVAL, "table_stride must be > 0");
    if (!len_dev || !rows_dev || !table_dev) return fail(QASR_EINVAL, "null device pointer");
    if (!ring_dev != !cursor_dev) return fail(QASR_EINVAL, "ring and cursor go together");
    const int ar = check_build_arrays(plan, nreq, len_dev, rows_dev, table_dev, table_stride, ring_dev, cursor_dev);
    if (ar) return ar;
    DeviceScope ds(ctx->device);
    if (ds.err != hipSuccess) return hip_fail(ds.err, "hipSetDevice");
    qasr::PagedPlanArgs a;
    a.len = len_dev;
    a.rows = rows_dev;
    a.table = table_dev;
    a.ring = ring_dev;
    a.cursor = cursor_dev;
    a.nreq = nreq;
    a.stride = table_stride;
    a.pages = plan->pool->pages;
    a.page_shift = plan->pool->shift;
    a.max_seq = ctx->cos ? std::min(ctx->cfg.max_seq, ctx->rope_rows) : ctx->cfg.max_seq;
    a.max_rows = plan->max_rows;
    a.status = plan->status;
    a.lens_out = plan->lens;
    a.row_start = plan->row_start;
    a.row_pos = plan->row_pos;
    a.row_slot = plan->row_slot;
    a.cursor_out = plan->cursor;
    a.n_items = plan->n_items;
    a.narrow = plan->narrow;
    a.wide = plan->wide;
    a.arrived = plan->arrived;
    const hipError_t e = qasr::launch_paged_plan(a, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "paged plan launch");
    plan->nreq = nreq;
    plan->stride = table_stride;
    return QASR_OK;
}

int qasr_paged_append(qasr_ctx* ctx, qasr_paged_plan* plan, int layer, int rows, const void* qkv_dev,
                      const void* q_gain_dev, const void* k_gain_dev, void* q_out_dev, void* stream) {
    const int rc = check_layer_rows(ctx, plan, layer, rows);
    if (rc) return rc;
    if (rows == 0) return QASR_OK;
    if (!qkv_dev || !q_gain_dev || !k_gain_dev || !q_out_dev) return fail(QASR_EINVAL, "null device pointer");
    const int nqh = ctx->cfg.num_attention_heads, heads = nqh + 2 * ctx->cfg.num_key_value_heads;
    const int64_t head_bytes = (int64_t)rows * qasr::kHeadDim * sizeof(f16);
    const int io = check_arrays(qkv_dev, heads * head_bytes, q_out_dev, nqh * head_bytes);
    if (io) return io;
    if (((uintptr_t)q_gain_dev | (uintptr_t)k_gain_dev) & 15) return fail(QASR_EINVAL, "gains must be 16-byte aligned");
    if (!ctx->cos) return fail(QASR_ESTATE, "RoPE tables not set (qasr_set_rope_tables)");
    DeviceScope ds(ctx->device);
    if (ds.err != hipSuccess) return hip_fail(ds.err, "hipSetDevice");
    qasr::RowMap P;
    P.pos = plan->row_pos;
    P.slot = plan->row_slot;
    P.slots = plan->pool->pages << plan->pool->shift;
    P.page_shift = plan->pool->shift;
    P.rope_rows = ctx->rope_rows;
    P.nqh = ctx->cfg.num_attention_heads;
    P.eps = ctx->cfg.rms_norm_eps;
    const hipError_t e = qasr::launch_paged_append(page_geom(plan->pool), layer, P, rows, (const f16*)qkv_dev,
                                                   (const f16*)q_gain_dev, (const f16*)k_gain_dev, ctx->cos, ctx->sin,
                                                   (f16*)q_out_dev, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "paged append launch");
    return QASR_OK;
}

int qasr_paged_attn(qasr_ctx* ctx, qasr_paged_plan* plan, int layer, int rows, const int32_t* table_dev,
                    int table_stride, const void* q_dev, void* out_dev, void* stream) {
    const int rc = check_layer_rows(ctx, plan, layer, rows);
    if (rc) return rc;
    if (table_stride != plan->stride)
        return fail(QASR_EINVAL, "table_stride %d, the plan was built with %d", table_stride, plan->stride);
    if (rows == 0) return QASR_OK;
    if (!table_dev || !q_dev || !out_dev) return fail(QASR_EINVAL, "null device pointer");
    const int64_t bytes = (int64_t)rows * ctx->cfg.num_attention_heads * qasr::kHeadDim * sizeof(f16);
    const int io = check_arrays(q_dev, bytes, out_dev, bytes);
    if (io) return io;
    DeviceScope ds(ctx->device);
    if (ds.err != hipSuccess) return hip_fail(ds.err, "hipSetDevice");
    const qasr::CacheGeom g = page_geom(plan->pool);
    qasr::PagedAttnArgs a;
    a.q = (const f16*)q_dev;
    a.out = (f16*)out_dev;
    a.base = g.base + layer * g.layer_stride;
    a.page_stride = g.slot_stride;
    a.kv_stride = g.kv_stride;
    a.head_stride = g.head_stride;
    a.table = table_dev;
    a.stride = table_stride;
    a.pages = plan->pool->pages;
    a.zero_page = a.pages * (ctx->cfg.num_hidden_layers - layer);
    a.page_shift = plan->pool->shift;
    a.nkvh = g.nkvh;
    a.rows = rows;
    a.scale_log2 = ctx->scale_log2;
    a.n_items = plan->n_items;
    a.narrow = plan->narrow;
    a.wide = plan->wide;
    a.max_narrow = plan->max_narrow;
    a.max_wide = qasr::paged_wide(plan->max_rows, (int64_t)plan->stride << plan->pool->shift) ? plan->max_wide : 0;
    a.ws_o = plan->ws_o;
    a.ws_ml = plan->ws_ml;
    a.counters = plan->counters;
    a.drawn = plan->drawn;
    const hipError_t e = qasr::launch_paged_attn(a, ctx->cus, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "paged attention launch");
    return QASR_OK;
}

int qasr_plan_paged(int len, int rows, int32_t* wide, int32_t* blocks, int32_t* splits) {
    if (len < 0 || len > 1 << 24 || rows < 1 || rows > QASR_PAGED_MAX_ROWS)
        return fail(QASR_EINVAL, "len %d / rows %d", len, rows);
    if (!wide || !blocks || !splits) return fail(QASR_EINVAL, "null pointer");
    const qasr::PagedShape s = qasr::paged_shape(len, rows);
    *wide = s.wide;
    *blocks = s.blocks;
    *splits = s.splits;
    return QASR_OK;
}

}  // extern "C"
