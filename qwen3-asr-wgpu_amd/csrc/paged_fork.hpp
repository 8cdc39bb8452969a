// paged_fork.hpp -- forks of paged requests: workspace, arguments and
// launcher, shared by the C ABI (paged_abi.hip) and the kernels
// (paged_fork.hip).
#pragma once

#include "paged.hpp"

namespace qasr {

constexpr int kForkColumns = 2;  // table columns of a workgroup

// What the first kernel finds out about each request, for the second.
struct ForkRow {
    int32_t parent;  // request it goes on from, -1: none
    int32_t used;    // pages that it holds (as a parent)
    int32_t whole;   // of them full ones; the next is unfinished if used > whole
    int32_t more;    // requests more that go on from it than itself: holders of its full pages
    int32_t more_last;  // and of its unfinished page, whose copies are pages of their own
    int32_t fresh;   // page for its copy of the parent's unfinished one, if `copy`
    int32_t copy;
    int32_t unused;
};
static_assert(sizeof(ForkRow) == 32, "");
struct ForkCopy {
    int32_t from, to, rows;  // rows 0: nothing to copy
    int32_t unused;
};
struct ForkHead {
    int32_t ok, copies, head, free;
    uint32_t arrived;  // zero at rest
    int32_t unused[3];
};

struct ForkArgs {
    int32_t* len;           // [nreq]
    const int32_t* parent;  // [nreq]
    int32_t* table;         // [nreq][stride]
    int32_t* shared;        // [pages] further requests that hold a page
    int32_t* ring;          // [pages]
    int32_t* cursor;        // {head, free}
    int32_t nreq, stride, pages, page_shift;
    int32_t* status;  // [nreq]
    // Workspace.
    ForkHead* w;
    ForkRow* rows;      // [nreq]
    ForkCopy* copies;   // [nreq]
    int32_t* gone;      // [column blocks][nreq * kForkColumns] pages that nobody holds any more
    int32_t* n_gone;    // [column blocks]
    // The pool.
    char* base;
    int64_t layer_bytes, page_bytes;
    int32_t row_bytes, layers, heads;  // heads: K's and V's of a page
    uint8_t* scales;  // or NULL
    int64_t layer_scales;
    int32_t page_scales;
};
hipError_t launch_paged_fork(const ForkArgs& a, int cus, hipStream_t stream);

}  // namespace qasr
