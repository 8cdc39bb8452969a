// beam_abi.hip -- C ABI of the beam selection (include/qasr_attn.h): its
// workspace, argument checks and dispatch.
//
// The reference decodes greedily (argmax, cpu_decoder.rs:514-532): nothing here
// has a counterpart in it.

#include <new>

#include "abi_internal.hpp"
#include "beam.hpp"

using qasr_abi::DeviceScope;
using qasr_abi::fail;
using qasr_abi::hip_fail;

struct qasr_beam {
    qasr_ctx* ctx;
    int device;
    int32_t max_groups, width, vocab, k;
    char* mem = nullptr;
    size_t bytes = 0;
    uint64_t *keys, *sums;
    uint32_t* arrived;
};

namespace {

struct Range {
    uintptr_t at;
    int64_t bytes;
    bool meets(const Range& o) const { return at && o.at && at < o.at + o.bytes && o.at < at + bytes; }
};

}  // namespace

extern "C" {

int qasr_beam_create(qasr_ctx* ctx, int max_groups, int width, int vocab, int k, qasr_beam** out) {
    if (!ctx || !out) return fail(QASR_EINVAL, "null argument");
    *out = nullptr;
    if (max_groups < 1 || max_groups > qasr::kBeamMaxGroups)
        return fail(QASR_EINVAL, "max_groups %d outside [1, %d]", max_groups, qasr::kBeamMaxGroups);
    if (width < 1 || width > qasr::kBeamMaxWidth)
        return fail(QASR_EINVAL, "width %d outside [1, %d]", width, qasr::kBeamMaxWidth);
    if (k < 1 || k > qasr::kBeamMaxK) return fail(QASR_EINVAL, "k %d outside [1, %d]", k, qasr::kBeamMaxK);
    if (vocab < 1 || vocab > qasr::kBeamMaxVocab)
        return fail(QASR_EINVAL, "vocab %d outside [1, %d]", vocab, qasr::kBeamMaxVocab);
    qasr_beam* b = new (std::nothrow) qasr_beam();
    if (!b) return fail(QASR_ENOMEM, "out of host memory");
    b->ctx = ctx;
    b->device = ctx->device;
    b->max_groups = max_groups;
    b->width = width;
    b->vocab = vocab;
    b->k = k;
    const size_t rows = (size_t)max_groups * width;
    const size_t o_sums = (size_t)max_groups * qasr::kBeamCounterStep * 4;
    const size_t o_keys = o_sums + rows * qasr::beam_tiles(vocab) * 8;
    b->bytes = o_keys + (size_t)qasr::beam_most_parts(rows, ctx->cus) * qasr::kBeamWaves * k * 8;
    DeviceScope ds(ctx->device);
    hipError_t e = ds.err;
    if (e == hipSuccess) e = hipMalloc(&b->mem, b->bytes);
    if (e == hipSuccess) e = hipMemset(b->mem, 0, o_sums);
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        if (b->mem) (void)hipFree(b->mem);
        delete b;
        (void)hipGetLastError();  // the next launch must not report it
        return hip_fail(e, "beam selection allocation");
    }
    b->arrived = (uint32_t*)b->mem;
    b->sums = (uint64_t*)(b->mem + o_sums);
    b->keys = (uint64_t*)(b->mem + o_keys);
    *out = b;
    return QASR_OK;
}

void qasr_beam_destroy(qasr_beam* b) {
    if (!b) return;
    DeviceScope ds(b->device);
    (void)hipDeviceSynchronize();
    if (b->mem) (void)hipFree(b->mem);
    delete b;
}

int qasr_beam_select(qasr_ctx* ctx, qasr_beam* beam, int groups, const float* logits_dev, int64_t logits_stride,
                     const float* scores_dev, const int32_t* done_dev, int eos, int32_t* parent_dev,
                     int32_t* token_dev, float* out_scores_dev, int32_t* out_done_dev, void* stream) {
    if (!ctx || !beam) return fail(QASR_EINVAL, "null context or beam selection");
    if (beam->ctx != ctx) return fail(QASR_EINVAL, "beam selection belongs to another context");
    if (groups < 1) return fail(QASR_EINVAL, "groups must be > 0");
    if (groups > beam->max_groups)
        return fail(QASR_ERANGE, "%d groups, the beam selection holds %d", groups, beam->max_groups);
    if (logits_stride < beam->vocab)
        return fail(QASR_EINVAL, "rows of %d logits are %lld apart", beam->vocab, (long long)logits_stride);
    if (logits_stride > (int64_t)1 << 40) return fail(QASR_EINVAL, "logits_stride %lld", (long long)logits_stride);
    if (eos < -1 || eos >= beam->vocab) return fail(QASR_EINVAL, "eos %d outside [-1, %d)", eos, beam->vocab);
    if (!logits_dev || !scores_dev || !parent_dev || !token_dev || !out_scores_dev)
        return fail(QASR_EINVAL, "null device pointer");
    const uintptr_t all = (uintptr_t)logits_dev | (uintptr_t)scores_dev | (uintptr_t)done_dev | (uintptr_t)parent_dev |
                          (uintptr_t)token_dev | (uintptr_t)out_scores_dev | (uintptr_t)out_done_dev;
    if (all & 3) return fail(QASR_EINVAL, "an array of 32-bit numbers is not 4-byte aligned");
    // A group's outputs are written when all of its inputs are read, other
    // groups' inputs may still be: in place only row for row.
    const int64_t in = (int64_t)groups * beam->width * 4, res = (int64_t)groups * beam->k * 4;
    const Range logits{(uintptr_t)logits_dev, ((int64_t)groups * beam->width - 1) * logits_stride * 4 + beam->vocab * 4ll};
    const Range ins[] = {{(uintptr_t)scores_dev, in}, {(uintptr_t)done_dev, in}};
    const Range outs[] = {{(uintptr_t)parent_dev, res}, {(uintptr_t)token_dev, res}, {(uintptr_t)out_scores_dev, res},
                          {(uintptr_t)out_done_dev, res}};
    const Range own{(uintptr_t)beam->mem, (int64_t)beam->bytes};
    for (const Range& o : outs) {
        if (o.meets(logits) || o.meets(own)) return fail(QASR_EINVAL, "an output lies in the logits or the workspace");
        for (const Range& i : ins)
            if (o.meets(i) && (o.at != i.at || beam->k != beam->width))
                return fail(QASR_EINVAL, "an output overlaps an input other than in place with as many candidates as beams");
        for (const Range& p : outs)
            if (&p != &o && o.meets(p)) return fail(QASR_EINVAL, "two outputs overlap");
    }
    DeviceScope ds(ctx->device);
    if (ds.err != hipSuccess) return hip_fail(ds.err, "hipSetDevice");
    qasr::BeamArgs a;
    a.logits = logits_dev;
    a.stride = logits_stride;
    a.scores = scores_dev;
    a.done = done_dev;
    a.groups = groups;
    a.width = beam->width;
    a.vocab = beam->vocab;
    a.k = beam->k;
    a.eos = eos;
    a.parent = parent_dev;
    a.token = token_dev;
    a.out_scores = out_scores_dev;
    a.out_done = out_done_dev;
    a.keys = beam->keys;
    a.sums = beam->sums;
    a.arrived = beam->arrived;
    const hipError_t e = qasr::launch_beam_select(a, ctx->cus, (hipStream_t)stream);
    if (e != hipSuccess) return hip_fail(e, "beam selection launch");
    return QASR_OK;
}

}  // extern "C"
