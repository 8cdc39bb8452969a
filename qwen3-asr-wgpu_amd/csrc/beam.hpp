// beam.hpp -- beam selection: limits, arguments and launcher, shared by the C
// ABI and the kernel (beam.hip).
#pragma once

#include "common.hpp"

namespace qasr {

constexpr int kBeamMaxGroups = 1024, kBeamMaxWidth = 32, kBeamMaxK = 32;
constexpr int kBeamThreads = 512;
constexpr int kBeamMaxSplits = 64;  // workgroups of a row: a lane each when they are merged
constexpr int kBeamMaxVocab = kBeamMaxSplits * kBeamThreads * 32;  // 2^20
constexpr int kBeamCounterStep = 32;  // words: a line each

// Logits of a thread: the fewest of 8, 16 and 32 with which kBeamMaxSplits
// workgroups cover a row.
inline int beam_values(int vocab) {
    int v = 8;
    while (v < 32 && (int64_t)kBeamMaxSplits * kBeamThreads * v < vocab) v *= 2;
    return v;
}
inline int beam_splits(int vocab) {
    const int tile = kBeamThreads * beam_values(vocab);
    return (vocab + tile - 1) / tile;
}

struct BeamArgs {
    const float* logits;  // [groups * width] rows, `stride` apart
    int64_t stride;
    const float* scores;   // [groups * width]
    const int32_t* done;   // [groups * width], or NULL
    int32_t groups, width, vocab, k, eos;
    int32_t* parent;  // [groups * k]
    int32_t* token;
    float* out_scores;
    int32_t* out_done;  // or NULL
    uint64_t* keys;     // [rows][splits][k], best first, 0: none
    float* sums;        // [rows][splits][2]: largest logit, sum of exp(logit - it); NaN: nothing of the row counts
    uint32_t* arrived;  // [groups], a line each, zero at rest
};
hipError_t launch_beam_select(const BeamArgs& a, hipStream_t stream);

}  // namespace qasr
