// beam.hpp -- beam selection: limits, arguments and launcher, shared by the C
// ABI and the kernel (beam.hip).
#pragma once

#include "common.hpp"

namespace qasr {

constexpr int kBeamMaxGroups = 1024, kBeamMaxWidth = 32, kBeamMaxK = 32;
constexpr int kBeamWaves = 8;      // of a workgroup
constexpr int kBeamValues = 32;    // logits of a lane
constexpr int kBeamTile = 64 * kBeamValues;  // of a wave
constexpr int kBeamMaxVocab = 1 << 20;
constexpr int kBeamMaxParts = 32;    // workgroups of a row
constexpr int kBeamCounterStep = 32;  // words: a line each

inline int beam_tiles(int vocab) { return (vocab + kBeamTile - 1) / kBeamTile; }
// Workgroups of a row.  A wave gets one tile more at a time once there are more
// than 16 tiles a CU.  (Two workgroups of the three that a CU holds: 8 and 24 waves
// a CU were slower.)
inline int beam_parts(int rows, int vocab, int cus) {
    const int64_t tiles = beam_tiles(vocab), turns = (rows * tiles + 16 * cus - 1) / (16 * cus);
    const int64_t parts = (tiles + turns * kBeamWaves - 1) / (turns * kBeamWaves);
    return (int)(parts < kBeamMaxParts ? parts : kBeamMaxParts);
}
// Of up to `rows` rows together: a row's parts are less than its share of
// 16 cus / kBeamWaves, and one.
inline int64_t beam_most_parts(int64_t rows, int cus) { return rows + 16 / kBeamWaves * cus; }

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
    uint64_t* keys;     // [rows][parts][kBeamWaves][k], best first, 0: none
    uint64_t* sums;     // [rows][tiles]: largest logit; sum of exp(logit - it), NaN: nothing of the row counts
    uint32_t* arrived;  // [groups], a line each, zero at rest
};
hipError_t launch_beam_select(const BeamArgs& a, int cus, hipStream_t stream);

}  // namespace qasr
