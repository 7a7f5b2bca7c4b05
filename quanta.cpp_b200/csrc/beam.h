// The selection of a beam search's next step (beam.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_cache.h"

namespace qb {

constexpr int kBeamMaxK = 64;

struct BeamArgs {
    const void* logits;  // row r = group * beams + beam at logits + r * stride (elements)
    long long stride;
    const float* scores;    // [groups][beams]
    const uint8_t* ended;   // [groups][beams] or null
    int groups, beams, vocab, k, end_id;
    float* out_scores;      // [groups][k]
    int* tokens;
    int* parents;
    KvType type;
};
size_t beam_ws_bytes(const BeamArgs& a);
cudaError_t launch_beam_select(const BeamArgs& a, void* ws, cudaStream_t st);

}  // namespace qb
