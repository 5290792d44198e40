// Host launcher of the selection over beams (beam_select.cu).
#pragma once

#include <cuda_runtime.h>
#include <cstdint>

#include "uf_b200.h"

namespace ufb {

// Code recorded in the device's status word.
constexpr int kStatusLogits = 51;

constexpr int kBeamMax = UFB_BEAM_MAX;
constexpr int kBeamCountMax = UFB_BEAM_COUNT_MAX;

struct BeamSelectArgs {
    const void* logits;                 // element (stream, beam, token) at stream * stream_stride + beam * beam_stride + token
    long long stream_stride, beam_stride;
    const float* scores;                // [streams][beams]
    const uint8_t* finished;            // [streams][beams] or null
    int streams, beams, vocab, count, pad;
    float* out_scores;                  // [streams][count]
    int32_t* parents;
    int32_t* tokens;
    int* status;
    void* workspace;                    // beam_select_workspace_bytes
};
int64_t beam_select_workspace_bytes(int streams, int beams, int vocab, int count, int dtype, int sms);
cudaError_t beam_select(const BeamSelectArgs& a, int dtype, int sms, cudaStream_t s);

}  // namespace ufb
