// C ABI of the selection over beams (include/uf_b200.h): argument checks, then
// the launcher of beam_select.cu.
#include "uf_b200.h"

#include "beam.h"
#include "capi_util.h"

#include <string>

using namespace ufb;

namespace {

bool check_sizes(int dtype, int streams, int beams, int vocab, int count) {
    if (dtype != UFB_F32 && dtype != UFB_F16 && dtype != UFB_BF16) return fail(UFB_EINVAL, "unsupported dtype");
    if (streams < 0 || beams < 1 || vocab < 1 || count < 1) return fail(UFB_EINVAL, "empty selection");
    if (beams > UFB_BEAM_MAX || count > UFB_BEAM_COUNT_MAX)
        return fail(UFB_ERANGE, "at most " + std::to_string(UFB_BEAM_MAX) + " beams and " +
                                    std::to_string(UFB_BEAM_COUNT_MAX) + " continuations of a stream");
    if (vocab > UFB_BEAM_VOCAB_MAX || static_cast<int64_t>(streams) * beams > (1 << 24)) return fail(UFB_ERANGE, "selection exceeds indexing bounds");
    return true;
}

}  // namespace

extern "C" {

int64_t ufb_beam_select_workspace(int dtype, int streams, int beams, int vocab, int count) {
    clear_error();
    if (!check_sizes(dtype, streams, beams, vocab, count)) return last_code();
    if (streams == 0) return 0;
    const int sms = current_sms();
    return sms > 0 ? beam_select_workspace_bytes(streams, beams, vocab, count, dtype, sms) : last_code();
}

int ufb_beam_select(const void* logits, int dtype, int64_t stream_stride, int64_t beam_stride, const float* scores,
                    const uint8_t* finished, int streams, int beams, int vocab, int count, int pad,
                    float* out_scores, int32_t* parents, int32_t* tokens, void* workspace, int64_t workspace_bytes,
                    void* stream) {
    clear_error();
    if (!check_sizes(dtype, streams, beams, vocab, count)) return last_code();
    if (pad < 0) return err(UFB_EINVAL, "pad must not be negative");
    if (stream_stride < 0 || beam_stride < 0) return err(UFB_EINVAL, "negative strides");
    if (streams == 0) return UFB_OK;
    if (!logits || !scores || !out_scores || !parents || !tokens)
        return err(UFB_EINVAL, "logits, scores and results must be non-null");
    const uintptr_t size = dtype == UFB_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) % size) return err(UFB_EINVAL, "logits must be aligned to their elements");
    const int sms = current_sms();
    if (sms <= 0) return last_code();
    const int64_t need = beam_select_workspace_bytes(streams, beams, vocab, count, dtype, sms);
    if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)
        return err(UFB_EINVAL, "selection needs " + std::to_string(need) + " bytes of 16-byte aligned workspace");
    int* status = current_status();
    if (!status) return last_code();
    const BeamSelectArgs a{logits, stream_stride, beam_stride, scores, finished, streams, beams, vocab, count,
                           pad, out_scores, parents, tokens, status, workspace};
    return cuda_ok(beam_select(a, dtype, sms, static_cast<cudaStream_t>(stream)), "beam select") ? UFB_OK : last_code();
}

}  // extern "C"
