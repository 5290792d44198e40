// Host launchers and the device view of the latent-attention operators
// (rotary.cu, kv_append.cu, kv_pages.cu, kv_attend*.cu).
#pragma once

#include <cuda_runtime.h>
#include <cstdint>

#include "uf_b200.h"

namespace ufb {

// Codes recorded in the device's status word.
constexpr int kStatusPosition = 21;
constexpr int kStatusPages = 31;
constexpr int kStatusIndex = 32;

constexpr int kRotaryMaxPairs = 128;

struct RotaryArgs {
    const float2* table;             // (cos, sin) of every axis, position and pair
    const int32_t* positions;        // [tokens, axes]
    long long tokens;
    int axes, head_dim, pairs;       // pairs = sum over the axes
    int layout, inverse;
    int extent[UFB_ROTARY_MAX_AXES];
    int first[UFB_ROTARY_MAX_AXES + 1];       // first pair of each axis
    long long base[UFB_ROTARY_MAX_AXES];      // first table entry of each axis
    int count;                       // tensors
    ufb_heads x[2], out[2];
};
cudaError_t rotary(const RotaryArgs& a, int dtype, int sms, int* status, cudaStream_t s);

// Marks of streams (one for each slot, behind the page operators' scratch in
// ufb_kv_cache.work): 1 from an extend that was refused to one that is granted.
__host__ __device__ inline int32_t* kv_refused(const ufb_kv_cache& c) {
    return c.work + 16 + 3ll * c.pages + c.slots;
}

// Streams of one call: new tokens [offsets[i], offsets[i + 1]) belong to slots[i].
struct KvBatch {
    const int32_t* slots;
    const int32_t* offsets;
    int n, max_new;
    long long tokens;
};

cudaError_t kv_append(const ufb_kv_cache& c, int layer, const KvBatch& b, int dtype, const ufb_heads& k,
                      const ufb_heads& v, int* status, cudaStream_t s);
cudaError_t kv_read(const ufb_kv_cache& c, int layer, const int32_t* pages, long long n, int dtype, void* out,
                    int* status, cudaStream_t s);

cudaError_t kv_extend(const ufb_kv_cache& c, const int32_t* slots, const int32_t* offsets, int n, int* status,
                      cudaStream_t s);
cudaError_t kv_release(const ufb_kv_cache& c, const int32_t* slots, int n, int* status, cudaStream_t s);
cudaError_t kv_fork(const ufb_kv_cache& c, const int32_t* src, const int32_t* dst, int n, int* status,
                    cudaStream_t s);
cudaError_t kv_trim(const ufb_kv_cache& c, const int32_t* slots, int n, int window, int sinks, int* status,
                    cudaStream_t s);
cudaError_t kv_compact(const ufb_kv_cache& c, int* status, cudaStream_t s);

struct AttendArgs {
    const int8_t* kv;                // this layer's pages
    const float* scale;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* refused;          // kv_refused
    const int32_t* slots;
    const int32_t* offsets;
    long long tokens;
    int n, max_new;
    int pages, heads, group, page_tokens, page_shift, head_dim, slots_total, table_width;
    int window, sinks, causal;
    float scale_log2;                // softmax scale * log2(e)
    ufb_heads q, out;
    float* lse;
    int* status;
    void* workspace;
};
cudaError_t kv_attend(const AttendArgs& a, int dtype, int sms, cudaStream_t s);
int64_t kv_attend_workspace_bytes(int sms);

}  // namespace ufb
