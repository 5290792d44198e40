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
constexpr int kStatusShare = 33;

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
// How many calls changed tables or lengths (the page operators' scratch begins with words of its own).
__host__ __device__ inline int32_t* kv_changes(const ufb_kv_cache& c) { return c.work + 2; }
// Behind the marks, one integer for each stream of a reorder.
__host__ __device__ inline int32_t* kv_last_entry(const ufb_kv_cache& c) { return kv_refused(c) + c.slots; }

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
cudaError_t kv_reorder(const ufb_kv_cache& c, const int32_t* slots, const int32_t* parents, int n, int width,
                       int* status, cudaStream_t s);
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

// What kv_share leaves of the groups of a batch (ufb_kv_groups.state).
struct KvGroupState {
    int32_t* shared;                       // [groups] tokens in common
    struct Group {
        int32_t token0, tokens, stream0, streams;
        int32_t shared, slot, low, high;   // slot: of a stream that has them; least and largest position
        int32_t own;                       // of all its streams' own keys: `units`
        int32_t seen;                      // kv_changes when it was written, and 1; its complement: turned away
        int32_t pad[2];
    };
    Group* group;                          // [groups], 16-byte aligned
    struct Token {
        int32_t position;                  // kNotWritten: its results are left alone
        int32_t own, end;                  // of the group's own keys, one after another: its stream's first, and the end
        int32_t stream;                    // number in the batch
    };
    Token* token;                          // [tokens], 16-byte aligned
    int32_t* units;                        // [n] kGroupUnit own keys each, of the group's streams up to this one
};
constexpr int kNotWritten = INT32_MIN;
constexpr int kGroupUnit = 16;             // own keys that begin together in a tile of kv_attend_groups
struct GroupArgs {
    int groups, max_tokens;
    const int32_t* first;                  // as in ufb_kv_groups
    const int32_t* offsets;
    const int32_t* changes;                // kv_changes
    KvGroupState state;
};
inline KvGroupState kv_group_state(const ufb_kv_groups& g, long long tokens) {
    KvGroupState s;
    s.shared = g.state;
    s.group = reinterpret_cast<KvGroupState::Group*>(s.shared + (g.groups + 3) / 4 * 4);
    s.token = reinterpret_cast<KvGroupState::Token*>(s.group + g.groups);
    s.units = reinterpret_cast<int32_t*>(s.token + tokens);
    return s;
}
cudaError_t kv_share(const ufb_kv_cache& c, const KvBatch& b, const ufb_kv_groups& g, int* status, cudaStream_t s);
cudaError_t kv_attend_groups(const AttendArgs& a, const GroupArgs& g, int dtype, int sms, cudaStream_t s);
int64_t kv_attend_workspace_bytes(int sms);

}  // namespace ufb
