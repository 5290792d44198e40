// Attention over the 8-bit cache (ufb_kv_attend): the choice of a kernel and its scratch.
#include "kv_attend.cuh"

#include <mutex>

namespace ufb {

namespace {

__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(__half& o, float v) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_float(__nv_bfloat16& o, float v) { o = __float2bfloat16_rn(v); }

template <typename T, int D>
__global__ void __launch_bounds__(128) attend_kernel(const AttendArgs a) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31;
    const long long unit = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int hq = a.heads * a.group;
    const long long token = unit / hq;
    const int head = static_cast<int>(unit % hq);
    if (token >= a.tokens) return;
    int lo = 0, hi = a.n;  // last stream whose first token is not after this one
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.offsets[mid] <= token) lo = mid;
        else hi = mid;
    }
    const int slot = a.slots[lo];
    const bool ok = slot >= 0 && slot < a.slots_total;
    if (!ok && lane == 0) atomicCAS(a.status, 0, kStatusIndex);
    const int length = ok ? a.lengths[slot] : 0;
    const long long at = static_cast<long long>(length) - (a.offsets[lo + 1] - token);
    const long long top = a.causal ? at : length - 1;
    float q[V], o[V], m = -INFINITY, l = 0.0f;
    const T* qp = static_cast<const T*>(a.q.data) + token * a.q.token_stride + head * a.q.head_stride + lane * V;
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = to_float(qp[i]), o[i] = 0.0f;
    for (long long j = 0; j <= top; ++j) {
        if (a.window && j <= at - a.window && j >= a.sinks) continue;
        const long long e = j / a.page_tokens;
        const int page = e < a.table_width ? a.table[static_cast<long long>(slot) * a.table_width + e] : -1;
        if (page < 0 || page >= a.pages) continue;
        const long long tile = static_cast<long long>(page) * 2 * a.heads + head / a.group;
        const long long row = (tile * a.page_tokens + j % a.page_tokens) * D;
        const int8_t* k = a.kv + row + lane * V;
        const int8_t* v = a.kv + row + static_cast<long long>(a.heads) * a.page_tokens * D + lane * V;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) s += q[i] * k[i];
#pragma unroll
        for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
        s *= a.scale[tile] * a.scale_log2;
        const float next = fmaxf(m, s);
        const float keep = exp2f(m - next), p = exp2f(s - next);
        l = l * keep + p;
        const float pv = p * a.scale[tile + a.heads];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = o[i] * keep + pv * v[i];
        m = next;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* op = static_cast<T*>(a.out.data) + token * a.out.token_stride + head * a.out.head_stride + lane * V;
#pragma unroll
    for (int i = 0; i < V; ++i) from_float(op[i], o[i] * inv);
    if (a.lse && lane == 0) a.lse[unit] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

template <typename T>
cudaError_t launch(const AttendArgs& a, cudaStream_t s) {
    const long long blocks = (a.tokens * a.heads * a.group + 3) / 4;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
    if (a.head_dim == 64) attend_kernel<T, 64><<<static_cast<unsigned>(blocks), 128, 0, s>>>(a);
    else attend_kernel<T, 128><<<static_cast<unsigned>(blocks), 128, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

int64_t kv_attend_workspace_bytes(int sms) {
    const int ctas = sms < kAttendMaxCtas ? sms : kAttendMaxCtas;
    const AttendScratch s = scratch_of(nullptr, ctas, kAttendManyRows);
    return reinterpret_cast<int64_t>(s.sums) + 2ll * ctas * kAttendManyRows * 128 * 4;
}

bool kv_tensor_map(CUtensorMap& map, const AttendArgs& a, int keys) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            encode = reinterpret_cast<Encode>(p);
    });
    if (!encode) return false;
    const cuuint64_t rows = static_cast<cuuint64_t>(a.pages) * 2 * a.heads * a.page_tokens * a.head_dim / 128;
    if (rows > 0x7fffffffull) return false;
    const cuuint64_t dims[2] = {128, rows};
    const cuuint64_t strides[1] = {128};
    const cuuint32_t box[2] = {128, static_cast<cuuint32_t>((a.page_tokens < keys ? a.page_tokens : keys) * a.head_dim / 128)};
    const cuuint32_t elem[2] = {1, 1};
    return encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(a.kv), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t kv_attend(const AttendArgs& a, int dtype, int sms, cudaStream_t s) {
    const long long rows = static_cast<long long>(a.max_new) * a.group;
    if (rows <= 16) return attend_few(a, dtype, sms, s);
    return dtype == UFB_F16 ? launch<__half>(a, s) : launch<__nv_bfloat16>(a, s);
}

}  // namespace ufb
