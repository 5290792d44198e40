// Attention over the 8-bit cache (ufb_kv_attend): the choice of a kernel and its scratch.
#include "kv_attend.cuh"

#include <mutex>

namespace ufb {

int64_t kv_attend_workspace_bytes(int sms) {
    static_assert(kAttendMaxCtas * sizeof(int32_t) <= UFB_KV_ATTEND_ZERO, "the counters begin the scratch");
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
    // rows of 128 bytes of a page's head, heads, key and value, pages
    const cuuint64_t rows = static_cast<cuuint64_t>(a.page_tokens) * a.head_dim / 128, heads = a.heads;
    const cuuint64_t dims[5] = {128, rows, heads, 2, static_cast<cuuint64_t>(a.pages)};
    const cuuint64_t strides[4] = {128, rows * 128, rows * 128 * heads, rows * 128 * heads * 2};
    const cuuint32_t box[5] = {128, static_cast<cuuint32_t>((a.page_tokens < keys ? a.page_tokens : keys) * a.head_dim / 128),
                               1, 2, 1};
    const cuuint32_t elem[5] = {1, 1, 1, 1, 1};
    return encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<int8_t*>(a.kv), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t kv_attend(const AttendArgs& a, int dtype, int sms, cudaStream_t s) {
    const long long rows = static_cast<long long>(a.max_new) * a.group;
    // Up to two tiles of 16 rows the keys may be read twice, the second time from L2.  At
    // 32 rows, head_dim 128, tiles of 256 rows in brackets: 1 stream x 4000 keys 21.6 [21.8]
    // us, 8 x 4000 36.8 [36.4], 64 x 16000 459 [511], 64 x 800 64 [54]; at 64 rows 64 x
    // 16000 889 [519].  The stream with the most rows decides for the whole call: 63
    // streams of one token beside one of 32, 16000 keys each, take 500 us together, 184 and
    // 41 us in calls of their own.
    return rows <= 32 ? attend_few(a, dtype, sms, s) : attend_many(a, dtype, sms, s);
}

}  // namespace ufb
