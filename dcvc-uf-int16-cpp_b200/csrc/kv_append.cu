// New keys and values into the 8-bit cache (ufb_kv_append) and the values that
// pages stand for (ufb_kv_read).
//
// One scale serves a page, head and side, so a CTA takes one (page, head, side)
// that a stream's new tokens reach: it finds max |x| over the new tokens of the
// page, s' = max(s, max * (1 / 127)), requantises the earlier tokens only when s' grew,
// and writes the new integers.  The new values stay in registers between the two
// steps (a page and head hold at most 16384 of them, 64 a thread), so HBM sees
// each input once and each byte of the cache at most once: the call is bound by
// those bytes, or by its latency when every stream brings one token.
// Every step is one IEEE operation in 32 bits (1 / 127 a constant, x / s' a
// division, done as a product wherever that cannot change the integer): the
// integers do not depend on the order of work.
#include "attention.h"

#include "capi_util.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ufb {

namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]);

template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&f)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__half>(const __half* p, float (&f)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&f)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// rint(x / scale), saturated; any float values.
__device__ __forceinline__ uint32_t quantise(float x, float scale) {
    if (scale == 0.0f) return 0;
    const float v = x / scale;
    return v == v ? static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(v, -127.0f), 127.0f))) & 0xff : 0;
}

// The same for finite x with |x / scale| <= 127.5 and a scale above 2^-100, inv =
// 1 / scale: x inv is within 127 * 3 * 2^-24 < 2^-15 of the quotient, so its
// nearest integer is the quotient's unless a tie is that close; those few are
// divided.  Adding 1.5 * 2^23 rounds to the nearest integer and leaves it in the
// low byte.
__device__ __forceinline__ uint32_t quantise_near(float x, float scale, float inv) {
    const float v = x * inv, t = v + 12582912.0f;
    uint32_t q = __float_as_uint(t);
    if (fabsf(v - (t - 12582912.0f)) > 0.5f - 3.0517578125e-5f) q = __float_as_uint(x / scale + 12582912.0f);
    return q & 0xff;
}

// A CTA to a (touched page of a stream, head, side): blockIdx.x = page * 2 heads +
// 2 head + side, so that neighbours read the same tokens; blockIdx.y = stream.
// G 8-element groups a thread hold a page's new values.
template <typename T, int D, int G>
__global__ void __launch_bounds__(kThreads) append_kernel(const ufb_kv_cache c, int layer, const KvBatch b,
                                                          const ufb_heads k, const ufb_heads v, int* status) {
    __shared__ float top_warp[kThreads / 32];
    constexpr int per = D / 8;
    const int stream = blockIdx.y;
    const int sides = 2 * c.heads;
    const int at_page = blockIdx.x / sides, part = blockIdx.x - at_page * sides;
    const int head = part >> 1, side = part & 1;
    const int slot = b.slots[stream];
    const long long t0 = b.offsets[stream];
    const long long count = b.offsets[stream + 1] - t0;
    if (count <= 0) return;
    const bool first_thread = threadIdx.x == 0;
    if (slot < 0 || slot >= c.slots || t0 < 0 || t0 + count > b.tokens || count > b.max_new) {
        if (first_thread) atomicCAS(status, 0, kStatusIndex);
        return;
    }
    const int P = c.page_tokens;
    const long long length = c.lengths[slot], start = length - count;
    if (start < 0) {
        if (first_thread) atomicCAS(status, 0, kStatusIndex);
        return;
    }
    const long long entry = start / P + at_page;
    if (entry * P >= length) return;
    const int page = entry < c.table_width ? c.table[static_cast<long long>(slot) * c.table_width + entry] : -1;
    if (page < 0 || page >= c.pages) {
        if (first_thread) atomicCAS(status, 0, kStatusIndex);
        return;
    }
    const int lo = static_cast<int>(max(start - entry * P, 0ll));
    const int hi = static_cast<int>(min(length - entry * P, static_cast<long long>(P)));
    const long long tile = ((static_cast<long long>(layer) * c.pages + page) * 2 + side) * c.heads + head;
    int8_t* q = c.kv + tile * P * D;
    const float before = lo > 0 ? c.scale[tile] : 0.0f;

    const ufb_heads& x = side ? v : k;
    const T* in = static_cast<const T*>(x.data) + (t0 + entry * P + lo - start) * x.token_stride + head * x.head_stride;
    const int groups = (hi - lo) * per;
    float f[G][8];
    float top = 0.0f;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < G; ++i) {
        const int g = threadIdx.x + i * kThreads;
        if (g < groups) load8<T>(in + (g / per) * x.token_stride + (g % per) * 8, f[i]);
    }
#pragma unroll
    for (int i = 0; i < G; ++i) {
        if (threadIdx.x + i * kThreads < groups) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float m = fabsf(f[i][j]);
                const bool finite = m < __int_as_float(0x7f800000);
                odd |= !finite;
                top = fmaxf(top, finite ? m : 0.0f);
            }
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) top_warp[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) top = fmaxf(top, top_warp[i]);
    const float scale = fmaxf(before, top * (1.0f / 127.0f));
    const bool near = scale > 7.888609052210118e-31f && !odd;  // 2^-100
    const float inv = 1.0f / scale;

#pragma unroll
    for (int i = 0; i < G; ++i) {
        const int g = threadIdx.x + i * kThreads;
        if (g < groups) {
            uint32_t w[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    o[j] = near ? quantise_near(f[i][4 * h + j], scale, inv) : quantise(f[i][4 * h + j], scale);
                w[h] = __byte_perm(__byte_perm(o[0], o[1], 0x0040), __byte_perm(o[2], o[3], 0x0040), 0x5410);
            }
            *reinterpret_cast<uint2*>(q + lo * D + g * 8) = make_uint2(w[0], w[1]);
        }
    }
    if (scale != before || lo == 0) {
        const float ratio = before / scale;  // used for earlier tokens only: lo > 0, scale > 0
        for (int i = threadIdx.x; i < lo * D / 16; i += kThreads) {
            uint4 w = reinterpret_cast<uint4*>(q)[i];
            int8_t* o = reinterpret_cast<int8_t*>(&w);
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = static_cast<int8_t>(__float2int_rn(static_cast<float>(o[j]) * ratio));
            reinterpret_cast<uint4*>(q)[i] = w;
        }
        if (first_thread) c.scale[tile] = scale;
    }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&f)[4]);
template <>
__device__ __forceinline__ void store4<float>(float* p, const float (&f)[4]) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(f[0], f[1], f[2], f[3]));
}
template <>
__device__ __forceinline__ void store4<__half>(__half* p, const float (&f)[4]) {
    const __half2 a = __floats2half2_rn(f[0], f[1]), b = __floats2half2_rn(f[2], f[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* p, const float (&f)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// grid (heads * 2, listed pages): one (page, side, head) to a CTA
template <typename T>
__global__ void __launch_bounds__(kThreads) read_kernel(const ufb_kv_cache c, int layer, const int32_t* pages, T* out,
                                                        int* status) {
    const long long item = static_cast<long long>(blockIdx.x);
    const int sides = 2 * c.heads;
    const long long which = item / sides;
    const int part = static_cast<int>(item % sides);
    const int page = pages[which];
    const bool ok = page >= 0 && page < c.pages;
    if (!ok && threadIdx.x == 0) atomicCAS(status, 0, kStatusIndex);
    const int n = c.page_tokens * c.head_dim / 4;
    const long long tile = (static_cast<long long>(layer) * c.pages + (ok ? page : 0)) * sides + part;
    const float scale = c.scale[tile];
    const uint32_t* q = reinterpret_cast<const uint32_t*>(c.kv) + tile * n;
    T* o = out + item * n * 4;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint32_t w = q[i];
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            f[j] = ok ? static_cast<float>(static_cast<int8_t>(w >> (8 * j))) * scale : __int_as_float(0x7fffffff);
        store4<T>(o + i * 4, f);
    }
}

template <typename T, int D>
cudaError_t append(const ufb_kv_cache& c, int layer, const KvBatch& b, const ufb_heads& k, const ufb_heads& v,
                   int* status, cudaStream_t s) {
    // max_new tokens reach at most this many pages, wherever the first one falls
    const long long touched = (static_cast<long long>(b.max_new) + c.page_tokens - 2) / c.page_tokens + 1;
    const long long blocks = touched * 2 * c.heads;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(blocks), b.n);
    // as many registers as a page's new values (or, with few, the call's) need
    const int tokens = b.max_new < c.page_tokens ? b.max_new : c.page_tokens;
    const int groups = (tokens * (D / 8) + kThreads - 1) / kThreads;
    if (groups <= 1) append_kernel<T, D, 1><<<grid, kThreads, 0, s>>>(c, layer, b, k, v, status);
    else if (groups <= 2) append_kernel<T, D, 2><<<grid, kThreads, 0, s>>>(c, layer, b, k, v, status);
    else if (groups <= 4) append_kernel<T, D, 4><<<grid, kThreads, 0, s>>>(c, layer, b, k, v, status);
    else append_kernel<T, D, 8><<<grid, kThreads, 0, s>>>(c, layer, b, k, v, status);
    return cudaGetLastError();
}

template <typename T>
cudaError_t append_dim(const ufb_kv_cache& c, int layer, const KvBatch& b, const ufb_heads& k, const ufb_heads& v,
                       int* status, cudaStream_t s) {
    return c.head_dim == 64 ? append<T, 64>(c, layer, b, k, v, status, s) : append<T, 128>(c, layer, b, k, v, status, s);
}

template <typename T>
cudaError_t read(const ufb_kv_cache& c, int layer, const int32_t* pages, long long n, void* out, int* status,
                 cudaStream_t s) {
    const long long items = n * 2 * c.heads;
    if (items > 0x7fffffffll) return cudaErrorInvalidValue;
    read_kernel<T><<<static_cast<unsigned>(items), kThreads, 0, s>>>(c, layer, pages, static_cast<T*>(out), status);
    return cudaGetLastError();
}

}  // namespace

cudaError_t kv_append(const ufb_kv_cache& c, int layer, const KvBatch& b, int dtype, const ufb_heads& k,
                      const ufb_heads& v, int* status, cudaStream_t s) {
    if (dtype == UFB_F32) return append_dim<float>(c, layer, b, k, v, status, s);
    if (dtype == UFB_F16) return append_dim<__half>(c, layer, b, k, v, status, s);
    return append_dim<__nv_bfloat16>(c, layer, b, k, v, status, s);
}

cudaError_t kv_read(const ufb_kv_cache& c, int layer, const int32_t* pages, long long n, int dtype, void* out,
                    int* status, cudaStream_t s) {
    if (dtype == UFB_F32) return read<float>(c, layer, pages, n, out, status, s);
    if (dtype == UFB_F16) return read<__half>(c, layer, pages, n, out, status, s);
    return read<__nv_bfloat16>(c, layer, pages, n, out, status, s);
}

}  // namespace ufb
