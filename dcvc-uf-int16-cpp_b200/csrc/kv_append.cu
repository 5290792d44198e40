// New keys and values into the 8-bit cache (ufb_kv_append) and the values that
// pages stand for (ufb_kv_read).
//
// One scale serves a page, head and side, so a team of threads takes one (page,
// head, side) that a stream's new tokens reach: it finds max |x| over the new
// tokens of the page, s' = max(s, max * (1 / 127)), requantises the earlier tokens
// only when s' grew, and writes the new integers.  The new values stay in
// registers between the two steps, so HBM sees each input once and each byte of
// the cache at most once: the call is bound by those bytes, or by its latency
// when every stream brings one token.  32640 tokens of 8 heads of 128: 53 us in float16
// (0.57 of a copy's rate), 64 in bfloat16, 68 in float32 (0.75); their pages read back to
// float32 in 55 us (0.94).  Neither the issue slots (53 %) nor the ALU (39 %) are full in
// float16: a team loads, joins its maximum, stores and ends, with no loads of a next
// tile under way.  One token of 64 streams: 11.7 us, 13.5 when it makes the scales grow
// and the earlier tokens of its pages are requantised.
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

// Eight elements as they lie in memory.
template <typename T>
struct Raw {
    uint4 v;
};
template <>
struct Raw<float> {
    uint4 v, w;
};

template <typename T>
__device__ __forceinline__ Raw<T> load8(const T* p) {
    Raw<T> r;
    r.v = *reinterpret_cast<const uint4*>(p);
    return r;
}
template <>
__device__ __forceinline__ Raw<float> load8<float>(const float* p) {
    return {reinterpret_cast<const uint4*>(p)[0], reinterpret_cast<const uint4*>(p)[1]};
}

__device__ __forceinline__ void unpack8(const Raw<float>& r, float (&f)[8]) {
    f[0] = __uint_as_float(r.v.x), f[1] = __uint_as_float(r.v.y), f[2] = __uint_as_float(r.v.z);
    f[3] = __uint_as_float(r.v.w), f[4] = __uint_as_float(r.w.x), f[5] = __uint_as_float(r.w.y);
    f[6] = __uint_as_float(r.w.z), f[7] = __uint_as_float(r.w.w);
}
__device__ __forceinline__ void unpack8(const Raw<__half>& r, float (&f)[8]) {
    const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
}
__device__ __forceinline__ void unpack8(const Raw<__nv_bfloat16>& r, float (&f)[8]) {
    const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// The largest magnitude so far, NaN when any value was: of 32-bit values, or of
// both halves of 16-bit pairs.
__device__ __forceinline__ void top_of(uint32_t& top, const Raw<float>& r) {
    const uint32_t w[8] = {r.v.x, r.v.y, r.v.z, r.v.w, r.w.x, r.w.y, r.w.z, r.w.w};
    // magnitudes order like their bits without the sign, infinities and NaN last
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, w[i] & 0x7fffffffu);
}
__device__ __forceinline__ void top_of(uint32_t& top, const Raw<__half>& r) {
    const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 m = __hmax2_nan(*reinterpret_cast<const __half2*>(&top), __habs2(*reinterpret_cast<const __half2*>(&w[i])));
        top = *reinterpret_cast<const uint32_t*>(&m);
    }
}
__device__ __forceinline__ void top_of(uint32_t& top, const Raw<__nv_bfloat16>& r) {
    const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&top),
                                             __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])));
        top = *reinterpret_cast<const uint32_t*>(&m);
    }
}
template <typename T>
__device__ __forceinline__ float top_value(uint32_t top);
template <>
__device__ __forceinline__ float top_value<float>(uint32_t top) { return __uint_as_float(top); }
template <>
__device__ __forceinline__ float top_value<__half>(uint32_t top) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(max(top & 0xffff, top >> 16))));
}
template <>
__device__ __forceinline__ float top_value<__nv_bfloat16>(uint32_t top) {
    return __uint_as_float(max(top & 0xffff, top >> 16) << 16);
}

// rint(x / scale) of eight values, saturated, one IEEE operation after another;
// any float values.
__device__ __noinline__ uint2 quantise_exact(float4 a, float4 b, float scale) {
    const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint32_t w[2] = {0, 0};
#pragma unroll 1
    for (int j = 0; j < 8; ++j) {
        const float v = scale == 0.0f ? 0.0f : x[j] / scale;
        const int q = v == v ? __float2int_rn(fminf(fmaxf(v, -127.0f), 127.0f)) : 0;
        w[j >> 2] |= (static_cast<uint32_t>(q) & 0xff) << (8 * (j & 3));
    }
    return make_uint2(w[0], w[1]);
}

// The same by products with inv = 1 / scale, for finite x with |x / scale| <=
// 127.5 and a scale above 2^-100: x inv is within 127 * 3 * 2^-24 < 2^-15 of the
// quotient, so its nearest integer is the quotient's unless a tie is that close.
// false: one is, and goes to quantise_ties.  Adding 1.5 * 2^23 rounds to the
// nearest integer and leaves it in the low byte.
constexpr float kRound = 12582912.0f, kNoTie = 0.5f - 3.0517578125e-5f;
__device__ __forceinline__ bool quantise_near(const float (&x)[8], float inv, uint2& out) {
    uint32_t q[8];
    float far = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float v = x[j] * inv, t = v + kRound;
        far = fmaxf(far, fabsf(v - (t - kRound)));
        q[j] = __float_as_uint(t);
    }
    out.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
    out.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
    return far <= kNoTie;
}

// quantise_near's integers, those of them at a tie by division (16-bit inputs meet
// ties often: half the largest value is one).
__device__ __noinline__ uint2 quantise_ties(float4 a, float4 b, float scale, float inv) {
    const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float v = x[j] * inv;
        float t = v + kRound;
        if (fabsf(v - (t - kRound)) > kNoTie) t = x[j] / scale + kRound;
        w[j >> 2] |= (__float_as_uint(t) & 0xff) << (8 * (j & 3));
    }
    return make_uint2(w[0], w[1]);
}

// `team` threads (a power of two, 32 to 256) to a tile (touched page of a stream,
// head, side); tile = page * 2 heads + 2 head + side, so that neighbours read the
// same tokens; blockIdx.y = stream.  G 8-element groups a thread hold a tile's new
// values: what a thread does once for its tile costs as much as about 20 elements.
template <typename T, int D, int G>
__global__ void __launch_bounds__(kThreads) append_kernel(const ufb_kv_cache c, int layer, const KvBatch b,
                                                          const ufb_heads k, const ufb_heads v, int tiles, int team,
                                                          int* status) {
    __shared__ float top_warp[kThreads / 32];
    constexpr int per = D / 8;
    const int stream = blockIdx.y;
    const int sides = 2 * c.heads;
    const int tile_index = (blockIdx.x * kThreads + threadIdx.x) / team, lane = threadIdx.x & (team - 1);
    const int at_page = tile_index / sides, part = tile_index - at_page * sides;
    const int head = part >> 1, side = part & 1;
    const int slot = b.slots[stream];
    const int t0 = b.offsets[stream], count = b.offsets[stream + 1] - t0;
    if (count <= 0) return;
    const int P = c.page_tokens, shift = 31 - __clz(P);  // a power of two
    int page = -1, lo = 0, hi = 0;
    long long first = 0;   // the tile's first new token
    if (slot < 0 || slot >= c.slots || t0 < 0 || t0 + static_cast<long long>(count) > b.tokens || count > b.max_new ||
        c.lengths[slot] < count) {
        if (threadIdx.x == 0) atomicCAS(status, 0, kStatusIndex);
    } else if (kv_refused(c)[slot]) {
        // no room was made for them: the stream's last tokens are stored ones, maybe on shared pages
        if (threadIdx.x == 0) atomicCAS(status, 0, kStatusPages);
    } else if (tile_index < tiles) {
        const int length = c.lengths[slot], start = length - count;
        const int entry = (start >> shift) + at_page;
        const long long begin = static_cast<long long>(entry) << shift;
        if (begin < length) {
            page = entry < c.table_width ? c.table[static_cast<long long>(slot) * c.table_width + entry] : -1;
            if (page < 0 || page >= c.pages) {
                page = -1;
                if (lane == 0) atomicCAS(status, 0, kStatusIndex);
            } else {
                lo = static_cast<int>(max(start - begin, 0ll));
                hi = static_cast<int>(min(length - begin, static_cast<long long>(P)));
                first = t0 + begin + lo - start;
            }
        }
    }
    const long long tile = ((static_cast<long long>(layer) * c.pages + (page < 0 ? 0 : page)) * 2 + side) * c.heads + head;
    int8_t* q = c.kv + tile * P * D;
    const float before = lo > 0 ? c.scale[tile] : 0.0f;

    const ufb_heads& x = side ? v : k;
    const T* in = static_cast<const T*>(x.data) + first * x.token_stride + head * x.head_stride +
                  (lane / per) * x.token_stride + (lane % per) * 8;
    const int groups = (hi - lo) * per;
    const long long step = (team / per) * x.token_stride;   // team is a multiple of per
    Raw<T> raw[G];
#pragma unroll
    for (int i = 0; i < G; ++i)
        if (lane + i * team < groups) raw[i] = load8<T>(in + i * step);
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < G; ++i)
        if (lane + i * team < groups) top_of(bits, raw[i]);
    float top = top_value<T>(bits);
    const bool odd = !(top < __int_as_float(0x7f800000));
    if (odd) {
        // not all finite: the largest of those that are
        top = 0.0f;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            if (lane + i * team >= groups) continue;
            float f[8];
            unpack8(raw[i], f);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fabsf(f[j]) < __int_as_float(0x7f800000) ? fmaxf(top, fabsf(f[j])) : top;
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (team > 32) {
        if ((threadIdx.x & 31) == 0) top_warp[threadIdx.x >> 5] = top;
        __syncthreads();
        const int warp0 = (threadIdx.x & ~(team - 1)) >> 5;
        for (int i = 0; i < team / 32; ++i) top = fmaxf(top, top_warp[warp0 + i]);
    }
    if (page < 0) return;
    const float scale = fmaxf(before, top * (1.0f / 127.0f));
    const bool near = scale > 7.888609052210118e-31f && !odd;  // 2^-100
    const float inv = 1.0f / scale;

#pragma unroll
    for (int i = 0; i < G; ++i) {
        const int g = lane + i * team;
        if (g < groups) {
            float f[8];
            unpack8(raw[i], f);
            uint2 w;
            const float4 a = make_float4(f[0], f[1], f[2], f[3]), z = make_float4(f[4], f[5], f[6], f[7]);
            if (!near) w = quantise_exact(a, z, scale);
            else if (!quantise_near(f, inv, w)) w = quantise_ties(a, z, scale, inv);
            *reinterpret_cast<uint2*>(q + lo * D + g * 8) = w;
        }
    }
    if (scale != before || lo == 0) {
        const float ratio = before / scale;  // used for earlier tokens only: lo > 0, scale > 0
        for (int i = lane; i < lo * D / 16; i += team) {
            uint4 w = reinterpret_cast<uint4*>(q)[i];
            int8_t* o = reinterpret_cast<int8_t*>(&w);
#pragma unroll 4
            for (int j = 0; j < 16; ++j) o[j] = static_cast<int8_t>(__float2int_rn(static_cast<float>(o[j]) * ratio));
            reinterpret_cast<uint4*>(q)[i] = w;
        }
        if (lane == 0) c.scale[tile] = scale;
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
    const long long tiles = touched * 2 * c.heads;
    if (tiles > 0x7fffffffll / 256) return cudaErrorInvalidValue;
    // 8 groups a thread (a page of 64 tokens x 128: 54 us for 32640 float16 tokens of 8
    // heads; 4 groups 58, 16 groups 87 us); calls of few tokens need their latency: 1
    constexpr int kMost = 8;
    const int tokens = b.max_new < c.page_tokens ? b.max_new : c.page_tokens;
    const int groups = tokens * (D / 8);
    const int most = groups <= kThreads ? 1 : kMost;
    int team = 32;
    while (team * most < groups) team *= 2;
    const dim3 grid(static_cast<unsigned>((tiles * team + kThreads - 1) / kThreads), b.n);
    if (most == 1)
        append_kernel<T, D, 1><<<grid, kThreads, 0, s>>>(c, layer, b, k, v, static_cast<int>(tiles), team, status);
    else
        append_kernel<T, D, kMost><<<grid, kThreads, 0, s>>>(c, layer, b, k, v, static_cast<int>(tiles), team, status);
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
