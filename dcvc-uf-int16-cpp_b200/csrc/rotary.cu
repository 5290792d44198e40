// Rotary positions over several axes (ufb_rotary).
//
// A head's pair j = (a, b) belongs to one axis and turns by the angle of its
// token's position there:  a' = a c - b s,  b' = a s + b c  (inverse: s -> -s).
// (c, s) come from a table of float pairs, one row for each position of an
// axis, computed once in 64 bits: large positions cost no accuracy and the
// kernel no sine.
//
// Bound by HBM: every element is read once and written once (130560 tokens x 20
// heads of 128 in bfloat16: 231 - 236 us, 5.7 TB/s, 0.88 of a plain copy's rate).  A
// thread owns one 16-byte column of a head (8 or 4 elements), reads that column's
// (c, s) once and applies them to the heads of the same token, since the table
// bytes of a column are four times its data in 16 bits (one to four heads a thread:
// 855 us).  In the half layout the partner column lies n elements away: where n is
// whole columns a thread reads and writes both members; otherwise the partner is
// read as the two aligned columns around it and shifted into place, so every access
// stays 16 bytes wide whatever the pair counts are: the same tokens with 61 or 63 pairs
// take 648 us (0.32: a column and the two around its partner are read, and the members of
// a pair belong to two threads; which of it bounds has not been measured), in float32 385
// us for 65280 tokens (0.54; whole columns 216 us, 0.96).  Interleaved: 291 us in bfloat16
// (0.71), 421 in float32 (0.98).
#include "attention.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ufb {

namespace {

constexpr int kThreads = 256;

template <typename T>
struct Column;  // 16 bytes of T as floats

template <>
struct Column<float> {
    static constexpr int n = 4;
    static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[4]) {
        f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y);
        f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};

template <>
struct Column<__half> {
    static constexpr int n = 8;
    static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = p.x, f[2 * i + 1] = p.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

template <>
struct Column<__nv_bfloat16> {
    static constexpr int n = 8;
    static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// 16 bytes that start at byte `at` (a multiple of the element size, possibly
// negative or past the row) of a row of `columns` aligned 16-byte columns;
// bytes outside the row are undefined and never used by the caller.
__device__ __forceinline__ uint4 window16(const uint4* row, int at, int columns) {
    const int first = at >> 4, rest = at & 15;
    const uint4 lo = row[min(max(first, 0), columns - 1)];
    if (rest == 0) return lo;
    const uint4 hi = row[min(max(first + 1, 0), columns - 1)];
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (rest & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (rest & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    if (rest & 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

enum Mode { kHalfPairs, kHalf, kInterleaved };

// Thread = (token, column), for heads [blockIdx.y * per, + per).  Columns of a head:
// kHalfPairs: n / N columns that hold the first of both members of N pairs (the
// second ones are n elements on), then the columns past 2 n; else all D / N.
template <typename T, Mode MODE>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a, int columns, int per, int* status) {
    constexpr int N = Column<T>::n;
    const unsigned slots = kThreads / columns;    // tokens of a block
    const unsigned slot = threadIdx.x / columns;
    const long long token = static_cast<long long>(blockIdx.x) * slots + slot;
    if (slot >= slots || token >= a.tokens) return;
    const int index = threadIdx.x - slot * columns;
    const int paired = a.pairs / N;
    const int col = MODE == kHalfPairs && index >= paired ? index + paired : index;
    const int e0 = col * N;

    // this column's (cos, sin): out = x c + partner s, s with the member's and the direction's sign
    float c[N], s[N];
    bool bad = false;
    int row[UFB_ROTARY_MAX_AXES];
#pragma unroll
    for (int ax = 0; ax < UFB_ROTARY_MAX_AXES; ++ax) {
        row[ax] = 0;
        if (ax < a.axes) {
            const int p = a.positions[token * a.axes + ax];
            bad |= p < 0 || p >= a.extent[ax];
            // a table holds less than 2^31 entries
            row[ax] = static_cast<int>(a.base[ax]) + (bad ? 0 : p) * (a.first[ax + 1] - a.first[ax]) - a.first[ax];
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = e0 + i;
        const int pair = MODE == kInterleaved ? e >> 1 : (e < a.pairs ? e : e - a.pairs);
        const bool second = MODE == kInterleaved ? (e & 1) : e >= a.pairs;
        c[i] = 1.0f, s[i] = -0.0f;  // x * 1 + 0 * -0 is x, zeros of both signs included
        if (pair < a.pairs) {
            int r = row[0];
#pragma unroll
            for (int ax = 1; ax < UFB_ROTARY_MAX_AXES; ++ax)
                if (ax < a.axes && pair >= a.first[ax]) r = row[ax];
            const float2 t = __ldg(a.table + r + pair);
            c[i] = t.x;
            s[i] = second != (a.inverse != 0) ? t.y : -t.y;
        }
        if (bad) c[i] = s[i] = __int_as_float(0x7fffffff);
    }
    if (bad && index == 0 && blockIdx.y == 0) atomicCAS(status, 0, kStatusPosition);

    const int vecs = a.head_dim / N;
    const int shift = a.pairs * static_cast<int>(sizeof(T));
    const bool tail = MODE == kHalfPairs && index >= paired;
    const bool plus = e0 < a.pairs, minus = e0 + N > a.pairs && e0 < 2 * a.pairs;
    const int total = a.x[0].heads + (a.count > 1 ? a.x[1].heads : 0);
    const int begin = blockIdx.y * per, end = min(total, begin + per);
    // all heads of one tensor, four at a time in flight
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int h0 = t ? max(begin - a.x[0].heads, 0) : begin;
        const int h1 = t ? end - a.x[0].heads : min(end, a.x[0].heads);
        const T* in = static_cast<const T*>(a.x[t].data) + token * a.x[t].token_stride + h0 * a.x[t].head_stride;
        T* out = static_cast<T*>(a.out[t].data) + token * a.out[t].token_stride + h0 * a.out[t].head_stride;
#pragma unroll 4
        for (int h = h0; h < h1; ++h, in += a.x[t].head_stride, out += a.out[t].head_stride) {
            const uint4* from = reinterpret_cast<const uint4*>(in);
            uint4* to = reinterpret_cast<uint4*>(out);
            float x[N], y[N], r[N];
            const uint4 own = __ldcs(from + col);
            Column<T>::unpack(own, x);
            if (MODE == kHalfPairs) {
                if (tail) {
                    __stcs(to + col, bad ? make_uint4(~0u, ~0u, ~0u, ~0u) : own);
                } else {
                    Column<T>::unpack(__ldcs(from + col + paired), y);
                    float q[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        r[i] = x[i] * c[i] + y[i] * s[i];
                        q[i] = y[i] * c[i] - x[i] * s[i];
                    }
                    __stcs(to + col, Column<T>::pack(r));
                    __stcs(to + col + paired, Column<T>::pack(q));
                }
                continue;
            }
            if (MODE == kHalf) {
                uint4 up = make_uint4(0, 0, 0, 0), down = make_uint4(0, 0, 0, 0);
                if (plus) up = window16(from, col * 16 + shift, vecs);
                if (minus) down = window16(from, col * 16 - shift, vecs);
                float u[N], d[N];
                Column<T>::unpack(up, u);
                Column<T>::unpack(down, d);
#pragma unroll
                for (int i = 0; i < N; ++i) y[i] = e0 + i < a.pairs ? u[i] : (e0 + i < 2 * a.pairs ? d[i] : 0.0f);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) y[i] = (e0 + i) >> 1 < a.pairs ? x[i ^ 1] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = x[i] * c[i] + y[i] * s[i];
            __stcs(to + col, Column<T>::pack(r));
        }
    }
}

template <typename T, Mode MODE>
cudaError_t launch(const RotaryArgs& a, int columns, int sms, int* status, cudaStream_t s) {
    const int heads = a.x[0].heads + (a.count > 1 ? a.x[1].heads : 0);
    const unsigned slots = kThreads / columns;
    const long long blocks = (a.tokens + slots - 1) / slots;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
    // All heads to a thread share its table values; while that leaves SMs without
    // two blocks, the heads are spread over more blocks.
    long long groups = (2ll * sms + blocks - 1) / blocks;
    if (groups > heads) groups = heads;
    const int per = static_cast<int>((heads + groups - 1) / groups);
    rotary_kernel<T, MODE><<<dim3(static_cast<unsigned>(blocks), (heads + per - 1) / per), kThreads, 0, s>>>(a, columns, per, status);
    return cudaGetLastError();
}

template <typename T>
cudaError_t dispatch(const RotaryArgs& a, int sms, int* status, cudaStream_t s) {
    constexpr int N = Column<T>::n;
    const int vecs = a.head_dim / N;
    if (a.layout == UFB_ROTARY_INTERLEAVED) return launch<T, kInterleaved>(a, vecs, sms, status, s);
    // pair counts that are whole columns: a thread reads and writes both members
    if (a.pairs % N == 0) return launch<T, kHalfPairs>(a, vecs - a.pairs / N, sms, status, s);
    return launch<T, kHalf>(a, vecs, sms, status, s);
}

}  // namespace

cudaError_t rotary(const RotaryArgs& a, int dtype, int sms, int* status, cudaStream_t s) {
    if (dtype == UFB_F32) return dispatch<float>(a, sms, status, s);
    if (dtype == UFB_F16) return dispatch<__half>(a, sms, status, s);
    return dispatch<__nv_bfloat16>(a, sms, status, s);
}

}  // namespace ufb
