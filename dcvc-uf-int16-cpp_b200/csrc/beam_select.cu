// The best continuations of each stream's beams (ufb_beam_select):
//
//   total[k][v] = f32(scores[k] + (logits[k][v] - ln sum_u exp logits[k][u])),
//
// the `count` best of a stream by total, then lower beam, larger logit, lower token.
//
// Bound by the bytes of the logits, which are read once from memory, and for 16-bit
// logits by the loop's instructions and what its warps wait for.  Two launches.  In the first a CTA
// takes a part of one row: it sums exp and finds the part's `count` largest logits.  With
// nothing between the loads but arithmetic every thread keeps its largest value and where
// it was; from these a threshold follows that at least `count` values reach and few more
// do, and the vectors that reach it are looked through again, from shared memory or
// cache: no running list and no barrier is in the loop.  The second launch, a CTA to a
// stream, joins the sums of each row's parts and finds the best of the parts' candidates
// in the same way.
//
// The order of candidates of different beams hangs on the rows' ln sum exp, and totals
// are next to each other: sums are in 64 bits, of exponentials good to 2^-27.
//
// Measured on 148 SMs, on the device: 64 streams x 8 beams x 32768 tokens of bfloat16 24.5 us
// (11.1 million warp instructions in the first launch, 13.5 a value in the loop, 900 a warp
// besides; 55 % of the issue slots, where the exponentials alone reach 6.7 values a cycle and
// SM), 32 x 16 x 131072 with a fifth of the beams ended 61 us; 24 x 5 x 65537 of float32 18 us;
// one stream of 4 x 256 tokens 6 us.  The second launch takes 5 us of each.
#include "beam.h"

#include "capi_util.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ufb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBatch = 4;         // vectors of a thread that are loaded together; two batches are under way
constexpr int kStretches = 8;     // of a thread's batches, whose largest values are kept
constexpr int kFound = 1024;      // candidates that are counted against each other
constexpr int kMostParts = 32;    // of a row
constexpr int kAhead = 4;         // candidates of a thread in the join that are loaded beside the sums
constexpr int kPartCost = 28;     // of a part, in values of a thread
// Sums are of exp itself while the part's largest logit is inside this, else of exp(x - largest).
constexpr float kPlain = 600.0f;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Order of floats as unsigned integers; equal zeros are equal.  0: none (below -infinity).
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
constexpr uint32_t kNone = 0x007fffffu;   // ordered(-infinity): no candidate is at or below it

// exp in two parts: 2^(k / 16) for k = rint(16 x / ln 2), from a table and the exponent,
// times 1 + p for the rest |r| <= a = ln 2 / 32.  k comes out of one multiply-add whose sum
// has no room for a fraction; r of two, whose products are exact.  p = r + (1/2 + a^2 / 24)
// r^2 + r^3 / 6: the series, whose r^4 / 24 is replaced by the parabola nearest to it,
// (a^2 r^2 - a^4 / 8) / 24; the constant is in the table (1 + p of it moves by 2^-57).  That
// errs by a^4 / 192 < 2^-29.6, the next term by 2^-34; three roundings of values below 2^-5
// add 3 * 2^-30 at most: 2^-27 in all.  The two parts are added up in 64 bits, T and T p
// apart.  16 entries of 64 bits lie one to each pair of shared memory's banks: a warp's
// look-up never conflicts.  x within [-700, 700] or NaN.
constexpr int kExpTable = 16;
constexpr float kExpScale = 23.083120654223414f;      // 16 / ln 2
constexpr float kExpRound = 12582912.0f;              // 1.5 * 2^23
constexpr double kExpStep = 0.043321698784996582;     // ln 2 / 16
constexpr float kExpHigh = static_cast<float>(kExpStep), kExpLow = static_cast<float>(kExpStep - static_cast<double>(kExpHigh));

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Of a vector: its largest value (NaN left out); its values, none below -700 and NaN kept;
// its i-th two values.  16-bit values are compared two at a time as they lie.
template <typename T>
struct Values;
template <>
struct Values<float> {
    static constexpr uint32_t kLowest = 0xff800000u;   // -infinity, as often as a word holds it
    static __device__ __forceinline__ float top(const uint4& w) {
        return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
    }
    static __device__ __forceinline__ uint32_t raise(uint32_t v) {
        return __float_as_uint(max_nan(__uint_as_float(v), -700.0f));
    }
    static __device__ __forceinline__ float2 two(const uint4& w, int i) {
        return i == 0 ? make_float2(__uint_as_float(w.x), __uint_as_float(w.y)) : make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
    }
};
template <>
struct Values<__half> {
    static constexpr uint32_t kLowest = 0xfc00fc00u;
    static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float top(const uint4& w) {
        const uint32_t m = most(most(w.x, w.y), most(w.z, w.w));
        const float2 f = __half22float2(reinterpret_cast<const __half2&>(m));
        return fmaxf(f.x, f.y);
    }
    static __device__ __forceinline__ uint32_t raise(uint32_t v) {
        uint32_t r;
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0xe178e178u));   // -700
        return r;
    }
    static __device__ __forceinline__ float2 two(const uint4& w, int i) {
        const uint32_t v = i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
        return __half22float2(reinterpret_cast<const __half2&>(v));
    }
};
template <>
struct Values<__nv_bfloat16> {
    static constexpr uint32_t kLowest = 0xff80ff80u;
    static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float top(const uint4& w) {
        const uint32_t m = most(most(w.x, w.y), most(w.z, w.w));
        return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t raise(uint32_t v) {
        uint32_t r;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0xc42fc42fu));   // -700
        return r;
    }
    static __device__ __forceinline__ float2 two(const uint4& w, int i) {
        const uint32_t v = i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
};

// Pairs of 32-bit floats.
__device__ __forceinline__ unsigned long long pair(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(unsigned long long v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// What add_exp multiplies by, as pairs: kept in registers, not made again for each value.
struct ExpPairs {
    unsigned long long scale, round, back, high, low, c3, c2;
    __device__ __forceinline__ ExpPairs() {
        auto twice = [](float v) {
            unsigned long long r;
            asm volatile("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(v));
            return r;
        };
        scale = twice(kExpScale), round = twice(kExpRound), back = twice(-kExpRound);
        high = twice(-kExpHigh), low = twice(-kExpLow);
        c3 = twice(1.0f / 6), c2 = twice(static_cast<float>(0.5 + kExpStep * kExpStep / 96));
    }
};

// sums[0, 1] += 2^(k / 16), sums[2, 3] += 2^(k / 16) p of x and y.
// table: its address in shared memory.
__device__ __forceinline__ void add_exp(uint32_t table, const ExpPairs& c, float x, float y, double (&sums)[4]) {
    const unsigned long long v = pair(x, y);
    const unsigned long long t = fma2(v, c.scale, c.round);
    const unsigned long long k = add2(t, c.back);
    unsigned long long r = fma2(k, c.high, v);
    r = fma2(k, c.low, r);
    const unsigned long long q = fma2(r, c.c3, c.c2);
    const float2 p = unpair(fma2(mul2(r, r), q, r));
    const float2 bits = unpair(t);
    auto power = [&](float b) {
        // k / 16 comes to the exponent, k % 16 below it, where the table's entry is less by
        // that; kExpRound's own bits leave with the shift
        const uint32_t w = __float_as_uint(b);
        uint32_t low, high;
        asm("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(low), "=r"(high) : "r"(table + (w & (kExpTable - 1)) * 8));
        return __hiloint2double(static_cast<int>(high + (w << 16)), static_cast<int>(low));
    };
    const double a = power(bits.x), b = power(bits.y);
    sums[0] += a;
    sums[1] += b;
    sums[2] = fma(a, static_cast<double>(p.x), sums[2]);
    sums[3] = fma(b, static_cast<double>(p.y), sums[3]);
}

// A part of one row.
struct Piece {
    const void* base;      // 16-byte boundary at or before the row's first element
    int head;              // elements between them
    int v0, v1;            // vectors
};

template <typename T>
constexpr int kElems = 16 / static_cast<int>(sizeof(T));   // of a vector
// CTAs of an SM: for 16-bit values 4 with 64 registers a thread measured better (64 streams x
// 8 beams x 32768 tokens 24.0 us, 29.4 with 3), for 32-bit ones 3 (24 x 5 x 65537 19.6, 22.2
// with 4).
template <typename T>
constexpr int kCtas = sizeof(T) == 4 ? 3 : 4;
template <typename T>
struct Vec {
    T v[kElems<T>];
};

// Vector i of a row; what lies outside of it is -infinity.
template <typename T>
__device__ __noinline__ uint4 load(const Piece& p, int vocab, int i) {
    constexpr int E = kElems<T>;
    const T* at = static_cast<const T*>(p.base) + static_cast<long long>(i) * E;
    const int first = i * E - p.head;
    if (first >= 0 && first <= vocab - E) return __ldg(reinterpret_cast<const uint4*>(at));
    uint4 w;
    Vec<T>& v = reinterpret_cast<Vec<T>&>(w);
#pragma unroll
    for (int e = 0; e < E; ++e) v.v[e] = first + e >= 0 && first + e < vocab ? at[e] : static_cast<T>(-INFINITY);
    return w;
}

// What a part leaves in the scratch, followed by `count` candidates: (ordered logit, ~token),
// falling, 0 where there are fewer.
struct Part {
    double ref, sum;       // sum exp(x - ref); ref -infinity: nothing there
};
__host__ __device__ inline long long part_bytes(int count) { return sizeof(Part) + 8ll * (count + (count & 1)); }

struct Shared {
    alignas(128) double powers[kExpTable];
    union {
        unsigned long long found[kFound];
        float tops[kStretches][kThreads];   // before: the largest value of each stretch of a thread's vectors
    };
    unsigned long long limit[kWarps];
    double part[kWarps];
    float top[kWarps];
    uint16_t reach[kStretches * kThreads];  // stretches that reach the threshold
    int reaches, finds;
    uint4 ring[2 * kBatch][kThreads];
};

// Sum of v over the block, the same in all threads.
__device__ __noinline__ double block_sum(Shared& sm, double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) sm.part[threadIdx.x / 32] = v;
    __syncthreads();
    v = sm.part[0];
    for (int w = 1; w < kWarps; ++w) v += sm.part[w];
    return v;
}

// sum exp(x - ref) of a part whose exp leaves the range of 64 bits.
template <typename T>
__device__ __noinline__ double far_sum(Shared& sm, const Piece& p, int vocab, double ref) {
    double sum = 0.0;
    for (int i = p.v0 + threadIdx.x; i < p.v1; i += kThreads) {
        const uint4 w = load<T>(p, vocab, i);
        const Vec<T>& v = reinterpret_cast<const Vec<T>&>(w);
#pragma unroll 1
        for (int e = 0; e < kElems<T>; ++e) sum += exp(static_cast<double>(to_float(v.v[e])) - ref);
    }
    return block_sum(sm, sum);
}

// Many equal values, or the large ones of the part in few threads: the count-th largest key
// bit by bit, then the `count` keys that reach it to sm.found.
template <typename T>
__device__ __noinline__ void find_by_bits(Shared& sm, const Piece& p, int vocab, int count) {
    auto each = [&](auto use) {
        for (int i = p.v0 + threadIdx.x; i < p.v1; i += kThreads) {
            const uint4 w = load<T>(p, vocab, i);
            const Vec<T>& v = reinterpret_cast<const Vec<T>&>(w);
#pragma unroll
            for (int e = 0; e < kElems<T>; ++e) {
                const float x = to_float(v.v[e]);
                const uint32_t o = ordered(x);
                if (o > kNone && x == x) use(static_cast<unsigned long long>(o) << 32 | (0xffffffffu - static_cast<uint32_t>(i * kElems<T> - p.head + e)));
            }
        }
    };
    unsigned long long least = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const unsigned long long trial = least | 1ull << bit;
        __syncthreads();
        if (threadIdx.x == 0) sm.finds = 0;
        __syncthreads();
        int n = 0;
        each([&](unsigned long long key) { n += key >= trial; });
        n = __reduce_add_sync(0xffffffffu, n);
        if (threadIdx.x % 32 == 0) atomicAdd(&sm.finds, n);
        __syncthreads();
        if (sm.finds >= count) least = trial;
    }
    __syncthreads();
    if (threadIdx.x == 0) sm.finds = 0;
    __syncthreads();
    each([&](unsigned long long key) {
        if (key >= least) sm.found[atomicAdd(&sm.finds, 1)] = key;
    });
    __syncthreads();
}

__device__ __forceinline__ void copy_async(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ uint4 load_shared(uint32_t from) {
    uint4 w;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(from));
    return w;
}
__device__ __forceinline__ void commit_async() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_async() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Beams at -infinity and NaN lead nowhere, ended ones stay as they are: their rows are not read.
__device__ __forceinline__ bool row_is_read(const BeamSelectArgs& a, long long row) {
    return a.scores[row] > -INFINITY && !(a.finished && a.finished[row]);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, kCtas<T>) part_kernel(const BeamSelectArgs a, int parts, int part_vecs) {
    constexpr int E = kElems<T>;
    extern __shared__ __align__(128) unsigned char raw[];
    Shared& sm = *reinterpret_cast<Shared*>(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int row = blockIdx.x / parts, stream = row / a.beams, beam = row - stream * a.beams;
    if (!row_is_read(a, row)) return;
    if (warp == kWarps - 1 && lane < kExpTable) {
        const double e = exp2(lane * (1.0 / kExpTable)) * (1.0 - kExpStep * kExpStep * kExpStep * kExpStep / (16 * 192));
        sm.powers[lane] = __hiloint2double(__double2hiint(e) - (lane << 16), __double2loint(e));
    }
    if (tid == 0) sm.reaches = sm.finds = 0;
    Piece p;
    const T* from = static_cast<const T*>(a.logits) + stream * a.stream_stride + beam * a.beam_stride;
    p.head = static_cast<int>((reinterpret_cast<uintptr_t>(from) & 15) / sizeof(T));
    p.base = from - p.head;
    p.v0 = (blockIdx.x - row * parts) * part_vecs;
    p.v1 = min(p.v0 + part_vecs, (p.head + a.vocab + E - 1) / E);     // the last part may be empty
    __syncthreads();
    // vectors that lie in the row wholly; the others, two at most, are thread 0's and 1's
    const int w0 = max(p.v0, p.head > 0 ? 1 : 0), w1 = max(w0, min(p.v1, (p.head + a.vocab) / E));
    const int edge = tid == 0 && p.v0 < w0 && p.v0 < p.v1 ? p.v0 : tid == 1 && w1 < p.v1 && w1 >= w0 && p.v1 - 1 >= w1 ? w1 : -1;
    const int per = max(w1 - w0 + kThreads - 1, 0) / kThreads;            // vectors of a thread at most
    const int stretch = ((per + kBatch - 1) / kBatch + kStretches - 1) / kStretches;   // batches of a stretch

    float best = -INFINITY, here = -INFINITY;             // of all, of the stretch so far
    int where = 0;
    double sum;
    {
        // each thread brings its own vectors, a batch ahead, and waits for nobody else's
        const uint4* next = static_cast<const uint4*>(p.base) + w0 + tid;
        const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(&sm.ring[0][tid]));
        constexpr uint32_t kRow = kThreads * 16, kHalf = kBatch * kRow;
        int left = max(w1 - w0 - tid + kThreads - 1, 0) / kThreads, coming = left;   // vectors to take, to bring
        double sums[4] = {0.0, 0.0, 0.0, 0.0};
        const ExpPairs pairs;
        const uint32_t powers = static_cast<uint32_t>(__cvta_generic_to_shared(sm.powers));
        auto bring = [&](uint32_t half) {
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
                if (u < coming) copy_async(ring + half + u * kRow, next + u * kThreads);
            commit_async();
            next += kBatch * kThreads;
            coming -= kBatch;
        };
        bring(0);
        bring(kHalf);
        uint32_t half = 0;
        int done = 0, batches = stretch, at = 0;
        for (; left > 0; left -= kBatch, at += kBatch) {
            wait_async<1>();
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                uint4 w = load_shared(ring + half + u * kRow);
                if (u > 0 && u >= left) w = make_uint4(Values<T>::kLowest, Values<T>::kLowest, Values<T>::kLowest, Values<T>::kLowest);
                const float top = Values<T>::top(w);
                if (top > best) best = top, where = at + u;
                here = fmaxf(here, top);
                w = make_uint4(Values<T>::raise(w.x), Values<T>::raise(w.y), Values<T>::raise(w.z), Values<T>::raise(w.w));
#pragma unroll
                for (int e = 0; e < E / 2; ++e) {
                    const float2 x = Values<T>::two(w, e);
                    add_exp(powers, pairs, x.x, x.y, sums);
                }
            }
            bring(half);
            half ^= kHalf;
            if (--batches == 0) {
                sm.tops[done++][tid] = here;
                here = -INFINITY;
                batches = stretch;
            }
        }
        where = w0 + tid + where * kThreads;
        // the stretch that the part ends in, and those that it has no vectors for
        for (; done < kStretches; ++done, here = -INFINITY) sm.tops[done][tid] = here;
        if (edge >= 0) {
            const uint4 w = load<T>(p, a.vocab, edge);
            const float top = Values<T>::top(w);
            if (top > best || (top == best && edge < where)) best = top, where = edge;
#pragma unroll 1
            for (int e = 0; e < E; ++e) {
                const float x = to_float(reinterpret_cast<const Vec<T>&>(w).v[e]);
                add_exp(powers, pairs, max_nan(x, -700.0f), -700.0f, sums);
            }
        }
        sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    }

    // ---- the part's sum; threshold: of `warps` warps whose lanes all have values, each gives
    // the rounds-th largest of its lanes' largest; the least of these is reached by rounds
    // values of each warp, count or more in all.  Values are told apart by the vector they
    // are in (lower first).
    const int warps = min((w1 - w0) / 32, kWarps);
    const int rounds = warps ? (a.count + warps - 1) / warps : 33;
    const uint32_t value = ordered(best);
    const uint32_t warp_top = __reduce_max_sync(0xffffffffu, value);
    unsigned long long limit = rounds > 32 ? 0 : ~0ull;
    if (warp < warps && rounds <= 32) {
        uint32_t left = value > kNone ? value : 0;
        for (int r = 0; r < rounds; ++r) {
            const uint32_t m = __reduce_max_sync(0xffffffffu, left);
            const uint32_t w = __reduce_min_sync(0xffffffffu, left == m ? static_cast<uint32_t>(where) : 0xffffffffu);
            if (left == m && static_cast<uint32_t>(where) == w) left = 0;
            limit = m ? static_cast<unsigned long long>(m) << 32 | (0xffffffffu - w) : 0;
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sm.limit[warp] = limit, sm.top[warp] = unordered(warp_top), sm.part[warp] = sum;
    __syncthreads();
    float top = sm.top[0];
    sum = sm.part[0];
    limit = sm.limit[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
        top = fmaxf(top, sm.top[w]);
        sum += sm.part[w];
        limit = min(limit, sm.limit[w]);
    }
    const uint32_t floor_value = max(static_cast<uint32_t>(limit >> 32), kNone);
    const int floor_at = limit >> 32 > kNone ? static_cast<int>(0xffffffffu - static_cast<uint32_t>(limit)) : -1;
    auto reaches = [&](uint32_t v, int i) { return v > floor_value || (v == floor_value && i <= floor_at); };
    if (reaches(value, where)) {
        for (int r = 0; r * stretch * kBatch < per; ++r) {
            const uint32_t v = ordered(sm.tops[r][tid]);
            // an equal value's place is not kept: it is looked at below
            if (v >= floor_value && v > kNone) sm.reach[atomicAdd(&sm.reaches, 1)] = static_cast<uint16_t>(r * kThreads + tid);
        }
    }
    double ref = 0.0;
    if (top == -INFINITY) {
        ref = -INFINITY;
        if (sum == sum) sum = 0.0;      // NaN stays
    } else if (!(top < INFINITY)) {
        sum = NAN;
    } else if (fabsf(top) > kPlain) {
        ref = top;
        sum = far_sum<T>(sm, p, a.vocab, ref);
    }
    __syncthreads();

    // ---- the values that reach it; a thread's last 2 kBatch vectors are in shared memory still
    auto look = [&](const uint4& w, int i) {
        if (!reaches(ordered(Values<T>::top(w)), i)) return;
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
            const float2 x = Values<T>::two(w, e);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float y = h ? x.y : x.x;
                const uint32_t v = ordered(y);
                if (v > kNone && y == y && reaches(v, i)) {
                    const int place = atomicAdd(&sm.finds, 1);
                    if (place < kFound)
                        sm.found[place] = static_cast<unsigned long long>(v) << 32 | (0xffffffffu - static_cast<uint32_t>(i * E - p.head + 2 * e + h));
                }
            }
        }
    };
    const int each = stretch * kBatch, vectors = sm.reaches * each;
    const float each_inv = 1.0f / each;
    for (int q = tid - 32; q < vectors; q += kThreads) {
        // threads 0 and 1 have the edges before; the float nearest to (q + 1/2) / each is on
        // the right side of whole numbers
        if (q < 0) {
            if (edge >= 0) look(load<T>(p, a.vocab, edge), edge);
            q += kThreads;
            if (q >= vectors) break;
        }
        const int r = vectors < (1 << 20) ? static_cast<int>((q + 0.5f) * each_inv) : q / each;
        const int t = sm.reach[r] % kThreads, j = sm.reach[r] / kThreads * each + q - r * each, i = w0 + t + j * kThreads;
        if (j >= per || i >= w1) continue;
        look(per <= 2 * kBatch ? sm.ring[j][t] : __ldg(static_cast<const uint4*>(p.base) + i), i);
    }
    __syncthreads();
    if (sm.finds > kFound) find_by_bits<T>(sm, p, a.vocab, a.count);
    const int finds = sm.finds;

    // ---- in falling order, `count` of them at most
    unsigned char* to = static_cast<unsigned char*>(a.workspace) + blockIdx.x * part_bytes(a.count);
    unsigned long long* list = reinterpret_cast<unsigned long long*>(to + sizeof(Part));
    for (int f = tid; f < finds; f += kThreads) {
        const unsigned long long key = sm.found[f];
        int place = 0;
#pragma unroll 4
        for (int g = 0; g < finds; ++g) place += sm.found[g] > key;
        if (place < a.count) list[place] = key;
    }
    for (int f = finds + tid; f < a.count; f += kThreads) list[f] = 0;
    if (tid == 0) *reinterpret_cast<Part*>(to) = Part{ref, sum};
}

struct alignas(16) Candidate {
    unsigned long long high, low;   // (total, ~beam), (logit, ~token); high 0: none
    __device__ __forceinline__ bool before(const Candidate& o) const {
        return (high > o.high) | ((high == o.high) & (low > o.low));
    }
};

// The result of stream blockIdx.x.
__global__ void __launch_bounds__(kThreads) join_kernel(const BeamSelectArgs a, int parts) {
    __shared__ Candidate found[kFound];
    __shared__ double lse[kBeamMax], score[kBeamMax];   // of the beams that go on
    __shared__ unsigned long long ended[kBeamMax];
    __shared__ uint32_t limit[kWarps];
    __shared__ int alive[kBeamMax];
    __shared__ int lives, endeds, finds;
    const int stream = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, count = a.count;
    const long long bytes = part_bytes(count);
    const unsigned char* work = static_cast<const unsigned char*>(a.workspace) + static_cast<long long>(stream) * a.beams * parts * bytes;
    if (tid == 0) lives = endeds = finds = 0;
    __syncthreads();
    if (tid < a.beams) {
        // the inputs are older than the launch before
        const long long row = static_cast<long long>(stream) * a.beams + tid;
        const float mine = a.scores[row];
        if (row_is_read(a, row)) {
            const int place = atomicAdd(&lives, 1);
            alive[place] = tid;
            score[place] = mine;
        } else if (mine > -INFINITY) {
            ended[atomicAdd(&endeds, 1)] = static_cast<unsigned long long>(ordered(mine)) << 32 | (0xffffffffu - tid);
        }
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // Candidates are numbered by their place in a part's list, then the part, then the row, and
    // dealt out by an odd multiple: neighbouring threads, and a thread's own, have different
    // places and rows, and the threshold below lets few more through than it has to.  (As they
    // lie, a row to a warp, hundreds pass where rows differ: 18 us for 9 of 32 streams x 16
    // beams x 32; with the rows in turn, where their number and the warps' have a factor in
    // common.)
    const int all = lives * parts * count;
    const int deals = all > 32 ? 1 << (32 - __clz(all - 1)) : 32;   // a power of two, all or more
    const int each = max(deals / kThreads, 1);                       // of a thread
    auto dealt = [&](int k) {   // the thread's k-th; all: none
        const uint32_t e = tid * each + k;
        return k < each && e < deals ? static_cast<int>(e * 0x9e3779b1u & (deals - 1)) : all;
    };
    const int warps = min(deals / 32, kWarps);
    const float lives_inv = 1.0f / lives, parts_inv = 1.0f / parts;
    static_assert(UFB_BEAM_MAX * UFB_BEAM_COUNT_MAX * kMostParts <= 1 << 17, "candidates of a stream");
    auto key_of = [&](int c, int& row) {   // (ordered logit, ~token)
        // below 2^17: (c + 1/2) times a reciprocal is on the right side of whole numbers
        const int in_beams = static_cast<int>((c + 0.5f) * lives_inv), place = static_cast<int>((in_beams + 0.5f) * parts_inv);
        row = c - in_beams * lives;
        return reinterpret_cast<const unsigned long long*>(work + (alive[row] * parts + in_beams - place * parts) * bytes + sizeof(Part))[place];
    };
    // a thread's first ones are on their way while the sums are worked out
    unsigned long long keys[kAhead];
    int rows[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
        keys[k] = 0, rows[k] = 0;
        const int c = dealt(k);
        if (c < all) keys[k] = key_of(c, rows[k]);
    }
    if (tid < lives) {
        // the row's sum, its parts in order
        double ref = -INFINITY, sum = 0.0;
        bool bad = false;
#pragma unroll 4
        for (int c = 0; c < parts; ++c) {
            const Part r = *reinterpret_cast<const Part*>(work + (alive[tid] * parts + c) * bytes);
            bad |= !(r.sum < INFINITY);
            if (!(r.sum > 0.0)) continue;
            // sums of one reference, as most are, are just added
            const double next = fmax(ref, r.ref);
            if (next != ref) sum = sum > 0.0 ? sum * exp(ref - next) : 0.0;
            sum += next == r.ref ? r.sum : r.sum * exp(r.ref - next);
            ref = next;
        }
        // NaN or +infinity in the row: no candidates of it
        if (bad) atomicCAS(a.status, 0, kStatusLogits);
        lse[tid] = !bad && sum > 0.0 ? ref + log(sum) : NAN;
    }
    __syncthreads();
    auto candidate_of = [&](unsigned long long key, int row) {
        Candidate x;
        x.low = key;
        const float logit = unordered(static_cast<uint32_t>(key >> 32));
        const float t = static_cast<float>(score[row] + (static_cast<double>(logit) - lse[row]));
        x.high = key && t > -INFINITY ? static_cast<unsigned long long>(ordered(t)) << 32 | (0xffffffffu - alive[row]) : 0;
        return x;
    };
    auto candidate = [&](int c) {
        int row;
        const unsigned long long key = key_of(c, row);
        return candidate_of(key, row);
    };
    uint32_t totals[kAhead];   // ordered; 0: none
#pragma unroll
    for (int k = 0; k < kAhead; ++k) totals[k] = keys[k] ? static_cast<uint32_t>(candidate_of(keys[k], rows[k]).high >> 32) : 0;
    // a threshold on the totals as in the parts, from each thread's largest
    uint32_t best = 0;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) best = max(best, totals[k]);
#pragma unroll 4
    for (int k = kAhead; k < each; ++k)
        if (dealt(k) < all) best = max(best, static_cast<uint32_t>(candidate(dealt(k)).high >> 32));
    uint32_t least = warp < warps ? 0 : 0xffffffffu;
    for (int r = 0; warp < warps && r * warps < count; ++r) {
        least = __reduce_max_sync(0xffffffffu, best);
        const unsigned same = __ballot_sync(0xffffffffu, best == least);
        if (lane == __ffs(same) - 1) best = 0;
    }
    if (lane == 0) limit[warp] = least;
    __syncthreads();
    least = limit[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) least = min(least, limit[w]);
    least = max(least, 1u);
    auto keep = [&](const Candidate& x) {
        const int place = atomicAdd(&finds, 1);
        if (place < kFound - kBeamMax) found[place] = x;
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
        if (totals[k] >= least)
            keep(Candidate{static_cast<unsigned long long>(totals[k]) << 32 | (0xffffffffu - alive[rows[k]]), keys[k]});
#pragma unroll 4
    for (int k = kAhead; k < each; ++k) {
        if (dealt(k) >= all) continue;
        const Candidate x = candidate(dealt(k));
        if (static_cast<uint32_t>(x.high >> 32) >= least) keep(x);
    }
    __syncthreads();
    if (finds > kFound - kBeamMax) {
        // many equal totals: the count-th largest key bit by bit
        Candidate limit_key = {0, 0};
        for (int bit = 127; bit >= 0; --bit) {
            Candidate trial = limit_key;
            (bit < 64 ? trial.low : trial.high) |= 1ull << (bit & 63);
            __syncthreads();
            if (tid == 0) finds = 0;
            __syncthreads();
            int n = 0;
            for (int c = tid; c < all; c += kThreads) {
                const Candidate x = candidate(c);
                n += x.high != 0 && !trial.before(x);
            }
            n = __reduce_add_sync(0xffffffffu, n);
            if (lane == 0) atomicAdd(&finds, n);
            __syncthreads();
            if (finds >= count) limit_key = trial;
        }
        __syncthreads();
        if (tid == 0) finds = 0;
        __syncthreads();
        for (int c = tid; c < all; c += kThreads) {
            const Candidate x = candidate(c);
            if (x.high != 0 && !limit_key.before(x)) found[atomicAdd(&finds, 1)] = x;
        }
        __syncthreads();
    }
    // the ended beams' after them
    const int n = finds + endeds;
    if (tid < endeds) found[finds + tid] = Candidate{ended[tid], 0xffffffffu - static_cast<uint32_t>(a.pad)};
    __syncthreads();
    const long long out = static_cast<long long>(stream) * count;
    for (int f = tid; f < n; f += kThreads) {
        const Candidate x = found[f];
        int place = 0;
#pragma unroll 4
        for (int g = 0; g < n; ++g) place += found[g].before(x);
        if (place >= count) continue;
        a.out_scores[out + place] = unordered(static_cast<uint32_t>(x.high >> 32));
        a.parents[out + place] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(x.high));
        a.tokens[out + place] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(x.low));
    }
    for (int place = n + tid; place < count; place += kThreads) {
        a.out_scores[out + place] = -INFINITY;
        a.parents[out + place] = min(place, a.beams - 1);
        a.tokens[out + place] = 0;
    }
}

// Parts of a row: the number with the least time of the SM that has the most CTAs.  An SM
// takes about as long for each value whether one CTA or four are on it (a row of 65537 floats
// alone 10 us, 3.3 values a cycle; the exponentials alone reach 6.7, and what the warps wait for
// besides was not told apart), so what counts is how evenly the work lies, against what a part costs
// besides.  Measured with other numbers of parts: 64 streams x 8 beams x 32768
// 24 us (2 parts 31, 4: 40), 48 x 8 x 50257 27.5 (2: 30, 3: 34), 32 x 16 x 131072 with a
// fifth of the beams ended 61 (1: 69, 4: 74), 8 x 8 x 131072 18 (1: 25, 4: 19), 1 x 8 x 131072
// 12 (1: 23, 4: 14), 16 x 4 x 50000 floats 11.4 (1: 14.4, 3: 13.2), 24 x 5 x 65537 floats 17.3
// (3: 18.7, 6: 23.6).  No more candidates than the join's threads have at hand (17 parts of the
// 8 rows take 15.7 us, 13 12.2), unless the rows are whole: x 131072, 1 x 16 beams, 32 best 20.5 us in
// the 2 parts that this leaves (1: 26.8, 4: 20.9), 2 x 20, 25 best 21.4 in 2 (4: 24.5), 1 x 64, 64
// best 40 in 1 (2: 43, 4: 70); 1 x 32, 32 best 27.4 in 1, where 2 would take 24.2 (4: 26.2).
struct Division {
    int parts, vecs;
};
template <typename T>
Division divide(int streams, int beams, int vocab, int count, int sms) {
    constexpr int elements = kElems<T>;
    const int row_vecs = (vocab + 2 * elements - 2) / elements;    // of any alignment
    const long long rows = static_cast<long long>(streams) * beams;
    Division d{1, row_vecs};
    double least = 1e300;
    for (int parts = 1; parts <= kMostParts && (parts == 1 || row_vecs / parts >= kThreads / 2); ++parts) {
        // whole sweeps of a CTA's threads, unless the row has less than one
        int vecs = (row_vecs + parts - 1) / parts;
        if (vecs > kThreads) vecs = (vecs + kThreads - 1) / kThreads * kThreads;
        const double cost = static_cast<double>((rows * parts + sms - 1) / sms) *
                            (static_cast<double>((vecs + kThreads - 1) / kThreads) * elements + kPartCost);
        const int made = (row_vecs + vecs - 1) / vecs;
        if (cost < least && (made == 1 || beams * made * count <= kAhead * kThreads)) {
            least = cost;
            d.vecs = vecs;
            d.parts = made;
        }
    }
    return d;
}

template <typename T>
cudaError_t launch(const BeamSelectArgs& a, int sms, cudaStream_t s) {
    const Division d = divide<T>(a.streams, a.beams, a.vocab, a.count, sms);
    static std::atomic<uint64_t> allowed;
    cudaError_t e = allow_smem(part_kernel<T>, sizeof(Shared), allowed);
    if (e != cudaSuccess) return e;
    part_kernel<T><<<static_cast<unsigned>(a.streams) * a.beams * d.parts, kThreads, sizeof(Shared), s>>>(a, d.parts, d.vecs);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(a.streams);
    config.blockDim = dim3(kThreads);
    config.stream = s;
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, join_kernel, a, d.parts);
}

}  // namespace

int64_t beam_select_workspace_bytes(int streams, int beams, int vocab, int count, int dtype, int sms) {
    const Division d = dtype == UFB_F32 ? divide<float>(streams, beams, vocab, count, sms) : divide<__half>(streams, beams, vocab, count, sms);
    return static_cast<int64_t>(streams) * beams * d.parts * part_bytes(count);
}

cudaError_t beam_select(const BeamSelectArgs& a, int dtype, int sms, cudaStream_t s) {
    return dtype == UFB_F32   ? launch<float>(a, sms, s)
           : dtype == UFB_F16 ? launch<__half>(a, sms, s)
                              : launch<__nv_bfloat16>(a, sms, s);
}

}  // namespace ufb
