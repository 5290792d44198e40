// The best continuations of each stream's beams (ufb_beam_select):
//
//   total[k][v] = f32(scores[k] + (logits[k][v] - ln sum_u exp logits[k][u])),
//
// the `count` best of a stream by total, then lower beam, larger logit, lower token.
//
// Bound by the bytes of the logits, which are read once from memory.  A cluster of
// CTAs serves a stream: the 16-byte vectors of its live beams' rows make one sequence
// that the CTAs share equally.  A CTA goes through the piece of each row in its share
// with nothing between the loads but arithmetic: every thread sums exp and keeps its
// largest value and where it was.  From the threads' largest values a threshold
// follows that at least `count` values reach and few more do (see threshold below);
// the threads that reach it are looked through again, from cache.  So no running list
// and no barrier is in the loop.  Then the CTAs exchange the rows' sums and each
// one's best `count`, by distributed shared memory, and the first writes the result:
// one launch, no scratch in global memory.
//
// The order of candidates of different beams hangs on the rows' ln sum exp, and totals
// are next to each other: sums are in 64 bits.
#include "beam.h"

#include "capi_util.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

namespace cg = cooperative_groups;

namespace ufb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kUnroll = 4;        // vectors a thread has under way
constexpr int kFound = 1024;      // candidates of a piece before they are cut to `count`
// Sums are of exp itself while the row's largest logit is inside this, else of exp(x - largest).
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

template <typename T>
struct Vec {
    static constexpr int kElems = 16 / sizeof(T);
    T v[kElems];
};

// A stretch of one row.
struct Piece {
    const void* base;      // 16-byte boundary at or before the row's first element
    int head;              // elements between them
    int beam;
    int v0, v1;            // vectors, v0 < v1
};

// Vector i of a row; what lies outside of it is -infinity.
template <typename T>
__device__ __forceinline__ void load(const Piece& p, int vocab, int i, float (&x)[Vec<T>::kElems]) {
    constexpr int E = Vec<T>::kElems;
    const T* at = static_cast<const T*>(p.base) + static_cast<long long>(i) * E;
    const int first = i * E - p.head;
    if (first >= 0 && first <= vocab - E) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(at));
        const Vec<T>& v = reinterpret_cast<const Vec<T>&>(w);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = to_float(v.v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = first + e >= 0 && first + e < vocab ? to_float(at[e]) : -INFINITY;
    }
}

// What a CTA knows of a row.
struct RowSum {
    double ref, sum;       // sum exp(x - ref) of its piece; ref -infinity: nothing there
};

struct Candidate {
    unsigned long long high, low;   // (total, ~beam), (logit, ~token)
    __device__ __forceinline__ bool before(const Candidate& o) const {
        return high > o.high || (high == o.high && low > o.low);
    }
};

struct Shared {
    RowSum rows[kBeamMax];              // by beam
    double lse[kBeamMax];
    float score[kBeamMax];
    int live[kBeamMax];                 // the beams whose rows are read, in order
    int lives, ended;
    Candidate over[kBeamMax];           // ended beams, each its own only candidate
    unsigned long long found[kFound];
    unsigned long long limit[kWarps];
    double part[kWarps];
    float top[kWarps];
    int reach[kThreads];                // threads whose largest value reaches the threshold
    int reaches, finds;
    int best;                           // candidates this CTA offers
    int poisoned;
};

// Of a list in falling order: how many come before c.
__device__ __forceinline__ int count_before(const Candidate* list, int n, const Candidate& c) {
    int low = 0, high = n;
    while (low < high) {
        const int mid = (low + high) >> 1;
        if (list[mid].before(c)) low = mid + 1;
        else high = mid;
    }
    return low;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) select_kernel(const BeamSelectArgs a, int most_pieces) {
    constexpr int E = Vec<T>::kElems;
    extern __shared__ __align__(16) unsigned char raw[];
    Shared& sm = *reinterpret_cast<Shared*>(raw);
    // [most_pieces][count] the pieces' best, then [count] the CTA's, then (first CTA) [cluster][count] all of them
    Candidate* lists = reinterpret_cast<Candidate*>(raw + (sizeof(Shared) + 15) / 16 * 16);
    __shared__ int list_beam[kBeamMax + 1], list_n[kBeamMax + 1];
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int stream = blockIdx.x / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Candidate* mine = lists + static_cast<long long>(most_pieces) * a.count;

    if (warp == 0) {
        // beams at -infinity and NaN lead nowhere; ended ones stay as they are
        int lives = 0, ended = 0;
        for (int k0 = 0; k0 < a.beams; k0 += 32) {
            const int k = k0 + lane;
            const float s = k < a.beams ? a.scores[static_cast<long long>(stream) * a.beams + k] : -INFINITY;
            const bool over = k < a.beams && a.finished && a.finished[static_cast<long long>(stream) * a.beams + k];
            const unsigned l = __ballot_sync(0xffffffffu, s > -INFINITY && !over);
            const unsigned o = __ballot_sync(0xffffffffu, s > -INFINITY && over);
            const unsigned below = (1u << lane) - 1;
            if (l >> lane & 1) sm.live[lives + __popc(l & below)] = k;
            if (o >> lane & 1) {
                Candidate& c = sm.over[ended + __popc(o & below)];
                c.high = static_cast<unsigned long long>(ordered(s)) << 32 | (0xffffffffu - k);
                c.low = 0xffffffffu - static_cast<uint32_t>(a.pad);
            }
            if (k < a.beams) {
                sm.score[k] = s;
                sm.rows[k].ref = -INFINITY;
                sm.rows[k].sum = 0.0;
            }
            lives += __popc(l);
            ended += __popc(o);
        }
        if (lane == 0) sm.lives = lives, sm.ended = ended, sm.poisoned = 0;
    }
    __syncthreads();

    // ---- the pieces of this CTA's share
    const int row_vecs = (a.vocab + 2 * E - 2) / E;    // of any alignment
    const long long total = static_cast<long long>(sm.lives) * row_vecs;
    const long long begin = total * rank / ctas, end = total * (rank + 1) / ctas;
    int pieces = 0;
    for (long long at = begin; at < end; ++pieces) {
        const int row = static_cast<int>(at / row_vecs);
        const long long row0 = static_cast<long long>(row) * row_vecs;
        Piece p;
        p.beam = sm.live[row];
        const T* from = static_cast<const T*>(a.logits) + stream * a.stream_stride + p.beam * a.beam_stride;
        p.head = static_cast<int>((reinterpret_cast<uintptr_t>(from) & 15) / sizeof(T));
        p.base = from - p.head;
        p.v0 = static_cast<int>(at - row0);
        p.v1 = static_cast<int>(min(end - row0, static_cast<long long>(row_vecs)));
        at = row0 + p.v1;
        p.v1 = min(p.v1, (p.head + a.vocab + E - 1) / E);
        const int vecs = p.v1 - p.v0;      // the row may end before row_vecs: none then

        float best = -INFINITY;
        int where = 0;
        double sum = 0.0;
        auto take = [&](const float (&x)[E], int i) {
            float top = x[0];
#pragma unroll
            for (int e = 1; e < E; ++e) top = fmaxf(top, x[e]);
            if (top > best) best = top, where = i;
#pragma unroll
            for (int e = 0; e < E; ++e) sum += exp(static_cast<double>(x[e]));
        };
        const int whole0 = p.head > 0 ? 1 : 0, whole1 = (p.head + a.vocab) / E;   // vectors inside the row
        int i = p.v0 + tid;
        for (; i - tid + kThreads * kUnroll <= p.v1 && i - tid >= whole0 && i - tid + kThreads * kUnroll <= whole1;
             i += kThreads * kUnroll) {
            uint4 w[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                w[u] = __ldg(static_cast<const uint4*>(p.base) + i + u * kThreads);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const Vec<T>& v = reinterpret_cast<const Vec<T>&>(w[u]);
                float x[E];
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = to_float(v.v[e]);
                take(x, i + u * kThreads);
            }
        }
        for (; i < p.v1; i += kThreads) {
            float x[E];
            load<T>(p, a.vocab, i, x);
            take(x, i);
        }

        // ---- the piece's sum and largest value
        float top = best;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if (lane == 0) sm.top[warp] = top, sm.part[warp] = sum;

        // ---- threshold: of `warps` warps whose lanes all have values, each gives the
        // rounds-th largest of its lanes' largest; the least of these is reached by
        // rounds values of each warp, count or more in all.  Values are told apart by
        // the vector they are in (lower first).
        const int warps = min(vecs / 32, kWarps);
        const int rounds = warps ? (a.count + warps - 1) / warps : 33;
        uint32_t value = ordered(best);
        unsigned long long limit = ~0ull;
        if (warp < warps && rounds <= 32) {
            uint32_t left = value > kNone ? value : 0;
            limit = 0;
            for (int r = 0; r < rounds; ++r) {
                const uint32_t m = __reduce_max_sync(0xffffffffu, left);
                const uint32_t w = __reduce_min_sync(0xffffffffu, left == m ? static_cast<uint32_t>(where) : 0xffffffffu);
                if (left == m && static_cast<uint32_t>(where) == w) left = 0;
                limit = m ? static_cast<unsigned long long>(m) << 32 | (0xffffffffu - w) : 0;
            }
        }
        if (rounds > 32) limit = 0;
        if (lane == 0) sm.limit[warp] = limit;
        if (tid == 0) sm.reaches = 0, sm.finds = 0;
        __syncthreads();
        top = sm.top[0];
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
        if (reaches(value, where)) sm.reach[atomicAdd(&sm.reaches, 1)] = tid;

        // ---- rows whose exp leaves the range of 64 bits: once more, less the largest value
        double ref = 0.0;
        if (top == -INFINITY) {
            ref = -INFINITY;
            if (sum == sum) sum = 0.0;      // NaN stays
        } else if (!(fabsf(top) <= kPlain) && top < INFINITY) {
            ref = top;
            sum = 0.0;
            for (int j = p.v0 + tid; j < p.v1; j += kThreads) {
                float x[E];
                load<T>(p, a.vocab, j, x);
#pragma unroll
                for (int e = 0; e < E; ++e) sum += exp(static_cast<double>(x[e]) - ref);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            __syncthreads();
            if (lane == 0) sm.part[warp] = sum;
            __syncthreads();
            sum = sm.part[0];
            for (int w = 1; w < kWarps; ++w) sum += sm.part[w];
        }
        if (!(top < INFINITY)) sum = NAN;
        if (tid == 0) sm.rows[p.beam].ref = ref, sm.rows[p.beam].sum = sum;
        __syncthreads();

        // ---- the values that reach it
        const int per = (vecs + kThreads - 1) / kThreads;   // vectors of a thread at most
        const int pairs = sm.reaches * per;
        for (int q = tid; q < pairs; q += kThreads) {
            const int j = p.v0 + sm.reach[q / per] + (q % per) * kThreads;
            if (j >= p.v1) continue;
            float x[E];
            load<T>(p, a.vocab, j, x);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint32_t v = ordered(x[e]);
                if (v > kNone && x[e] == x[e] && reaches(v, j)) {
                    const int at = atomicAdd(&sm.finds, 1);
                    if (at < kFound)
                        sm.found[at] = static_cast<unsigned long long>(v) << 32 | (0xffffffffu - static_cast<uint32_t>(j * E - p.head + e));
                }
            }
        }
        __syncthreads();
        int finds = sm.finds;
        if (finds > kFound) {
            // many equal values, or the large ones of the row in few threads: the count-th largest
            // value by bisection, then of the values equal to it the lowest tokens
            auto number = [&](auto test) {
                int n = 0;
                for (int j = p.v0 + tid; j < p.v1; j += kThreads) {
                    float x[E];
                    load<T>(p, a.vocab, j, x);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const uint32_t v = ordered(x[e]);
                        n += v > kNone && x[e] == x[e] && test(v, j * E - p.head + e);
                    }
                }
                n = __reduce_add_sync(0xffffffffu, n);
                if (lane == 0) atomicAdd(&sm.finds, n);
            };
            auto sum_up = [&](auto test) {
                __syncthreads();
                if (tid == 0) sm.finds = 0;
                __syncthreads();
                number(test);
                __syncthreads();
                return sm.finds;
            };
            uint32_t low = kNone + 1, high = 0xffffffffu;   // the largest v that count values reach
            while (low < high) {
                const uint32_t mid = low + (high - low + 1) / 2;
                if (sum_up([&](uint32_t v, int) { return v >= mid; }) >= a.count) low = mid;
                else high = mid - 1;
            }
            const int above = sum_up([&](uint32_t v, int) { return v > low; });
            int token0 = 0, token1 = a.vocab - 1;           // the lowest token up to which there are enough
            while (token0 < token1) {
                const int mid = token0 + (token1 - token0) / 2;
                if (above + sum_up([&](uint32_t v, int t) { return v == low && t <= mid; }) >= a.count) token1 = mid;
                else token0 = mid + 1;
            }
            __syncthreads();
            if (tid == 0) sm.finds = 0;
            __syncthreads();
            for (int j = p.v0 + tid; j < p.v1; j += kThreads) {
                float x[E];
                load<T>(p, a.vocab, j, x);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const uint32_t v = ordered(x[e]);
                    const int t = j * E - p.head + e;
                    if (v > kNone && x[e] == x[e] && (v > low || (v == low && t <= token0)))
                        sm.found[atomicAdd(&sm.finds, 1)] = static_cast<unsigned long long>(v) << 32 | (0xffffffffu - static_cast<uint32_t>(t));
                }
            }
            __syncthreads();
            finds = sm.finds;
        }
        // ---- in falling order, `count` of them at most
        Candidate* list = lists + static_cast<long long>(pieces) * a.count;
        for (int f = tid; f < finds; f += kThreads) {
            const unsigned long long key = sm.found[f];
            int place = 0;
            for (int g = 0; g < finds; ++g) place += sm.found[g] > key;
            if (place < a.count) list[place].low = key;
        }
        if (tid == 0) list_beam[pieces] = p.beam, list_n[pieces] = min(finds, a.count);
        __syncthreads();
    }

    // ---- the rows' sums over all CTAs
    if (ctas > 1) cluster.sync();
    if (tid < sm.lives) {
        const int beam = sm.live[tid];
        double ref = -INFINITY, sum = 0.0;
        const long long row0 = static_cast<long long>(tid) * row_vecs;
        RowSum parts[kMaxCluster];
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) {
            parts[c].ref = -INFINITY, parts[c].sum = 0.0;
            // the row's pieces only
            if (c < ctas && total * c / ctas < row0 + row_vecs && total * (c + 1) / ctas > row0)
                parts[c] = ctas > 1 ? cluster.map_shared_rank(&sm, c)->rows[beam] : sm.rows[beam];
            ref = fmax(ref, parts[c].ref);
        }
        bool bad = false;
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) {
            bad |= !(parts[c].sum < INFINITY);
            if (parts[c].sum > 0.0) sum += parts[c].sum * (parts[c].ref == ref ? 1.0 : exp(parts[c].ref - ref));
        }
        // NaN or +infinity in the row: no candidates of it
        sm.lse[beam] = bad ? NAN : ref + log(sum);
        if (bad && rank == 0) atomicCAS(a.status, 0, kStatusLogits);
    }
    __syncthreads();

    // ---- this CTA's best
    for (int c = tid; c < pieces * a.count; c += kThreads) {
        const int l = c / a.count, beam = list_beam[l];
        if (c - l * a.count >= list_n[l]) continue;
        const float logit = unordered(static_cast<uint32_t>(lists[c].low >> 32));
        const float t = static_cast<float>(static_cast<double>(sm.score[beam]) + (static_cast<double>(logit) - sm.lse[beam]));
        // the order of a list stays: totals do not fall where logits rise
        lists[c].high = t > -INFINITY ? static_cast<unsigned long long>(ordered(t)) << 32 | (0xffffffffu - beam) : 0;
    }
    if (tid == 0) sm.best = 0;
    __syncthreads();
    Candidate* offered = ctas > 1 ? mine : lists + static_cast<long long>(most_pieces + 1) * a.count;
    for (int c = tid; c < pieces * a.count; c += kThreads) {
        const int l = c / a.count;
        if (c - l * a.count >= list_n[l] || lists[c].high == 0) continue;
        int place = c - l * a.count;
        for (int o = 0; o < pieces && place < a.count; ++o)
            if (o != l) place += count_before(lists + static_cast<long long>(o) * a.count, list_n[o], lists[c]);
        if (place < a.count) {
            offered[place] = lists[c];
            atomicMax(&sm.best, place + 1);
        }
    }
    if (ctas > 1) {
        cluster.sync();
        if (rank == 0) {
            // all CTAs' offers side by side
            Candidate* all = lists + static_cast<long long>(most_pieces + 1) * a.count;
            for (int c = tid; c < ctas * a.count; c += kThreads) {
                const int o = c / a.count;
                if (c - o * a.count < cluster.map_shared_rank(&sm, o)->best) all[c] = cluster.map_shared_rank(mine, o)[c - o * a.count];
            }
            if (tid < ctas) list_n[tid] = cluster.map_shared_rank(&sm, tid)->best;
        }
        cluster.sync();
        if (rank != 0) return;
    } else {
        __syncthreads();
        if (tid == 0) list_n[0] = sm.best;
    }
    __syncthreads();

    // ---- the stream's result
    const Candidate* all = lists + static_cast<long long>(most_pieces + 1) * a.count;
    const long long out = static_cast<long long>(stream) * a.count;
    auto put = [&](int place, const Candidate& c) {
        a.out_scores[out + place] = unordered(static_cast<uint32_t>(c.high >> 32));
        a.parents[out + place] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(c.high));
        a.tokens[out + place] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(c.low));
    };
    int have = sm.ended;
    for (int o = 0; o < ctas; ++o) have += list_n[o];
    for (int c = tid; c < ctas * a.count; c += kThreads) {
        const int l = c / a.count;
        if (c - l * a.count >= list_n[l]) continue;
        int place = c - l * a.count;
        for (int o = 0; o < ctas && place < a.count; ++o)
            if (o != l) place += count_before(all + static_cast<long long>(o) * a.count, list_n[o], all[c]);
        for (int f = 0; f < sm.ended && place < a.count; ++f) place += sm.over[f].before(all[c]);
        if (place < a.count) put(place, all[c]);
    }
    for (int f = tid; f < sm.ended; f += kThreads) {
        int place = 0;
        for (int g = 0; g < sm.ended; ++g) place += sm.over[g].before(sm.over[f]);
        for (int o = 0; o < ctas && place < a.count; ++o)
            place += count_before(all + static_cast<long long>(o) * a.count, list_n[o], sm.over[f]);
        if (place < a.count) put(place, sm.over[f]);
    }
    for (int place = have + tid; place < a.count; place += kThreads) {
        a.out_scores[out + place] = -INFINITY;
        a.parents[out + place] = min(place, a.beams - 1);
        a.tokens[out + place] = 0;
    }
}

template <typename T>
cudaError_t launch(const BeamSelectArgs& a, int sms, cudaStream_t s) {
    constexpr int E = Vec<T>::kElems;
    // CTAs of a stream: as many as keep the GPU busy with four to an SM, while each has work
    const long long vecs = static_cast<long long>(a.beams) * ((a.vocab + 2 * E - 2) / E);
    int ctas = 1;
    while (ctas < kMaxCluster && static_cast<long long>(a.streams) * ctas < 4ll * sms && vecs / (2 * ctas) >= 64) ctas *= 2;
    // rows that a share touches at most
    const int pieces = (a.beams + ctas - 1) / ctas + (ctas > 1 ? 1 : 0);
    const int smem = (sizeof(Shared) + 15) / 16 * 16 +
                     (pieces + 1 + ctas) * a.count * static_cast<int>(sizeof(Candidate));
    auto kernel = select_kernel<T>;
    static std::atomic<uint64_t> allowed;
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
    if (!(allowed.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(sizeof(Shared)) + 16 + (kBeamMax + 2 + kMaxCluster) * kBeamCountMax * static_cast<int>(sizeof(Candidate)));
        if (e != cudaSuccess) return e;
        allowed.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(a.streams) * ctas);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ctas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, a, pieces);
}

}  // namespace

cudaError_t beam_select(const BeamSelectArgs& a, int dtype, int sms, cudaStream_t s) {
    return dtype == UFB_F32   ? launch<float>(a, sms, s)
           : dtype == UFB_F16 ? launch<__half>(a, sms, s)
                              : launch<__nv_bfloat16>(a, sms, s);
}

}  // namespace ufb
