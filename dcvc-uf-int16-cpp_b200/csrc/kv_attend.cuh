// Shared parts of the attention kernels: which keys a tile of rows sees, how the
// work of a call is divided over the CTAs, and the scratch of split items.
//
// Rows.  The new tokens of a stream times the query heads of one key head are
// rows r = token * group + query head; a tile of TM rows with one key head and
// its keys is an item.  The tiles of BK keys of all items, in the order stream,
// row tile, key head, make one sequence, and every CTA takes an equal share of
// it, wherever items begin and end: streams of very different lengths load all
// SMs alike and the division depends on nothing but the lengths, so results do
// not vary from run to run.  A CTA writes the rows of an item it holds whole; of
// one that it shares it writes partial sums to its scratch, at most two a CTA
// (the item its share begins in and the one it ends in).
#pragma once

#include "attention.h"
#include "capi_util.h"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ufb {

constexpr int kAttendMaxCtas = 160;     // CTAs of a launch at most (scratch is sized by the SMs)
constexpr int kAttendManyRows = 256;    // rows of the widest tile
constexpr int kGroupKeys = 16;          // keys that share a page, and so a scale, at every page size

// Value scales below this act as this: such a page's values vanish beside any
// other, but its keys still carry weight.  A row's weight, the sum of P / scale with
// P up to 2^15 over up to 2^30 keys, stays inside 32 bits.
constexpr float kTinyScale = 8.271806125530277e-25f;  // 2^-80

// Keys [0, sink) and [low, hi) hold every key that a tile of rows sees; in tiles
// of BK keys: [0, sink_tiles) and from low_tile on, nt in all.
struct KeyRange {
    int sink, low, hi;
    int sink_tiles, low_tile, nt;
    __device__ __forceinline__ int tile(int t) const { return t < sink_tiles ? t : low_tile + t - sink_tiles; }
    // any of the keys [k, k + kGroupKeys) inside
    __device__ __forceinline__ bool touches(int k) const { return k < sink || (k < hi && k + kGroupKeys > low); }
};

// Tokens first..last (of n_new) of a stream of `length` keys.
template <int BK>
__device__ __forceinline__ KeyRange key_range(const AttendArgs& a, int length, int n_new, int first, int last) {
    KeyRange r;
    const long long base = static_cast<long long>(length) - n_new;
    const long long top = a.causal ? base + last + 1 : length;
    r.hi = static_cast<int>(top < 0 ? 0 : (top > length ? length : top));
    const long long low = a.window ? base + first - a.window + 1 : 0;
    r.low = static_cast<int>(low < 0 ? 0 : (low > length ? length : low));
    r.sink = a.window ? min(a.sinks, min(r.low, r.hi)) : 0;
    const int hi_tile = (r.hi + BK - 1) / BK;
    r.low_tile = min(r.low / BK, hi_tile);
    r.sink_tiles = (r.sink + BK - 1) / BK;
    if (r.sink_tiles > 0 && r.sink_tiles >= r.low_tile) r.sink_tiles = r.low_tile = 0;
    r.nt = r.sink_tiles + hi_tile - r.low_tile;
    // rows that see nothing are still written: one tile, all of it hidden
    if (r.nt <= 0) r.nt = 1, r.low_tile = 0, r.sink_tiles = 0;
    return r;
}

// One stream's row tile.
struct RowTile {
    int slot, length, n_new;
    long long token0;       // the stream's first new token
    int row0, rows;         // rows of the tile
    KeyRange keys;
};

// false: the pair (stream, row tile) does not exist.
template <int BK, int TM>
__device__ __forceinline__ bool row_tile(const AttendArgs& a, int stream, int rt, RowTile& t) {
    const int o0 = a.offsets[stream], o1 = a.offsets[stream + 1];
    t.slot = a.slots[stream];
    const bool ok = t.slot >= 0 && t.slot < a.slots_total && o0 >= 0 && o1 >= o0 && o1 <= a.tokens && o1 - o0 <= a.max_new;
    t.n_new = ok ? o1 - o0 : 0;
    t.token0 = o0;
    t.row0 = rt * TM;
    t.rows = min(TM, t.n_new * a.group - t.row0);
    if (!ok && rt == 0) atomicCAS(a.status, 0, kStatusIndex);
    if (t.rows <= 0) return false;
    t.length = max(a.lengths[t.slot], 0);
    if (a.refused[t.slot]) {
        // its new tokens were not taken in: no position is theirs, they see no key
        t.length = 0;
        if (rt == 0) atomicCAS(a.status, 0, kStatusPages);
    }
    t.keys = key_range<BK>(a, t.length, t.n_new, t.row0 / a.group, (t.row0 + t.rows - 1) / a.group);
    return true;
}

// a / b of values that nearly always fit 32 bits, where a division is much shorter.
__device__ __forceinline__ long long quotient(long long a, long long b) {
    return ((a | b) >> 31) == 0 ? static_cast<long long>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}

// Where a CTA's share of the sequence begins.
struct Share {
    long long total;        // tiles of the call
    long long per;          // tiles of a CTA's share
    long long pair_start;   // first tile of the pair the share begins in
    int pair;
};

struct ShareSmem {
    long long warp[32];
    long long pair_start;
    int pair;
};

// Every thread of the block calls it.  tiles(p): the tiles of pair p.
template <int THREADS, class Tiles>
__device__ __forceinline__ Share share_out(int pairs, int min_share, Tiles tiles_of, ShareSmem& sm) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Share s;
    auto tiles = [&](int p) -> long long { return p < pairs ? tiles_of(p) : 0; };
    long long first = 0, sum = 0;
    for (int base = 0; base < pairs; base += THREADS) {
        const long long v = tiles(base + threadIdx.x);
        if (base == 0) first = v;
        sum += v;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sm.warp[warp] = sum;
    if (threadIdx.x == 0) sm.pair = pairs, sm.pair_start = 0;
    __syncthreads();
    s.total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) s.total += sm.warp[w];
    s.per = quotient(s.total + gridDim.x - 1, gridDim.x);
    if (s.per < min_share) s.per = min_share;
    const long long start = s.per * blockIdx.x;
    long long before = 0;
    for (int base = 0; base < pairs && before <= start; base += THREADS) {
        const long long v = base == 0 ? first : tiles(base + threadIdx.x);
        long long inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        __syncthreads();
        if (lane == 31) sm.warp[warp] = inc;
        __syncthreads();
        long long skip = before;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) skip += sm.warp[w];
            before += sm.warp[w];
        }
        const long long at = skip + inc - v;
        if (v > 0 && at <= start && start < at + v) sm.pair = base + threadIdx.x, sm.pair_start = at;
    }
    __syncthreads();
    s.pair = sm.pair;
    s.pair_start = sm.pair_start;
    return s;
}

// row_tiles: row tiles of a stream at most.
template <int BK, int TM, int THREADS>
__device__ __forceinline__ Share locate_share(const AttendArgs& a, int row_tiles, int min_share, ShareSmem& sm) {
    RowTile t;
    return share_out<THREADS>(
        a.n * row_tiles, min_share,
        [&](int p) -> long long {
            return row_tile<BK, TM>(a, p / row_tiles, p % row_tiles, t) ? static_cast<long long>(t.keys.nt) * a.heads : 0;
        },
        sm);
}

// The part of one item that a CTA holds.
struct Piece {
    RowTile t;
    int head;
    int first, end;             // its key tiles, of t.keys.nt
    long long item_start;       // the item's first tile in the sequence
    __device__ __forceinline__ bool whole() const { return first == 0 && end == t.keys.nt; }
};

// Walks the pieces of this CTA's share; every role of a kernel has its own.
template <int BK, int TM>
struct Walker {
    int row_tiles, pair, pairs;
    long long pos, end, pair_start;
    bool loaded;
    RowTile t;

    __device__ __forceinline__ Walker(const AttendArgs& a, const Share& s, int rts) {
        row_tiles = rts;
        pairs = a.n * rts;
        pos = s.per * blockIdx.x;
        end = min(pos + s.per, s.total);
        pair = s.pair;
        pair_start = s.pair_start;
        loaded = false;
    }
    __device__ __forceinline__ bool next(const AttendArgs& a, Piece& p) {
        if (pos >= end) return false;
        while (true) {
            if (pair >= pairs) return false;
            if (!loaded) {
                if (!row_tile<BK, TM>(a, pair / row_tiles, pair % row_tiles, t)) {
                    pair = (pair / row_tiles + 1) * row_tiles;  // no further row tiles of this stream
                    continue;
                }
                loaded = true;
            }
            const long long size = static_cast<long long>(t.keys.nt) * a.heads;
            if (pos < pair_start + size) break;
            pair_start += size;
            ++pair;
            loaded = false;
        }
        p.t = t;
        p.head = static_cast<int>(quotient(pos - pair_start, t.keys.nt));
        p.item_start = pair_start + static_cast<long long>(p.head) * t.keys.nt;
        p.first = static_cast<int>(pos - p.item_start);
        p.end = static_cast<int>(min(static_cast<long long>(t.keys.nt), end - p.item_start));
        pos = p.item_start + p.end;
        return true;
    }
};

// Scratch of split items: 2 parts a CTA (0: of the item its share begins in, if
// that began earlier; 1: of the item it ends in), each [rows][D] sums, [rows]
// maxima and [rows] weights.
struct AttendScratch {
    int32_t* counters;   // [kAttendMaxCtas] arrivals at the item that CTA's share ends in; zero between calls
    int32_t* items;      // [kAttendMaxCtas][8] that item's description for the join launch
    float* stats;        // [parts][2][rows]
    float* sums;         // [parts][rows][D]
};

__host__ __device__ inline AttendScratch scratch_of(void* workspace, int ctas, int rows) {
    AttendScratch s;
    s.counters = static_cast<int32_t*>(workspace);
    s.items = s.counters + kAttendMaxCtas;
    s.stats = reinterpret_cast<float*>(s.items + kAttendMaxCtas * 8);
    s.sums = s.stats + static_cast<long long>(2 * ctas) * 2 * rows;
    return s;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Four stored integers to float16, exactly: an integer plus 128 in the low byte
// of 0x64xx is 1024 + 128 + integer.
__device__ __forceinline__ uint32_t half2_minus_1152(uint32_t v) {
    const uint32_t c = 0x64806480u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void int8x4_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    w ^= 0x80808080u;
    lo = half2_minus_1152(__byte_perm(w, 0x64646464u, 0x4140));
    hi = half2_minus_1152(__byte_perm(w, 0x64646464u, 0x4342));
}

// Power of two that brings a row's largest |q| into [2^15, 2^16), float16's last
// binade: values of float16 rows stay what they are, down to the smallest beside the
// largest, and bfloat16 values keep their bits down to 2^-32 of the largest.
// Products with the integers, 128 of them, stay below 2^30.  NaN for a row that is not
// finite.
__device__ __forceinline__ float row_unit(float top) {
    if (!(top < __int_as_float(0x7f800000))) return __int_as_float(0x7fffffff);
    if (top < 1.1754943508222875e-38f) return 8.507059173023462e37f;  // 2^126
    const int e = (__float_as_int(top) >> 23) - 126;                    // top in [2^(e-1), 2^e)
    // 2^(16 - e), kept where its inverse is a normal number too
    return __int_as_float((127 + min(16 - e, 126)) << 23);
}

// 1 / u of a power of two u (NaN stays NaN).
__device__ __forceinline__ float unit_inverse(float u) {
    return u == u ? __int_as_float((254 << 23) - __float_as_int(u)) : u;
}

__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __half) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// The layer's integers as (128 bytes, rows of a head, heads, key and value, pages),
// in boxes of the keys (at most `keys`) that lie together in a page and their
// values, with TMA's 128-byte swizzle.
bool kv_tensor_map(CUtensorMap& map, const AttendArgs& a, int keys);

cudaError_t attend_few(const AttendArgs& a, int dtype, int sms, cudaStream_t s);
cudaError_t attend_many(const AttendArgs& a, int dtype, int sms, cudaStream_t s);

}  // namespace ufb
