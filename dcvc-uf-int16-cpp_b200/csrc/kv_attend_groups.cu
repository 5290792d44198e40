// Attention of groups of streams that begin with common pages (ufb_kv_attend_groups):
// the branches of one stream, which go on by few tokens of their own.
//
//   S = Q K^T,  P = 2^(S f + log2 vs - M),  O = P V,  l = sum P / vs,  out = O / l
//
// as in kv_attend_many.cu, in tiles of 128 rows x 128 keys on the fifth-generation tensor
// cores.  The rows of a group -- all its streams' new tokens times the query heads of a
// key head -- go through the common keys once; then, in the same accumulators, through
// the streams' own keys, which only that stream's rows see.  Own keys lie in the tiles one
// stream's behind the other's, from every 16th key on: 19 branches with 9 own tokens each
// fill 3 tiles, not 19 (10 such groups, 8 heads of 128, 1324 common keys, 2 layers: 74 us
// where a tile to each stream took 98).  Nothing has to be joined but what CTAs share, and
// a step of a search is one launch and its join.
//
// One CTA an SM, six roles:
//   walker (1 warp)      divides the work, and says of the tiles ahead (four at a time, a
//                        lane to 16 keys) which pages hold their keys and who sees them
//   converter (8 warps)  integers from global memory through registers to float16 in
//                        shared memory, keys and values double buffered; a register takes
//                        the next tile's integers as soon as this one's are stored
//   MMA (1 warp)         S of the next tile before P V of this one: two tiles of scores
//                        in tensor memory, two of sums
//   softmax (2 x 4 warps) a thread to a row; the two sets take every other tile, each
//                        with a maximum and sums of its own, so that one exponentiates
//                        while the other loads or waits.  P goes back over S in float16.
//   scales (1 warp)      of each 16 keys, three tiles ahead
// Up to 64 rows are in the tile two times, up to 32 four times: a copy takes a half or a
// quarter of each tile's keys, its other weights are zeros, so all softmax warps work and
// a thread has 32 scores where it had 128.  The sums of both sets and all copies of a row
// become one at a piece's end.  Warps whose rows are padding, or no rows of an own tile's
// stream, skip the softmax.  A window leaves out tiles of common keys only; own keys behind
// it are loaded and masked.
//
// Measured on 148 SMs: 64 branches x 65320 keys, 64 query heads over 8 of 128: 213 us among
// calls of its own kind, 640 TFLOP/s, 3100 cycles a tile (217 to 228 us with its share, 600
// TFLOP/s); 8 streams x 8 branches, to 16381 keys, 4 heads of 128: 40 us a layer, 2700 cycles
// a tile.  The products of a tile take 1300 alone, its exponentials 1024, its integers 1400
// from HBM.  What bounds a tile is the chain S -> softmax -> P V -> S of a set (S and P share
// their columns; at 128 dims tensor memory is full), half a period each: of 128 scores a
// thread the softmax takes 4800 cycles, of 32 still 2800, in which a warp issues every 5 to 7
// cycles.  The roles share the instruction caches, and code counts: 126 KB of
// it ran 240 us where 108 KB take 226.  A call's start takes 6 us (division, look-ups of
// pages, the first loads), its end 3, the join 3 to 4.
#include "kv_attend.cuh"
#include "umma.cuh"

#include <type_traits>

namespace ufb {

namespace {

constexpr int kRows = 128;
constexpr int kKeys = 128;
constexpr int kGroups = kKeys / kGroupKeys;
static_assert(kGroupUnit == kGroupKeys, "own keys begin where pages and scales are looked up");
constexpr int kMmaWarp = 16, kWalkWarp = 17, kScaleWarp = 18;
constexpr int kThreads = 640;         // warps: softmax 0-7, converter 8-15, MMA 16, walker 17, scales 18; 19 idle
constexpr int kPieces = 4;            // pieces announced ahead
constexpr int kTiles = 8;             // tiles announced ahead
constexpr int kScaleRing = 4;
constexpr int kWarpPairs = 128;       // (group, row tile) pairs up to which one warp divides the work
constexpr int kCode = 45;
// A wait gives up after so many looks at its barrier; the hardware holds each for about 300
// cycles, so that is a second or so.  (A clock in every wait took three times the instructions,
// and the roles share the instruction caches.)
constexpr int kPolls = 1 << 22;
// As in kv_attend_many.cu: a running maximum stays while it grows by less than 2^kSlack, P is
// taken times 2^kShift, rows with scores beyond kFar round the score before the maximum is
// taken off.
constexpr float kSlack = 2.0f, kShift = 13.0f;
constexpr float kFar = 1048576.0f;   // 2^20

struct alignas(16) GroupScales {
    float key, log2_value, inv_value, pad;   // log2_value -inf: the 16 keys are not there
};

// One row tile of a group.
struct GroupTile {
    int token0;             // the group's first token
    int row0, rows;
    int low, high;          // first and last position of the group's tokens
    int shared, slot;       // common keys, and a stream that has them
    KeyRange keys;          // of the common ones
    int common, nt;         // tiles of common keys, of all
    int stream, last, own;  // the row tile's streams, their first tile among the group's of own keys
    int before;             // units of own keys of the streams before
};

// A piece of an item as the walker announces it; rows 0: there is none any more.
struct Announced {
    int rows, row0, token0, head, parts, part, shared;
    int count;              // its tiles
};
// A tile of a piece.
struct Tile {
    int key0, head;         // key0: of the common keys, or of the group's own ones
    int row_low, row_high;  // rows that may see it
    int place[kGroups];     // of each 16 keys among the pool's; -1: not looked at, or not there
    int flags;              // kClear: all its rows see all of it; kOwnKeys; kNone: there is no further tile
};
constexpr int kClear = 1, kOwnKeys = 2, kNone = 4;

template <int D>
struct Smem {
    alignas(1024) uint8_t q[kRows * D * 2];        // [64 dims][row][128 bytes]
    alignas(1024) uint8_t k[2][kKeys * D * 2];
    alignas(1024) uint8_t v[2][kKeys * D * 2];
    GroupScales scales[kScaleRing][kGroups];
    float2 stored[kTiles][kGroups];                // scales of keys and values as the pages have them
    float row[2][2][kRows];                        // maxima, weights: by parity
    float unit[kRows];                             // what a line's products count
    alignas(8) uint64_t k_full[2], v_empty[2], s_full[2], p_full[2][2];   // s_full: and the keys' place is free
    uint64_t q_full, o_full, drained, pair[4], all;
    uint64_t piece_full[kPieces], piece_empty[kPieces], tile_full[kTiles], tile_empty[kTiles];
    Announced pieces[kPieces];
    Tile tiles[kTiles];
    ShareSmem share;
    uint32_t tmem;
    int dead;
};

template <int D>
struct Tmem {
    __device__ static constexpr uint32_t s(int b) { return b * 128; }
    __device__ static constexpr uint32_t o(int b) { return 256 + b * D; }
};

// Address of row `row`, 16-byte chunk `chunk` (8 float16) of a [D / 64][128][128 bytes] tile.
__device__ __forceinline__ uint32_t tile_at(int row, int chunk) {
    return (chunk >> 3) * (128 * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

// The lowest n bits (none below 0, all from 32 on).
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u); }

__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

// Two 32-bit multiply-adds (x, y) = (x, y) f + add, two additions (a, b) += (x, y).
__device__ __forceinline__ void fma2(float& x, float& y, float f, float add) {
    asm("{\n\t.reg .b64 v, m, c;\n\t"
        "mov.b64 v, {%0, %1};\n\tmov.b64 m, {%2, %2};\n\tmov.b64 c, {%3, %3};\n\t"
        "fma.rn.f32x2 v, v, m, c;\n\tmov.b64 {%0, %1}, v;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(f), "f"(add));
}
__device__ __forceinline__ void add2(float& a, float& b, float x, float y) {
    asm("{\n\t.reg .b64 v, w;\n\t"
        "mov.b64 v, {%0, %1};\n\tmov.b64 w, {%2, %3};\n\t"
        "add.rn.f32x2 v, v, w;\n\tmov.b64 {%0, %1}, v;\n\t}"
        : "+f"(a), "+f"(b)
        : "f"(x), "f"(y));
}

// (x, y) = (x, y) f + (u, v) g
__device__ __forceinline__ void weigh2(float& x, float& y, float f, float u, float v, float g) {
    asm("{\n\t.reg .b64 a, b, m, n;\n\t"
        "mov.b64 a, {%0, %1};\n\tmov.b64 m, {%2, %2};\n\tmov.b64 b, {%3, %4};\n\tmov.b64 n, {%5, %5};\n\t"
        "mul.rn.f32x2 b, b, n;\n\tfma.rn.f32x2 a, a, m, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(f), "f"(u), "f"(v), "f"(g));
}

// The larger of two pairs, entry by entry, of their absolute values; NaN if there is one.
__device__ __forceinline__ uint32_t top2(uint32_t a, uint32_t b, __half) {
    const __half2 m = __hmax2_nan(__habs2(*reinterpret_cast<const __half2*>(&a)), __habs2(*reinterpret_cast<const __half2*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t top2(uint32_t a, uint32_t b, __nv_bfloat16) {
    const __nv_bfloat162 m = __hmax2_nan(__habs2(*reinterpret_cast<const __nv_bfloat162*>(&a)), __habs2(*reinterpret_cast<const __nv_bfloat162*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&m);
}

// One lane of a whole warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}
// Products by the elected lane; a descriptor's address is in its lower word.
__device__ __forceinline__ void product(uint32_t d, uint32_t a, uint32_t a_high, uint32_t b, uint32_t b_high, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tmov.b64 x, {%1, %2};\n\tmov.b64 y, {%3, %4};\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, p;\n\t}" ::"r"(d), "r"(a), "r"(a_high), "r"(b), "r"(b_high), "r"(idesc),
        "r"(static_cast<uint32_t>(accumulate))
        : "memory");
}
// A in tensor memory.
__device__ __forceinline__ void product_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t b_high, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tmov.b64 y, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(b_high), "r"(idesc),
        "r"(static_cast<uint32_t>(accumulate))
        : "memory");
}

__device__ __forceinline__ void cp_async4(void* to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}

__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Once all blocks have said so the next launch's may take what room there is; they wait for this one's end.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// false: the pair (group, row tile) does not exist, or ufb_kv_share has turned the group away or not
// seen it as it is.
__device__ __forceinline__ bool group_tile(const AttendArgs& a, const GroupArgs& g, int group, int rt, GroupTile& t) {
    const int4* record = reinterpret_cast<const int4*>(g.state.group + group);
    const int4 place = record[0], keys = record[1], rest = record[2];   // KvGroupState::Group
    if (rest.y != *g.changes + 1) return false;
    int own = rest.x;
    t.token0 = place.x;
    t.row0 = rt * kRows;
    const int rows = place.y * a.group;
    t.rows = min(kRows, rows - t.row0);
    if (t.rows <= 0) return false;
    t.shared = keys.x;
    t.slot = keys.y;
    t.low = keys.z;
    t.high = keys.w;
    t.stream = place.z;
    t.last = place.z + place.w - 1;
    t.before = 0;
    if (rows > kRows) {
        // the streams of these rows only
        t.stream = g.state.token[t.token0 + t.row0 / a.group].stream;
        t.last = g.state.token[t.token0 + (t.row0 + t.rows - 1) / a.group].stream;
        if (t.stream > place.z) t.before = g.state.units[t.stream - 1];
        own = g.state.units[t.last];
    }
    t.own = t.before / kGroups;
    t.keys = key_range<kKeys>(a, t.shared, 0, t.low - t.shared, t.high - t.shared);
    t.common = t.keys.hi > 0 ? t.keys.nt : 0;
    // rows that see nothing are still written: one tile, all of it hidden
    t.nt = max(t.common + (own > t.before ? (own + kGroups - 1) / kGroups - t.own : 0), 1);
    return true;
}

// Walks the pieces of this CTA's share.
struct GroupWalker {
    int row_tiles, pair, pairs;
    long long pos, end, pair_start;
    bool loaded;
    GroupTile t;
    int head, first, last;      // the piece: key head, key tiles [first, last)
    long long item_start;

    __device__ __forceinline__ bool next(const AttendArgs& a, const GroupArgs& g) {
        if (pos >= end) return false;
        while (true) {
            if (pair >= pairs) return false;
            if (!loaded) {
                if (!group_tile(a, g, pair / row_tiles, pair % row_tiles, t)) {
                    pair = (pair / row_tiles + 1) * row_tiles;
                    continue;
                }
                loaded = true;
            }
            const long long size = static_cast<long long>(t.nt) * a.heads;
            if (pos < pair_start + size) break;
            pair_start += size;
            ++pair;
            loaded = false;
        }
        head = static_cast<int>(quotient(pos - pair_start, t.nt));
        item_start = pair_start + static_cast<long long>(head) * t.nt;
        first = static_cast<int>(pos - item_start);
        last = static_cast<int>(min(static_cast<long long>(t.nt), end - item_start));
        pos = item_start + last;
        return true;
    }
};

// share_out by one warp, which needs no other: for few pairs (lanes take 32 at a time).
// item: the tile that the share begins in.  tiles_of(p, t): the tiles of pair p, which is t.
template <class Tiles>
__device__ __forceinline__ Share share_of_warp(int pairs, Tiles tiles_of, GroupTile& item) {
    const int lane = threadIdx.x & 31;
    Share s;
    GroupTile t;
    long long v = 0;
    s.total = 0;
#pragma unroll 1
    for (int base = 0; base < pairs; base += 32) {
        v = base + lane < pairs ? tiles_of(base + lane, t) : 0;
        s.total += v;
    }
#pragma unroll 1
    for (int o = 16; o; o >>= 1) s.total += __shfl_xor_sync(0xffffffffu, s.total, o);
    s.per = max(quotient(s.total + gridDim.x - 1, gridDim.x), 1ll);
    s.pair = pairs, s.pair_start = 0;
    const long long start = s.per * blockIdx.x;
    long long before = 0;
#pragma unroll 1
    for (int base = 0; base < pairs; base += 32) {
        if (pairs > 32) v = base + lane < pairs ? tiles_of(base + lane, t) : 0;
        long long at = v;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += u;
        }
        const long long sum = __shfl_sync(0xffffffffu, at, 31);
        at += before - v;
        const uint32_t hit = __ballot_sync(0xffffffffu, at <= start && start < at + v);
        if (hit) {
            const int from = __ffs(hit) - 1;
            s.pair = base + from;
            s.pair_start = __shfl_sync(0xffffffffu, at, from);
            static_assert(sizeof(GroupTile) % 4 == 0, "words");
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(GroupTile) / 4); ++i)
                reinterpret_cast<int*>(&item)[i] = __shfl_sync(0xffffffffu, reinterpret_cast<const int*>(&t)[i], from);
            break;
        }
        before += sum;
    }
    return s;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) groups_kernel(const AttendArgs a, const GroupArgs g, int row_tiles) {
    // aligned by declaration, so that descriptors are constants (checked below)
    extern __shared__ __align__(1024) uint8_t raw[];
    Smem<D>& sm = *reinterpret_cast<Smem<D>*>(raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.k_full[i], 129);
            mbar_init(&sm.v_empty[i], 1);
            mbar_init(&sm.p_full[i][0], 256);   // the first half of the weights, and the values
            mbar_init(&sm.p_full[i][1], 128);
            mbar_init(&sm.s_full[i], 1);
        }
        mbar_init(&sm.q_full, 256);
        mbar_init(&sm.o_full, 1);
        mbar_init(&sm.drained, 1);
        for (int i = 0; i < 4; ++i) mbar_init(&sm.pair[i], 64);
        mbar_init(&sm.all, 256);
        for (int i = 0; i < kPieces; ++i) {
            mbar_init(&sm.piece_full[i], 1);
            mbar_init(&sm.piece_empty[i], 9);
        }
        for (int i = 0; i < kTiles; ++i) {
            mbar_init(&sm.tile_full[i], 1);
            mbar_init(&sm.tile_empty[i], 13);
        }
        fence_mbar_init();
        sm.dead = (smem_u32(raw) & 1023) != 0;
    }
    if (warp == kMmaWarp) {
        tmem_alloc(&sm.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    const int pairs = g.groups * row_tiles;
    auto tiles_of = [&](int p, GroupTile& t) -> long long {
        const int group = row_tiles == 1 ? p : p / row_tiles;
        return group_tile(a, g, group, p - group * row_tiles, t) ? static_cast<long long>(t.nt) * a.heads : 0;
    };
    __syncthreads();
    wait_for_previous();
    let_next_start();
    // Only the walker needs to know this CTA's share.  For few pairs its warp alone has the first
    // piece 5300 cycles after the start, where with the block's scan it had it after 7400; beyond
    // four rounds of 32 loads the block divides.
    Share share;
    if (pairs > kWarpPairs)
        share = share_out<kThreads>(
            pairs, 1,
            [&](int p) {
                GroupTile t;
                return tiles_of(p, t);
            },
            sm.share);
    tc_fence_after();
    // all 512 columns are this CTA's: its tensor memory begins at 0
    constexpr uint32_t tmem = 0;
    volatile int* dead = &sm.dead;
    // after a wait gave up nobody waits any more, and no further tile is begun
    auto wait = [&](uint64_t* bar, int phase) {
        for (int polls = 0; !mbar_try_wait(bar, phase & 1); ++polls) {
            if (*dead) return;
            if (polls == kPolls) *dead = 1;   // reported at the end
        }
    };
    // Tiles one after another; a reader gives each back when it is done with it.
    auto tile_info = [&](int n) -> const Tile& {
        wait(&sm.tile_full[n % kTiles], n / kTiles);
        __syncwarp();
        return sm.tiles[n % kTiles];
    };
    // what the warp's lanes did before is seen by those that wait
    auto arrive = [&](uint64_t* bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    auto tile_done = [&](int n) { arrive(&sm.tile_empty[n % kTiles]); };

    // the registers of 640 threads at 96: 2 x 128 + 2 x 72 + 80 = 5 x 96
    if (warp < 8) {
        regs_inc<128>();
        // ---- softmax: the tiles of parity t, each into sums of its own
        const int t = warp >> 2, quarter = warp & 3, line = quarter * 32 + lane;   // line: of tensor memory
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t ts = tmem + lanes + Tmem<D>::s(t), to = tmem + lanes + Tmem<D>::o(t);
        const AttendScratch scratch = scratch_of(a.workspace, gridDim.x, kRows);
        if (threadIdx.x == 0) scratch.items[blockIdx.x * 8] = 0;
        // the two warps that share lines meet, in tensor memory too; all eight
        auto meet = [&](uint64_t* bar, int& met) {
            tc_fence_before();
            mbar_arrive(bar);
            wait(bar, met++);
            __syncwarp();
            tc_fence_after();
        };
        int pair_met = 0, all_met = 0;
        auto pair_sync = [&] { meet(&sm.pair[quarter], pair_met); };
        auto all_sync = [&] { meet(&sm.all, all_met); };
        int first = 0;   // number of the piece's first tile among this CTA's
        for (int piece = 0;; ++piece) {
            wait(&sm.piece_full[piece % kPieces], piece / kPieces);
            __syncwarp();
            const Announced& p = sm.pieces[piece % kPieces];
            if (p.rows == 0 || *dead) break;
            const int count = p.count;
            // up to 64 rows lie in the tile two times, up to 32 four times: copy `copy` takes
            // `wide` of each tile's chunks of 32 keys
            const int wide = p.rows > 64 ? 4 : p.rows > 32 ? 2 : 1;
            const int copy = wide == 4 ? 0 : wide == 2 ? quarter >> 1 : quarter;
            const int row0 = (quarter - copy * wide) * 32, row = row0 + lane;
            const bool real = row < p.rows;
            const bool busy = row0 < p.rows;
            const int in_group = p.row0 + (real ? row : 0);
            int token = in_group / a.group;
            const int head = p.head * a.group + in_group - token * a.group;
            token += p.token0;
            int4 seat = make_int4(-1, 0, 0, 0);   // KvGroupState::Token
            if (real) seat = reinterpret_cast<const int4*>(g.state.token)[token];
            const bool write = real && seat.x != kNotWritten;
            const int pos = write ? seat.x : -1;
            float m = -INFINITY, l = 0.0f;
            bool far = false;   // a row of the warp has scores beyond kFar
            // The queries: a warp takes 16 lines, D / 8 lanes to a line.  To [2^15, 2^16) and
            // float16; the softmax scale's sign goes with it.
            {
                constexpr int kLanes = D / 8, kLines = 32 / kLanes;
                const int mine = (warp * 16 + (lane & 15)) & (wide * 32 - 1);   // a row for each lane's sake
                const uint32_t there = __ballot_sync(0xffffffffu, mine < p.rows);
                const int of_group = p.row0 + mine, of_token = of_group / a.group;
                const long long at = (p.token0 + of_token) * a.q.token_stride + (p.head * a.group + of_group - of_token * a.group) * a.q.head_stride;
                uint4 v[16 / kLines];
#pragma unroll
                for (int i = 0; i < 16 / kLines; ++i) {
                    const int j = i * kLines + lane / kLanes;
                    const long long from = __shfl_sync(0xffffffffu, at, j);
                    v[i] = make_uint4(0, 0, 0, 0);
                    if (there >> j & 1) v[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q.data) + from + lane % kLanes * 8);
                }
#pragma unroll
                for (int i = 0; i < 16 / kLines; ++i) {
                    const int j = warp * 16 + i * kLines + lane / kLanes;
                    uint32_t largest = top2(top2(v[i].x, v[i].y, T()), top2(v[i].z, v[i].w, T()), T());
#pragma unroll
                    for (int o = 1; o < kLanes; o <<= 1) largest = top2(largest, __shfl_xor_sync(0xffffffffu, largest, o), T());
                    const float2 f = unpack2(largest, T());
                    const float u = row_unit(f.x == f.x && f.y == f.y ? fmaxf(f.x, f.y) : __int_as_float(0x7fffffff));
                    const float mul = u == u ? (a.scale_log2 < 0.0f ? -u : u) : 0.0f;
                    const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
                    uint32_t y[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2 d = unpack2(x[k], T());
                        y[k] = pack2(d.x * mul, d.y * mul, __half());
                    }
                    *reinterpret_cast<uint4*>(sm.q + tile_at(j, lane % kLanes)) = make_uint4(y[0], y[1], y[2], y[3]);
                    if (lane % kLanes == 0) sm.unit[j] = unit_inverse(u) * fabsf(a.scale_log2);
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(&sm.q_full);
            for (int n = first + ((first ^ t) & 1); n < first + count; n += 2) {
                const Tile& tile = tile_info(n);
                const int flags = tile.flags;
                // columns below high are seen by this row that are from low on, or from first on and below sink
                int high = 0, low = 0, sink = 0, begin = 0;
                bool mine = busy;   // rows of this warp that the tile is for
                if (!(flags & kClear)) {
                    const int row_low = tile.row_low, row_high = tile.row_high;
                    mine = busy && row_low < row0 + 32 && row_high > row0;
                    // column of key 0
                    const int zero = (flags & kOwnKeys ? seat.y - p.shared : 0) - tile.key0;
                    begin = flags & kOwnKeys ? seat.y - tile.key0 : 0;
                    const int end = flags & kOwnKeys ? seat.z - tile.key0 : p.shared - tile.key0;
                    high = a.causal || !(flags & kOwnKeys) ? min(end, pos + 1 + zero) : end;
                    low = begin;
                    // sinks that reach past the end act as the end: of any number of them the sum stays in 32 bits
                    if (a.window) low = max(begin, pos - a.window + 1 + zero), sink = min(a.sinks, end - zero) + zero;
                }
                tile_done(n);
                wait(&sm.s_full[t], n >> 1);
                __syncwarp();
                tc_fence_after();
                if (!mine) {
                    // rows of other streams: no weight.  (Padding's weights do not matter.)
                    if (busy) {
                        uint32_t w[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) w[j] = 0;
#pragma unroll
                        for (int c = 0; c < 4; ++c) tmem_st16(ts + c * 16, w);
                        tmem_wait_st();
                    }
                    tc_fence_before();
                    mbar_arrive(&sm.p_full[t][0]);
                    mbar_arrive(&sm.p_full[t][1]);
                    continue;
                }
                const GroupScales* sc = sm.scales[n % kScaleRing];
                const float unit = sm.unit[line];
                auto seen = [&](int c) {   // of 32 columns, a bit each
                    return bits_below(high - c * 32) & (~bits_below(low - c * 32) | (bits_below(sink - c * 32) & ~bits_below(begin - c * 32)));
                };
                // 64 columns at a time, the later ones first: the others stay for their weights
                uint32_t s0[32], s1[32];
                float top = -INFINITY;
                auto maximum = [&](auto masked) {
                    auto chunk = [&](int c, const uint32_t (&s)[32]) {
                        const uint32_t bits = decltype(masked)::value ? seen(c) : 0u;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            auto f = [&](int j) {
                                return decltype(masked)::value && !(bits & (1u << (h * 16 + j))) ? -INFINITY : __uint_as_float(s[h * 16 + j]);
                            };
                            float y = max3(f(0), f(1), f(2)), z = max3(f(3), f(4), f(5));
                            y = max3(y, f(6), f(7)), z = max3(z, f(8), f(9));
                            y = max3(y, f(10), f(11)), z = max3(z, f(12), f(13));
                            y = max3(y, f(14), f(15));
                            y = fmaxf(y, z);
                            const GroupScales gs = sc[c * 2 + h];
                            const float v = fmaf(y, unit * gs.key, gs.log2_value);
                            // -infinity: nothing of the group is seen
                            top = fmaxf(top, decltype(masked)::value && y == -INFINITY ? y : v);
                        }
                    };
#pragma unroll 1
                    for (int c = wide == 4 ? 2 : copy * wide; c >= copy * wide; c -= 2) {
                        tmem_ld32(ts + c * 32, s0);
                        if (wide > 1) tmem_ld32(ts + c * 32 + 32, s1);
                        tmem_wait_ld();
                        tmem_tie32(s0);
                        tmem_tie32(s1);
                        chunk(c, s0);
                        if (wide > 1) chunk(c + 1, s1);
                    }
                };
                const bool clear = flags & kClear;
                if (clear) maximum(std::false_type());
                else maximum(std::true_type());
                if (wide < 4) {
                    // the keys of the other copies have no weight in this one
                    uint32_t w[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) w[j] = 0;
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (c < copy * wide || c >= copy * wide + wide) tmem_st16(ts + c * 16, w);
                }
                // the maximum stays while it is within 2^kSlack; these sums' last product was before these scores
                const bool grow = top > __fadd_rd(m, kSlack);
                if (__any_sync(0xffffffffu, grow)) {
                    if (__any_sync(0xffffffffu, grow && m != -INFINITY)) {
                        const float keep = grow && m != -INFINITY ? ex2(m - top) : 1.0f;
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16];
                            tmem_ld16(to + c * 16, o);
                            tmem_wait_ld_regs(o);
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
                            tmem_st16(to + c * 16, o);
                        }
                        l *= keep;
                    }
                    if (grow) m = top;
                    far = __any_sync(0xffffffffu, fabsf(m) >= kFar && m != -INFINITY);
                }
                const float base = m == -INFINITY ? 0.0f : __fsub_ru(m, kShift);
                auto weights = [&](auto masked) {
                    // 32 columns: P, the row's weight
                    auto chunk = [&](int c, uint32_t (&s)[32]) {
                        const uint32_t bits = decltype(masked)::value ? seen(c) : 0u;
                        uint32_t w[16];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const GroupScales gs = sc[c * 2 + h];
                            const float f = unit * gs.key, add = decltype(masked)::value ? gs.log2_value : gs.log2_value - base;
                            float sum[2] = {0.0f, 0.0f};
#pragma unroll
                            for (int j = 0; j < 16; j += 2) {
                                float x = __uint_as_float(s[h * 16 + j]), y = __uint_as_float(s[h * 16 + j + 1]);
                                fma2(x, y, f, add);
                                if (decltype(masked)::value) {
                                    add2(x, y, -base, -base);
                                    if (!(bits & (1u << (h * 16 + j)))) x = -INFINITY;
                                    if (!(bits & (1u << (h * 16 + j + 1)))) y = -INFINITY;
                                }
                                x = ex2(x);
                                y = ex2(y);
                                add2(sum[0], sum[1], x, y);
                                w[h * 8 + j / 2] = pack2(x, y, __half());
                            }
                            sum[0] += sum[1];
                            if (sum[0] != 0.0f) l = fmaf(sum[0], gs.inv_value, l);
                        }
                        tmem_st16(ts + c * 16, w);
                    };
                    // the next columns are on their way while these are worked on
#pragma unroll 1
                    for (int c = copy * wide; c < copy * wide + wide; c += 2) {
                        const bool more = wide == 4 && c == 0;
                        tmem_wait_ld();
                        tmem_tie32(s0);
                        tmem_tie32(s1);
                        chunk(c, s0);
                        if (more) tmem_ld32(ts + 64, s0);
                        if (wide > 1) chunk(c + 1, s1);
                        if (more) tmem_ld32(ts + 96, s1);
                        // P V starts on the first 64 keys while the others are in the works
                        tmem_wait_st();
                        tc_fence_before();
                        if (more || wide < 4) mbar_arrive(&sm.p_full[t][0]);
                        if (!more) mbar_arrive(&sm.p_full[t][1]);
                    }
                };
                if (clear && !far) weights(std::false_type());
                else weights(std::true_type());
            }
            // sets that had no tile have no sums
            const int sums0 = count > 1 || !(first & 1) ? 0 : 1, sums1 = count > 1 || (first & 1) ? 1 : 0;
            first += count;

            // ---- the piece's rows: the sums of both sets and all copies, half of the dims each
            if (busy) {
                sm.row[0][t][line] = m;
                sm.row[1][t][line] = l;
            }
            wait(&sm.o_full, piece);
            __syncwarp();
            tc_fence_after();
            if (busy) {
                if (wide == 4) pair_sync();
                else all_sync();
                // of the lines that have this row
                auto copy_of = [&](int i) { return ((i ^ quarter) & (wide - 1)) == 0; };
                float tops[4][2], top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        tops[i][u] = copy_of(i) ? sm.row[0][u][i * 32 + lane] : -INFINITY;
                        top = fmaxf(top, tops[i][u]);
                    }
                float weight = 0.0f, e0 = 0.0f, e1 = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const float l = copy_of(i) ? sm.row[1][u][i * 32 + lane] : 0.0f;
                        // a part that saw nothing has no weight; one that is not finite spoils its row
                        const float e = tops[i][u] == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : ex2(tops[i][u] - top);
                        if (e != 0.0f) weight += l * e;
                        if (i == quarter) (u ? e1 : e0) = e;
                    }
                const bool whole = p.part < 0;
                const int part = 2 * blockIdx.x + p.part;
                const float inv = !whole ? 1.0f : weight == 0.0f ? 0.0f : 1.0f / weight;
                e0 *= inv, e1 *= inv;
                T* out = static_cast<T*>(a.out.data) + head * a.out.head_stride;   // of a row: behind its token
                float* sums = scratch.sums + static_cast<long long>(part) * kRows * D;
                // 16 dims of this line
                auto sum16 = [&](int c, float (&o)[16]) {
                    uint32_t x[16], y[16];
                    tmem_ld16(tmem + lanes + Tmem<D>::o(0) + sums0 * D + c * 16, x);
                    tmem_ld16(tmem + lanes + Tmem<D>::o(0) + sums1 * D + c * 16, y);
                    tmem_wait_ld_regs(x);
                    tmem_wait_ld_regs(y);
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        o[j] = __uint_as_float(x[j]), o[j + 1] = __uint_as_float(x[j + 1]);
                        weigh2(o[j], o[j + 1], e0, __uint_as_float(y[j]), __uint_as_float(y[j + 1]), e1);
                    }
                };
                auto store4 = [&](T* to, float4 v) { *reinterpret_cast<uint2*>(to) = make_uint2(pack2(v.x, v.y, T()), pack2(v.z, v.w, T())); };
                if (wide == 4) {
                    T* to = out + static_cast<long long>(token) * a.out.token_stride;
#pragma unroll 1
                    for (int c = t * (D / 32); c < (t + 1) * (D / 32); ++c) {
                        float o[16];
                        sum16(c, o);
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            const float4 v = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                            if (write && whole) store4(to + c * 16 + j, v);
                            else if (real && !whole) __stcg(reinterpret_cast<float4*>(sums + row * D + c * 16 + j), v);
                        }
                        __syncwarp();
                    }
                } else {
                    // a quarter of the dims of all lines at a time through the queries' place, where
                    // neighbouring threads then add up neighbouring dims of a row
                    constexpr int kChunks = D / 16;   // of 4 dims, in a step of a set
                    float4* place = reinterpret_cast<float4*>(sm.q) + t * kRows * kChunks;
#pragma unroll 1
                    for (int step = 0; step < 2; ++step) {
                        const int dim0 = t * (D / 2) + step * (D / 4);
#pragma unroll 1
                        for (int c = 0; c < D / 64; ++c) {
                            float o[16];
                            sum16(dim0 / 16 + c, o);
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                place[line * kChunks + ((c * 4 + j) ^ (lane & (kChunks - 1)))] =
                                    make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                        }
                        all_sync();
#pragma unroll 1
                        for (int i = line; i < wide * 32 * kChunks; i += kRows) {
                            const int r = i / kChunks, c = i % kChunks;
                            if (r >= p.rows) break;
                            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if (k * wide < 4) {
                                    const float4 x = place[(k * wide * 32 + r) * kChunks + (c ^ (r & (kChunks - 1)))];
                                    v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
                                }
                            if (!whole) {
                                __stcg(reinterpret_cast<float4*>(sums + r * D + dim0 + c * 4), v);
                            } else {
                                const int of_group = p.row0 + r, of_token = of_group / a.group;
                                if (g.state.token[p.token0 + of_token].position != kNotWritten)
                                    store4(static_cast<T*>(a.out.data) + (p.token0 + of_token) * a.out.token_stride +
                                               (p.head * a.group + of_group - of_token * a.group) * a.out.head_stride + dim0 + c * 4, v);
                            }
                        }
                        if (step == 0) all_sync();
                    }
                }
                if (t == 0 && copy == 0 && write && whole && a.lse)
                    a.lse[static_cast<long long>(token) * (a.heads * a.group) + head] =
                        weight == 0.0f ? -INFINITY : (top - kShift + log2f(weight)) * 0.6931471805599453f;
                if (t == 0 && copy == 0 && real && !whole) {
                    __stcg(scratch.stats + (part * 2) * kRows + row, top);
                    __stcg(scratch.stats + (part * 2 + 1) * kRows + row, weight);
                }
                // the next piece's queries and sums wait until all have read these
                if (wide == 4) pair_sync();
                else all_sync();
            }
            if (p.parts && threadIdx.x == 0) {
                int32_t* item = scratch.items + blockIdx.x * 8;
                item[1] = p.token0;
                item[2] = p.row0;
                item[3] = p.rows;
                item[4] = p.head;
                item[0] = p.parts;
            }
            arrive(&sm.piece_empty[piece % kPieces]);
            tc_fence_before();
        }
    } else if (warp < kMmaWarp) {
        regs_dec<72>();
        // ---- converter: warps 8-11 the keys and the scales, 12-15 the values, 32 keys each
        constexpr int kLoads = D / 16;   // 16-byte loads of a thread for a tile
        const int side = (warp - 8) >> 2, w = warp & 3;
        const int chunk = D == 128 ? (lane & 3) + ((lane >> 3) & 1) * 4 : lane & 3;
        const int sub = D == 128 ? ((lane >> 2) & 1) + ((lane >> 4) & 1) * 2 : lane >> 2;
        constexpr int kStep = D == 128 ? 4 : 8;   // rows of one load of a warp
        uint64_t* empty = side ? sm.v_empty : sm.s_full;
        uint8_t* tiles = side ? sm.v[0] : sm.k[0];
        // this thread's two 16-byte pieces of its first row; row & 7 repeats every kStep * 2 rows
        uint32_t at0[2], at1[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            at0[i] = tile_at(w * 32 + i * kStep + sub, chunk * 2);
            at1[i] = tile_at(w * 32 + i * kStep + sub, chunk * 2 + 1);
        }
        uint4 buf[kLoads];
        const uint8_t* from[2] = {};   // of this warp's two groups of 16 keys
        int place[2] = {-1, -1};
        // what is not there keeps what was: its weights are 0
        auto load = [&](int i) {
            if (place[(i * kStep) >> 4] >= 0)   // sub < kStep, a divisor of 16
                buf[i] = __ldg(reinterpret_cast<const uint4*>(from[(i * kStep) >> 4] + ((i * kStep) & 15) * D));
        };
        bool more = true;
        // tile n from its registers, which then take tile n + 1: a tile's time until it is looked at
#pragma unroll 1
        for (int n = -1; more; ++n) {
            const Tile& t = tile_info(n + 1);
            more = !(t.flags & kNone) && !*dead;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                place[i] = more ? t.place[w * 2 + i] : -1;
                const int row = (place[i] & (a.page_tokens / 16 - 1)) * 16 + sub;
                const long long tile = (static_cast<long long>(place[i] >> (a.page_shift - 4)) * 2 + side) * a.heads + t.head;
                from[i] = reinterpret_cast<const uint8_t*>(a.kv) + ((tile << a.page_shift) + row) * D + chunk * 16;
            }
            if (more) tile_done(n + 1);
            if (n < 0) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    buf[i] = make_uint4(0, 0, 0, 0);
                    load(i);
                }
                continue;
            }
            const int b = n & 1;
            if (n >= 2) wait(&empty[b], (n >> 1) - 1);
            uint8_t* to = tiles + b * (kKeys * D * 2);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint32_t x[4] = {buf[i].x, buf[i].y, buf[i].z, buf[i].w};
                uint32_t y[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) int8x4_to_half(x[j], y[2 * j], y[2 * j + 1]);
                const int step = (i / 2) * 2 * kStep * 128;
                *reinterpret_cast<uint4*>(to + at0[i & 1] + step) = make_uint4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<uint4*>(to + at1[i & 1] + step) = make_uint4(y[4], y[5], y[6], y[7]);
                load(i);
            }
            fence_proxy_async_smem();
            mbar_arrive(side ? &sm.p_full[b][0] : &sm.k_full[b]);
        }
    } else {
        regs_dec<80>();
        if (warp == kWalkWarp) {
            // ---- walker: announces this CTA's pieces and their tiles
            GroupWalker walk;
            if (pairs <= kWarpPairs) share = share_of_warp(pairs, tiles_of, walk.t);
            walk.row_tiles = row_tiles;
            walk.pairs = pairs;
            walk.pos = share.per * blockIdx.x;
            walk.end = min(walk.pos + share.per, share.total);
            walk.pair = share.pair;
            walk.pair_start = share.pair_start;
            walk.loaded = pairs <= kWarpPairs;
            int n = 0, piece = 0;
            for (; !*dead && walk.next(a, g); ++piece) {
                const GroupTile& t = walk.t;
                if (piece >= kPieces) wait(&sm.piece_empty[piece % kPieces], piece / kPieces - 1);
                if (lane == 0) {
                    Announced& o = sm.pieces[piece % kPieces];
                    o.rows = t.rows;
                    o.row0 = t.row0;
                    o.token0 = t.token0;
                    o.shared = t.shared;
                    o.head = walk.head;
                    o.count = walk.last - walk.first;
                    // the part of a shared item: 0 where an earlier CTA began it, 1 where this
                    // one does, which then tells how many parts there are
                    const bool whole = walk.first == 0 && walk.last == t.nt;
                    o.part = whole ? -1 : (walk.first > 0 ? 0 : 1);
                    o.parts = o.part == 1 ? static_cast<int>(quotient(walk.item_start + t.nt - 1, share.per)) - static_cast<int>(blockIdx.x) + 1 : 0;
                    mbar_arrive(&sm.piece_full[piece % kPieces]);
                }
                // four tiles at a time, a lane to 16 keys of one
                const int my_tile = lane / kGroups, my_key = (lane % kGroups) * kGroupKeys;
                // own keys: 32 streams at a time, from `seen` on, a lane to each; before: units ahead of them
                int seen = t.stream - 32, before = t.before, units = t.before, slot_of = 0, low_of = 0, high_of = 0;
                auto look_on = [&] {
                    before = __shfl_sync(0xffffffffu, units, 31);
                    seen += 32;
                    const int s = min(seen + lane, t.last);
                    units = g.state.units[s], slot_of = a.slots[s], low_of = a.offsets[s], high_of = a.offsets[s + 1];
                };
                for (int i0 = walk.first; i0 < walk.last; i0 += 4) {
                    const int i = min(i0 + my_tile, walk.last - 1);
                    Tile o;
                    o.head = walk.head;
                    o.flags = 0;
                    o.row_low = 0;
                    o.row_high = kRows;
                    int slot = t.slot, key = -1;          // lane's 16 keys; -1: not looked at
                    const bool own = i >= t.common;
                    if (!own) {
                        o.key0 = t.keys.tile(i) * kKeys;
                        if (t.keys.touches(o.key0 + my_key)) key = o.key0 + my_key;
                        if (o.key0 + kKeys - 1 <= t.low && o.key0 + kKeys <= t.shared &&
                            (!a.window || t.high - o.key0 < a.window || o.key0 + kKeys <= a.sinks))
                            o.flags |= kClear;
                    } else {
                        o.key0 = (t.own + i - t.common) * kKeys;
                        o.flags |= kOwnKeys;
                        o.row_low = kRows, o.row_high = 0;
                    }
                    const int unit = own ? (o.key0 + my_key) / kGroupUnit : INT_MAX;
                    bool wanted = own;
                    if (__any_sync(0xffffffffu, own) && seen < t.stream) look_on();
                    while (__any_sync(0xffffffffu, wanted)) {
                        // the first stream whose units reach beyond this one
                        int k = 0;
#pragma unroll
                        for (int d = 16; d; d >>= 1)
                            if (__shfl_sync(0xffffffffu, units, k + d - 1) <= unit) k += d;
                        const int until = __shfl_sync(0xffffffffu, units, k), ahead = __shfl_sync(0xffffffffu, units, max(k - 1, 0));
                        const int found = __shfl_sync(0xffffffffu, slot_of, k);
                        const int low = __shfl_sync(0xffffffffu, low_of, k), high = __shfl_sync(0xffffffffu, high_of, k);
                        const int from = k > 0 ? ahead : before;
                        if (wanted && unit < until) {
                            wanted = false;
                            if (unit >= from) {   // else of a stream before this row tile's
                                slot = found;
                                key = t.shared + (unit - from) * kGroupUnit;
                                o.row_low = (low - t.token0) * a.group - t.row0;
                                o.row_high = (high - t.token0) * a.group - t.row0;
                            }
                        }
                        if (seen + 32 > t.last || !__any_sync(0xffffffffu, wanted)) break;
                        look_on();
                    }
                    // all its streams' rows
#pragma unroll
                    for (int d = 1; d < kGroups; d <<= 1) {
                        o.row_low = min(o.row_low, __shfl_xor_sync(0xffffffffu, o.row_low, d));
                        o.row_high = max(o.row_high, __shfl_xor_sync(0xffffffffu, o.row_high, d));
                    }
                    int place = -1;
                    const int entry = key >> a.page_shift;
                    if (key >= 0 && entry < a.table_width) {
                        const int page = a.table[static_cast<long long>(slot) * a.table_width + entry];
                        if (page >= 0 && page < a.pages)
                            place = (page << (a.page_shift - 4)) + ((key & (a.page_tokens - 1)) >> 4);
                    }
                    const int tiles = min(walk.last - i0, 4);
                    for (int j = 0; j < tiles; ++j, ++n) {
                        if (n >= kTiles) wait(&sm.tile_empty[n % kTiles], n / kTiles - 1);
                        Tile& to = sm.tiles[n % kTiles];
                        if (my_tile == j) {
                            to.place[lane % kGroups] = place;
                            if (lane % kGroups == 0) {
                                to.key0 = o.key0, to.head = o.head, to.flags = o.flags;
                                to.row_low = o.row_low, to.row_high = o.row_high;
                            }
                        }
                        arrive(&sm.tile_full[n % kTiles]);
                    }
                }
            }
            if (n >= kTiles) wait(&sm.tile_empty[n % kTiles], n / kTiles - 1);
            if (piece >= kPieces) wait(&sm.piece_empty[piece % kPieces], piece / kPieces - 1);
            if (lane == 0) {
                sm.tiles[n % kTiles].flags = kNone;
                mbar_arrive(&sm.tile_full[n % kTiles]);
                sm.pieces[piece % kPieces].rows = 0;
                mbar_arrive(&sm.piece_full[piece % kPieces]);
            }
            __syncwarp();
            // No tile is made of groups that share has turned away or not seen as they are: their rows see
            // no key.  Here, while the others work on the last tiles, it costs 0 to 0.3 us; a warp of its
            // own, which looks beside the first look-ups, took 0.7 us of each call, the join 0.3.
            const int heads = a.heads * a.group;
            for (int group = blockIdx.x; group < g.groups; group += gridDim.x) {
                const int seen = g.state.group[group].seen, now = *g.changes + 1;
                if (seen == now) continue;
                if (lane == 0) atomicCAS(a.status, 0, seen == ~now ? kStatusIndex : kStatusShare);
                const int first = max(g.first[group], 0), end = min(g.first[group + 1], a.n);
                const int o0 = g.offsets[group], o1 = g.offsets[group + 1];
                // of the streams' tokens alone: where the bounds are not the batch's, rows may be another group's
                if (first > end || o0 < 0 || o1 > a.tokens || o0 != a.offsets[first] || o1 != a.offsets[end]) continue;
                for (long long token = o0; token < o1; ++token) {
                    T* to = static_cast<T*>(a.out.data) + token * a.out.token_stride;
                    for (int i = lane; i < heads * (D / 8); i += 32)
                        *reinterpret_cast<uint4*>(to + i / (D / 8) * a.out.head_stride + i % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
                    for (int h = lane; a.lse && h < heads; h += 32) a.lse[token * heads + h] = -INFINITY;
                }
            }
            __syncwarp();
        }
        if (warp == kScaleWarp) {
            // ---- scales: a lane to 16 keys, kAhead tiles ahead of what is written
            constexpr int kAhead = 3;
            bool more = true;
            int known = 0;
            auto fetch = [&](int n) {
                const Tile* t = more ? &tile_info(n) : nullptr;
                more = more && !(t->flags & kNone) && !*dead;
                if (more) {
                    if (lane < kGroups) {
                        float2* to = &sm.stored[n % kTiles][lane];
                        if (t->place[lane] >= 0) {
                            const float* s = a.scale + static_cast<long long>(t->place[lane] >> (a.page_shift - 4)) * 2 * a.heads + t->head;
                            cp_async4(&to->x, s);
                            cp_async4(&to->y, s + a.heads);
                        } else {
                            *to = make_float2(0.0f, -1.0f);   // -1: not there
                        }
                    }
                    ++known;
                    tile_done(n);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
#pragma unroll 1
            for (int n = -kAhead; n < known; ++n) {
                fetch(n + kAhead);
                if (n < 0) continue;
                asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
                const float2 got = sm.stored[n % kTiles][lane % kGroups];
                GroupScales s;
                const float v = got.y == -1.0f || !(got.y < kTinyScale) ? got.y : kTinyScale;
                s.key = got.x;
                s.log2_value = v == -1.0f ? -INFINITY : log2f(v);
                s.inv_value = v == -1.0f ? 0.0f : 1.0f / v;
                s.pad = 0.0f;
                // the scores two tiles back are made, so the weights four tiles back are: their place is free
                if (n >= 2) wait(&sm.s_full[n & 1], (n >> 1) - 1);
                if (lane < kGroups) sm.scales[n % kScaleRing][lane] = s;
                arrive(&sm.k_full[n & 1]);
            }
        }
        // ---- MMA: the warp waits together, one lane issues
        if (warp == kMmaWarp) {
            constexpr uint32_t qk = f16_idesc(128, kKeys, false), pv = f16_idesc(128, D, true);
            constexpr uint32_t kTile = (kKeys * D * 2) >> 4;   // descriptor step between the two buffers
            const uint64_t q_desc = sw128_desc(smem_u32(sm.q)), k_desc = sw128_desc(smem_u32(sm.k[0]));
            const uint64_t v_desc = sw128_n_major_desc(smem_u32(sm.v[0]), 128 * 128);
            const uint32_t q_low = static_cast<uint32_t>(q_desc), q_high = static_cast<uint32_t>(q_desc >> 32);
            const uint32_t v_high = static_cast<uint32_t>(v_desc >> 32);
            int n = 0;   // the piece's first tile
            for (int piece = 0;; ++piece) {
                wait(&sm.piece_full[piece % kPieces], piece / kPieces);
                __syncwarp();
                const int count = sm.pieces[piece % kPieces].rows ? sm.pieces[piece % kPieces].count : 0;
                arrive(&sm.piece_empty[piece % kPieces]);
                if (count == 0 || *dead) break;
                // the queries' place is free once the piece before is through
                wait(&sm.q_full, piece);
#pragma unroll 1
                for (int i = 0; i <= count; ++i) {
                    if (i < count) {
                        const int b = (n + i) & 1;
                        wait(&sm.k_full[b], (n + i) >> 1);
                        __syncwarp();
                        tc_fence_after();
                        if (elect_one()) {
                            const uint32_t kd = static_cast<uint32_t>(k_desc) + b * kTile;
#pragma unroll
                            for (int k = 0; k < D / 16; ++k) {
                                const uint32_t off = ((k >> 2) * (128 * 128) + (k & 3) * 32) >> 4;
                                product(tmem + Tmem<D>::s(b), q_low + off, q_high, kd + off, q_high, qk, k > 0);
                            }
                            mma_commit(&sm.s_full[b]);
                        }
                        __syncwarp();
                    }
                    if (i > 0) {
                        const int b = (n + i - 1) & 1;
                        const uint32_t vd = static_cast<uint32_t>(v_desc) + b * kTile;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            wait(&sm.p_full[b][h], (n + i - 1) >> 1);
                            __syncwarp();
                            tc_fence_after();
                            if (elect_one()) {
#pragma unroll
                                for (int k = h * 4; k < h * 4 + 4; ++k)
                                    product_ts(tmem + Tmem<D>::o(b), tmem + Tmem<D>::s(b) + k * 8, vd + k * (16 * 128 >> 4), v_high, pv,
                                               i > 2 || k > 0);   // a piece's first two tiles begin their sums
                                if (h == 1) {
                                    mma_commit(&sm.v_empty[b]);
                                    if (i == count) mma_commit(&sm.o_full);
                                }
                            }
                            __syncwarp();
                        }
                    }
                }
                n += count;
            }
            // nothing may be in flight when tensor memory is given back
            if (elect_one()) {
                mma_commit(&sm.drained);
                mbar_wait(&sm.drained, 0, a.status, kCode);
            }
            __syncwarp();
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *dead) atomicCAS(a.status, 0, kCode);
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(sm.tmem, 512);
    }
}

// Rows that several CTAs share: the item that CTA x's share ends in, a block's rows
// from kJoinRows * y on.  The parts' maxima and weights come first, once a row, by a
// warp; then a thread adds the parts of four columns, in the order of the CTAs.
constexpr int kJoinThreads = 256;
constexpr int kJoinAhead = 8;   // parts

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) groups_join_kernel(const AttendArgs a, const GroupArgs g, int ctas) {
    constexpr int kJoinRows = kJoinThreads / (D / 4);
    __shared__ float share[kAttendMaxCtas][kJoinRows];   // of a part in a row's sum
    __shared__ float tops[kJoinRows], weights[kJoinRows];
    const AttendScratch scratch = scratch_of(a.workspace, ctas, kRows);
    const int c0 = blockIdx.x, first = blockIdx.y * kJoinRows;
    let_next_start();
    wait_for_previous();
    const int32_t* item = scratch.items + c0 * 8;
    const int parts = item[0], rows = min(item[3] - first, kJoinRows);
    if (parts == 0 || rows <= 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r = threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4, row = first + r;
    auto part_sums = [&](int i) {
        const int from = 2 * (c0 + i) + (i == 0);
        return __ldcg(reinterpret_cast<const float4*>(scratch.sums + (static_cast<long long>(from) * kRows + row) * D + d));
    };
    // the first parts are on their way while the weights are worked out
    float4 ahead[kJoinAhead];
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i)
        if (i < parts && r < rows) ahead[i] = part_sums(i);
    for (int r = warp; r < rows; r += kJoinThreads / 32) {
        float top = -INFINITY;
        for (int i = lane; i < parts; i += 32)
            top = fmaxf(top, scratch.stats[(2 * (c0 + i) + (i == 0)) * 2 * kRows + first + r]);
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float weight = 0.0f;
        for (int i = lane; i < parts; i += 32) {
            const int from = 2 * (c0 + i) + (i == 0);
            const float m = scratch.stats[from * 2 * kRows + first + r], l = scratch.stats[(from * 2 + 1) * kRows + first + r];
            const float mul = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : ex2(m - top);
            share[i][r] = mul;
            weight += l * mul;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) weight += __shfl_xor_sync(0xffffffffu, weight, o);
        if (lane == 0) tops[r] = top, weights[r] = weight;
    }
    __syncthreads();
    if (r >= rows) return;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](int i, float4 x) {
        const float mul = share[i][r];
        v.x += x.x * mul, v.y += x.y * mul, v.z += x.z * mul, v.w += x.w * mul;
    };
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i)
        if (i < parts) add(i, ahead[i]);
#pragma unroll 8
    for (int i = kJoinAhead; i < parts; ++i) add(i, part_sums(i));
    const int in_group = item[2] + row;
    int token = in_group / a.group;
    const int head = item[4] * a.group + in_group - token * a.group;
    token += item[1];
    if (g.state.token[token].position == kNotWritten) return;
    const float top = tops[r], weight = weights[r];
    const float inv = weight == 0.0f ? 0.0f : 1.0f / weight;
    T* to = static_cast<T*>(a.out.data) + static_cast<long long>(token) * a.out.token_stride + head * a.out.head_stride + d;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2(v.x * inv, v.y * inv, T()), pack2(v.z * inv, v.w * inv, T()));
    if (a.lse && d == 0)
        a.lse[static_cast<long long>(token) * (a.heads * a.group) + head] =
            weight == 0.0f ? -INFINITY : (top - kShift + log2f(weight)) * 0.6931471805599453f;
}

template <typename T, int D>
cudaError_t launch(const AttendArgs& a, const GroupArgs& g, int sms, cudaStream_t s) {
    auto kernel = groups_kernel<T, D>;
    const int smem = sizeof(Smem<D>);
    static std::atomic<uint64_t> allowed;
    const cudaError_t attr = allow_smem(kernel, smem, allowed);
    if (attr != cudaSuccess) return attr;
    const long long row_tiles = (static_cast<long long>(g.max_tokens) * a.group + kRows - 1) / kRows;
    if (row_tiles * g.groups > 0x3fffffff) return cudaErrorInvalidValue;
    const int ctas = sms < kAttendMaxCtas ? sms : kAttendMaxCtas;
    // Both kernels may start before the one ahead of them has ended (each waits for that before it
    // reads anything): 16 branches 76.3 us for 78.8, a window 30.2 for 31.6.
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    config.stream = s;
    config.gridDim = dim3(ctas);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = smem;
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, a, g, static_cast<int>(row_tiles));
    if (e != cudaSuccess) return e;
    config.dynamicSmemBytes = 0;
    const long long rows = static_cast<long long>(g.max_tokens) * a.group;
    constexpr int kJoinRows = kJoinThreads / (D / 4);
    config.gridDim = dim3(ctas, static_cast<unsigned>(((rows < kRows ? rows : kRows) + kJoinRows - 1) / kJoinRows));
    config.blockDim = dim3(kJoinThreads);
    return cudaLaunchKernelEx(&config, groups_join_kernel<T, D>, a, g, ctas);
}

}  // namespace

cudaError_t kv_attend_groups(const AttendArgs& a, const GroupArgs& g, int dtype, int sms, cudaStream_t s) {
    if (a.head_dim == 64)
        return dtype == UFB_F16 ? launch<__half, 64>(a, g, sms, s) : launch<__nv_bfloat16, 64>(a, g, sms, s);
    return dtype == UFB_F16 ? launch<__half, 128>(a, g, sms, s) : launch<__nv_bfloat16, 128>(a, g, sms, s);
}

}  // namespace ufb
