// Attention over the 8-bit cache for few rows (new tokens x query heads of a key
// head, up to 32: one tile of 8, or one or two of 16): a decoding step.
//
//   S = Q K^T,  P = 2^(S f + log2 vs - M),  O = P V,  l = sum P / vs
//
// with f the page's key scale times the softmax scale times log2 e and vs its
// value scale.  Folding log2 vs into the running maximum M bounds P whatever the
// pages' scales are, so it can be rounded to float16 for the second
// product; l divides it out again, in 32 bits.  out = O / l.
//
// Bound by the bytes of the cache.  Work is divided by tiles of 64 keys
// (kv_attend.cuh), one CTA to an SM; two producer warps stream the integers by TMA
// into a ring (7 stages, 112 KB in flight at head_dim 128, against the 35 KB that
// HBM's latency needs), and the other warps take 32 keys of a stage each, in turn.
//
// The products are m16n8k16 tensor instructions on registers with the rows as the
// narrow side: S^T = K Q^T and O^T = V^T P^T in tiles of 8 rows.  A tile of 128
// rows, which tcgen05 needs, would be mostly padding here, and its operands would
// have to go back through shared memory as float16, while these integers are
// expanded in the registers they were loaded to.  8 rows (one token of up to 8
// query heads) leave registers for 14 consumer warps, 16 rows for 6: the
// expansion is a chain of dependent instructions, and warps are what hides it.
// Which dims and keys share an instruction is free as long as both operands agree;
// the order below makes every shared-memory read 16 (or 8) bytes wide and free of
// bank conflicts under TMA's 128-byte swizzle.
//
// 64 streams x 16000 keys x 4 heads of 128: 188 us, 5.6 TB/s, 0.87 of a plain
// copy's rate (8 consumer warps with the rows as the wide side: 160 us for 127 on 64
// ragged streams up to 16320 keys);
// head_dim 64 at 3.3 TB/s: half the bytes a key, and scores, weights and their exchange
// cost as much a key (not the expansion: a form with two instructions less for four keys
// took as long); one token over 1760 keys 12 us.
//
// Parts of an item that several CTAs share are joined by the CTA that arrives
// last, in the order of the CTAs, so the sum does not depend on which one it is.
#include "kv_attend.cuh"
#include "umma.cuh"

#include <type_traits>

namespace ufb {

namespace {

constexpr int kKeys = 64;             // keys of a stage
constexpr int kWarpKeys = 32;         // keys of a consumer warp's step
constexpr int kProducers = 2;         // producer warps; a slot of the ring always has the same one
constexpr int kGroups = kKeys / kGroupKeys;
constexpr int kMinShare = 7;          // tiles of a CTA's share at least: as many as its warps take at once
// With 8 (NT 1) or 16 (NT 2) rows: consumer warps, and stages of the ring.  A warp
// comes back to every (consumers / 2)-th stage, and the ring is a multiple of that:
// a warp has seen each earlier use of a stage it waits for, which a barrier's parity
// needs (copies may land out of order).
__host__ __device__ constexpr int consumers(int nt) { return nt == 1 ? 14 : 6; }
__host__ __device__ constexpr int stages(int nt) { return nt == 1 ? 7 : 9; }
// P is taken times 2^kShift: at most 2^15, inside float16, and weights down to
// 2^-29 of the largest keep all 11 bits.  (The maximum less kShift is rounded up, or
// scores spaced by more than 1, from 2^24 on, would give weights of 2^16.)
constexpr float kShift = 15.0f;
constexpr int kCodeFull = 41, kCodeEmpty = 42, kCodeDrain = 43;

struct PageScales {
    float key, log2_value, inv_value;  // log2_value -inf: the 16 keys are not there
    float pad;
};

template <int D, int NT>
struct Smem {
    alignas(1024) uint8_t ring[stages(NT)][2 * kKeys * D];     // copies of key, then value integers
    float sums[consumers(NT)][8 * NT][D];
    float stats[2][2][consumers(NT)][8 * NT];               // by piece parity: maxima, weights
    PageScales scales[stages(NT)][kGroups];
    alignas(8) uint64_t full[stages(NT)], empty[stages(NT)];
    ShareSmem share;
    int last;
    int dead;
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The transpose of an 8 x 8 matrix of float16, a row to four lanes.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

template <int N>
__device__ __forceinline__ void consumers_sync() {
    asm volatile("bar.sync 1, %0;" ::"n"(N * 32) : "memory");
}

__device__ __forceinline__ void joiners_sync(int warps) { asm volatile("bar.sync 2, %0;" ::"r"(warps * 32) : "memory"); }

// The dims of lane quarter c in k step t, four in a row (also Q's fragments).
template <int D>
__device__ __forceinline__ int key_dim(int c, int t) {
    return D == 128 ? (t >> 2) * 64 + c * 16 + (t & 3) * 4 : (t >> 1) * 32 + c * 8 + (t & 1) * 4;
}
// The first of the D / 8 dims that lane row n (0..7) has of a value row.
template <int D>
__device__ __forceinline__ int value_dim(int n) {
    if (D == 128) return (((n & 1) << 2) | (n >> 1)) * 16;
    const int pair = n >> 1;  // 16-byte chunks 0, 2, 1, 3
    return ((((pair & 1) << 1) | (pair >> 1)) * 2 + (n & 1)) * 8;
}
// The key (of 8) that lane row n of a score tile stands for.
__device__ __forceinline__ int key_of(int n) { return ((n & 1) << 2) | (n >> 1); }

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * (consumers(NT) + kProducers), 1)
    few_kernel(const __grid_constant__ CUtensorMap map, const AttendArgs a, int row_tiles, int min_share) {
    constexpr int kWarps = consumers(NT), kRows = 8 * NT, kThreads = 32 * (kWarps + kProducers), kStages = stages(NT);
    static_assert(kStages % (kWarps * kWarpKeys / kKeys) == 0, "see consumers");
    extern __shared__ uint8_t raw[];
    Smem<D, NT>& sm = *reinterpret_cast<Smem<D, NT>*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == kThreads - 1) prefetch_tmap(&map);
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.empty[i], kKeys / kWarpKeys);
        }
        fence_mbar_init();
        sm.dead = 0;
    }
    const Share share = locate_share<kKeys, kRows, kThreads>(a, row_tiles, min_share, sm.share);
    Walker<kKeys, kRows> walk(a, share, row_tiles);
    volatile int* dead = &sm.dead;

    if (warp >= kWarps) {
        // ---- producers: a batch is up to 8 stages of one piece, lane = (stage, group of 16
        // keys).  Pages are looked up two batches ahead, scales one, so no load is waited
        // for; the four lanes of a stage wait for it and start its copies by themselves.
        // Both producers look at every batch and fill the slots that are theirs.
        // no more than the ring: a batch must not wait for its own stages
        constexpr int kBatch = kStages < 32 / kGroups ? kStages : 32 / kGroups;
        struct Batch {
            int count, page, row, head;  // page -1: not there; row: the group's first token slot in it
            float key, value;
        };
        Piece p;
        bool have = walk.next(a, p);
        int at = have ? p.first : 0;
        auto look_up = [&](Batch& b) {
            b.count = 0;
            b.page = -1;
            if (!have) return;
            b.count = min(kBatch, p.end - at);
            b.head = p.head;
            if (lane / kGroups < b.count) {
                const int key = p.t.keys.tile(at + lane / kGroups) * kKeys + (lane % kGroups) * kGroupKeys;
                const int entry = key >> a.page_shift;
                b.row = key & (a.page_tokens - 1);
                if (p.t.keys.touches(key) && entry < a.table_width)
                    b.page = a.table[static_cast<long long>(p.t.slot) * a.table_width + entry];
            }
            at += b.count;
            if (at == p.end) {
                have = walk.next(a, p);
                at = have ? p.first : 0;
            }
        };
        auto load_scales = [&](Batch& b) {
            if (b.page >= a.pages) b.page = -1;
            if (b.page < 0) return;
            const float* s = a.scale + static_cast<long long>(b.page) * 2 * a.heads + b.head;
            b.key = s[0];
            b.value = s[a.heads];
        };
        // one copy brings the 16-key groups that lie together in a page, when any of them is there
        const int box = min(a.page_tokens, kKeys), per = box / kGroupKeys;
        const bool lead = lane % kGroups % per == 0;
        Batch now, next, later;
        look_up(now);
        load_scales(now);
        look_up(next);
        int it = 0;
        bool ok = true;
        while (now.count) {
            load_scales(next);
            look_up(later);
            PageScales sc;
            sc.key = sc.inv_value = 0.0f;
            sc.log2_value = -INFINITY;
            if (now.page >= 0) {
                const float v = now.value < kTinyScale ? kTinyScale : now.value;
                sc.key = now.key;
                sc.log2_value = log2f(v);
                sc.inv_value = 1.0f / v;
            }
            const int mine = lane / kGroups, stage_it = it + mine, stage = stage_it % kStages;
            const bool fill = mine < now.count && stage % kProducers == warp - kWarps;
            const unsigned there = __ballot_sync(0xffffffffu, now.page >= 0);
            const unsigned near = (there >> lane) & ((1u << per) - 1);
            const int from = near ? __ffs(near) - 1 : 0;
            const int page = __shfl_sync(0xffffffffu, now.page, (lane + from) & 31);
            const int row = __shfl_sync(0xffffffffu, now.row, (lane + from) & 31) - from * kGroupKeys;
            const bool copy = lead && near != 0;
            const unsigned copies = __ballot_sync(0xffffffffu, copy);
            const int bytes = __popc((copies >> (mine * kGroups)) & ((1u << kGroups) - 1)) * 2 * box * D;
            // a copy's place: [copy][key, value][16-key groups of it]
            const int off = (lane % kGroups) * kGroupKeys * 2 * D, map_row = row * D / 128;
            const unsigned group = ((1u << kGroups) - 1) << (lane & ~(kGroups - 1));
            for (int s = 0; s < now.count; ++s) {
                if (mine != s || !fill) continue;
                if (stage_it >= kStages) ok = mbar_wait(&sm.empty[stage], (stage_it / kStages - 1) & 1, a.status, kCodeEmpty);
                // the four agree, or those that go on would miss the others below
                ok = __shfl_sync(group, ok, lane & ~(kGroups - 1));
                if (!ok) break;
                sm.scales[stage][lane % kGroups] = sc;
                __syncwarp(group);
                if (lane % kGroups == 0) {
                    if (bytes) mbar_arrive_expect_tx(&sm.full[stage], bytes);
                    else mbar_arrive(&sm.full[stage]);
                }
                if (copy) tma_load_5d(&sm.ring[stage][off], &map, &sm.full[stage], 0, map_row, now.head, 0, page);
            }
            __syncwarp();
            if (__any_sync(0xffffffffu, !ok) || *dead) {
                // somebody gave up: copies still in flight must land before the CTA's shared
                // memory goes, those of this batch's filled stages and of the ones before
                *dead = 1;
                if (ok && fill) mbar_wait(&sm.full[stage], (stage_it / kStages) & 1, a.status, kCodeDrain);
                __syncwarp();
                for (int i = max(0, it - kStages); i < it; ++i)
                    if (i % kStages % kProducers == warp - kWarps) mbar_wait(&sm.full[i % kStages], (i / kStages) & 1, a.status, kCodeDrain);
                return;
            }
            it += now.count;
            now = next;
            next = later;
        }
        return;
    }

    // ---- consumers
    const int g = lane >> 2, c = lane & 3;
    constexpr int kSteps = D / 16, kTiles = D / 16;   // of keys' dims; of output dims
    const AttendScratch scratch = scratch_of(a.workspace, gridDim.x, kRows);
    int it = 0, parity = 0;
    Piece p;
    while (walk.next(a, p)) {
        // Q fragments: row 8 n + g, brought to [2^15, 2^16) and rounded to float16; then what
        // the scores of rows 8 n + 2 c and + 1 need
        uint32_t q[NT][kSteps][2];
        float unit[NT][2];
        int pos[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = n * 8 + g;
            const bool real = row < p.t.rows;
            const int in_stream = p.t.row0 + row;
            const int token = real ? in_stream / a.group : 0;
            const T* src = static_cast<const T*>(a.q.data) + (p.t.token0 + token) * a.q.token_stride +
                           (p.head * a.group + in_stream - token * a.group) * a.q.head_stride;
            float top = 0.0f, odd = 0.0f;
            uint2 w[kSteps];
#pragma unroll
            for (int t = 0; t < kSteps; ++t) {
                w[t] = make_uint2(0, 0);
                if (real) w[t] = *reinterpret_cast<const uint2*>(src + key_dim<D>(c, t));
            }
#pragma unroll
            for (int t = 0; t < kSteps; ++t) {
                const float2 x = unpack2(w[t].x, T()), y = unpack2(w[t].y, T());
                top = fmaxf(top, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))));
                odd += (x.x - x.x) + (x.y - x.y) + (y.x - y.x) + (y.y - y.y);  // NaN for what is not finite
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                odd += __shfl_xor_sync(0xffffffffu, odd, o);
            }
            const float u = row_unit(odd == odd ? top : odd);
            const float mul = u == u ? u : 0.0f;
#pragma unroll
            for (int t = 0; t < kSteps; ++t) {
                const float2 x = unpack2(w[t].x, T()), y = unpack2(w[t].y, T());
                q[n][t][0] = pack2(x.x * mul, x.y * mul, __half());
                q[n][t][1] = pack2(y.x * mul, y.y * mul, __half());
            }
            const float f = unit_inverse(u) * a.scale_log2;
            const int at = p.t.length - p.t.n_new + token;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int from = (2 * c + r) * 4;
                unit[n][r] = __shfl_sync(0xffffffffu, f, from);
                pos[n][r] = __shfl_sync(0xffffffffu, at, from);
            }
        }
        float o[NT][kTiles][4];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < kTiles; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.0f;
            m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.0f;
        }
        const int last_pos = p.t.length - p.t.n_new + (p.t.row0 + p.t.rows - 1) / a.group;
        const int first_pos = p.t.length - p.t.n_new + p.t.row0 / a.group;

        // steps of 32 keys go round the warps
        const int steps_before = it * (kKeys / kWarpKeys);
        const int steps = (p.end - p.first) * (kKeys / kWarpKeys);
        int step = (warp - steps_before % kWarps + kWarps) % kWarps;
#pragma unroll 1
        for (; step < steps; step += kWarps) {
            const int index = it + step / (kKeys / kWarpKeys), stage = index % kStages;
            const int part = (step % (kKeys / kWarpKeys)) * kWarpKeys;
            // after a wait gave up the warps go on without waiting: they meet at barriers, and
            // every join still counts all its CTAs, so the counters end at zero
            if (!mbar_try_wait(&sm.full[stage], (index / kStages) & 1) && !*dead &&
                !mbar_wait(&sm.full[stage], (index / kStages) & 1, a.status, kCodeFull))
                *dead = 1;
            __syncwarp();
            constexpr int kM = kWarpKeys / 16;    // score tiles of 16 keys
            const PageScales* sc = &sm.scales[stage][part / kGroupKeys];
            // where the step's 16-key groups lie, less their offset in the stage
            const int box = min(a.page_tokens, kKeys);
            const uint8_t *keys[kM], *values[kM];
#pragma unroll
            for (int x = 0; x < kM; ++x) {
                const int first = part + x * 16, copy = first & ~(box - 1);
                keys[x] = sm.ring[stage] + (copy * 2 + first - copy) * D;
                values[x] = keys[x] + box * D;
            }
            float s[kM][NT][4];
#pragma unroll
            for (int x = 0; x < kM; ++x)
#pragma unroll
                for (int n = 0; n < NT; ++n) s[x][n][0] = s[x][n][1] = s[x][n][2] = s[x][n][3] = 0.0f;
            // S^T, half the dims at a time
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t w[kM][2][kSteps / 2];
#pragma unroll
                for (int x = 0; x < kM; ++x)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int key = h * 8 + key_of(g);
                        if (D == 128) {
                            const uint4 v = *reinterpret_cast<const uint4*>(keys[x] + key * 128 + (((c + i * 4) ^ (key & 7)) << 4));
                            w[x][h][0] = v.x, w[x][h][1] = v.y;
                            w[x][h][2 % (kSteps / 2)] = v.z, w[x][h][3 % (kSteps / 2)] = v.w;
                        } else {
                            const int row = key >> 1;
                            const uint2 v = *reinterpret_cast<const uint2*>(
                                keys[x] + row * 128 + ((((key & 1) * 4 + i * 2 + (c >> 1)) ^ (row & 7)) << 4) + (c & 1) * 8);
                            w[x][h][0] = v.x, w[x][h][1] = v.y;
                        }
                    }
#pragma unroll
                for (int k = 0; k < kSteps / 2; ++k)
#pragma unroll
                    for (int x = 0; x < kM; ++x) {
                        uint32_t f[4];
                        int8x4_to_half(w[x][0][k], f[0], f[2]);
                        int8x4_to_half(w[x][1][k], f[1], f[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            mma16816(s[x][n], f, q[n][i * (kSteps / 2) + k][0], q[n][i * (kSteps / 2) + k][1]);
                    }
            }
            // scores in base 2 with the value scale, the maximum, P
            const int key0 = p.t.keys.tile(p.first + step / (kKeys / kWarpKeys)) * kKeys + part;
            const bool clear = (!a.causal || key0 + kWarpKeys - 1 <= first_pos) && key0 + kWarpKeys <= p.t.length &&
                               (!a.window || last_pos - key0 < a.window || key0 + kWarpKeys <= a.sinks);
            uint32_t pb[kM][NT][2];
            auto softmax = [&](auto masked) {
                constexpr bool kMasked = decltype(masked)::value;
                uint32_t hidden = 0;   // of this thread's scores, a bit each
                float top[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    top[n][0] = top[n][1] = -INFINITY;
#pragma unroll
                    for (int x = 0; x < kM; ++x) {
                        const float f[2] = {unit[n][0] * sc[x].key, unit[n][1] * sc[x].key};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[x][n][e] = fmaf(s[x][n][e], f[e & 1], sc[x].log2_value);
                            if (kMasked) {
                                const int key = key0 + x * 16 + (e >> 1) * 8 + key_of(g), at = pos[n][e & 1];
                                const bool seen = key < p.t.length && (!a.causal || key <= at) &&
                                                  (!a.window || at - key < a.window || key < a.sinks);
                                if (!seen) s[x][n][e] = -INFINITY, hidden |= 1u << ((x * NT + n) * 4 + e);
                            }
                            top[n][e & 1] = fmaxf(top[n][e & 1], s[x][n][e]);
                        }
                    }
                }
                bool grew = false;
                float keep[NT][2], base[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float x = top[n][r];
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                        const float next = fmaxf(m[n][r], x);
                        grew |= next > m[n][r];
                        keep[n][r] = next == -INFINITY ? 1.0f : ex2(m[n][r] - next);
                        base[n][r] = next == -INFINITY ? 0.0f : __fsub_ru(next, kShift);
                        m[n][r] = next;
                    }
                if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int j = 0; j < kTiles; ++j) {
                            o[n][j][0] *= keep[n][0], o[n][j][1] *= keep[n][1];
                            o[n][j][2] *= keep[n][0], o[n][j][3] *= keep[n][1];
                        }
                        l[n][0] *= keep[n][0], l[n][1] *= keep[n][1];
                    }
                }
#pragma unroll
                for (int x = 0; x < kM; ++x)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[x][n][e] = ex2(s[x][n][e] - base[n][e & 1]);
                            // a hidden weight is 0 also where its row or scale is not finite
                            if (kMasked && (hidden & (1u << ((x * NT + n) * 4 + e)))) s[x][n][e] = 0.0f;
                        }
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const float sum = s[x][n][r] + s[x][n][2 + r];
                            if (sum != 0.0f) l[n][r] = fmaf(sum, sc[x].inv_value, l[n][r]);
                        }
                        // from (key, two rows) to (two keys, row)
                        pb[x][n][0] = transpose8(pack2(s[x][n][0], s[x][n][1], __half()));
                        pb[x][n][1] = transpose8(pack2(s[x][n][2], s[x][n][3], __half()));
                    }
            };
            if (clear) softmax(std::false_type());
            else softmax(std::true_type());
            // O^T += V^T P^T, 16 keys at a time
#pragma unroll
            for (int x = 0; x < kM; ++x) {
                uint32_t v[4][D / 32];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = (i >> 1) * 8 + (i & 1) * 4 + c;
                    if (D == 128) {
                        const uint4 y = *reinterpret_cast<const uint4*>(values[x] + key * 128 + (((value_dim<D>(g) >> 4) ^ (key & 7)) << 4));
                        v[i][0] = y.x, v[i][1] = y.y, v[i][2 % (D / 32)] = y.z, v[i][3 % (D / 32)] = y.w;
                    } else {
                        const int row = key >> 1, chunk = (key & 1) * 4 + (value_dim<D>(g) >> 4);
                        const uint2 y = *reinterpret_cast<const uint2*>(values[x] + row * 128 + ((chunk ^ (row & 7)) << 4) + (g & 1) * 8);
                        v[i][0] = y.x, v[i][1] = y.y;
                    }
                }
                if (x == kM - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.empty[stage]);
                }
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const uint32_t w0 = v[0][i] ^ 0x80808080u, w1 = v[1][i] ^ 0x80808080u;
                    const uint32_t w2 = v[2][i] ^ 0x80808080u, w3 = v[3][i] ^ 0x80808080u;
                    // (key, key') pairs of dims 0, 1 and of dims 2, 3 of the word
                    const uint32_t e[2][2] = {{__byte_perm(w0, w1, 0x5140), __byte_perm(w2, w3, 0x5140)},
                                              {__byte_perm(w0, w1, 0x7362), __byte_perm(w2, w3, 0x7362)}};
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t f[4] = {half2_minus_1152(__byte_perm(e[j][0], 0x64646464u, 0x4140)),
                                               half2_minus_1152(__byte_perm(e[j][0], 0x64646464u, 0x4342)),
                                               half2_minus_1152(__byte_perm(e[j][1], 0x64646464u, 0x4140)),
                                               half2_minus_1152(__byte_perm(e[j][1], 0x64646464u, 0x4342))};
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma16816(o[n][i * 2 + j], f, pb[x][n][0], pb[x][n][1]);
                    }
                }
            }
        }
        it += p.end - p.first;

        // ---- the warps' sums become one
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[n][r] += __shfl_xor_sync(0xffffffffu, l[n][r], d);
                if (g == 0) {
                    sm.stats[parity][0][warp][n * 8 + 2 * c + r] = m[n][r];
                    sm.stats[parity][1][warp][n * 8 + 2 * c + r] = l[n][r];
                }
            }
        consumers_sync<kWarps>();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = n * 8 + 2 * c + r;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm.stats[parity][0][w][row]);
                const float mul = m[n][r] == -INFINITY ? (l[n][r] == 0.0f ? 0.0f : 1.0f) : ex2(m[n][r] - top);
                if (row < p.t.rows) {
                    float* to = &sm.sums[warp][row][value_dim<D>(g)];
#pragma unroll
                    for (int j = 0; j < kTiles; j += 2)
                        *reinterpret_cast<float4*>(to + j * 2) = make_float4(o[n][j][r] * mul, o[n][j][2 + r] * mul,
                                                                             o[n][j + 1][r] * mul, o[n][j + 1][2 + r] * mul);
                }
            }
        consumers_sync<kWarps>();
        const bool whole = p.whole();
        const int part = 2 * blockIdx.x + (p.first > 0 ? 0 : 1);
        auto finish = [&](int row, int d, float4 v, float top, float weight) {
            const int in_stream = p.t.row0 + row, token = in_stream / a.group;
            const int head = p.head * a.group + in_stream - token * a.group;
            const float inv = weight == 0.0f ? 0.0f : 1.0f / weight;
            T* to = static_cast<T*>(a.out.data) + (p.t.token0 + token) * a.out.token_stride + head * a.out.head_stride + d;
            *reinterpret_cast<uint2*>(to) = make_uint2(pack2(v.x * inv, v.y * inv, T()), pack2(v.z * inv, v.w * inv, T()));
            if (a.lse && d == 0)
                a.lse[(p.t.token0 + token) * (a.heads * a.group) + head] =
                    weight == 0.0f ? -INFINITY : (top - kShift + log2f(weight)) * 0.6931471805599453f;
        };
        // as many warps as there is to sum; the others go on to the next piece
        const int joiners = min(kWarps, (p.t.rows * (D / 4) + 31) / 32);
        if (warp < joiners) {
            for (int e = threadIdx.x; e < p.t.rows * (D / 4); e += joiners * 32) {
                const int row = e / (D / 4), d = e % (D / 4) * 4;
                float top = -INFINITY, weight = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm.stats[parity][0][w][row]);
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float mw = sm.stats[parity][0][w][row], lw = sm.stats[parity][1][w][row];
                    if (lw != 0.0f) weight += lw * (mw == -INFINITY ? 1.0f : ex2(mw - top));
                    const float4 x = *reinterpret_cast<const float4*>(&sm.sums[w][row][d]);
                    v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
                }
                if (whole) {
                    finish(row, d, v, top, weight);
                } else {
                    __stcg(reinterpret_cast<float4*>(scratch.sums + (static_cast<long long>(part) * kRows + row) * D + d), v);
                    if (d == 0) {
                        __stcg(scratch.stats + (part * 2) * kRows + row, top);
                        __stcg(scratch.stats + (part * 2 + 1) * kRows + row, weight);
                    }
                }
            }
            if (!whole) {
                // CTAs of this item: the one its first tile falls to .. the one its last tile falls to
                const int c0 = static_cast<int>(p.item_start / share.per);
                const int c1 = static_cast<int>((p.item_start + p.t.keys.nt - 1) / share.per);
                __threadfence();
                joiners_sync(joiners);
                if (threadIdx.x == 0) {
                    const int before = atomicAdd(scratch.counters + c0, 1);
                    sm.last = before == c1 - c0;
                    if (sm.last) scratch.counters[c0] = 0;
                }
                joiners_sync(joiners);
                if (sm.last) {
                    __threadfence();
                    for (int e = threadIdx.x; e < p.t.rows * (D / 4); e += joiners * 32) {
                        const int row = e / (D / 4), d = e % (D / 4) * 4;
                        float top = -INFINITY, weight = 0.0f;
#pragma unroll 4
                        for (int i = c0; i <= c1; ++i)
                            top = fmaxf(top, __ldcg(scratch.stats + (2 * i + (i == c0)) * 2 * kRows + row));
                        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                        for (int i = c0; i <= c1; ++i) {
                            const int from = 2 * i + (i == c0);
                            const float mi = __ldcg(scratch.stats + from * 2 * kRows + row);
                            const float li = __ldcg(scratch.stats + (from * 2 + 1) * kRows + row);
                            const float4 x = __ldcg(reinterpret_cast<const float4*>(
                                scratch.sums + (static_cast<long long>(from) * kRows + row) * D + d));
                            const float mul = mi == -INFINITY ? (li == 0.0f ? 0.0f : 1.0f) : ex2(mi - top);
                            weight += li * mul;
                            v.x += x.x * mul, v.y += x.y * mul, v.z += x.z * mul, v.w += x.w * mul;
                        }
                        finish(row, d, v, top, weight);
                    }
                }
            }
        }
        parity ^= 1;
    }
}

template <typename T, int D, int NT>
cudaError_t launch(const AttendArgs& a, int sms, cudaStream_t s) {
    auto kernel = few_kernel<T, D, NT>;
    const int smem = sizeof(Smem<D, NT>) + 1024;
    static std::atomic<uint64_t> allowed;
    const cudaError_t attr = allow_smem(kernel, smem, allowed);
    if (attr != cudaSuccess) return attr;
    CUtensorMap map;
    // boxes of the keys that lie together in a page, 64 at most
    if (!kv_tensor_map(map, a, kKeys)) return cudaErrorInvalidValue;
    const int row_tiles = static_cast<int>((static_cast<long long>(a.max_new) * a.group + 8 * NT - 1) / (8 * NT));
    kernel<<<sms < kAttendMaxCtas ? sms : kAttendMaxCtas, 32 * (consumers(NT) + kProducers), smem, s>>>(map, a, row_tiles, kMinShare);
    return cudaGetLastError();
}

template <typename T, int D>
cudaError_t launch_rows(const AttendArgs& a, int sms, cudaStream_t s) {
    const long long rows = static_cast<long long>(a.max_new) * a.group;
    return rows <= 8 ? launch<T, D, 1>(a, sms, s) : launch<T, D, 2>(a, sms, s);
}

}  // namespace

cudaError_t attend_few(const AttendArgs& a, int dtype, int sms, cudaStream_t s) {
    if (a.head_dim == 64)
        return dtype == UFB_F16 ? launch_rows<__half, 64>(a, sms, s) : launch_rows<__nv_bfloat16, 64>(a, sms, s);
    return dtype == UFB_F16 ? launch_rows<__half, 128>(a, sms, s) : launch_rows<__nv_bfloat16, 128>(a, sms, s);
}

}  // namespace ufb
