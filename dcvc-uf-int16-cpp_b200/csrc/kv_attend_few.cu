// Attention over the 8-bit cache for few rows (new tokens x query heads of a key
// head <= 16 or so): a decoding step.
//
//   S = Q K^T,  P = 2^(S f + log2 vs - M),  O = P V,  l = sum P / vs
//
// with f the page's key scale times the softmax scale times log2 e and vs its
// value scale.  Folding log2 vs into the running maximum M bounds P whatever the
// pages' scales are, so it can be rounded to float16 for the second
// product; l divides it out again, in 32 bits.  out = O / l.
//
// Bound by the bytes of the cache.  Work is divided by tiles of 64 keys
// (kv_attend.cuh), one CTA to an SM; a producer warp streams the integers by TMA
// into a ring (8 stages, 128 KB in flight at head_dim 128, against the 35 KB that
// HBM's latency needs), and two groups of four warps take the stages in turn, 16
// keys a warp.  With at most 16 rows the products are m16n8k16 tensor
// instructions on registers: a tile of 128 rows, which tcgen05 needs, would be
// seven eighths padding and its operands would have to go back through shared
// memory as float16, while here the integers are expanded in the registers they
// were loaded to.  Which dims and keys share an instruction is free as long as
// both operands agree; the order below makes every shared-memory read 16 (or 8)
// bytes wide and free of bank conflicts under TMA's 128-byte swizzle.
//
// Parts of an item that several CTAs share are joined by the CTA that arrives
// last, in the order of the CTAs, so the sum does not depend on which one it is.
#include "kv_attend.cuh"
#include "umma.cuh"

#include <mutex>

namespace ufb {

namespace {

constexpr int kRows = 16;
constexpr int kKeys = 64;             // keys of a stage
constexpr int kWarps = 8;             // consumer warps
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kStages = 8;
constexpr int kGroups = kKeys / kGroupKeys;
// P is taken times 2^kShift: at most 2^15, inside float16, and weights down to
// 2^-29 of the largest keep all 11 bits.
constexpr float kShift = 15.0f;
constexpr int kCodeFull = 41, kCodeEmpty = 42, kCodeDrain = 43;

struct PageScales {
    float key, log2_value, inv_value;  // log2_value -inf: the 16 keys are not there
    float pad;
};

template <int D>
struct Smem {
    alignas(1024) uint8_t ring[kStages][2][kKeys * D];   // key, value integers
    float sums[kWarps][kRows][D];
    float stats[2][2][kWarps][kRows];                    // by piece parity: maxima, weights
    PageScales scales[kStages][kGroups];
    alignas(8) uint64_t full[kStages], empty[kStages];
    ShareSmem share;
    int last;
    int dead;
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); }

// The dims of lane quarter c in k step t, four in a row (also Q's fragments).
template <int D>
__device__ __forceinline__ int key_dim(int c, int t) {
    return D == 128 ? (t >> 2) * 64 + c * 16 + (t & 3) * 4 : (t >> 1) * 32 + c * 8 + (t & 1) * 4;
}
// The first of the D / 8 dims of output column n (0..7), one a value tile.
template <int D>
__device__ __forceinline__ int value_dim(int n) {
    if (D == 128) return (((n & 1) << 2) | (n >> 1)) * 16;
    const int pair = n >> 1;  // 16-byte chunks 0, 2, 1, 3
    return ((((pair & 1) << 1) | (pair >> 1)) * 2 + (n & 1)) * 8;
}
// The key (of 8) that column n of a score tile stands for.
__device__ __forceinline__ int key_of(int n) { return ((n & 1) << 2) | (n >> 1); }

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) few_kernel(const __grid_constant__ CUtensorMap map, const AttendArgs a,
                                                          int row_tiles, int min_share) {
    extern __shared__ uint8_t raw[];
    Smem<D>& sm = *reinterpret_cast<Smem<D>*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.empty[i], kWarps / 2);
        }
        fence_mbar_init();
        sm.dead = 0;
    }
    const Share share = locate_share<kKeys, kRows, kThreads>(a, row_tiles, min_share, sm.share);
    Walker<kKeys, kRows> walk(a, share, row_tiles);
    volatile int* dead = &sm.dead;

    if (warp == kWarps) {
        // ---- producer: a batch is up to 8 stages of one piece, lane = (stage, group of 16 keys)
        if (lane == 0) prefetch_tmap(&map);
        struct Batch {
            int count, page, row, head;  // row: the group's first token slot in its page
            float key, value;
        };
        Piece p;
        bool have = walk.next(a, p);
        int at = have ? p.first : 0;
        auto fetch = [&](Batch& b) {
            b.count = 0;
            if (!have) return;
            b.count = min(32 / kGroups, p.end - at);
            b.page = -1;
            b.head = p.head;
            const int t = at + lane / kGroups;
            if (lane / kGroups < b.count) {
                const int key = p.t.keys.tile(t) * kKeys + (lane % kGroups) * kGroupKeys;
                const int entry = key >> a.page_shift;
                if (p.t.keys.touches(key) && entry < a.table_width) {
                    const int page = a.table[static_cast<long long>(p.t.slot) * a.table_width + entry];
                    if (page >= 0 && page < a.pages) {
                        b.page = page;
                        b.row = key & (a.page_tokens - 1);
                        const float* s = a.scale + static_cast<long long>(page) * 2 * a.heads + p.head;
                        b.key = s[0];
                        b.value = s[a.heads];
                    }
                }
            }
            at += b.count;
            if (at == p.end) {
                have = walk.next(a, p);
                at = have ? p.first : 0;
            }
        };
        Batch now, next;
        fetch(now);
        int it = 0;
        bool ok = true;
        while (now.count && ok) {
            fetch(next);
            PageScales sc;
            sc.key = sc.inv_value = 0.0f;
            sc.log2_value = -INFINITY;
            if (now.page >= 0) {
                const float v = now.value < kTinyScale ? kTinyScale : now.value;
                sc.key = now.key;
                sc.log2_value = log2f(v);
                sc.inv_value = 1.0f / v;
            }
            // one copy brings the 16-key groups that lie together in a page
            const int box = min(a.page_tokens, kKeys);                   // keys of a copy
            const bool lead = (lane % kGroups) * kGroupKeys % box == 0;  // first group of its copy
            // a page is loaded when any of its groups is there
            unsigned there = __ballot_sync(0xffffffffu, now.page >= 0);
            const int per = box / kGroupKeys;
            const unsigned mine = (there >> lane) & ((1u << per) - 1);
            const int from = mine ? __ffs(mine) - 1 : 0;
            const int page = __shfl_sync(0xffffffffu, now.page, (lane + from) & 31);
            const int row = __shfl_sync(0xffffffffu, now.row, (lane + from) & 31) - from * kGroupKeys;
            const bool copy = lead && mine != 0;
            const unsigned copies = __ballot_sync(0xffffffffu, copy);
            for (int s = 0; s < now.count; ++s, ++it) {
                const int stage = it % kStages;
                if (it >= kStages) ok = mbar_wait(&sm.empty[stage], (it / kStages - 1) & 1, a.status, kCodeEmpty);
                ok = __shfl_sync(0xffffffffu, ok, 0) && !*dead;
                if (!ok) break;
                if (lane / kGroups == s) {
                    sm.scales[stage][lane % kGroups] = sc;
                }
                __syncwarp();
                const int n = __popc((copies >> (s * kGroups)) & ((1u << kGroups) - 1));
                if (lane == 0) {
                    if (n) mbar_arrive_expect_tx(&sm.full[stage], n * 2 * box * D);
                    else mbar_arrive(&sm.full[stage]);
                }
                __syncwarp();
                if (lane / kGroups == s && copy) {
                    // the cache as rows of 128 bytes
                    const long long tile = static_cast<long long>(page) * 2 * a.heads + now.head;
                    const int off = (lane % kGroups) * kGroupKeys * D;
                    const long long key_row = (tile * a.page_tokens + row) * D / 128;
                    const long long value_row = ((tile + a.heads) * a.page_tokens + row) * D / 128;
                    tma_load_2d(&sm.ring[stage][0][off], &map, &sm.full[stage], 0, static_cast<int>(key_row));
                    tma_load_2d(&sm.ring[stage][1][off], &map, &sm.full[stage], 0, static_cast<int>(value_row));
                }
                __syncwarp();
            }
            now = next;
        }
        if (!ok) {
            *dead = 1;
            // copies still in flight must land before the CTA's shared memory goes
            if (lane == 0)
                for (int i = max(0, it - kStages); i < it; ++i)
                    mbar_wait(&sm.full[i % kStages], (i / kStages) & 1, a.status, kCodeDrain);
        }
        return;
    }

    // ---- consumers
    const int g = lane >> 2, c = lane & 3;
    const int half = warp >> 2, quarter = warp & 3;
    constexpr int kSteps = D / 16, kTiles = D / 8;
    const AttendScratch scratch = scratch_of(a.workspace, gridDim.x, kRows);
    int it = 0, parity = 0;
    Piece p;
    while (walk.next(a, p)) {
        // Q fragments: rows g and g + 8, brought to [1/2, 1) and rounded to float16
        uint32_t q[kSteps][4];
        float unit[2];
        int pos[2];   // where the row stands
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = g + r * 8;
            const bool real = row < p.t.rows;
            const int in_stream = p.t.row0 + row;
            const int token = real ? in_stream / a.group : 0;
            pos[r] = p.t.length - p.t.n_new + token;
            const T* src = static_cast<const T*>(a.q.data) + (p.t.token0 + token) * a.q.token_stride +
                           (p.head * a.group + in_stream - token * a.group) * a.q.head_stride;
            float top = 0.0f;
            uint2 w[kSteps];
#pragma unroll
            for (int t = 0; t < kSteps; ++t) {
                w[t] = make_uint2(0, 0);
                if (real) w[t] = *reinterpret_cast<const uint2*>(src + key_dim<D>(c, t));
            }
#pragma unroll
            for (int t = 0; t < kSteps; ++t) {
                const float2 x = unpack2(w[t].x, T()), y = unpack2(w[t].y, T());
                const float m = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y)));
                // fmaxf drops NaN: x - x is NaN for what is not finite
                const float odd = (x.x - x.x) + (x.y - x.y) + (y.x - y.x) + (y.y - y.y);
                top = odd == odd && top == top ? fmaxf(top, m) : __int_as_float(0x7fffffff);
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                const float other = __shfl_xor_sync(0xffffffffu, top, o);
                top = top == top && other == other ? fmaxf(top, other) : __int_as_float(0x7fffffff);
            }
            const float u = row_unit(top);
            unit[r] = unit_inverse(u) * a.scale_log2;
            const float mul = u == u ? u : 0.0f;
#pragma unroll
            for (int t = 0; t < kSteps; ++t) {
                const float2 x = unpack2(w[t].x, T()), y = unpack2(w[t].y, T());
                q[t][r] = pack2(x.x * mul, x.y * mul, __half());
                q[t][2 + r] = pack2(y.x * mul, y.y * mul, __half());
            }
        }
        float o[kTiles][4];
#pragma unroll
        for (int j = 0; j < kTiles; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        const int last_pos = p.t.length - p.t.n_new + (p.t.row0 + p.t.rows - 1) / a.group;
        const int first_pos = p.t.length - p.t.n_new + p.t.row0 / a.group;

        for (int t = p.first; t < p.end; ++t, ++it) {
            if ((it & 1) != half) continue;
            const int stage = it % kStages;
            // after a wait gave up the warps go on without waiting: they meet at barriers
            if (!*dead && !mbar_wait(&sm.full[stage], (it / kStages) & 1, a.status, kCodeFull)) *dead = 1;
            const PageScales sc = sm.scales[stage][quarter];
            // S: two tiles of 8 keys
            const uint8_t* keys = sm.ring[stage][0];
            const uint8_t* values = sm.ring[stage][1];
            float s[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                s[h][0] = s[h][1] = s[h][2] = s[h][3] = 0.0f;
                const int key = quarter * 16 + h * 8 + key_of(g);
                uint32_t w[kSteps];
                if (D == 128) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint4 v = *reinterpret_cast<const uint4*>(keys + key * 128 + (((c + i * 4) ^ (key & 7)) << 4));
                        w[i * 4] = v.x, w[i * 4 + 1] = v.y, w[i * 4 + 2] = v.z, w[i * 4 + 3] = v.w;
                    }
                } else {
                    const int row = key >> 1, base = (key & 1) * 4;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint2 v = *reinterpret_cast<const uint2*>(
                            keys + row * 128 + (((base + i * 2 + (c >> 1)) ^ (row & 7)) << 4) + (c & 1) * 8);
                        w[i * 2] = v.x, w[i * 2 + 1] = v.y;
                    }
                }
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    uint32_t b0, b1;
                    int8x4_to_half(w[k], b0, b1);
                    mma16816(s[h], q[k], b0, b1);
                }
            }
            // scores in base 2, with the value scale
            const int key0 = p.t.keys.tile(t) * kKeys + quarter * kGroupKeys;
            const bool clear = (!a.causal || key0 + kGroupKeys - 1 <= first_pos) && key0 + kGroupKeys <= p.t.length &&
                               (!a.window || last_pos - key0 < a.window || key0 + kGroupKeys <= a.sinks);
            const float f[2] = {unit[0] * sc.key, unit[1] * sc.key};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[h][e] = fmaf(s[h][e], f[e >> 1], sc.log2_value);
            bool hidden[2][4];
            if (!clear || sc.log2_value == -INFINITY) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key0 + h * 8 + key_of(2 * c + (e & 1)), at = pos[e >> 1];
                        const bool seen = key < p.t.length && (!a.causal || key <= at) &&
                                          (!a.window || at - key < a.window || key < a.sinks);
                        hidden[h][e] = !seen || sc.log2_value == -INFINITY;
                        if (hidden[h][e]) s[h][e] = -INFINITY;
                    }
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) hidden[h][e] = false;
            }
            float keep[2];
            bool grew = false;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float top = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float next = fmaxf(m[r], top);
                grew |= next > m[r];
                keep[r] = next == -INFINITY ? 1.0f : ex2(m[r] - next);
                m[r] = next;
            }
            if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                for (int j = 0; j < kTiles; ++j) {
                    o[j][0] *= keep[0], o[j][1] *= keep[0];
                    o[j][2] *= keep[1], o[j][3] *= keep[1];
                }
                l[0] *= keep[0], l[1] *= keep[1];
            }
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[h][e] = hidden[h][e] ? 0.0f : ex2(s[h][e] - (m[e >> 1] - kShift));
                    if (!hidden[h][e]) sum[e >> 1] += s[h][e];
                }
            if (sum[0] != 0.0f) l[0] = fmaf(sum[0], sc.inv_value, l[0]);
            if (sum[1] != 0.0f) l[1] = fmaf(sum[1], sc.inv_value, l[1]);
            // O += P V
            const uint32_t pa[4] = {pack2(s[0][0], s[0][1], __half()), pack2(s[0][2], s[0][3], __half()),
                                    pack2(s[1][0], s[1][1], __half()), pack2(s[1][2], s[1][3], __half())};
            uint32_t v[4][kTiles / 4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = quarter * 16 + (i >> 1) * 8 + (i & 1) * 4 + c;
                if (D == 128) {
                    const uint4 x = *reinterpret_cast<const uint4*>(values + key * 128 + (((value_dim<D>(g) >> 4) ^ (key & 7)) << 4));
                    v[i][0] = x.x, v[i][1] = x.y, v[i][2 % (kTiles / 4)] = x.z, v[i][3 % (kTiles / 4)] = x.w;
                } else {
                    const int row = key >> 1, chunk = (key & 1) * 4 + (value_dim<D>(g) >> 4);
                    const uint2 x = *reinterpret_cast<const uint2*>(values + row * 128 + ((chunk ^ (row & 7)) << 4) + (g & 1) * 8);
                    v[i][0] = x.x, v[i][1] = x.y;
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.empty[stage]);
#pragma unroll
            for (int i = 0; i < kTiles / 4; ++i) {
                const uint32_t w0 = v[0][i] ^ 0x80808080u, w1 = v[1][i] ^ 0x80808080u;
                const uint32_t w2 = v[2][i] ^ 0x80808080u, w3 = v[3][i] ^ 0x80808080u;
                const uint32_t x0 = __byte_perm(w0, w1, 0x5140), y0 = __byte_perm(w0, w1, 0x7362);
                const uint32_t x1 = __byte_perm(w2, w3, 0x5140), y1 = __byte_perm(w2, w3, 0x7362);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t b0 = half2_minus_1152(__byte_perm(j < 2 ? x0 : y0, 0x64646464u, (j & 1) ? 0x4342 : 0x4140));
                    const uint32_t b1 = half2_minus_1152(__byte_perm(j < 2 ? x1 : y1, 0x64646464u, (j & 1) ? 0x4342 : 0x4140));
                    mma16816(o[i * 4 + j], pa, b0, b1);
                }
            }
        }

        // ---- the eight warps' sums become one
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (c == 0) {
                sm.stats[parity][0][warp][g + 8 * r] = m[r];
                sm.stats[parity][1][warp][g + 8 * r] = l[r];
            }
        }
        consumers_sync();
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = g + 8 * r;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm.stats[parity][0][w][row]);
            const float mul = m[r] == -INFINITY ? 0.0f : ex2(m[r] - top);
            if (row < p.t.rows) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    float* to = &sm.sums[warp][row][value_dim<D>(2 * c + n)];
#pragma unroll
                    for (int j = 0; j < kTiles; j += 4)
                        *reinterpret_cast<float4*>(to + j) =
                            m[r] == -INFINITY && l[r] == 0.0f
                                ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                : make_float4(o[j][2 * r + n] * mul, o[j + 1][2 * r + n] * mul, o[j + 2][2 * r + n] * mul,
                                              o[j + 3][2 * r + n] * mul);
                }
            }
        }
        consumers_sync();
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
        for (int e = threadIdx.x; e < p.t.rows * (D / 4); e += kWarps * 32) {
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
            consumers_sync();
            if (threadIdx.x == 0) {
                const int before = atomicAdd(scratch.counters + c0, 1);
                sm.last = before == c1 - c0;
                if (sm.last) scratch.counters[c0] = 0;
            }
            consumers_sync();
            if (sm.last) {
                __threadfence();
                for (int e = threadIdx.x; e < p.t.rows * (D / 4); e += kWarps * 32) {
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
        parity ^= 1;
    }
}

template <typename T, int D>
cudaError_t launch(const AttendArgs& a, int sms, cudaStream_t s) {
    auto kernel = few_kernel<T, D>;
    const int smem = sizeof(Smem<D>) + 1024;
    static std::once_flag once;
    static cudaError_t attr = cudaSuccess;
    std::call_once(once, [&] { attr = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (attr != cudaSuccess) return attr;
    CUtensorMap map;
    // boxes of the keys that lie together in a page, 64 at most
    if (!kv_tensor_map(map, a, kKeys)) return cudaErrorInvalidValue;
    const int row_tiles = static_cast<int>((static_cast<long long>(a.max_new) * a.group + kRows - 1) / kRows);
    few_kernel<T, D><<<sms < kAttendMaxCtas ? sms : kAttendMaxCtas, kThreads, smem, s>>>(map, a, row_tiles, 1);
    return cudaGetLastError();
}

}  // namespace

cudaError_t attend_few(const AttendArgs& a, int dtype, int sms, cudaStream_t s) {
    if (a.head_dim == 64)
        return dtype == UFB_F16 ? launch<__half, 64>(a, sms, s) : launch<__nv_bfloat16, 64>(a, sms, s);
    return dtype == UFB_F16 ? launch<__half, 128>(a, sms, s) : launch<__nv_bfloat16, 128>(a, sms, s);
}

}  // namespace ufb
