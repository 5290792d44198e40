// Attention over the 8-bit cache for many rows (more new tokens x query heads of a
// key head than kv_attend_few.cu takes): frames, pieces of streams.
//
//   S = Q K^T,  P = 2^(S f + log2 vs - M),  O = P V,  l = sum P / vs,  out = O / l
//
// as there, in tiles of 256 rows x 128 keys on the fifth-generation tensor cores:
// the rows of all query heads of a key head lie in one tile, so the integers of a
// key tile are expanded to float16 once for 256 rows.
//
// One CTA an SM, four roles:
//   converter (8 warps)  integers from global memory through registers to float16
//                        in shared memory, keys and values double buffered, with
//                        128-byte swizzle; the page scales of each 16 keys
//   MMA (1 warp)         S_t = Q_t K^T and O_t += P_t V for the two halves t of
//                        128 rows, in the order O_0 S_0 O_1 S_1, so that one half
//                        multiplies while the other is in its softmax
//   softmax (2 x 4 warps) a thread owns a row: S from tensor memory, P back to it
//                        in float16 over S, where it is the A operand of P V
// Tensor memory: S_0, S_1 (128 columns each), O_0, O_1.
//
// Its floor at head_dim 128: 2048 cycles a tile for the exponentials (16 an SM and
// cycle) and 2200 for the products (measured alone), side by side.  A tile takes
// about 4900: the chain S, softmax, P V, S of a half, whose S and P share columns,
// and four roles' instructions on the same schedulers; which of them bounds it is not
// settled (at head_dim 64 a form without the chain took as long).  8160 tokens x 24480
// keys, 16 heads: 1.82 - 1.87 ms, 875 - 900 TFLOP/s, 0.52 - 0.53 of cuBLAS's rate in
// bfloat16; the first form of this kernel took 3.66 ms.  A running maximum that grows little is kept, so O is
// rescaled rarely and by the softmax threads themselves.
//
// The key tiles of all items are divided equally over the CTAs (kv_attend.cuh);
// rows shared by CTAs are joined by a second launch.
#include "kv_attend.cuh"
#include "umma.cuh"

#include <type_traits>

namespace ufb {

namespace {

constexpr int kRows = kAttendManyRows;
constexpr int kHalf = 128;
constexpr int kKeys = 128;
constexpr int kGroups = kKeys / kGroupKeys;
constexpr int kMmaWarp = 16, kWalkWarp = 17;
constexpr int kThreads = 640;         // warps: softmax 0-7, converter 8-15, MMA 16, walker 17; 18, 19 idle
constexpr int kPieces = 4;            // pieces announced ahead
constexpr int kReaders = 17;          // warps that read them
constexpr int kScaleRing = 4;
constexpr int kCode = 44;
// A running maximum stays while it grows by less than 2^kSlack, and P is taken
// times 2^kShift: it reaches 2^15 at most, inside float16, and weights down to
// 2^-27 of the largest keep all 11 bits.
constexpr float kSlack = 2.0f, kShift = 13.0f;
// Scores less their row's maximum in one multiply-add keep what the maximum lost in
// rounding: up to 2^-4 from this maximum on, and past float16's range from 2^26 on.
// Warps with such a row, and those with masked keys, round the score first, as the
// maximum was.  (Sums with the maximum are
// rounded so that P stays at or below 2^15 whatever the spacing of the scores is.)
constexpr float kFar = 1048576.0f;   // 2^20

struct alignas(16) GroupScales {
    float key, log2_value, inv_value, pad;   // log2_value -inf: the 16 keys are not there
};

// A piece of an item as the walker announces it; rows 0: there is none any more.
struct Announced {
    KeyRange keys;
    int rows, row0, first, end, slot, length, start, token0, head, parts, part;  // start: where token 0 stands
};

template <int D>
struct Smem {
    alignas(1024) uint8_t q[2][kHalf * D * 2];     // [64 dims][row][128 bytes]
    alignas(1024) uint8_t k[2][kKeys * D * 2];
    alignas(1024) uint8_t v[2][kKeys * D * 2];
    GroupScales scales[kScaleRing][kGroups];
    alignas(8) uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t q_full[2], s_full[2], p_full[2][2], o_full[2], drained;
    uint64_t piece_full[kPieces], piece_empty[kPieces];
    Announced pieces[kPieces];
    ShareSmem share;
    uint32_t tmem;
    int dead;
};

template <int D>
struct Tmem {
    __device__ static constexpr uint32_t s(int t) { return t * 128; }
    __device__ static constexpr uint32_t o(int t) { return 256 + t * D; }
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

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) many_kernel(const AttendArgs a, int row_tiles, int min_share) {
    // aligned by declaration, so that descriptors are constants (checked below)
    extern __shared__ __align__(1024) uint8_t raw[];
    Smem<D>& sm = *reinterpret_cast<Smem<D>*>(raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.k_full[i], 128);
            mbar_init(&sm.v_full[i], 128);
            mbar_init(&sm.k_empty[i], 1);
            mbar_init(&sm.v_empty[i], 1);
            mbar_init(&sm.q_full[i], 128);
            mbar_init(&sm.p_full[i][0], 128);
            mbar_init(&sm.p_full[i][1], 128);
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.o_full[i], 1);
        }
        mbar_init(&sm.drained, 1);
        for (int i = 0; i < kPieces; ++i) {
            mbar_init(&sm.piece_full[i], 1);
            mbar_init(&sm.piece_empty[i], kReaders);
        }
        fence_mbar_init();
        sm.dead = (smem_u32(raw) & 1023) != 0;
        if (sm.dead) atomicCAS(a.status, 0, kCode);
    }
    if (warp == kMmaWarp) {
        tmem_alloc(&sm.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    const Share share = locate_share<kKeys, kRows, kThreads>(a, row_tiles, min_share, sm.share);
    tc_fence_after();
    // all 512 columns are this CTA's: its tensor memory begins at 0
    constexpr uint32_t tmem = 0;
    volatile int* dead = &sm.dead;
    // after a wait gave up nobody waits any more, and no further piece is begun
    auto wait = [&](uint64_t* bar, int phase) {
        if (mbar_try_wait(bar, phase & 1)) return;
        if (!*dead && !mbar_wait(bar, phase & 1, a.status, kCode)) *dead = 1;
    };
    // Pieces one after another; a reader gives each back when it is done with it.
    auto piece_at = [&](int n) -> const Announced& {
        wait(&sm.piece_full[n % kPieces], n / kPieces);
        __syncwarp();
        return sm.pieces[n % kPieces];
    };
    auto piece_done = [&](int n) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.piece_empty[n % kPieces]);
    };

    // the registers of 640 threads at 96: 2 x 128 + 2 x 72 + 80 = 5 x 96
    if (warp < 8) {
        regs_inc<128>();
        // ---- softmax: half t, row of the half = thread
        const int t = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + Tmem<D>::s(t), to = tmem + lanes + Tmem<D>::o(t);
        int tiles = 0, s_n = 0, o_n = 0;   // key tiles of this CTA so far; phases of this half
        const AttendScratch scratch = scratch_of(a.workspace, gridDim.x, kRows);
        if (t == 0 && row == 0) scratch.items[blockIdx.x * 8] = 0;
        for (int n = 0;; ++n) {
            const Announced& p = piece_at(n);
            if (p.rows == 0 || *dead) break;
            if (t * kHalf >= p.rows) {
                tiles += p.end - p.first;
                piece_done(n);
                continue;
            }
            const int r = t * kHalf + row;
            const bool real = r < p.rows;
            const int in_stream = p.row0 + (real ? r : 0);
            const int token = in_stream / a.group, head = p.head * a.group + in_stream - token * a.group;
            const int pos = p.start + token;
            const long long out_row = p.token0 + static_cast<long long>(token);
            float unit;
            {
                // the row to [2^15, 2^16) and float16; the softmax scale's sign goes with it
                const T* src = static_cast<const T*>(a.q.data) + out_row * a.q.token_stride +
                               head * a.q.head_stride;
                const uint4* vec = reinterpret_cast<const uint4*>(src);
                float top = 0.0f, odd = 0.0f;
#pragma unroll 4
                for (int i = 0; i < D / 8; ++i) {
                    const uint4 v = real ? vec[i] : make_uint4(0, 0, 0, 0);
                    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 f = unpack2(x[j], T());
                        top = max3(top, fabsf(f.x), fabsf(f.y));
                        odd += (f.x - f.x) + (f.y - f.y);  // NaN for what is not finite
                    }
                }
                const float u = row_unit(odd == odd ? top : odd);
                unit = unit_inverse(u) * fabsf(a.scale_log2);
                const float mul = u == u ? (a.scale_log2 < 0.0f ? -u : u) : 0.0f;
#pragma unroll 4
                for (int i = 0; i < D / 8; ++i) {
                    const uint4 v = real ? vec[i] : make_uint4(0, 0, 0, 0);
                    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
                    uint32_t y[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 f = unpack2(x[j], T());
                        y[j] = pack2(f.x * mul, f.y * mul, __half());
                    }
                    *reinterpret_cast<uint4*>(sm.q[t] + tile_at(row, i)) = make_uint4(y[0], y[1], y[2], y[3]);
                }
                fence_proxy_async_smem();
                mbar_arrive(&sm.q_full[t]);
            }
            float m = -INFINITY, l = 0.0f;
            bool far = false;   // a row of the warp has scores beyond kFar
            const int first_pos = p.start + (p.row0 + t * kHalf) / a.group;
            const int last_pos = p.start + (p.row0 + min(p.rows, (t + 1) * kHalf) - 1) / a.group;
            const int length = p.length, end = p.end;
            for (int tile = p.first; tile < end; ++tile, ++tiles) {
                wait(&sm.s_full[t], s_n++);
                __syncwarp();
                tc_fence_after();
                const GroupScales* sc = sm.scales[tiles % kScaleRing];
                const int key0 = p.keys.tile(tile) * kKeys;
                const bool clear = (!a.causal || key0 + kKeys - 1 <= first_pos) && key0 + kKeys <= length &&
                                   (!a.window || last_pos - key0 < a.window || key0 + kKeys <= a.sinks);
                // columns [0, high) that are from low on or below sink are seen by this row
                const int high = min(length, a.causal ? pos + 1 : length) - key0;
                const int low = a.window ? max(pos - a.window + 1, 0) - key0 : 0;
                const int sink = a.window ? a.sinks - key0 : 0;
                auto seen = [&](int c) {   // of 32 columns, a bit each
                    return bits_below(high - c * 32) & (~bits_below(low - c * 32) | bits_below(sink - c * 32));
                };
                // 64 columns at a time, the later ones first: the others stay for their
                // weights.  Loops are not unrolled: three roles share each scheduler's
                // instruction cache.
                uint32_t s0[32], s1[32];
                float top = -INFINITY;
                auto maximum = [&](auto masked) {
                    auto chunk = [&](int c, const uint32_t (&s)[32]) {
                        const uint32_t bits = decltype(masked)::value ? seen(c) : 0u;
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            auto f = [&](int j) {
                                return decltype(masked)::value && !(bits & (1u << (g * 16 + j))) ? -INFINITY
                                                                                              : __uint_as_float(s[g * 16 + j]);
                            };
                            float y = max3(f(0), f(1), f(2)), z = max3(f(3), f(4), f(5));
                            y = max3(y, f(6), f(7)), z = max3(z, f(8), f(9));
                            y = max3(y, f(10), f(11)), z = max3(z, f(12), f(13));
                            y = max3(y, f(14), f(15));
                            y = fmaxf(y, z);
                            const GroupScales gs = sc[c * 2 + g];
                            const float v = fmaf(y, unit * gs.key, gs.log2_value);
                            // -infinity: nothing of the group is seen
                            top = fmaxf(top, decltype(masked)::value && y == -INFINITY ? y : v);
                        }
                    };
#pragma unroll 1
                    for (int c = 2; c >= 0; c -= 2) {
                        tmem_ld32(ts + c * 32, s0);
                        tmem_ld32(ts + c * 32 + 32, s1);
                        tmem_wait_ld();
                        tmem_tie32(s0);
                        tmem_tie32(s1);
                        chunk(c, s0);
                        chunk(c + 1, s1);
                    }
                };
                if (clear) maximum(std::false_type());
                else maximum(std::true_type());
                // the maximum stays while it is within 2^kSlack
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
                    for (int half = 0; half < 2; ++half) {
                        tmem_wait_ld();
                        tmem_tie32(s0);
                        tmem_tie32(s1);
                        chunk(half * 2, s0);
                        if (half == 0) tmem_ld32(ts + 64, s0);
                        chunk(half * 2 + 1, s1);
                        if (half == 0) tmem_ld32(ts + 96, s1);
                        // P V starts on the first 64 keys while the others are in the works
                        tmem_wait_st();
                        tc_fence_before();
                        mbar_arrive(&sm.p_full[t][half]);
                    }
                };
                if (clear && !far) weights(std::false_type());
                else weights(std::true_type());
            }
            wait(&sm.o_full[t], o_n++);
            __syncwarp();
            tc_fence_after();
            const bool whole = p.part < 0;
            const int part = 2 * blockIdx.x + p.part;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            T* out = static_cast<T*>(a.out.data) + out_row * a.out.token_stride + head * a.out.head_stride;
            float* sums = scratch.sums + (static_cast<long long>(part) * kRows + r) * D;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(to + c * 32, o);
                tmem_wait_ld();
                if (real && whole) {
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float x = __uint_as_float(o[j + 2 * i]) * inv, y = __uint_as_float(o[j + 2 * i + 1]) * inv;
                            w[i] = pack2(x, y, T());
                        }
                        reinterpret_cast<uint4*>(out)[c * 4 + j / 8] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else if (real) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        __stcg(reinterpret_cast<uint4*>(sums + c * 32 + j), make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]));
                }
                __syncwarp();
            }
            if (real && whole && a.lse)
                a.lse[out_row * (a.heads * a.group) + head] =
                    l == 0.0f ? -INFINITY : (m - kShift + log2f(l)) * 0.6931471805599453f;
            if (real && !whole) {
                __stcg(scratch.stats + (part * 2) * kRows + r, m);
                __stcg(scratch.stats + (part * 2 + 1) * kRows + r, l);
            }
            if (p.parts && t == 0 && row == 0) {
                int32_t* item = scratch.items + blockIdx.x * 8;
                item[1] = p.token0;
                item[2] = p.row0;
                item[3] = p.rows;
                item[4] = p.head;
                item[0] = p.parts;
            }
            piece_done(n);
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
        uint64_t* full = side ? sm.v_full : sm.k_full;
        uint64_t* empty = side ? sm.v_empty : sm.k_empty;
        uint8_t* tiles = side ? sm.v[0] : sm.k[0];
        // this thread's two 16-byte pieces of its first row; row & 7 repeats every kStep * 2 rows
        uint32_t at0[2], at1[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            at0[i] = tile_at(w * 32 + i * kStep + sub, chunk * 2);
            at1[i] = tile_at(w * 32 + i * kStep + sub, chunk * 2 + 1);
        }
        struct Next {
            int page[2], row[2], head;   // of this warp's two groups of 16 keys
            bool tile;                   // false: no further tile
        };
        int piece = 0, at = -1;   // the piece being looked up and its next tile; -1: not begun
        bool have = true;
        auto fetch = [&](Next& n) {
            n.tile = false;
            n.page[0] = n.page[1] = -1;
            if (!have) return;
            const Announced& p = piece_at(piece);
            have = p.rows > 0 && !*dead;
            if (!have) return;
            if (at < 0) at = p.first;
            n.tile = true;
            n.head = p.head;
            const int key0 = p.keys.tile(at) * kKeys + w * 32;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int key = key0 + g * kGroupKeys, entry = key >> a.page_shift;
                n.row[g] = key & (a.page_tokens - 1);
                if (p.keys.touches(key) && entry < a.table_width)
                    n.page[g] = a.table[static_cast<long long>(p.slot) * a.table_width + entry];
            }
            if (++at == p.end) {
                piece_done(piece++);
                at = -1;
            }
        };
        uint4 buf[kLoads];
        float key_scale = 0.0f, value_scale = -1.0f;   // of the warp's group `lane` (0, 1); -1: not there
        auto load = [&](const Next& n) {
            if (!n.tile) return;
            const int8_t* from[2];
            bool there[2];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                there[g] = n.page[g] >= 0 && n.page[g] < a.pages;
                const long long tile = (static_cast<long long>(n.page[g]) * 2 + side) * a.heads + n.head;
                from[g] = a.kv + ((tile << a.page_shift) + n.row[g] + sub) * D + chunk * 16;
            }
            if (there[0] && there[1]) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i)  // sub < kStep, a divisor of 16
                    buf[i] = __ldg(reinterpret_cast<const uint4*>(from[(i * kStep) >> 4] + ((i * kStep) & 15) * D));
            } else {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    buf[i] = make_uint4(0, 0, 0, 0);
                    if (there[(i * kStep) >> 4])
                        buf[i] = __ldg(reinterpret_cast<const uint4*>(from[(i * kStep) >> 4] + ((i * kStep) & 15) * D));
                }
            }
            if (side == 0 && lane < 2) {
                key_scale = 0.0f, value_scale = -1.0f;
                if (lane == 0 ? there[0] : there[1]) {
                    const int page = lane == 0 ? n.page[0] : n.page[1];
                    const float* s = a.scale + static_cast<long long>(page) * 2 * a.heads + n.head;
                    key_scale = s[0];
                    value_scale = s[a.heads];
                    if (value_scale < kTinyScale) value_scale = kTinyScale;
                }
            }
        };
        Next now, next;
        fetch(now);
        load(now);
        fetch(next);
        for (int n = 0; now.tile; ++n) {
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
            }
            if (side == 0 && lane < 2) {
                GroupScales g;
                g.key = key_scale;
                g.log2_value = value_scale == -1.0f ? -INFINITY : log2f(value_scale);
                g.inv_value = value_scale == -1.0f ? 0.0f : 1.0f / value_scale;
                g.pad = 0.0f;
                sm.scales[n % kScaleRing][w * 2 + lane] = g;
            }
            fence_proxy_async_smem();
            mbar_arrive(&full[b]);
            load(next);
            now = next;
            fetch(next);
        }
    } else {
        regs_dec<80>();
        if (warp == kWalkWarp) {
            // ---- walker: announces this CTA's pieces
            Walker<kKeys, kRows> walk(a, share, row_tiles);
            Piece p;
            bool more = true;
            for (int n = 0; more; ++n) {
                more = walk.next(a, p) && !*dead;
                if (n >= kPieces) wait(&sm.piece_empty[n % kPieces], n / kPieces - 1);
                if (lane == 0) {
                    Announced& o = sm.pieces[n % kPieces];
                    o.rows = more ? p.t.rows : 0;
                    if (more) {
                        o.keys = p.t.keys;
                        o.row0 = p.t.row0;
                        o.first = p.first;
                        o.end = p.end;
                        o.slot = p.t.slot;
                        o.length = p.t.length;
                        o.start = p.t.length - p.t.n_new;
                        o.token0 = static_cast<int>(p.t.token0);
                        o.head = p.head;
                        // the part of a shared item: 0 where an earlier CTA began it, 1 where this
                        // one does, which then tells how many parts there are
                        o.part = p.whole() ? -1 : (p.first > 0 ? 0 : 1);
                        o.parts = o.part == 1 ? static_cast<int>(quotient(p.item_start + p.t.keys.nt - 1, share.per)) -
                                                    static_cast<int>(blockIdx.x) + 1
                                              : 0;
                    }
                    mbar_arrive(&sm.piece_full[n % kPieces]);
                }
                __syncwarp();
            }
        }
        // ---- MMA: the warp waits together, one lane issues
        if (warp == kMmaWarp) {
            constexpr uint32_t qk = f16_idesc(128, kKeys, false), pv = f16_idesc(128, D, true);
            constexpr uint64_t kTile = (kKeys * D * 2) >> 4;   // descriptor step between the two buffers
            const uint64_t q_desc = sw128_desc(smem_u32(sm.q[0])), k_desc = sw128_desc(smem_u32(sm.k[0]));
            const uint64_t v_desc = sw128_n_major_desc(smem_u32(sm.v[0]), 128 * 128);
            int n = 0;                    // key tiles so far
            int q_n[2] = {0, 0}, p_n[2] = {0, 0};
            const uint32_t issue = lane == 0;
            auto scores = [&](int t, int b) {
                const uint64_t qd = q_desc + t * kTile, kd = k_desc + b * kTile;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const int off = ((k >> 2) * (128 * 128) + (k & 3) * 32) >> 4;
                    mma_f16(tmem + Tmem<D>::s(t), qd + off, kd + off, qk, k > 0, issue);
                }
                mma_commit_if(&sm.s_full[t], issue);
            };
            for (int piece = 0;; ++piece) {
                const Announced& p = piece_at(piece);
                if (p.rows == 0 || *dead) break;
                const int halves = p.rows > kHalf ? 2 : 1;
                const int count = p.end - p.first;
                piece_done(piece);
                wait(&sm.k_full[n & 1], n >> 1);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (t >= halves) continue;
                    wait(&sm.q_full[t], q_n[t]++);
                    __syncwarp();
                    tc_fence_after();
                    scores(t, n & 1);
                }
                mma_commit_if(&sm.k_empty[n & 1], issue);
#pragma unroll 1
                for (int i = 0; i < count; ++i, ++n) {
                    const int b = n & 1, c = (n + 1) & 1;
                    const bool more = i + 1 < count;
                    wait(&sm.v_full[b], n >> 1);
                    if (more) wait(&sm.k_full[c], (n + 1) >> 1);
                    const uint64_t vd = v_desc + b * kTile;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (t >= halves) continue;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            wait(&sm.p_full[t][h], p_n[t]);
                            __syncwarp();
                            tc_fence_after();
#pragma unroll
                            for (int k = h * 4; k < h * 4 + 4; ++k)
                                mma_f16_ts(tmem + Tmem<D>::o(t), tmem + Tmem<D>::s(t) + k * 8, vd + k * (16 * 128 >> 4),
                                           pv, i > 0 || k > 0, issue);
                        }
                        ++p_n[t];
                        if (more) scores(t, c);
                        else mma_commit_if(&sm.o_full[t], issue);
                    }
                    mma_commit_if(&sm.v_empty[b], issue);
                    if (more) mma_commit_if(&sm.k_empty[c], issue);
                }
            }
            // nothing may be in flight when tensor memory is given back
            if (lane == 0) {
                mma_commit(&sm.drained);
                mbar_wait(&sm.drained, 0, a.status, kCode);
            }
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(sm.tmem, 512);
    }
}

// Rows that several CTAs share: the item that CTA x's share ends in, a block's rows
// from kJoinRows * y on.  The parts' maxima and weights come first, once a row, by a
// warp; then a thread adds the parts of four columns, in the order of the CTAs.
constexpr int kJoinThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const AttendArgs a, int ctas) {
    constexpr int kJoinRows = kJoinThreads / (D / 4);
    __shared__ float share[kAttendMaxCtas][kJoinRows];   // of a part in a row's sum
    __shared__ float tops[kJoinRows], weights[kJoinRows];
    const AttendScratch scratch = scratch_of(a.workspace, ctas, kRows);
    const int c0 = blockIdx.x, first = blockIdx.y * kJoinRows;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int32_t* item = scratch.items + c0 * 8;
    const int parts = item[0], rows = min(item[3] - first, kJoinRows);
    if (parts == 0 || rows <= 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
    const int r = threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
    if (r >= rows) return;
    const int row = first + r;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int i = 0; i < parts; ++i) {
        const int from = 2 * (c0 + i) + (i == 0);
        const float4 x = *reinterpret_cast<const float4*>(scratch.sums + (static_cast<long long>(from) * kRows + row) * D + d);
        const float mul = share[i][r];
        v.x += x.x * mul, v.y += x.y * mul, v.z += x.z * mul, v.w += x.w * mul;
    }
    const int in_stream = item[2] + row, token = in_stream / a.group;
    const int head = item[4] * a.group + in_stream - token * a.group;
    const float top = tops[r], weight = weights[r];
    const float inv = weight == 0.0f ? 0.0f : 1.0f / weight;
    const long long out_row = item[1] + static_cast<long long>(token);
    T* to = static_cast<T*>(a.out.data) + out_row * a.out.token_stride + head * a.out.head_stride + d;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2(v.x * inv, v.y * inv, T()), pack2(v.z * inv, v.w * inv, T()));
    if (a.lse && d == 0)
        a.lse[out_row * (a.heads * a.group) + head] =
            weight == 0.0f ? -INFINITY : (top - kShift + log2f(weight)) * 0.6931471805599453f;
}

template <typename T, int D>
cudaError_t launch(const AttendArgs& a, int sms, cudaStream_t s) {
    auto kernel = many_kernel<T, D>;
    const int smem = sizeof(Smem<D>);
    static std::atomic<uint64_t> allowed;
    const cudaError_t attr = allow_smem(kernel, smem, allowed);
    if (attr != cudaSuccess) return attr;
    const long long row_tiles = (static_cast<long long>(a.max_new) * a.group + kRows - 1) / kRows;
    if (row_tiles * a.n > 0x3fffffff) return cudaErrorInvalidValue;
    const int ctas = sms < kAttendMaxCtas ? sms : kAttendMaxCtas;
    many_kernel<T, D><<<ctas, kThreads, smem, s>>>(a, static_cast<int>(row_tiles), 1);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    // its blocks may start once the CTAs have exited, before that kernel's end is signalled
    // (it gives no earlier trigger): they wait for that
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(ctas, kRows * (D / 4) / kJoinThreads);
    config.blockDim = dim3(kJoinThreads);
    config.stream = s;
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, join_kernel<T, D>, a, ctas);
}

}  // namespace

cudaError_t attend_many(const AttendArgs& a, int dtype, int sms, cudaStream_t s) {
    if (a.head_dim == 64)
        return dtype == UFB_F16 ? launch<__half, 64>(a, sms, s) : launch<__nv_bfloat16, 64>(a, sms, s);
    return dtype == UFB_F16 ? launch<__half, 128>(a, sms, s) : launch<__nv_bfloat16, 128>(a, sms, s);
}

}  // namespace ufb
