// Pages of the 8-bit cache: extend, release, fork, trim, compact.
//
// Tables, lengths and reference counts live on the device and the host never
// waits for them.  What has to be decided in order (which free page goes to
// which stream) is done by one CTA with block-wide prefix sums over the
// requests and over the reference counts, lowest free page first, so the result
// does not depend on timing; the bytes of a decision (page copies over all
// layers) are moved by a second launch that fills the GPU and reads the list of
// moves from the cache's scratch.
#include "attention.h"

#include "capi_util.h"

namespace ufb {

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

// Scratch layout (int32): [0] moves to make, [16, 16 + pages) free pages found,
// in order; then [pages) moves' sources / [pages) token counts; then one offset
// per request (slots).  Behind it lie the marks of refused streams (kv_refused).
struct Work {
    int32_t* moves;
    int32_t* found;
    int32_t* source;
    int32_t* rest;
    int32_t* start;
};

__host__ __device__ inline Work work_of(const ufb_kv_cache& c) {
    Work w;
    w.moves = c.work;
    w.found = c.work + 16;
    w.source = w.found + c.pages;
    w.rest = w.source + c.pages;
    w.start = w.rest + c.pages;
    return w;
}

// Block-wide exclusive prefix sum of one value a thread; total to every thread.
__device__ __forceinline__ int block_scan(int value, int* warp_sum, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = value;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
    }
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        int s = warp_sum[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += t;
        }
        warp_sum[lane] = s;
    }
    __syncthreads();
    total = warp_sum[kWarps - 1];
    const int base = warp ? warp_sum[warp - 1] : 0;
    __syncthreads();
    return base + inc - value;
}

// The first `need` free pages, in order, to found[]; returns how many there are
// (at most need).  Four pages a thread and step; stops when there are enough.
// refs are read past the L1 cache: this CTA's own atomics changed them.
__device__ int find_free(const ufb_kv_cache& c, int need, int32_t* found, int* warp_sum) {
    int have = 0;
    for (int base = 0; base < c.pages && have < need; base += kThreads * 4) {
        const int p0 = base + threadIdx.x * 4;
        bool free_page[4];
        int count = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            free_page[j] = p0 + j < c.pages && __ldcg(c.refs + p0 + j) == 0;
            count += free_page[j];
        }
        int total;
        int at = have + block_scan(count, warp_sum, total);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (free_page[j]) {
                if (at < need) found[at] = p0 + j;
                ++at;
            }
        have += total;
    }
    __syncthreads();
    return min(have, need);
}

__device__ __forceinline__ bool valid_slot(const ufb_kv_cache& c, int slot) { return slot >= 0 && slot < c.slots; }

__global__ void __launch_bounds__(kThreads) extend_kernel(const ufb_kv_cache c, const int32_t* slots,
                                                          const int32_t* offsets, int n, int* status) {
    __shared__ int warp_sum[kWarps];
    const Work w = work_of(c);
    const int P = c.page_tokens;
    long long need = 0;
    int bad = 0;
    for (int base = 0; base < n; base += kThreads) {
        const int i = base + threadIdx.x;
        int want = 0;
        if (i < n) {
            const int slot = slots[i], count = offsets[i + 1] - offsets[i];
            if (!valid_slot(c, slot) || count < 0 || c.lengths[slot] < 0)
                bad = kStatusIndex;
            else {
                const long long have = c.lengths[slot], after = have + count;
                const long long entries = (after + P - 1) / P;
                if (entries > c.table_width || after > 0x7fffffffll)
                    bad = bad ? bad : kStatusPages;
                else
                    want = static_cast<int>(entries - (have + P - 1) / P);
            }
        }
        int total;
        const int at = block_scan(want, warp_sum, total);
        if (i < n) w.start[i] = static_cast<int>(min(need + at, 0x7fffffffll));
        need += total;
    }
    const int any_index = __syncthreads_or(bad == kStatusIndex), any_pages = __syncthreads_or(bad == kStatusPages);
    if (!any_index && !any_pages && need <= c.pages) {
        const int found = find_free(c, static_cast<int>(need), w.found, warp_sum);
        if (found == need) {
            const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
            for (int i = warp; i < n; i += kWarps) {
                const int slot = slots[i], count = offsets[i + 1] - offsets[i];
                const int have = c.lengths[slot], first = (have + P - 1) / P;
                const int entries = static_cast<int>((static_cast<long long>(have) + count + P - 1) / P) - first;
                __syncwarp();
                for (int e = lane; e < entries; e += 32) {
                    const int page = w.found[w.start[i] + e];
                    c.table[static_cast<long long>(slot) * c.table_width + first + e] = page;
                    c.refs[page] = 1;
                }
                if (lane == 0) {
                    c.lengths[slot] = have + count;
                    kv_refused(c)[slot] = 0;
                }
            }
            return;
        }
    }
    // the lengths stay, so the last tokens of these streams are no new ones: append and
    // attend of the step that goes on regardless must not take them for such
    for (int i = threadIdx.x; i < n; i += kThreads)
        if (valid_slot(c, slots[i]) && offsets[i + 1] > offsets[i]) kv_refused(c)[slots[i]] = 1;
    if (threadIdx.x == 0) atomicCAS(status, 0, any_index ? kStatusIndex : kStatusPages);
}

// A warp drops every page of table row `slot` (all 32 lanes call it).
__device__ __forceinline__ void drop_row(const ufb_kv_cache& c, int slot, long long first, long long end) {
    for (long long e = first + (threadIdx.x & 31); e < end; e += 32) {
        int32_t* entry = c.table + static_cast<long long>(slot) * c.table_width + e;
        const int page = *entry;
        if (page >= 0) {
            if (page < c.pages) atomicSub(c.refs + page, 1);
            *entry = -1;
        }
    }
}

// One warp to a stream.  window 0: release everything; else trim.
__global__ void __launch_bounds__(128) drop_kernel(const ufb_kv_cache c, const int32_t* slots, int n, int window,
                                                   int sinks, int* status) {
    const int i = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (i >= n) return;
    const int slot = slots[i];
    if (!valid_slot(c, slot)) {
        if ((threadIdx.x & 31) == 0) atomicCAS(status, 0, kStatusIndex);
        return;
    }
    if (window == 0) {
        drop_row(c, slot, 0, c.table_width);
        if ((threadIdx.x & 31) == 0) c.lengths[slot] = kv_refused(c)[slot] = 0;
        return;
    }
    // the next query stands at length or later: keys below length - window + 1
    // that are no sinks are seen by nobody any more
    const long long unseen = static_cast<long long>(c.lengths[slot]) - window + 1;
    const long long end = unseen > 0 ? min(unseen / c.page_tokens, static_cast<long long>(c.table_width)) : 0;
    drop_row(c, slot, (static_cast<long long>(sinks) + c.page_tokens - 1) / c.page_tokens, end);
}

__global__ void __launch_bounds__(kThreads) fork_kernel(const ufb_kv_cache c, const int32_t* src, const int32_t* dst,
                                                        int n, int* status) {
    __shared__ int warp_sum[kWarps];
    const Work w = work_of(c);
    const int P = c.page_tokens;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) *w.moves = 0;
    int bad = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) bad |= !valid_slot(c, src[i]) || !valid_slot(c, dst[i]);
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) atomicCAS(status, 0, kStatusIndex);
        return;
    }
    // release the destinations and share the sources' full pages
    for (int i = warp; i < n; i += kWarps) {
        const int s = src[i], d = dst[i];
        const int32_t* from = c.table + static_cast<long long>(s) * c.table_width;
        int32_t* to = c.table + static_cast<long long>(d) * c.table_width;
        const int full = min(c.lengths[s] / P, c.table_width);
        for (int e = lane; e < c.table_width; e += 32) {
            const int held = to[e], shared = e < full ? from[e] : -1;
            if (held >= 0 && held < c.pages) atomicSub(c.refs + held, 1);
            if (shared >= 0 && shared < c.pages) atomicAdd(c.refs + shared, 1);
            if (held != shared) to[e] = shared;
        }
    }
    __syncthreads();
    int need = 0;
    for (int base = 0; base < n; base += kThreads) {
        const int i = base + threadIdx.x;
        int want = 0;
        if (i < n) {
            const int length = c.lengths[src[i]], full = length / P;
            want = length % P > 0 && full < c.table_width &&
                   c.table[static_cast<long long>(src[i]) * c.table_width + full] >= 0;
        }
        int total;
        const int at = block_scan(want, warp_sum, total);
        if (i < n) w.start[i] = want ? need + at : -1;
        need += total;
    }
    const int found = need <= c.pages ? find_free(c, need, w.found, warp_sum) : -1;
    if (found != need) {
        for (int i = warp; i < n; i += kWarps) {
            drop_row(c, dst[i], 0, c.table_width);
            if (lane == 0) c.lengths[dst[i]] = kv_refused(c)[dst[i]] = 0;
        }
        if (threadIdx.x == 0) atomicCAS(status, 0, kStatusPages);
        return;
    }
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int length = c.lengths[src[i]], full = length / P, at = w.start[i];
        if (at >= 0) {
            const int page = w.found[at];
            c.table[static_cast<long long>(dst[i]) * c.table_width + full] = page;
            c.refs[page] = 1;
            w.source[at] = c.table[static_cast<long long>(src[i]) * c.table_width + full];
            w.rest[at] = length % P;
        }
        c.lengths[dst[i]] = length;
        kv_refused(c)[dst[i]] = kv_refused(c)[src[i]];
    }
    if (threadIdx.x == 0) *w.moves = need;
}

__global__ void __launch_bounds__(kThreads) compact_kernel(const ufb_kv_cache c) {
    __shared__ int warp_sum[kWarps];
    const Work w = work_of(c);
    int live = 0;
    for (int p = threadIdx.x; p < c.pages; p += kThreads) live += c.refs[p] > 0;
    int total;
    block_scan(live, warp_sum, total);
    live = total;
    // free pages below the live count, live pages from it on: as many of either
    int holes = 0, movers = 0;
    for (int base = 0; base < c.pages; base += kThreads) {
        const int p = base + threadIdx.x;
        const bool used = p < c.pages && c.refs[p] > 0;
        const bool hole = p < c.pages && p < live && !used, mover = p >= live && used;
        // a page is one or the other: both counts in one sum of at most 1024 each
        const int at = block_scan(hole + (mover << 16), warp_sum, total);
        if (hole) w.found[holes + (at & 0xffff)] = p;
        if (mover) w.source[movers + (at >> 16)] = p;
        if (p < c.pages) w.rest[p] = p;   // the page's new id, for the tables
        holes += total & 0xffff;
        movers += total >> 16;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < movers; i += kThreads) {
        const int from = w.source[i], to = w.found[i];
        w.rest[from] = to;
        c.refs[to] = c.refs[from];
        c.refs[from] = 0;
    }
    if (threadIdx.x == 0) *w.moves = movers;
}

// Waits for the kernel before this one.  Launched with programmatic serialization,
// this one's blocks may start once that one's have exited, without its end being
// flushed and signalled first: that hides part of a launch's latency, no work (the
// kernel before gives no earlier trigger).
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Moves of the list: grid (moves upper bound or less, layers * 2 sides).  A CTA
// copies the tokens of every head of one side.  PARTIAL: rest[move] tokens of each
// head.  Else whole pages, and one more row of blocks (y = layers * 2) takes the
// moved pages' new ids (rest[page]) into the tables.
template <bool PARTIAL>
__global__ void __launch_bounds__(256) move_kernel(const ufb_kv_cache c) {
    const Work w = work_of(c);
    const int side = blockIdx.y & 1, layer = blockIdx.y >> 1;
    const int head_vecs = c.page_tokens * c.head_dim / 16;
    wait_for_previous();
    const int moves = *w.moves;
    if (!PARTIAL && layer == c.layers) {
        const long long entries = static_cast<long long>(c.slots) * c.table_width;
        for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; moves && i < entries; i += gridDim.x * 256ll) {
            const int page = c.table[i];
            if (page >= 0 && page < c.pages) {
                const int to = w.rest[page];
                if (to != page) c.table[i] = to;
            }
        }
        return;
    }
    for (int m = blockIdx.x; m < moves; m += gridDim.x) {
        const long long from = ((static_cast<long long>(layer) * c.pages + w.source[m]) * 2 + side) * c.heads;
        const long long to = ((static_cast<long long>(layer) * c.pages + w.found[m]) * 2 + side) * c.heads;
        const uint4* in = reinterpret_cast<const uint4*>(c.kv) + from * head_vecs;
        uint4* out = reinterpret_cast<uint4*>(c.kv) + to * head_vecs;
        const int vecs = PARTIAL ? w.rest[m] * c.head_dim / 16 : head_vecs;
        const int total = vecs * c.heads;
        constexpr int kBatch = 8;
        for (int base = threadIdx.x; base < total; base += 256 * kBatch) {
            uint4 v[kBatch];
            int at[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int i = base + j * 256;
                const int head = PARTIAL ? i / vecs : 0;
                at[j] = PARTIAL ? head * head_vecs + i - head * vecs : i;
                if (i < total) v[j] = __ldcs(in + at[j]);
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (base + j * 256 < total) out[at[j]] = v[j];
        }
        for (int h = threadIdx.x; h < c.heads; h += 256) c.scale[to + h] = c.scale[from + h];
    }
}

template <bool PARTIAL>
cudaError_t move(const ufb_kv_cache& c, int most, cudaStream_t s) {
    // layers are checked: gridDim.y stays below 65536
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(most < 1024 ? most : 1024, c.layers * 2 + (PARTIAL ? 0 : 1));
    config.blockDim = dim3(256);
    config.stream = s;
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, move_kernel<PARTIAL>, c);
}

}  // namespace

cudaError_t kv_extend(const ufb_kv_cache& c, const int32_t* slots, const int32_t* offsets, int n, int* status,
                      cudaStream_t s) {
    extend_kernel<<<1, kThreads, 0, s>>>(c, slots, offsets, n, status);
    return cudaGetLastError();
}

cudaError_t kv_release(const ufb_kv_cache& c, const int32_t* slots, int n, int* status, cudaStream_t s) {
    drop_kernel<<<(n + 3) / 4, 128, 0, s>>>(c, slots, n, 0, 0, status);
    return cudaGetLastError();
}

cudaError_t kv_trim(const ufb_kv_cache& c, const int32_t* slots, int n, int window, int sinks, int* status,
                    cudaStream_t s) {
    drop_kernel<<<(n + 3) / 4, 128, 0, s>>>(c, slots, n, window, sinks, status);
    return cudaGetLastError();
}

cudaError_t kv_fork(const ufb_kv_cache& c, const int32_t* src, const int32_t* dst, int n, int* status,
                    cudaStream_t s) {
    fork_kernel<<<1, kThreads, 0, s>>>(c, src, dst, n, status);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? move<true>(c, n, s) : e;
}

cudaError_t kv_compact(const ufb_kv_cache& c, int*, cudaStream_t s) {
    compact_kernel<<<1, kThreads, 0, s>>>(c);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? move<false>(c, c.pages, s) : e;
}

}  // namespace ufb
