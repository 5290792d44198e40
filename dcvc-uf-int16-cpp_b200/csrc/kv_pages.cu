// Pages of the 8-bit cache: extend, release, fork, reorder, trim, compact, and what
// groups of streams have in common.
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

#include <climits>

namespace ufb {

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kApplyThreads = 256;
constexpr int kColumns = 128;   // table columns of a block of reorder_apply_kernel

// Scratch layout (int32): [0] moves to make, [1] whether a reorder goes ahead, [2] the
// calls that changed tables or lengths (kv_changes), [16, 16 + pages) free pages found, in order; then [pages) moves' sources / [pages) token counts;
// then one offset per request (slots).  Behind it lie the marks of refused streams
// (kv_refused) and the entries of last pages (kv_last_entry).
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

// By one thread of a kernel that changes tables, lengths or marks (page ids apart): what
// ufb_kv_share found before holds no more.
__device__ __forceinline__ void count_change(const ufb_kv_cache& c) {
    *kv_changes(c) = static_cast<int32_t>(static_cast<uint32_t>(*kv_changes(c)) + 1u);
}

__device__ __forceinline__ bool valid_slot(const ufb_kv_cache& c, int slot) { return slot >= 0 && slot < c.slots; }

__global__ void __launch_bounds__(kThreads) extend_kernel(const ufb_kv_cache c, const int32_t* slots,
                                                          const int32_t* offsets, int n, int* status) {
    __shared__ int warp_sum[kWarps];
    const Work w = work_of(c);
    const int P = c.page_tokens;
    if (threadIdx.x == 0) count_change(c);
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
    if (blockIdx.x == 0 && threadIdx.x == 0) count_change(c);
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
    if (threadIdx.x == 0) *w.moves = 0, count_change(c);
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
__device__ __forceinline__ void move_page(const ufb_kv_cache& c, const Work& w, int m, int layer, int side) {
    const int head_vecs = c.page_tokens * c.head_dim / 16;
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

template <bool PARTIAL>
__global__ void __launch_bounds__(256) move_kernel(const ufb_kv_cache c) {
    const Work w = work_of(c);
    const int side = blockIdx.y & 1, layer = blockIdx.y >> 1;
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
    for (int m = blockIdx.x; m < moves; m += gridDim.x) move_page<PARTIAL>(c, w, m, layer, side);
}

// ---- reorder: stream i of the list goes on from what stream parent(i) held.
//
// The decision, by one CTA, writes nothing that it reads: which stream keeps its
// parent's last page, which get a copy, and the pages for these -- first those that
// streams without a child leave, so that the pool is looked through only where their
// number does not suffice.  A second launch takes the rows of a group through shared
// memory, a column of all its streams to a thread (a row may be read by several and
// is overwritten itself), and moves the copies' bytes.
//
// Bound by the latency of the two launches, of which the second reads its rows while the
// first decides (4 branches of one stream, 2 layers: 5.5 us on the device, 6.8 one after the
// other); 16 streams x 8 branches, 8 layers of 4 heads of 128, 10.8 us, of which the copies
// (29 MB read and written) would take 4.5 from memory.

// The page of a stream's last, partly filled entry; -1: it has none.
__device__ __forceinline__ int last_page(const ufb_kv_cache& c, int slot, int length) {
    const int full = length / c.page_tokens;
    if (length <= 0 || length % c.page_tokens == 0 || full >= c.table_width) return -1;
    const int page = c.table[static_cast<long long>(slot) * c.table_width + full];
    return page < c.pages ? page : -1;
}

__global__ void __launch_bounds__(kThreads) reorder_kernel(const ufb_kv_cache c, const int32_t* slots,
                                                           const int32_t* parents, int n, int width, int* status) {
    __shared__ int warp_sum[kWarps];
    __shared__ int children[kThreads], first[kThreads], page_of[kThreads], rest_of[kThreads];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const Work w = work_of(c);
    int32_t* last_entry = kv_last_entry(c);
    if (threadIdx.x == 0) w.moves[0] = w.moves[1] = 0;
    // whole groups at a time
    const int tile = kThreads / width * width;
    int need = 0, left = 0, bad = 0;
    for (int base = 0; base < n; base += tile) {
        const int t = threadIdx.x, i = base + t, group = t / width * width;
        const bool mine = t < tile && i < n;
        int parent = t, page = -1, rest = 0;
        children[t] = 0;
        first[t] = kThreads;
        __syncthreads();
        if (mine) {
            const int p = parents[i], slot = slots[i];
            if (p < 0 || p >= width || !valid_slot(c, slot)) {
                bad = 1;
            } else {
                parent = group + p;
                const int length = c.lengths[slot];
                page = last_page(c, slot, length);
                rest = length % c.page_tokens;
                last_entry[i] = page >= 0 ? length / c.page_tokens : -1;
                atomicAdd(children + parent, 1);
                // the parent itself comes before its other children
                atomicMin(first + parent, parent == t ? -1 : t);
            }
        }
        page_of[t] = page;
        rest_of[t] = rest;
        __syncthreads();
        const bool copy = mine && !bad && page_of[parent] >= 0 && first[parent] != (parent == t ? -1 : t);
        const bool leaves = mine && !bad && children[t] == 0 && page >= 0 && c.refs[page] == 1;
        int copies, leavers;
        const int at = need + block_scan(copy, warp_sum, copies), from = left + block_scan(leaves, warp_sum, leavers);
        if (mine) w.start[i] = copy ? at : -1;
        if (copy && at < c.pages) {
            w.source[at] = page_of[parent];
            w.rest[at] = rest_of[parent];
        }
        if (leaves && from < c.pages) w.found[from] = page;
        need += copies;
        left += leavers;
        __syncthreads();
    }
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) atomicCAS(status, 0, kStatusIndex);
        return;
    }
    if (need > left) {
        const int more = need - left;
        if (need > c.pages || find_free(c, more, w.found + left, warp_sum) != more) {
            if (threadIdx.x == 0) atomicCAS(status, 0, kStatusPages);
            return;
        }
    }
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int at = w.start[i];
        if (at < 0) continue;
        const int page = w.found[at];
        // a page that a stream leaves loses that stream's count with its row
        c.refs[page] = at < left ? 2 : 1;
        w.start[i] = page;
    }
    if (threadIdx.x == 0) w.moves[0] = need, w.moves[1] = 1, count_change(c);
}

// Blocks below row_blocks: kColumns columns of one group's rows; the others: copies, by
// (layer, side).
__global__ void __launch_bounds__(kApplyThreads) reorder_apply_kernel(const ufb_kv_cache c, const int32_t* slots,
                                                                      const int32_t* parents, int width, int row_blocks,
                                                                      int chunks) {
    extern __shared__ int rows[];   // [width][kColumns]
    __shared__ int slot[UFB_BEAM_MAX], parent[UFB_BEAM_MAX], page[UFB_BEAM_MAX], entry[UFB_BEAM_MAX];
    __shared__ int children[UFB_BEAM_MAX], length[UFB_BEAM_MAX], refused[UFB_BEAM_MAX];
    const Work w = work_of(c);
    if (blockIdx.x >= row_blocks) {
        wait_for_previous();
        if (w.moves[1] == 0) return;
        const int moves = w.moves[0], parts = c.layers * 2;
        for (long long j = blockIdx.x - row_blocks; j < static_cast<long long>(moves) * parts; j += gridDim.x - row_blocks)
            move_page<true>(c, w, static_cast<int>(j / parts), static_cast<int>(j % parts) >> 1, static_cast<int>(j & 1));
        return;
    }
    const int group = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
    const int i = group * width + threadIdx.x;
    // the decision writes none of this: it is read while that is made
    if (threadIdx.x < width) {
        const int from = slots[i];
        slot[threadIdx.x] = valid_slot(c, from) ? from : 0;   // out of range: the call is refused
        parent[threadIdx.x] = parents[i];
        children[threadIdx.x] = 0;
        if (chunk == 0) {
            length[threadIdx.x] = c.lengths[slot[threadIdx.x]];
            refused[threadIdx.x] = kv_refused(c)[slot[threadIdx.x]];
        }
    }
    __syncthreads();
    // half of the block's threads have the even rows, the other half the odd ones
    const int column = threadIdx.x % kColumns, half = threadIdx.x / kColumns, e = chunk * kColumns + column;
    const bool there = e < c.table_width;
    for (int r = half; there && r < width; r += kApplyThreads / kColumns)
        rows[r * kColumns + column] = c.table[static_cast<long long>(slot[r]) * c.table_width + e];
    wait_for_previous();
    if (w.moves[1] == 0) return;
    if (threadIdx.x < width) {
        page[threadIdx.x] = w.start[i];
        entry[threadIdx.x] = kv_last_entry(c)[i];
        atomicAdd(children + parent[threadIdx.x], 1);
        if (chunk == 0) {
            c.lengths[slot[threadIdx.x]] = length[parent[threadIdx.x]];
            kv_refused(c)[slot[threadIdx.x]] = refused[parent[threadIdx.x]];
        }
    }
    __syncthreads();
    if (!there) return;
    bool same = true;   // one page in all rows: nothing changes, nor does its count
    for (int r = 1; r < width; ++r) same &= rows[r * kColumns + column] == rows[column];
    for (int r = 0; r < width; ++r) same &= entry[r] != e;
    if (same) return;
    for (int r = half; r < width; r += kApplyThreads / kColumns) {
        const int held = rows[r * kColumns + column], p = parent[r];
        // of a last page that is partly filled one child at most goes on with it
        const int more = (entry[r] == e ? min(children[r], 1) : children[r]) - 1;
        if (more != 0 && held >= 0 && held < c.pages) atomicAdd(c.refs + held, more);
        const int now = page[r] >= 0 && entry[p] == e ? page[r] : rows[p * kColumns + column];
        if (now != held) c.table[static_cast<long long>(slot[r]) * c.table_width + e] = now;
    }
}

// What the streams of group blockIdx.x have in common: the leading entries that are equal
// in all their tables, inside of every one's earlier tokens.  Streams that bring no tokens,
// or whose extend was refused, do not count.  Then where each stream's own keys lie among
// the group's, one stream's behind the other's in units of kGroupUnit, and the tokens'
// positions.  Latency of three passes over the streams: 4.2 us for 4 streams of 1769 tokens,
// 5.1 for 8 groups of 8, 8.9 for 64 streams of 65320 (2 a warp, 511 entries each; 14 where
// 32 registers made the loads of a row wait for one another).
__global__ void __launch_bounds__(kThreads, 1) share_kernel(const ufb_kv_cache c, const KvBatch b, const ufb_kv_groups g,
                                                         const KvGroupState out, int* status) {
    __shared__ int warp_sum[kWarps];
    __shared__ int width, lowest, highest, members, chosen;
    __shared__ long long warp_units[kWarps];
    const int group = blockIdx.x, first = max(g.first[group], 0), end = min(g.first[group + 1], b.n);
    // attention over the groups may start; it waits for this launch's end
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int seen = *kv_changes(c) + 1;
    if (threadIdx.x == 0) width = c.table_width, lowest = INT_MAX, highest = -1, members = 0, chosen = INT_MAX;
    __syncthreads();
    // of stream i: its slot, -1 when something is out of range, -2 when it does not count
    int start = 0, count = 0;
    auto look = [&](int i) {
        const int slot = b.slots[i], o0 = b.offsets[i], o1 = b.offsets[i + 1];
        if (!valid_slot(c, slot) || o0 < 0 || o1 < o0 || o1 > b.tokens || o1 - o0 > b.max_new) return -1;
        count = o1 - o0;
        start = c.lengths[slot] - count;
        return kv_refused(c)[slot] != 0 || count == 0 ? -2 : slot;
    };
    for (int i = first + threadIdx.x; i < end; i += kThreads) {
        const int slot = look(i);
        if (slot == -1) {
            atomicCAS(status, 0, kStatusIndex);
        } else if (slot >= 0) {
            atomicAdd(&members, 1);
            atomicMin(&chosen, i);
            atomicMin(&width, max(start, 0) / c.page_tokens);
            atomicMin(&lowest, start);
            atomicMax(&highest, start + count - 1);
        } else if (count > 0) {
            atomicMin(&lowest, -1);
            atomicCAS(status, 0, kStatusPages);
        }
    }
    __syncthreads();
    const int most = width;
    // a warp to a stream: where its table first differs from the chosen one's
    for (int i = first + warp; i < end; i += kWarps) {
        const int slot = look(i);
        if (slot < 0 || members < 2 || i == chosen) continue;
        const int32_t* own = c.table + static_cast<long long>(slot) * c.table_width;
        const int32_t* other = c.table + static_cast<long long>(b.slots[chosen]) * c.table_width;
        for (int e0 = 0; e0 < most; e0 += 256) {
            // all loads before the first comparison
            int a[8], d[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = min(e0 + j * 32 + lane, most - 1);
                a[j] = own[e], d[j] = other[e];
            }
            int differs = INT_MAX;
#pragma unroll
            for (int j = 7; j >= 0; --j)
                if (a[j] != d[j]) differs = min(e0 + j * 32 + lane, most - 1);
            differs = __reduce_min_sync(0xffffffffu, differs);
            if (differs != INT_MAX) {
                if (lane == 0) atomicMin(&width, differs);
                break;
            }
        }
    }
    __syncthreads();
    const int shared = members > 1 ? width * c.page_tokens : 0;
    // tokens from..., `step` apart, of stream i, whose own keys are behind `before` units
    auto seat = [&](int i, int slot, int before, int from, int step) {
        KvGroupState::Token r;
        r.own = before * kGroupUnit;
        r.end = slot >= 0 ? r.own + start + count - shared : r.own;
        r.stream = i;
        const int o0 = b.offsets[i], o1 = min(b.offsets[i + 1], static_cast<int>(min(b.tokens, static_cast<long long>(INT_MAX))));
        for (int t = max(o0, 0) + from; t < o1; t += step) {
            r.position = slot == -1 ? kNotWritten : slot == -2 ? -1 : start + t - o0;
            out.token[t] = r;
        }
    };
    const bool few = b.max_new <= 4;   // tokens of a stream: its thread writes them, else a warp
    int sum = 0;
    long long many = 0;
    for (int i0 = first; i0 < end; i0 += kThreads) {
        const int i = i0 + threadIdx.x, slot = i < end ? look(i) : -1;
        int total;
        const int units = slot >= 0 ? (start + count - shared + kGroupUnit - 1) / kGroupUnit : 0;
        many += units;
        const int before = block_scan(units, warp_sum, total);
        if (i < end) out.units[i] = sum + before + units;
        if (i < end && few) seat(i, slot, sum + before, 0, 1);
        sum += total;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) many += __shfl_xor_sync(0xffffffffu, many, o);
    if (lane == 0) warp_units[warp] = many;
    __syncthreads();
    for (int i = first + warp; !few && i < end; i += kWarps) seat(i, look(i), i > first ? out.units[i - 1] : 0, lane, 32);
    if (warp == 0) {
        many = warp_units[lane];
#pragma unroll
        for (int o = 16; o; o >>= 1) many += __shfl_xor_sync(0xffffffffu, many, o);
    }
    if (threadIdx.x == 0) {
        out.shared[group] = shared;
        const int o0 = g.offsets[group], o1 = g.offsets[group + 1];
        // the tokens are those of the streams: every one of them has its record
        const bool ok = first <= end && o0 == b.offsets[first] && o1 == b.offsets[end] && o0 >= 0 && o1 >= o0 && o1 <= b.tokens &&
                        o1 - o0 <= g.max_tokens && many <= INT_MAX / kGroupUnit - 8;
        if (!ok) atomicCAS(status, 0, kStatusIndex);
        KvGroupState::Group r;
        r.token0 = o0, r.tokens = ok ? o1 - o0 : 0, r.stream0 = first, r.streams = end - first;
        r.shared = shared, r.slot = members ? b.slots[chosen] : 0;
        r.low = lowest == INT_MAX ? -1 : lowest, r.high = highest;
        r.own = sum, r.seen = ok ? seen : ~seen, r.pad[0] = r.pad[1] = 0;
        out.group[group] = r;
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

cudaError_t kv_reorder(const ufb_kv_cache& c, const int32_t* slots, const int32_t* parents, int n, int width,
                       int* status, cudaStream_t s) {
    reorder_kernel<<<1, kThreads, 0, s>>>(c, slots, parents, n, width, status);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const int chunks = (c.table_width + kColumns - 1) / kColumns, row_blocks = n / width * chunks;
    // at most a copy for each stream but one of a group; blocks take further ones in turn
    const long long copies = static_cast<long long>(n - n / width) * c.layers * 2;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(row_blocks + static_cast<unsigned>(copies < 2368 ? copies : 2368));
    config.blockDim = dim3(kApplyThreads);
    config.dynamicSmemBytes = width * kColumns * sizeof(int);
    config.stream = s;
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, reorder_apply_kernel, c, slots, parents, width, row_blocks, chunks);
}

cudaError_t kv_share(const ufb_kv_cache& c, const KvBatch& b, const ufb_kv_groups& g, int* status, cudaStream_t s) {
    share_kernel<<<g.groups, kThreads, 0, s>>>(c, b, g, kv_group_state(g, b.tokens), status);
    return cudaGetLastError();
}

cudaError_t kv_compact(const ufb_kv_cache& c, int*, cudaStream_t s) {
    compact_kernel<<<1, kThreads, 0, s>>>(c);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? move<false>(c, c.pages, s) : e;
}

}  // namespace ufb
