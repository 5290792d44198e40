// C ABI of the latent-attention operators (include/uf_b200.h): argument checks,
// then the launchers of rotary.cu, kv_append.cu, kv_pages.cu and kv_attend.cu.
#include "uf_b200.h"

#include "attention.h"
#include "capi_util.h"

#include <climits>
#include <cmath>
#include <cstdint>
#include <string>

using namespace ufb;

namespace {

constexpr int kMostKeys = 1 << 30;  // of a stream

int element_size(int dtype) { return dtype == UFB_F32 ? 4 : 2; }

int done(cudaError_t e, const char* what) { return cuda_ok(e, what) ? UFB_OK : last_code(); }

bool check_heads(const ufb_heads* t, int heads, int head_dim, int dtype, const char* what) {
    const int64_t lanes = 16 / element_size(dtype);
    if (!t || !t->data) return fail(UFB_EINVAL, std::string(what) + " must be non-null");
    if (t->heads <= 0 || (heads > 0 && t->heads != heads))
        return fail(UFB_EINVAL, std::string(what) + " has a wrong number of heads");
    if (reinterpret_cast<uintptr_t>(t->data) % 16 || t->token_stride % lanes || t->head_stride % lanes)
        return fail(UFB_EINVAL, std::string(what) + " must be aligned to 16 bytes, strides included");
    if (t->token_stride < 0 || (t->heads > 1 && t->head_stride < head_dim))
        return fail(UFB_EINVAL, std::string(what) + " has overlapping or negative strides");
    return true;
}

// The heads of one tensor lie in [data, data + span) bytes.
int64_t span_bytes(const ufb_heads& t, int64_t tokens, int head_dim, int dtype) {
    return ((tokens - 1) * t.token_stride + (t.heads - 1) * t.head_stride + head_dim) * element_size(dtype);
}

bool overlap(const ufb_heads& a, const ufb_heads& b, int64_t tokens, int head_dim, int dtype) {
    const auto x = reinterpret_cast<uintptr_t>(a.data), y = reinterpret_cast<uintptr_t>(b.data);
    return x < y + span_bytes(b, tokens, head_dim, dtype) && y < x + span_bytes(a, tokens, head_dim, dtype);
}

// Rows of two heads `apart` elements from one another: whether token t of one and any
// token t + dt of the other share elements (dt 0 left out for a head and itself).
bool rows_meet(int64_t apart, int64_t token_stride, int64_t tokens, int head_dim, bool same) {
    const int64_t most = tokens - 1, at = token_stride > 0 ? -apart / token_stride : 0;
    const int64_t near = at < -most ? -most : at > most ? most : at;
    for (int64_t dt = near - 1; dt <= near + 1; ++dt) {
        const int64_t x = apart + dt * token_stride;
        if (dt >= -most && dt <= most && !(same && dt == 0) && x < head_dim && x > -head_dim) return true;
    }
    return false;
}

// A tensor that is written: its rows share no memory.
bool check_output(const ufb_heads* t, int heads, int64_t tokens, int head_dim, int dtype, const char* what) {
    if (!check_heads(t, heads, head_dim, dtype, what)) return false;
    if (t->token_stride >= (t->heads - 1) * t->head_stride + head_dim) return true;
    for (int h = 0; h < t->heads; ++h)
        if (rows_meet(h * t->head_stride, t->token_stride, tokens, head_dim, h == 0))
            return fail(UFB_EINVAL, std::string(what) + " has heads that overlap");
    return true;
}

// Two tensors that are written: parts of one buffer with one token stride, or apart.
bool check_outputs(const ufb_heads& a, const ufb_heads& b, int64_t tokens, int head_dim, int dtype, const char* what) {
    if (!overlap(a, b, tokens, head_dim, dtype)) return true;
    const int64_t apart = (static_cast<const char*>(b.data) - static_cast<const char*>(a.data)) / element_size(dtype);
    bool meet = tokens > 1 && a.token_stride != b.token_stride;
    for (int h = 0; h < a.heads && !meet; ++h)
        for (int g = 0; g < b.heads && !meet; ++g)
            meet = rows_meet(apart + g * b.head_stride - h * a.head_stride, a.token_stride, tokens, head_dim, false);
    return !meet || fail(UFB_EINVAL, std::string(what) + " overlap");
}

bool check_cache(const ufb_kv_cache* c) {
    if (!c || !c->kv || !c->scale || !c->table || !c->lengths || !c->refs || !c->work)
        return fail(UFB_EINVAL, "cache tensors must be non-null");
    if (c->layers <= 0 || c->pages <= 0 || c->heads <= 0 || c->slots <= 0 || c->table_width <= 0)
        return fail(UFB_EINVAL, "empty cache");
    if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128)
        return fail(UFB_EINVAL, "page_tokens must be 16, 32, 64 or 128");
    if (c->head_dim != 64 && c->head_dim != 128) return fail(UFB_EINVAL, "head_dim must be 64 or 128");
    if (reinterpret_cast<uintptr_t>(c->kv) % 128) return fail(UFB_EINVAL, "cache kv must be 128-byte aligned");
    if (c->layers > 32766 || c->heads > 32767) return fail(UFB_ERANGE, "cache exceeds grid bounds");
    if (static_cast<int64_t>(c->table_width) * c->page_tokens > kMostKeys)
        return fail(UFB_ERANGE, "a stream may hold 2^30 tokens at most");
    return true;
}

bool check_layer(const ufb_kv_cache* c, int layer) {
    if (!check_cache(c)) return false;
    if (layer < 0 || layer >= c->layers) return fail(UFB_EINVAL, "layer out of range");
    return true;
}

bool check_list(const ufb_kv_cache* c, const void* list, int n) {
    if (!check_cache(c)) return false;
    if (n < 0 || n > c->slots) return fail(UFB_EINVAL, "more streams than slots");
    if (n > 0 && !list) return fail(UFB_EINVAL, "slot list is null");
    return true;
}

bool check_batch(const ufb_kv_cache* c, int layer, const int32_t* slots, const int32_t* offsets, int n, int max_new,
                 int64_t tokens) {
    if (!check_layer(c, layer) || !check_list(c, slots, n)) return false;
    if (n > 0 && !offsets) return fail(UFB_EINVAL, "token offsets are null");
    if (tokens < 0 || max_new < 0 || max_new > tokens) return fail(UFB_EINVAL, "invalid token counts");
    if (tokens > INT32_MAX) return fail(UFB_ERANGE, "too many tokens");
    if (n > 65535) return fail(UFB_ERANGE, "too many streams in one call");
    return true;
}

// Groups of the streams of a batch that check_batch has passed.
bool check_groups(const ufb_kv_groups* g, int n, int max_new, int64_t tokens) {
    if (!g || g->groups < 0 || g->groups > n || (n > 0 && g->groups == 0))
        return fail(UFB_EINVAL, "a batch has between one group and one for each stream");
    if (g->groups > 0 && (!g->first || !g->offsets || !g->state)) return fail(UFB_EINVAL, "group tensors must be non-null");
    if (reinterpret_cast<uintptr_t>(g->state) % 16) return fail(UFB_EINVAL, "group state must be 16-byte aligned");
    if (g->max_tokens < max_new || g->max_tokens > tokens) return fail(UFB_EINVAL, "invalid token count of a group");
    return true;
}

}  // namespace

extern "C" {

int64_t ufb_rotary_table(int axes, const int32_t* pairs, const int32_t* extents, const double* bases, float* table) {
    clear_error();
    if (axes < 1 || axes > UFB_ROTARY_MAX_AXES || !pairs || !extents || !bases)
        return err(UFB_EINVAL, "rotary positions have 1 to 4 axes");
    int64_t total = 0;
    for (int a = 0; a < axes; ++a) {
        if (pairs[a] <= 0 || pairs[a] > kRotaryMaxPairs || extents[a] <= 0 || !(bases[a] > 0.0) || std::isinf(bases[a]))
            return err(UFB_EINVAL, "invalid rotary axis");
        total += 2ll * pairs[a] * extents[a];
    }
    if (!table) return total;
    for (int a = 0; a < axes; ++a) {
        for (int64_t p = 0; p < extents[a]; ++p)
            for (int i = 0; i < pairs[a]; ++i) {
                const double angle = static_cast<double>(p) * std::pow(bases[a], -static_cast<double>(i) / pairs[a]);
                *table++ = static_cast<float>(std::cos(angle));
                *table++ = static_cast<float>(std::sin(angle));
            }
    }
    return total;
}

int ufb_rotary(const float* table, int axes, const int32_t* pairs, const int32_t* extents, int layout, int inverse,
               const int32_t* positions, int64_t tokens, int head_dim, int dtype, int count, const ufb_heads* x,
               const ufb_heads* out, void* stream) {
    clear_error();
    if (axes < 1 || axes > UFB_ROTARY_MAX_AXES || !pairs || !extents)
        return err(UFB_EINVAL, "rotary positions have 1 to 4 axes");
    if (dtype != UFB_F32 && dtype != UFB_F16 && dtype != UFB_BF16) return err(UFB_EINVAL, "unsupported dtype");
    if (layout != UFB_ROTARY_HALF && layout != UFB_ROTARY_INTERLEAVED) return err(UFB_EINVAL, "unknown rotary layout");
    if (head_dim < 16 || head_dim > 256 || head_dim % 16)
        return err(UFB_EINVAL, "head_dim must be a multiple of 16 up to 256");
    if (count < 1 || count > 2 || !x || !out) return err(UFB_EINVAL, "rotary takes 1 or 2 tensors");
    if (tokens < 0 || tokens > INT32_MAX) return err(UFB_ERANGE, "invalid token count");
    RotaryArgs a{};
    for (int i = 0; i < axes; ++i) {
        if (pairs[i] <= 0 || extents[i] <= 0) return err(UFB_EINVAL, "invalid rotary axis");
        a.extent[i] = extents[i];
        a.first[i + 1] = a.first[i] + pairs[i];
        if (a.first[i + 1] > head_dim / 2) return err(UFB_EINVAL, "more rotary pairs than the head holds");
        if (i + 1 < UFB_ROTARY_MAX_AXES) a.base[i + 1] = a.base[i] + static_cast<long long>(pairs[i]) * extents[i];
        if (a.base[i] + static_cast<long long>(pairs[i]) * extents[i] > INT32_MAX)
            return err(UFB_ERANGE, "rotary table exceeds indexing bounds");
    }
    a.pairs = a.first[axes];
    if (tokens == 0) return UFB_OK;
    if (!table || !positions) return err(UFB_EINVAL, "rotary table and positions must be non-null");
    for (int i = 0; i < count; ++i) {
        if (!check_heads(x + i, 0, head_dim, dtype, "rotary input") ||
            !check_output(out + i, x[i].heads, tokens, head_dim, dtype, "rotary output"))
            return last_code();
        a.x[i] = x[i];
        a.out[i] = out[i];
    }
    for (int i = 0; i < count; ++i)
        for (int j = 0; j < count; ++j)
            if (overlap(out[i], x[j], tokens, head_dim, dtype))
                return err(UFB_EINVAL, "rotary output must not overlap its input");
    if (count == 2 && !check_outputs(out[0], out[1], tokens, head_dim, dtype, "rotary outputs")) return last_code();
    a.table = reinterpret_cast<const float2*>(table);
    a.positions = positions;
    a.tokens = tokens;
    a.axes = axes;
    a.head_dim = head_dim;
    a.layout = layout;
    a.inverse = inverse != 0;
    a.count = count;
    const int sms = current_sms();
    if (sms <= 0) return last_code();
    int* status = current_status();
    if (!status) return last_code();
    return done(rotary(a, dtype, sms, status, static_cast<cudaStream_t>(stream)), "rotary");
}

int64_t ufb_kv_work_ints(int32_t pages, int32_t slots) {
    clear_error();
    if (pages <= 0 || slots <= 0) return err(UFB_EINVAL, "empty cache");
    return 16 + 3ll * pages + 3ll * slots;
}

int ufb_kv_extend(const ufb_kv_cache* c, const int32_t* slots, const int32_t* offsets, int n, void* stream) {
    clear_error();
    if (!check_list(c, slots, n)) return last_code();
    if (n == 0) return UFB_OK;
    if (!offsets) return err(UFB_EINVAL, "token offsets are null");
    int* status = current_status();
    if (!status) return last_code();
    return done(kv_extend(*c, slots, offsets, n, status, static_cast<cudaStream_t>(stream)), "kv extend");
}

int ufb_kv_release(const ufb_kv_cache* c, const int32_t* slots, int n, void* stream) {
    clear_error();
    if (!check_list(c, slots, n)) return last_code();
    if (n == 0) return UFB_OK;
    int* status = current_status();
    if (!status) return last_code();
    return done(kv_release(*c, slots, n, status, static_cast<cudaStream_t>(stream)), "kv release");
}

int ufb_kv_fork(const ufb_kv_cache* c, const int32_t* src, const int32_t* dst, int n, void* stream) {
    clear_error();
    if (!check_list(c, src, n) || !check_list(c, dst, n)) return last_code();
    if (n == 0) return UFB_OK;
    int* status = current_status();
    if (!status) return last_code();
    return done(kv_fork(*c, src, dst, n, status, static_cast<cudaStream_t>(stream)), "kv fork");
}

int ufb_kv_reorder(const ufb_kv_cache* c, const int32_t* slots, const int32_t* parents, int n, int width,
                   void* stream) {
    clear_error();
    if (!check_list(c, slots, n)) return last_code();
    if (width < 1 || n % width) return err(UFB_EINVAL, "a reorder takes whole groups of streams");
    if (width > UFB_BEAM_MAX) return err(UFB_ERANGE, "at most " + std::to_string(UFB_BEAM_MAX) + " streams to a group");
    if (n == 0) return UFB_OK;
    if (!parents) return err(UFB_EINVAL, "parent list is null");
    if (n / width * ((c->table_width + 127ll) / 128) > (1 << 30)) return err(UFB_ERANGE, "cache exceeds grid bounds");
    int* status = current_status();
    if (!status) return last_code();
    return done(kv_reorder(*c, slots, parents, n, width, status, static_cast<cudaStream_t>(stream)), "kv reorder");
}

int ufb_kv_trim(const ufb_kv_cache* c, const int32_t* slots, int n, int window, int sinks, void* stream) {
    clear_error();
    if (!check_list(c, slots, n)) return last_code();
    if (window < 1 || sinks < 0) return err(UFB_EINVAL, "trim needs a window of at least one key and sinks >= 0");
    if (n == 0) return UFB_OK;
    int* status = current_status();
    if (!status) return last_code();
    return done(kv_trim(*c, slots, n, window, sinks, status, static_cast<cudaStream_t>(stream)), "kv trim");
}

int ufb_kv_compact(const ufb_kv_cache* c, void* stream) {
    clear_error();
    if (!check_cache(c)) return last_code();
    int* status = current_status();
    if (!status) return last_code();
    return done(kv_compact(*c, status, static_cast<cudaStream_t>(stream)), "kv compact");
}

int ufb_kv_append(const ufb_kv_cache* c, int layer, const int32_t* slots, const int32_t* offsets, int n, int max_new,
                  int64_t tokens, int dtype, const ufb_heads* k, const ufb_heads* v, void* stream) {
    clear_error();
    if (!check_batch(c, layer, slots, offsets, n, max_new, tokens)) return last_code();
    if (dtype != UFB_F32 && dtype != UFB_F16 && dtype != UFB_BF16) return err(UFB_EINVAL, "unsupported dtype");
    if (n == 0 || max_new == 0) return UFB_OK;
    if (!check_heads(k, c->heads, c->head_dim, dtype, "keys") || !check_heads(v, c->heads, c->head_dim, dtype, "values"))
        return last_code();
    int* status = current_status();
    if (!status) return last_code();
    const KvBatch b{slots, offsets, n, max_new, tokens};
    return done(kv_append(*c, layer, b, dtype, *k, *v, status, static_cast<cudaStream_t>(stream)), "kv append");
}

int ufb_kv_read(const ufb_kv_cache* c, int layer, const int32_t* pages, int64_t n, int dtype, void* out,
                void* stream) {
    clear_error();
    if (!check_layer(c, layer)) return last_code();
    if (dtype != UFB_F32 && dtype != UFB_F16 && dtype != UFB_BF16) return err(UFB_EINVAL, "unsupported dtype");
    if (n < 0 || n > INT32_MAX / (2ll * c->heads)) return err(UFB_ERANGE, "invalid page count");
    if (n == 0) return UFB_OK;
    if (!pages || !out || reinterpret_cast<uintptr_t>(out) % 16)
        return err(UFB_EINVAL, "page list and 16-byte aligned output required");
    int* status = current_status();
    if (!status) return last_code();
    return done(kv_read(*c, layer, pages, n, dtype, out, status, static_cast<cudaStream_t>(stream)), "kv read");
}

int64_t ufb_kv_attend_workspace(void) {
    clear_error();
    const int sms = current_sms();
    return sms > 0 ? kv_attend_workspace_bytes(sms) : last_code();
}

int64_t ufb_capture_id(void* stream) {
    clear_error();
    cudaStreamCaptureStatus state;
    unsigned long long id = 0;
    if (!cuda_ok(cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &state, &id), "capture info"))
        return last_code();
    return state == cudaStreamCaptureStatusActive ? static_cast<int64_t>(id) : 0;
}

int64_t ufb_kv_group_ints(int groups, int n, int64_t tokens) {
    clear_error();
    if (groups < 0 || n < 0 || tokens < 0 || tokens > INT32_MAX) return err(UFB_EINVAL, "invalid counts");
    return (groups + 3ll) / 4 * 4 + 12ll * groups + n + 4 * tokens;
}

int ufb_kv_share(const ufb_kv_cache* c, const int32_t* slots, const int32_t* offsets, int n, int max_new,
                 int64_t tokens, const ufb_kv_groups* groups, void* stream) {
    clear_error();
    if (!check_batch(c, 0, slots, offsets, n, max_new, tokens) || !check_groups(groups, n, max_new, tokens))
        return last_code();
    if (groups->groups == 0) return UFB_OK;
    int* status = current_status();
    if (!status) return last_code();
    const KvBatch b{slots, offsets, n, max_new, tokens};
    return done(kv_share(*c, b, *groups, status, static_cast<cudaStream_t>(stream)), "kv share");
}

// Checks of ufb_kv_attend and ufb_kv_attend_groups, and the kernels' arguments; nothing
// to do: go is left false.
static bool attend_args(AttendArgs& a, bool& go, int& sms, const ufb_kv_cache* c, int layer, const int32_t* slots,
                        const int32_t* offsets, int n, int max_new, int64_t tokens, int dtype, const ufb_heads* q,
                        const ufb_heads* out, float* lse, int window, int sinks, int causal, float scale,
                        void* workspace, int64_t workspace_bytes) {
    go = false;
    if (!check_batch(c, layer, slots, offsets, n, max_new, tokens)) return false;
    if (dtype != UFB_F16 && dtype != UFB_BF16) return fail(UFB_EINVAL, "attention takes float16 or bfloat16 queries");
    if (window < 0 || sinks < 0) return fail(UFB_EINVAL, "window and sinks must not be negative");
    if (!std::isfinite(scale)) return fail(UFB_EINVAL, "softmax scale must be finite");
    if (n == 0 || max_new == 0) return true;
    if (!check_heads(q, 0, c->head_dim, dtype, "queries") ||
        !check_output(out, q->heads, tokens, c->head_dim, dtype, "attention output"))
        return false;
    if (q->heads % c->heads) return fail(UFB_EINVAL, "query heads must be a multiple of the cache's heads");
    if (q->heads / c->heads > 128) return fail(UFB_ERANGE, "more than 128 query heads to a key head");
    sms = current_sms();
    if (sms <= 0) return false;
    const int64_t need = kv_attend_workspace_bytes(sms);
    if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256)
        return fail(UFB_EINVAL, "attention needs " + std::to_string(need) + " bytes of 256-byte aligned workspace");
    int* status = current_status();
    if (!status) return false;
    const int64_t page_heads = 2ll * c->heads * c->pages;
    a.kv = c->kv + layer * page_heads * c->page_tokens * c->head_dim;
    a.scale = c->scale + layer * page_heads;
    a.table = c->table;
    a.lengths = c->lengths;
    a.refused = kv_refused(*c);
    a.slots = slots;
    a.offsets = offsets;
    a.tokens = tokens;
    a.n = n;
    a.max_new = max_new;
    a.pages = c->pages;
    a.heads = c->heads;
    a.group = q->heads / c->heads;
    a.page_tokens = c->page_tokens;
    a.page_shift = c->page_tokens == 16 ? 4 : c->page_tokens == 32 ? 5 : c->page_tokens == 64 ? 6 : 7;
    a.head_dim = c->head_dim;
    a.slots_total = c->slots;
    a.table_width = c->table_width;
    a.window = window < kMostKeys ? window : kMostKeys;  // positions less the window stay in 32 bits
    a.sinks = sinks;
    a.causal = causal != 0;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.q = *q;
    a.out = *out;
    a.lse = lse;
    a.status = status;
    a.workspace = workspace;
    go = true;
    return true;
}

int ufb_kv_attend(const ufb_kv_cache* c, int layer, const int32_t* slots, const int32_t* offsets, int n, int max_new,
                  int64_t tokens, int dtype, const ufb_heads* q, const ufb_heads* out, float* lse, int window,
                  int sinks, int causal, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    AttendArgs a{};
    bool go;
    int sms;
    if (!attend_args(a, go, sms, c, layer, slots, offsets, n, max_new, tokens, dtype, q, out, lse, window, sinks, causal,
                     scale, workspace, workspace_bytes))
        return last_code();
    if (!go) return UFB_OK;
    return done(kv_attend(a, dtype, sms, static_cast<cudaStream_t>(stream)), "kv attend");
}

int ufb_kv_attend_groups(const ufb_kv_cache* c, int layer, const int32_t* slots, const int32_t* offsets, int n,
                         int max_new, int64_t tokens, int dtype, const ufb_heads* q, const ufb_heads* out, float* lse,
                         int window, int sinks, int causal, float scale, const ufb_kv_groups* groups,
                         void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    AttendArgs a{};
    bool go;
    int sms;
    if (!attend_args(a, go, sms, c, layer, slots, offsets, n, max_new, tokens, dtype, q, out, lse, window, sinks,
                     causal, scale, workspace, workspace_bytes) ||
        !check_groups(groups, n, max_new, tokens))
        return last_code();
    if (!go || groups->groups == 0) return UFB_OK;
    const GroupArgs g{groups->groups, groups->max_tokens, groups->first, groups->offsets, kv_changes(*c),
                      kv_group_state(*groups, tokens)};
    return done(kv_attend_groups(a, g, dtype, sms, static_cast<cudaStream_t>(stream)), "kv attend groups");
}

}  // extern "C"
