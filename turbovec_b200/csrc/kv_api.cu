// Entry points of the paged key/value cache: argument checks, tensor maps, workspaces, launches.  Nothing is kept between calls but
// what belongs to a device (its number of multiprocessors).
#include <atomic>
#include <cmath>
#include <cstdio>
#include <utility>

#include "kv_cache.cuh"
#include "search.cuh"

namespace tv {
int set_create_error(int code, const char *message);          // index.cu: the message of tv_last_error(NULL)
}

namespace {

using namespace tv;

constexpr int64_t kMaxCount = 1 << 30;                        // tokens, pages, places of a table: 32-bit indices with room

// The caller's current device is put back when the call ends.
struct DeviceScope {
    int before = -1;
    bool ok = false;
    explicit DeviceScope(int device) {
        if (cudaGetDevice(&before) != cudaSuccess) before = -1;
        ok = before == device || cudaSetDevice(device) == cudaSuccess;
        if (before == device) before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
};

int sm_count_of(int device) {
    static std::atomic<int> known[kKvMaxDevices];
    if (device < 0 || device >= kKvMaxDevices) return 0;
    int n = known[device].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) { cudaGetLastError(); return 0; }
        known[device].store(n, std::memory_order_relaxed);
    }
    return n;
}

int refuse(const char *message) { return set_create_error(TV_ERR_INVALID_ARGUMENT, message); }
int unsupported(const char *message) { return set_create_error(TV_ERR_UNSUPPORTED, message); }
int cuda_error(const char *what, cudaError_t e) {
    char text[256];
    cudaGetLastError();                                        // reported here: it does not wait for the caller's next call
    std::snprintf(text, sizeof text, "%s: %s", what, cudaGetErrorString(e));
    return set_create_error(TV_ERR_CUDA, text);
}

bool aligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
bool stride_ok(int64_t s) { return s > 0 && s % 8 == 0 && s < (int64_t(1) << 38); }

int check_common(const tv_kv_cache *c, const tv_kv_batch *b, int64_t tokens, int heads) {
    if (!c || !b) return refuse("the cache and the batch must be given");
    if (c->dtype != TV_KV_BF16 && c->dtype != TV_KV_F16) return unsupported("dtype must be bfloat16 or float16");
    if (c->head_dim != 64 && c->head_dim != 128) return unsupported("head_dim must be 64 or 128");
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return unsupported("page_size must be 16, 32, 64 or 128");
    if (c->kv_heads < 1 || c->kv_heads > 65535) return refuse("kv_heads must be between 1 and 65535");
    if (c->pages < 1 || c->pages > kMaxCount) return refuse("pages must be between 1 and 2^30");
    if (!c->k || !c->v || !aligned(c->k, 16) || !aligned(c->v, 16)) return refuse("k and v must be given and 16-byte aligned");
    if (!stride_ok(c->k_page_stride) || !stride_ok(c->k_head_stride) || !stride_ok(c->k_token_stride) || !stride_ok(c->v_page_stride) ||
        !stride_ok(c->v_head_stride) || !stride_ok(c->v_token_stride))
        return refuse("strides of k and v must be positive multiples of 8 elements");
    if ((c->bounds == nullptr) != (c->scales == nullptr)) return refuse("bounds and scales must be given together");
    if (!aligned(c->bounds, 32) || !aligned(c->scales, 4)) return refuse("bounds must be 32-byte aligned");
    if (b->sequences < 0 || b->sequences > kMaxCount || b->table_width < 0 || b->table_width > kMaxCount || b->table_stride < b->table_width)
        return refuse("sequences and table_width must be at most 2^30, and table_stride at least table_width");
    if (b->sequences > 0 && (!b->lens || !b->offsets || (b->table_width > 0 && !b->table))) return refuse("table, lens and offsets must be given");
    if (!aligned(b->table, 4) || !aligned(b->lens, 4) || !aligned(b->offsets, 4)) return refuse("table, lens and offsets must be 4-byte aligned");
    if (tokens < 0 || tokens > kMaxCount) return refuse("tokens must be between 0 and 2^30");
    if (heads < c->kv_heads || heads % c->kv_heads != 0 || heads > 65535) return refuse("heads must be a positive multiple of kv_heads, at most 65535");
    if (int64_t(tokens) * heads > (int64_t(1) << 31)) return unsupported("tokens * heads must be at most 2^31");
    return TV_OK;
}
int check_rows(const tv_kv_rows *r, const char *message) {
    if (!r || !r->data || !aligned(r->data, 16) || !stride_ok(r->token_stride) || !stride_ok(r->head_stride)) return refuse(message);
    return TV_OK;
}
// Runs of `run` bytes: count[0] times stride[0] apart, each time count[1] of them stride[1] apart, the larger stride first.
struct Runs {
    intptr_t at;
    int64_t count[2], stride[2], run;
};
Runs runs_of(const tv_kv_rows *r, int64_t tokens, int64_t heads, int64_t dim) {
    Runs v{reinterpret_cast<intptr_t>(r->data), {tokens, heads}, {2 * r->token_stride, 2 * r->head_stride}, 2 * dim};
    for (int i = 0; i < 2; ++i)
        if (v.count[i] == 1) v.stride[i] = 0;                  // whatever it says
    if (v.stride[0] < v.stride[1]) { std::swap(v.count[0], v.count[1]); std::swap(v.stride[0], v.stride[1]); }
    return v;
}
Runs bytes_of(const void *p, size_t bytes) { return {reinterpret_cast<intptr_t>(p), {1, 1}, {0, 0}, int64_t(bytes)}; }
// Whether `na` runs sa apart from 0 on and `nb` runs sb apart from `at` on share a byte.
bool meet(int64_t na, int64_t sa, int64_t ra, __int128 at, int64_t nb, int64_t sb, int64_t rb) {
    constexpr int64_t kMost = 1 << 18;
    if (na > kMost || nb > kMost) return true;                 // not worth the time
    for (int64_t i = 0, j = 0; i < na && j < nb;) {
        const __int128 x = __int128(i) * sa, y = at + __int128(j) * sb;
        if (x + ra <= y) ++i;
        else if (y + rb <= x) ++j;
        else return true;
    }
    return false;
}
// Whether two views share a byte.  Views of one buffer that interleave (heads of a fused projection, say) do not; where strides
// have nothing in common and the views lie in the same range, they are taken to.
bool overlap(const Runs &a, const Runs &b) {
    auto extent = [](const Runs &v) { return __int128(v.count[0] - 1) * v.stride[0] + __int128(v.count[1] - 1) * v.stride[1] + v.run; };
    if (a.at + extent(a) <= b.at || b.at + extent(b) <= a.at) return false;
    const int64_t outer = a.stride[0] > b.stride[0] ? a.stride[0] : b.stride[0];
    if (outer == 0) return true;                               // a run each
    // rows `outer` apart, of runs within a row
    struct Rows { int64_t rows, count, stride; bool ok; };
    auto rows_in = [&](const Runs &v) {
        const Rows r = v.stride[0] == outer ? Rows{v.count[0], v.count[1], v.stride[1], true} : Rows{1, v.count[0], v.stride[0], v.count[1] == 1};
        return Rows{r.rows, r.count, r.stride, r.ok && __int128(r.count - 1) * r.stride + v.run <= outer};
    };
    const Rows ra = rows_in(a), rb = rows_in(b);
    if (!ra.ok || !rb.ok) return true;
    int64_t apart = (b.at - a.at) / outer, within = (b.at - a.at) % outer;
    if (within < 0) { within += outer; --apart; }
    // row j of b begins `within` after row j + apart of a, and ends in that or the next
    auto both = [&](int64_t shift) { return shift < ra.rows && shift > -rb.rows; };
    return (both(apart) && meet(ra.count, ra.stride, a.run, within, rb.count, rb.stride, b.run)) ||
           (both(apart + 1) && meet(ra.count, ra.stride, a.run, __int128(within) - outer, rb.count, rb.stride, b.run));
}
KvRows rows_of(const tv_kv_rows *r) { return r ? KvRows{r->data, r->token_stride, r->head_stride} : KvRows{nullptr, 0, 0}; }
KvBatch batch_of(const tv_kv_batch *b) { return {b->table, b->lens, b->offsets, b->table_stride, int(b->table_width), int(b->sequences)}; }
int shift_of(int page_size) { return page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7; }

// Tensor map of four dimensions, channels first (strides of the others in elements); boxes of 64 channels (128 bytes, swizzled) by
// box1 x 1 x box3.
bool make_map(CUtensorMap *map, const tv_kv_cache *c, void *base, const int64_t (&dims)[3], const int64_t (&strides)[3], int box1, int box3) {
    typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                      const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    const EncodeTiledFn enc = reinterpret_cast<EncodeTiledFn>(tensor_map_encoder());
    if (!enc) return false;
    const cuuint64_t d[4] = {cuuint64_t(c->head_dim), cuuint64_t(dims[0]), cuuint64_t(dims[1]), cuuint64_t(dims[2])};
    const cuuint64_t st[3] = {cuuint64_t(2 * strides[0]), cuuint64_t(2 * strides[1]), cuuint64_t(2 * strides[2])};
    const cuuint32_t box[4] = {64, cuuint32_t(box1), 1, cuuint32_t(box3)}, step[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = c->dtype == TV_KV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return enc(map, type, 4, base, d, st, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// (channel, token, key head, page) of K and V
bool make_maps(KvMaps *m, const tv_kv_cache *c, int box_tokens) {
    const int64_t dims[3] = {c->page_size, c->kv_heads, c->pages};
    return make_map(&m->k, c, c->k, dims, {c->k_token_stride, c->k_head_stride, c->k_page_stride}, box_tokens, 1) &&
           make_map(&m->v, c, c->v, dims, {c->v_token_stride, c->v_head_stride, c->v_page_stride}, box_tokens, 1);
}
// (channel, head of the group, key head, token) of Q, whole tokens to a tile of rows
bool make_query_map(KvMaps *m, const tv_kv_cache *c, const tv_kv_rows *q, int64_t tokens, int group, int rows) {
    const int64_t dims[3] = {group, c->kv_heads, tokens};
    return make_map(&m->q, c, q->data, dims, {q->head_stride, group * q->head_stride, q->token_stride}, group, rows / group);
}

// Cuts a workspace into arrays, each on a 256-byte boundary; with a null base it only counts.
struct Carver {
    char *base;
    size_t used = 0;
    template <typename T>
    T *take(int64_t count) {
        T *p = base ? reinterpret_cast<T *>(base + used) : nullptr;
        used += (size_t(count) * sizeof(T) + 255) & ~size_t(255);
        return p;
    }
};
// Whether a prefix goes to the tensor-memory kernel.  The warp-level kernel reads it once for every 16 rows, which costs 3.1 us for a million
// (row, key, key head) triples; the other costs 8 us more to begin with and 0.09 us for a thousand (key, key head) pairs, up to 128
// rows.  They meet where keys * key heads * (rows - 29) is 2.6 million.  Measured (8 key heads of 128 channels, us, warp-level / tensor):
// 32 rows, 16,000 keys 27 / 29; 64 rows 41 / 33; 128 rows, 4,000 keys 31 / 31; 256 rows, 500 keys 29 / 33, 2,000 keys 38 / 36, 8,000
// keys 72 / 42; 64 channels: 64 rows, 8,000 keys 25 / 25, 256 rows, 2,000 keys 27 / 28.
constexpr int64_t kTensorFrom = 2600000;
std::atomic<int64_t> g_tensor_prefix{-1};                 // TV_KV_OPT_TENSOR_PREFIX
void plan_prefix(KvAttendParams &p, const tv_kv_cache *c, int64_t tokens, int heads, int64_t prefix_len, int sm_count) {
    const int group = heads / c->kv_heads;
    const int64_t option = g_tensor_prefix.load(std::memory_order_relaxed);
    const bool worth = option < 0 ? tokens * group > 29 && prefix_len * c->kv_heads > kTensorFrom / (tokens * group - 29) : option > 0;
    p.tensor_prefix = prefix_len > 0 && worth && group <= kKvPrefixRows;     // a tile holds whole tokens
    if (p.tensor_prefix) p.plan = kv_prefix_plan(tokens, group, c->kv_heads, int(prefix_len), sm_count);
}
size_t carve_attend(KvAttendParams &p, char *base, int64_t slots, int64_t rows, const tv_kv_cache *c, bool prefix) {
    Carver w{base};
    const int head_dim = c->head_dim;
    if (p.tensor_prefix) {
        const int64_t blocks = int64_t(c->kv_heads + p.plan.groups) * p.plan.units * 2;
        p.pre_o = w.take<float>(blocks * kKvPrefixRows * head_dim);
        p.pre_ml = w.take<float2>(blocks * kKvPrefixRows);
    }
    p.part_o = w.take<float>(slots * kKvRows * head_dim);
    p.part_ml = w.take<float2>(slots * kKvRows);
    p.own_pieces = w.take<KvPieces>(rows);
    p.prefix_pieces = prefix ? w.take<KvPieces>(rows) : nullptr;
    p.slots = int(slots);
    return w.used;
}
size_t carve_chosen(KvAttendParams &p, KvSelectParams &q, char *base, int64_t slots, int64_t tokens, int64_t rows, int64_t lists, const tv_kv_cache *c) {
    const size_t first = carve_attend(p, base, slots, rows, c, false);
    Carver w{base, first};
    q.chosen_pool = w.take<int32_t>(lists);
    q.token_pos = w.take<int32_t>(tokens);
    return w.used;
}
int64_t attend_slots(const tv_kv_cache *c, const tv_kv_batch *b, int64_t tokens, int heads, bool prefix, int sm_count) {
    return kv_attend_slots(tokens, b->sequences, heads / c->kv_heads, c->kv_heads, prefix, kv_attend_grid(sm_count));
}
int64_t chosen_slots(const tv_kv_cache *c, int64_t tokens, int heads, int sm_count) {
    return kv_chosen_slots(tokens, heads / c->kv_heads, c->kv_heads, kv_attend_grid(sm_count));
}

int fill_attend(KvAttendParams &p, const tv_kv_cache *c, const tv_kv_batch *b, int64_t tokens, int heads, const tv_kv_rows *q, const tv_kv_rows *out, float *lse, float scale) {
    int rc = check_rows(q, "q must be given, 16-byte aligned, with strides that are positive multiples of 8 elements");
    if (rc == TV_OK) rc = check_rows(out, "out must be given, 16-byte aligned, with strides that are positive multiples of 8 elements");
    if (rc != TV_OK) return rc;
    if (overlap(runs_of(q, tokens, heads, c->head_dim), runs_of(out, tokens, heads, c->head_dim))) return refuse("out must not overlap q");
    if (!aligned(lse, 4)) return refuse("lse must be 4-byte aligned");
    if (lse) {
        const Runs sums = bytes_of(lse, size_t(tokens) * heads * 4);
        if (overlap(sums, runs_of(q, tokens, heads, c->head_dim)) || overlap(sums, runs_of(out, tokens, heads, c->head_dim))) return refuse("lse must not overlap q or out");
    }
    if (!(scale > 0.0f) || !std::isfinite(scale)) return refuse("scale must be positive and finite");
    p.batch = batch_of(b);
    p.q = rows_of(q);
    p.out = rows_of(out);
    p.lse = lse;
    p.tokens = int(tokens);
    p.group = heads / c->kv_heads;
    p.kv_heads = c->kv_heads;
    p.heads = heads;
    p.page_shift = shift_of(c->page_size);
    p.pages = int(c->pages);
    p.scale_log2 = scale * 1.4426950408889634f;
    p.item_cost = 4;
    return TV_OK;
}
int check_workspace(const void *ws, size_t have, size_t need) {
    if (!ws || !aligned(ws, 256)) return refuse("the workspace must be given and 256-byte aligned");
    if (have < need) return refuse("the workspace is too small");
    return TV_OK;
}

}  // namespace

extern "C" {

int tv_kv_append(const tv_kv_cache *c, const tv_kv_batch *b, int64_t tokens, int heads, const tv_kv_rows *k_new, const tv_kv_rows *v_new,
                 const tv_kv_rows *q, const tv_kv_rows *q_out, const float *cos, const float *sin, int64_t positions, int rotary, int interleaved,
                 int64_t position_offset, void *stream) {
    int rc = check_common(c, b, tokens, heads);
    if (rc != TV_OK) return rc;
    if (tokens == 0 || b->sequences == 0) return TV_OK;
    rc = check_rows(k_new, "k_new must be given, 16-byte aligned, with strides that are positive multiples of 8 elements");
    if (rc == TV_OK) rc = check_rows(v_new, "v_new must be given, 16-byte aligned, with strides that are positive multiples of 8 elements");
    if (rc == TV_OK && (q != nullptr) != (q_out != nullptr)) rc = refuse("q and q_out must be given together");
    if (rc == TV_OK && q) rc = check_rows(q, "q must be 16-byte aligned, with strides that are positive multiples of 8 elements");
    if (rc == TV_OK && q) rc = check_rows(q_out, "q_out must be 16-byte aligned, with strides that are positive multiples of 8 elements");
    if (rc != TV_OK) return rc;
    if (q) {
        const Runs to = runs_of(q_out, tokens, heads, c->head_dim);
        if (!(q->data == q_out->data && q->token_stride == q_out->token_stride && q->head_stride == q_out->head_stride) && overlap(runs_of(q, tokens, heads, c->head_dim), to))
            return refuse("q_out must be q itself or not overlap it");
        if (overlap(runs_of(k_new, tokens, c->kv_heads, c->head_dim), to) || overlap(runs_of(v_new, tokens, c->kv_heads, c->head_dim), to))
            return refuse("q_out must not overlap k_new or v_new");
    }
    if (rotary < 0 || rotary > c->head_dim || rotary % 16 != 0) return refuse("rotary must be a multiple of 16 up to head_dim");
    if (rotary > 0 && (!cos || !sin || !aligned(cos, 16) || !aligned(sin, 16) || positions < 0 || positions > (int64_t(1) << 40)))
        return refuse("cos and sin must be given and 16-byte aligned, and positions not negative");
    if (position_offset < -(int64_t(1) << 40) || position_offset > (int64_t(1) << 40)) return refuse("position_offset is out of range");
    const int64_t most = tokens / c->page_size + 2 * b->sequences;
    if ((most < tokens ? most : tokens) > INT_MAX) return unsupported("too many pages for one call");
    DeviceScope scope(c->device);
    if (!scope.ok) return cuda_error("no such CUDA device", cudaGetLastError());
    KvAppendParams p{};
    p.batch = batch_of(b);
    p.k_new = rows_of(k_new); p.v_new = rows_of(v_new); p.q = rows_of(q); p.q_out = rows_of(q_out);
    p.k = static_cast<char *>(c->k); p.v = static_cast<char *>(c->v);
    p.k_page = c->k_page_stride; p.k_head = c->k_head_stride; p.k_token = c->k_token_stride;
    p.v_page = c->v_page_stride; p.v_head = c->v_head_stride; p.v_token = c->v_token_stride;
    p.bounds = c->bounds; p.scales = c->scales;
    p.cos = cos; p.sin = sin; p.positions = positions; p.position_offset = position_offset;
    p.pages = c->pages; p.tokens = int(tokens); p.group = heads / c->kv_heads; p.kv_heads = c->kv_heads;
    p.page_shift = shift_of(c->page_size); p.rotary = rotary; p.interleaved = interleaved != 0;
    const cudaError_t e = launch_kv_append(p, c->dtype, c->head_dim, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? int(TV_OK) : cuda_error("append kernel", e);
}

size_t tv_kv_attend_workspace(const tv_kv_cache *c, const tv_kv_batch *b, int64_t tokens, int heads, int64_t prefix_len) {
    if (check_common(c, b, tokens, heads) != TV_OK) return 0;
    if (prefix_len < 0 || prefix_len > kMaxCount) { refuse("prefix_len must be between 0 and 2^30"); return 0; }
    const int sms = sm_count_of(c->device);
    if (sms == 0) { set_create_error(TV_ERR_CUDA, "no such CUDA device"); return 0; }
    KvAttendParams p{};
    plan_prefix(p, c, tokens, heads, prefix_len, sms);
    const bool items = prefix_len > 0 && !p.tensor_prefix;
    return carve_attend(p, nullptr, attend_slots(c, b, tokens, heads, items, sms), tokens * heads, c, items);
}

int tv_kv_attend(const tv_kv_cache *c, const tv_kv_batch *b, int64_t tokens, int heads, const tv_kv_rows *q, const int32_t *prefix_pages,
                 int64_t prefix_width, int64_t prefix_len, float scale, const tv_kv_rows *out, float *lse, void *workspace, size_t workspace_bytes,
                 void *stream) {
    int rc = check_common(c, b, tokens, heads);
    if (rc != TV_OK) return rc;
    if (prefix_len < 0 || prefix_width < 0 || prefix_width > kMaxCount || prefix_len > prefix_width * c->page_size || prefix_len > kMaxCount)
        return refuse("prefix_len must be between 0 and prefix_width pages of tokens, at most 2^30");
    if (prefix_len > 0 && !prefix_pages) return refuse("prefix_pages must be given with prefix_len");
    if (!aligned(prefix_pages, 4)) return refuse("prefix_pages must be 4-byte aligned");
    if (tokens == 0 || b->sequences == 0) return TV_OK;
    KvAttendParams p{};
    rc = fill_attend(p, c, b, tokens, heads, q, out, lse, scale);
    if (rc != TV_OK) return rc;
    const int sms = sm_count_of(c->device);
    if (sms == 0) return set_create_error(TV_ERR_CUDA, "no such CUDA device");
    plan_prefix(p, c, tokens, heads, prefix_len, sms);
    const bool items = prefix_len > 0 && !p.tensor_prefix;
    const int64_t slots = attend_slots(c, b, tokens, heads, items, sms);
    if (slots > INT_MAX) return unsupported("too many rows for one call");
    rc = check_workspace(workspace, workspace_bytes, carve_attend(p, static_cast<char *>(workspace), slots, tokens * heads, c, items));
    if (rc != TV_OK) return rc;
    p.prefix_pages = prefix_pages; p.prefix_len = int(prefix_len); p.prefix_width = int(prefix_width);
    DeviceScope scope(c->device);
    if (!scope.ok) return cuda_error("no such CUDA device", cudaGetLastError());
    p.timeouts = kv_timeouts_symbol(c->device);
    KvMaps maps;
    if (!p.timeouts || !make_maps(&maps, c, c->page_size < kKvTile ? c->page_size : kKvTile)) return set_create_error(TV_ERR_CUDA, "the tensor maps of the cache cannot be made");
    cudaError_t e;
    if (p.tensor_prefix) {
        KvMaps wide;
        if (!make_maps(&wide, c, c->page_size) || !make_query_map(&wide, c, q, tokens, p.group, p.plan.rows)) return set_create_error(TV_ERR_CUDA, "the tensor maps of the cache cannot be made");
        e = launch_kv_prefix(p, wide, c->dtype, c->head_dim, c->device, static_cast<cudaStream_t>(stream));
        if (e != cudaSuccess) return cuda_error("prefix kernel", e);
    }
    e = launch_kv_attend(p, maps, c->dtype, c->head_dim, false, c->device, sms, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? int(TV_OK) : cuda_error("attention kernel", e);
}

size_t tv_kv_attend_selected_workspace(const tv_kv_cache *c, const tv_kv_batch *b, int64_t tokens, int heads, int64_t budget) {
    if (check_common(c, b, tokens, heads) != TV_OK) return 0;
    if (budget < 1 || budget > kKvMaxScored) { refuse("budget must be between 1 and 32,768"); return 0; }
    const int sms = sm_count_of(c->device);
    if (sms == 0) { set_create_error(TV_ERR_CUDA, "no such CUDA device"); return 0; }
    KvAttendParams p{};
    KvSelectParams s{};
    return carve_chosen(p, s, nullptr, chosen_slots(c, tokens, heads, sms), tokens, tokens * heads, tokens * c->kv_heads * budget, c);
}

int tv_kv_attend_selected(const tv_kv_cache *c, const tv_kv_batch *b, int64_t tokens, int heads, const tv_kv_rows *q, int64_t budget, int64_t first,
                          int64_t recent, float scale, const tv_kv_rows *out, float *lse, int32_t *pages_out, void *workspace, size_t workspace_bytes,
                          void *stream) {
    int rc = check_common(c, b, tokens, heads);
    if (rc != TV_OK) return rc;
    if (!c->bounds) return refuse("the cache has no bounds to choose pages by");
    if (budget < 1 || budget > kKvMaxScored || first < 0 || recent < 0 || first > budget || recent > budget - first)
        return refuse("budget must be between 1 and 32,768, and first + recent at most budget");
    if (b->table_width > kKvMaxScored) return unsupported("table_width must be at most 32,768 pages");
    if (tokens == 0 || b->sequences == 0) return TV_OK;
    if (!pages_out || !aligned(pages_out, 4)) return refuse("pages_out must be given and 4-byte aligned");
    KvAttendParams p{};
    KvSelectParams s{};
    rc = fill_attend(p, c, b, tokens, heads, q, out, lse, scale);
    if (rc != TV_OK) return rc;
    const int sms = sm_count_of(c->device);
    if (sms == 0) return set_create_error(TV_ERR_CUDA, "no such CUDA device");
    const int64_t slots = chosen_slots(c, tokens, heads, sms);
    if (slots > INT_MAX) return unsupported("too many rows for one call");
    rc = check_workspace(workspace, workspace_bytes,
                         carve_chosen(p, s, static_cast<char *>(workspace), slots, tokens, tokens * heads, tokens * c->kv_heads * budget, c));
    if (rc != TV_OK) return rc;
    const Runs list = bytes_of(pages_out, size_t(tokens) * c->kv_heads * budget * 4);
    if (overlap(list, runs_of(q, tokens, heads, c->head_dim)) || overlap(list, runs_of(out, tokens, heads, c->head_dim)) ||
        (lse && overlap(list, bytes_of(lse, size_t(tokens) * heads * 4))))
        return refuse("pages_out must not overlap q, out or lse");
    s.batch = p.batch; s.q = p.q; s.bounds = c->bounds; s.scales = c->scales; s.chosen = pages_out;
    s.tokens = p.tokens; s.group = p.group; s.kv_heads = p.kv_heads; s.page_shift = p.page_shift; s.pages = p.pages;
    s.budget = int(budget); s.first = int(first); s.recent = int(recent);
    p.chosen = pages_out; p.chosen_pool = s.chosen_pool; p.token_pos = s.token_pos; p.budget = int(budget);
    DeviceScope scope(c->device);
    if (!scope.ok) return cuda_error("no such CUDA device", cudaGetLastError());
    p.timeouts = kv_timeouts_symbol(c->device);
    KvMaps maps;
    if (!p.timeouts || !make_maps(&maps, c, c->page_size < kKvTile ? c->page_size : kKvTile)) return set_create_error(TV_ERR_CUDA, "the tensor maps of the cache cannot be made");
    cudaError_t e = launch_kv_select(s, c->dtype, c->head_dim, c->device, sms, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_error("selection kernel", e);
    e = launch_kv_attend(p, maps, c->dtype, c->head_dim, true, c->device, sms, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? int(TV_OK) : cuda_error("attention kernel", e);
}

int tv_kv_set_option(int option, int64_t value) {
    if (option != TV_KV_OPT_TENSOR_PREFIX || value < -1 || value > 1) return refuse("no such option, or no such value of it");
    g_tensor_prefix.store(value, std::memory_order_relaxed);
    return TV_OK;
}

int tv_kv_status(int device) {
    if (device < 0 || device >= kKvMaxDevices) return set_create_error(TV_ERR_CUDA, "no such CUDA device");
    DeviceScope scope(device);
    if (!scope.ok) return cuda_error("no such CUDA device", cudaGetLastError());
    uint32_t *flag = kv_timeouts_symbol(device), value = 0;
    cudaError_t e = flag ? cudaDeviceSynchronize() : cudaGetLastError();
    if (flag && e == cudaSuccess) e = cudaMemcpy(&value, flag, 4, cudaMemcpyDeviceToHost);
    if (flag && e == cudaSuccess && value) e = cudaMemset(flag, 0, 4);
    if (!flag || e != cudaSuccess) return cuda_error("reading the state of the cache's kernels", e);
    return value ? set_create_error(TV_ERR_DEVICE_TIMEOUT, "a kernel of the key/value cache gave up a wait") : int(TV_OK);
}

}  // extern "C"
