// Paged key/value cache: what its kernels (kv_append.cu, kv_attend.cu, kv_select.cu) and its entry points (kv_api.cu) share.
//
// A pool holds `pages` pages; a page holds page_size tokens for every key head.  The views K and V are indexed
// [page][key head][token][channel] with any strides (channels adjacent), so that both usual orders of heads and tokens work.
// Row t of a call is token j of sequence b, offsets[b] <= t < offsets[b + 1]; it stands at position
// lens[b] - (offsets[b + 1] - offsets[b]) + j of the sequence's own pages.  All three arrays are device data that the host
// never sees, so every index derived from them is clamped or checked where it is used: page numbers outside the pool hold
// no keys, positions outside the table do not exist.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <climits>
#include <cstdint>
#include <type_traits>

#include "../../include/turbovec_b200.h"
#include "tv_common.cuh"

namespace tv {

constexpr int kKvTile = 64;                  // keys of one step of the warp-level attention
constexpr int kKvRows = 16;                  // query rows (tokens x heads of one key head) of one item: M of mma.sync
constexpr int kKvScaleMin = -24, kKvScaleMax = 40;   // powers of two that the page bounds and the int8 queries may be multiples of

struct KvBatch {
    const int32_t *table, *lens, *offsets;
    int64_t table_stride;
    int table_width, sequences;
};
struct KvRows {                              // [token][head][channel], strides in elements
    void *data;
    int64_t token_stride, head_stride;
};

// Rows of sequence b: [first, first + count).  Offsets that decrease or leave [0, tokens] give empty or shortened sequences.
struct KvSpan {
    int first, count;
};
__host__ __device__ inline KvSpan kv_span(int from, int to, int tokens) {
    const int a = from < 0 ? 0 : (from > tokens ? tokens : from);
    const int z = to < a ? a : (to > tokens ? tokens : to);
    return {a, z - a};
}
__host__ __device__ inline int64_t kv_capacity(int table_width, int page_shift) { return int64_t(table_width) << page_shift; }
// Keys that a token at position `pos` sees among its sequence's own: the positions 0 .. pos that the table covers.
__host__ __device__ inline int kv_visible(int64_t pos, int64_t capacity) {
    const int64_t n = pos + 1 < capacity ? pos + 1 : capacity;
    return n < 0 ? 0 : (n > INT_MAX - 2 * kKvTile ? INT_MAX - 2 * kKvTile : int(n));
}

// Weights of a softmax are 2^(logit - base) in the type, with a running base that is set to kLift below the largest logit and stays until a
// logit is more than kLift + kRescaleAt above it.  bfloat16 has float's range: 2^8 is no matter to it.  float16 ends at 2^-24, with few bits below 2^-14:
// under a base that is the largest logit itself, keys of less than 2^-25 of its weight would count for nothing, however many there are
// of them (as beside a first key that takes most of the weight); times 2^11, and up to 2^15, they have all their bits down to 2^-25 of the largest.
template <typename T> struct KvType;
template <> struct KvType<__nv_bfloat16> {
    static constexpr float kLift = 0.0f, kRescaleAt = 8.0f;
    static __device__ __forceinline__ float2 unpack(uint32_t x) { return {__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)}; }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t d;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
        return d;
    }
    static constexpr uint32_t kExponents = 0x7f807f80u;
};
template <> struct KvType<__half> {
    static constexpr float kLift = 11.0f, kRescaleAt = 4.0f;
    static __device__ __forceinline__ float2 unpack(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2 *>(&x)); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t d;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
        return d;
    }
    static constexpr uint32_t kExponents = 0x7c007c00u;
};

// Smallest e in [kKvScaleMin, kKvScaleMax] with amax <= 127 * 2^e; amax >= 0 (infinite: the largest).
__host__ __device__ inline int kv_exponent(float amax) {
#ifdef __CUDA_ARCH__
    const uint32_t u = __float_as_uint(amax);
#else
    union { float f; uint32_t u; } cvt; cvt.f = amax; const uint32_t u = cvt.u;
#endif
    const int biased = int(u >> 23);
    if (biased < 104) return kKvScaleMin;                     // below 2^-23: far below 127 * 2^-24
    const int e = biased - 127 - 6 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);   // 127 * 2^e = 1.984375 * 2^(e + 6), mantissa 0x7e0000
    return e < kKvScaleMin ? kKvScaleMin : (e > kKvScaleMax ? kKvScaleMax : e);
}
__device__ __forceinline__ float kv_pow2(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }
__device__ __forceinline__ float kv_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Lets a kernel have all of a block's shared memory, once per device: the call costs as much as a launch's arguments.
constexpr int kKvMaxDevices = 64;
template <typename Kernel>
inline cudaError_t kv_allow_shared(Kernel *kern, std::atomic<uint64_t> &done, int device, int static_bytes = 0) {
    const uint64_t bit = uint64_t(1) << device;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    const cudaError_t e = allow_dynamic_shared(kern, static_bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// Launches a kernel that may begin before the one in front of it in the stream has ended.  Every block of every kernel waits
// (griddepcontrol.wait) before it ends, so that what follows a kernel that has ended follows all before it too, and waits before it touches
// memory, with one exception: a kernel may read and write first if the kernel in front of it waits before it lets this one begin
// (griddepcontrol.launch_dependents) and neither touches what the other writes.  The attention behind a prefix kernel does.
template <typename... Params, typename... Args>
inline cudaError_t kv_launch(void (*kern)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t s, const Args &...args) {
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Index of the work unit `at` (block-uniform) of a list in which sequence b has cost(b) units, b ascending: gives b and the
// unit's place within it; b = sequences when the list is shorter.  All threads of the block call this; `scratch` holds one
// int64 per warp and two more.
template <int THREADS, typename Cost>
__device__ __forceinline__ void kv_locate(int64_t at, int sequences, Cost cost, int64_t *scratch, int &b_out, int64_t &place_out) {
    constexpr int kWarps = THREADS / 32;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    __syncthreads();
    if (tid == 0) scratch[kWarps] = -1;
    int64_t base = 0;
    for (int b0 = 0; b0 < sequences; b0 += THREADS) {
        const int b = b0 + tid;
        const int64_t c = b < sequences ? cost(b) : 0;
        int64_t sum = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(kFullMask, sum, o);
            if (lane >= o) sum += up;
        }
        if (lane == 31) scratch[warp] = sum;
        __syncthreads();
        int64_t before = base, total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += scratch[w];
            total += scratch[w];
        }
        const int64_t start = before + sum - c;
        if (at >= start && at < start + c) { scratch[kWarps] = b; scratch[kWarps + 1] = at - start; }
        __syncthreads();
        base += total;
        if (at < base) break;
    }
    __syncthreads();
    const int64_t found = scratch[kWarps];
    b_out = found < 0 ? sequences : int(found);
    place_out = found < 0 ? at - base : scratch[kWarps + 1];
}

struct KvAppendParams {
    KvBatch batch;
    KvRows k_new, v_new, q, q_out;
    char *k, *v;
    int64_t k_page, k_head, k_token, v_page, v_head, v_token;     // elements
    int8_t *bounds;
    float *scales;
    const float *cos, *sin;
    int64_t positions, position_offset, pages;
    int tokens, group, kv_heads, page_shift, rotary, interleaved;
};
cudaError_t launch_kv_append(const KvAppendParams &p, int dtype, int head_dim, cudaStream_t s);

// Keys that an item of the attention reads, as tiles of kKvTile keys; a row of partial results for every part of it that a block
// computes.  The parts of an item lie in consecutive slots (kv_attend.cu).
struct KvPieces {
    int64_t first_row;                       // first slot * kKvRows + the row within the item
    int count, unused;                       // count 0: the row was written where it belongs
};
// Partial results of the tensor-memory form for a prefix (kv_prefix.cu): blocks of 128 rows.
constexpr int kKvPrefixRows = 128;           // M of tcgen05.mma
constexpr int kKvPrefixTile = 128;           // keys of one step
struct KvPrefixPlan {                        // computed alike on host and device
    int rows;                                // rows of a tile: whole tokens
    bool paired;                             // two row tiles to a block, which share its keys; else one, its keys dealt to two streams
    int units;                               // row tiles (or pairs) of a key head
    int tiles;                               // key tiles
    int groups;                              // blocks of one unit: they share the (key head, tile) list
    int64_t places;                          // places of a key head in the list: its tiles, and none behind them
    int64_t per;                             // places of a block
};
inline KvPrefixPlan kv_prefix_plan(int64_t tokens, int group, int kv_heads, int prefix_len, int sm_count) {
    KvPrefixPlan w;
    w.rows = kKvPrefixRows / group * group;
    const int64_t row_tiles = (tokens * group + w.rows - 1) / w.rows;
    w.paired = row_tiles > 1;
    w.units = int(w.paired ? (row_tiles + 1) / 2 : 1);
    w.tiles = (prefix_len + kKvPrefixTile - 1) / kKvPrefixTile;
    int64_t groups = w.units < sm_count ? sm_count / w.units : 1;
    const int64_t steps = int64_t(kv_heads) * w.tiles;
    if (groups > steps) groups = steps;
    w.places = w.tiles;
    w.per = (steps + groups - 1) / groups;
    // A block whose run crosses from one key head to the next has a second part: loading Q, starting and ending cost it about four
    // steps.  If the runs are hardly longer when each lies within a head, they do.
    const int64_t per_head = groups / kv_heads;
    if (per_head > 0) {
        const int64_t within = (w.tiles + per_head - 1) / per_head;
        if (within <= w.per + 4) { w.per = within; w.places = per_head * within; groups = per_head * kv_heads; }
    }
    w.groups = int(groups);
    return w;
}
struct KvAttendParams {
    KvBatch batch;
    KvRows q, out;
    float *lse;                              // [token][head], or null
    const int32_t *prefix_pages;
    int prefix_len, prefix_width;
    int tokens, group, kv_heads, heads, page_shift, pages;
    float scale_log2;                        // scale * log2(e)
    // attention over chosen pages: [token][key head][budget] page numbers of the sequence (ascending, then -1) and of the pool, and
    // the position of every token
    const int32_t *chosen, *chosen_pool;
    const int32_t *token_pos;
    int budget;
    int item_cost;                           // what an item costs beside its tiles, in tiles
    // partial results: unnormalised sums, and (base, sum of weights) in powers of two
    float *part_o;                           // [slot][kKvRows][head_dim]
    float2 *part_ml;                         // [slot][kKvRows]
    KvPieces *own_pieces, *prefix_pieces;    // [token][head]
    int slots;
    uint32_t *timeouts;
    // prefix by the tensor-memory form: its results instead of prefix items
    bool tensor_prefix;
    KvPrefixPlan plan;
    float *pre_o;                            // [key head + group][unit][2][kKvPrefixRows][head_dim]
    float2 *pre_ml;                          // [key head + group][unit][2][kKvPrefixRows]
};
struct KvMaps {
    CUtensorMap k, v;                        // (channel, token, key head, page), boxes of 64 channels
    CUtensorMap q;                           // (channel, head of the group, key head, token); for the prefix kernel alone
};
// Upper bound of the slots that `grid` blocks can use.
inline int64_t kv_attend_slots(int64_t tokens, int64_t sequences, int group, int kv_heads, bool prefix, int grid) {
    const int64_t own = (tokens * group) / kKvRows + (sequences < tokens ? sequences : tokens);
    const int64_t pre = prefix ? (tokens * group + kKvRows - 1) / kKvRows : 0;
    return (own + pre) * kv_heads + grid;
}
inline int64_t kv_chosen_slots(int64_t tokens, int group, int kv_heads, int grid) { return tokens * ((group + kKvRows - 1) / kKvRows) * kv_heads + grid; }
int kv_attend_grid(int sm_count);
cudaError_t launch_kv_attend(const KvAttendParams &p, const KvMaps &maps, int dtype, int head_dim, bool chosen, int device, int sm_count, cudaStream_t s);
// The prefix by tcgen05 (kv_prefix.cu); launched before launch_kv_attend with the same parameters.
cudaError_t launch_kv_prefix(const KvAttendParams &p, const KvMaps &maps, int dtype, int head_dim, int device, cudaStream_t s);
uint32_t *kv_timeouts_symbol(int device);    // address on `device`, which is the current one; null if it cannot be had

constexpr int kKvMaxScored = 32768;          // pages of a sequence whose scores fit a block's shared memory
struct KvSelectParams {
    KvBatch batch;
    KvRows q;
    const int8_t *bounds;
    const float *scales;
    int32_t *chosen, *chosen_pool, *token_pos;
    int tokens, group, kv_heads, page_shift, pages, budget, first, recent;
};
cudaError_t launch_kv_select(const KvSelectParams &p, int dtype, int head_dim, int device, int sm_count, cudaStream_t s);

}  // namespace tv
