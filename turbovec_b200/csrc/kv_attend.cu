// Attention of a few query rows over the keys of a paged cache: a shared prefix, a sequence's own pages, or chosen pages.
//
// An item is up to 16 query rows of one key head (the heads that share it, times the tokens of one sequence; for a prefix the
// rows of all sequences) and the keys they read, in tiles of 64.  All items' tiles are laid end to end and every block takes an equal
// run of them, so that batches of any lengths fill the device evenly: lengths are known on the device alone.  A run that begins or
// ends inside an item leaves partial results, (base of the weights, their sum, weighted sum of values), in slot
// item + block, a number that is different for every pair of the two that meet; a second kernel joins them.
//
// Bound by memory: a tile of 128 channels is 32 KB and 3 * 64 * 128 * 16 multiply-adds (Q K^T, the weights times V, and what rounding the
// weights left times V), most of them padding where rows are few.  One warp
// keeps the ring of tiles full by tensor copies; four warps take 16 keys of each tile: no exchange between warps until the end of a
// part.  What a part costs beside its tiles is weighed as four tiles when the list is divided (2, 3, 4, 5, 6: attend_48_ragged 60.0, 54.2, 54.8,
// 55.4, 55.7 us a call, attend_24_drafts_prefix_8200 57.1, 55.4, 52.8, 53.0, 52.5).  attend_48_ragged, 48 sequences of 1 to 12,000 keys,
// 274 MB: 52.6 us for this kernel, 5.2 TB/s.
#include <cfloat>

#include "kv_cache.cuh"
#include "scan_tc_common.cuh"

namespace tv {
namespace {

constexpr int kConsumers = 4;
constexpr int kAttendThreads = (kConsumers + 1) * 32;
constexpr int kLeastTiles = 2;                           // tiles of a run: joining more parts takes longer than these
constexpr int kNothing = INT_MAX - kKvTile;              // first position of a group of keys that nobody sees

__device__ uint32_t g_kv_timeouts;

template <int D>
struct Geometry {
    static constexpr int kStages = D == 128 ? 2 : 4;      // 64 KB in flight a block, two blocks to a multiprocessor
    static constexpr int kHalfBytes = kKvTile * 128;      // 64 channels of a tile
    static constexpr int kOperandBytes = kHalfBytes * (D / 64);
    static constexpr int kStageBytes = 2 * kOperandBytes;
};
template <int D>
struct AttendShared {
    float o[kConsumers][kKvRows][D + 8];
    uint16_t q[kKvRows][D + 8];                          // rows of Q, a row's banks four words from the one before it
    float2 ml[kConsumers][kKvRows], total[kKvRows];
    int first_key[Geometry<D>::kStages][kConsumers];
    int64_t scratch[2 * (kAttendThreads / 32) + 3];
    uint64_t full[Geometry<D>::kStages], empty[Geometry<D>::kStages];
};

// A run of tiles of one item.  In the list an item is p.item_cost places without tiles, which stand for what an item costs beside them
// (its rows of Q, and joining the warps' results), and then its tiles.
struct Part {
    int item, row0, rows;          // rows of the call's q: (token, head of the group) pairs row0 .. row0 + rows of `first_token` on
    int first_token, h, b;         // b = -1: prefix
    int tile0, tile1, item_tiles;  // tiles of this part, and of the item
    int64_t pos;                   // position of first_token in its sequence
    int64_t item_start;            // place of the item's first tile in the whole list
};

// Quotient of two numbers that are not negative: a 64-bit division costs several times a 32-bit one.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
    return ((a | b) >> 31) == 0 ? int64_t(uint32_t(a) / uint32_t(b)) : a / b;
}

// Walks the parts of a block's run [at, end) of the list.  Order of items: prefix by (key head, rows); then by (sequence, key head,
// rows).  With chosen pages: by (token, key head, rows).
template <bool CHOSEN>
struct Walk {
    const KvAttendParams &p;
    int64_t at, end, prefix_total;
    int live_first, live;           // tokens that belong to a sequence
    int prefix_tiles, prefix_mt;
    int b, item_of_b;               // sequence, its first item
    int64_t start_of_b;

    __device__ __forceinline__ int tiles_of(int len) const {
        const int64_t cap = kv_capacity(p.batch.table_width, p.page_shift);
        const int keys = kv_visible(int64_t(len) - 1, cap);
        return keys < 1 ? 1 : (keys + kKvTile - 1) / kKvTile;        // an item without keys is one empty tile
    }
    __device__ __forceinline__ int row_tiles(int count) const { return int((int64_t(count) * p.group + kKvRows - 1) / kKvRows); }
    __device__ __forceinline__ KvSpan span(int i) const { return kv_span(p.batch.offsets[i], p.batch.offsets[i + 1], p.tokens); }
    __device__ __forceinline__ int64_t items(int i) const { return int64_t(row_tiles(span(i).count)) * p.kv_heads; }

    // the next part; false when the run is over
    __device__ __forceinline__ bool next(Part &out) {
        while (at < end) {
            int64_t begin;                                  // the item's first place
            if constexpr (CHOSEN) {
                const int places = p.item_cost + chosen_tiles(), mt = row_tiles(1);
                const int item = int(divide(at, places));
                const int m = item % mt, th = item / mt;
                begin = int64_t(item) * places;
                out.item = item; out.b = 0; out.item_tiles = chosen_tiles();
                out.h = th % p.kv_heads; out.first_token = live_first + th / p.kv_heads; out.pos = p.token_pos[out.first_token];
                out.row0 = m * kKvRows; out.rows = min(kKvRows, p.group - out.row0);
            } else if (at < prefix_total) {
                const int places = p.item_cost + prefix_tiles, item = int(divide(at, places));
                const int m = item % prefix_mt;
                begin = int64_t(item) * places;
                out.item = item; out.b = -1; out.h = item / prefix_mt; out.first_token = live_first; out.item_tiles = prefix_tiles; out.pos = 0;
                out.row0 = m * kKvRows; out.rows = int(min(int64_t(kKvRows), int64_t(live) * p.group - out.row0));
            } else {
                KvSpan sp = span(b);
                int len = p.batch.lens[b], mt = row_tiles(sp.count), places = p.item_cost + tiles_of(len);
                while (at - start_of_b >= int64_t(mt) * p.kv_heads * places) {
                    if (b + 1 >= p.batch.sequences) return false;
                    start_of_b += int64_t(mt) * p.kv_heads * places;
                    item_of_b += mt * p.kv_heads;
                    ++b;
                    sp = span(b); len = p.batch.lens[b]; mt = row_tiles(sp.count); places = p.item_cost + tiles_of(len);
                }
                const int item = int(divide(at - start_of_b, places));
                const int m = item % mt;
                begin = start_of_b + int64_t(item) * places;
                out.item = item_of_b + item; out.b = b; out.h = item / mt; out.first_token = sp.first; out.item_tiles = places - p.item_cost; out.pos = int64_t(len) - sp.count;
                out.row0 = m * kKvRows; out.rows = int(min(int64_t(kKvRows), int64_t(sp.count) * p.group - out.row0));
            }
            out.item_start = begin + p.item_cost;
            const int64_t stop = min(end, out.item_start + out.item_tiles);
            out.tile0 = int(max(at, out.item_start) - out.item_start);
            out.tile1 = int(stop - out.item_start);
            at = min(end, out.item_start + out.item_tiles);
            if (out.tile1 > out.tile0) return true;         // else the run ended before the item's first tile
        }
        return false;
    }
    __device__ __forceinline__ int chosen_tiles() const { return ((p.budget << p.page_shift) + kKvTile - 1) / kKvTile; }
    // keys that token `j` (of first_token on) of the part sees: those before this position
    __device__ __forceinline__ int limit(const Part &w, int j) const {
        if constexpr (CHOSEN) return int(w.pos) + 1;
        if (w.b < 0) return p.prefix_len;
        return kv_visible(w.pos + j, kv_capacity(p.batch.table_width, p.page_shift));
    }
    // one past the last tile of the part that some row sees a key of
    __device__ __forceinline__ int last_tile(const Part &w) const {
        if constexpr (CHOSEN) {                              // the list is shorter where the sequence has fewer pages
            const int64_t keys = ((w.pos >> p.page_shift) + 1) << p.page_shift;
            return int(min(int64_t(w.tile1), (keys + kKvTile - 1) / kKvTile));
        }
        return min(w.tile1, (limit(w, (w.row0 + w.rows - 1) / p.group) + kKvTile - 1) / kKvTile);
    }
};

// Sets the walk of this block up; `per` = tiles of a run.  All threads.
template <bool CHOSEN>
__device__ __forceinline__ void set_up(Walk<CHOSEN> &w, int64_t *scratch, int64_t &per) {
    const KvAttendParams &p = w.p;
    const KvSpan all = kv_span(p.batch.offsets[0], p.batch.offsets[p.batch.sequences], p.tokens);
    w.live_first = all.first; w.live = all.count;
    int64_t total;
    w.b = w.item_of_b = 0;
    w.start_of_b = 0;
    if constexpr (CHOSEN) {
        w.prefix_total = 0; w.prefix_tiles = w.prefix_mt = 1;
        total = int64_t(w.live) * p.kv_heads * w.row_tiles(1) * (p.item_cost + w.chosen_tiles());
    } else {
        w.prefix_tiles = max(1, (p.prefix_len + kKvTile - 1) / kKvTile);
        w.prefix_mt = max(1, w.row_tiles(w.live));
        w.prefix_total = p.prefix_len > 0 && !p.tensor_prefix && w.live > 0 ? int64_t(w.prefix_mt) * p.kv_heads * (p.item_cost + w.prefix_tiles) : 0;
        w.item_of_b = w.prefix_total > 0 ? w.prefix_mt * p.kv_heads : 0;
        w.start_of_b = w.prefix_total;
    }
    // (cost, items) before this thread's sequence of the run of sequences that begins at b0, and of the whole run
    struct Sums { int64_t cost, items, before_cost, before_items, all_cost, all_items; };
    auto sums = [&](int b0) {
        const int i = b0 + int(threadIdx.x), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        Sums x{};
        if (i < p.batch.sequences) { x.items = w.items(i); x.cost = x.items * (p.item_cost + w.tiles_of(p.batch.lens[i])); }
        int64_t c = x.cost, n = x.items;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t uc = __shfl_up_sync(kFullMask, c, o), un = __shfl_up_sync(kFullMask, n, o);
            if (lane >= o) { c += uc; n += un; }
        }
        __syncthreads();
        if (lane == 31) { scratch[2 * warp] = c; scratch[2 * warp + 1] = n; }
        __syncthreads();
        x.before_cost = c - x.cost; x.before_items = n - x.items;
#pragma unroll
        for (int v = 0; v < kAttendThreads / 32; ++v) {
            if (v < warp) { x.before_cost += scratch[2 * v]; x.before_items += scratch[2 * v + 1]; }
            x.all_cost += scratch[2 * v]; x.all_items += scratch[2 * v + 1];
        }
        return x;
    };
    Sums mine{};
    if constexpr (!CHOSEN) {
        total = w.prefix_total;
        for (int b0 = 0; b0 < p.batch.sequences; b0 += kAttendThreads) {
            mine = sums(b0);
            total += mine.all_cost;
        }
    }
    per = max(int64_t(p.item_cost + kLeastTiles), divide(total + gridDim.x - 1, gridDim.x));
    w.at = min(total, int64_t(blockIdx.x) * per);
    w.end = min(total, w.at + per);
    if constexpr (!CHOSEN) {
        if (w.at < w.end && w.at > w.prefix_total) {             // the sequence that the run begins in
            int64_t *found = scratch + 2 * (kAttendThreads / 32);
            int64_t base_cost = w.prefix_total, base_items = w.item_of_b;
            for (int b0 = 0; b0 < p.batch.sequences; b0 += kAttendThreads) {
                if (p.batch.sequences > kAttendThreads) mine = sums(b0);
                if (w.at < base_cost + mine.all_cost) {
                    const int64_t start = base_cost + mine.before_cost;
                    if (w.at >= start && w.at < start + mine.cost) { found[0] = b0 + int(threadIdx.x); found[1] = start; found[2] = base_items + mine.before_items; }
                    break;
                }
                base_cost += mine.all_cost; base_items += mine.all_items;
            }
            __syncthreads();
            w.b = int(found[0]); w.start_of_b = found[1]; w.item_of_b = int(found[2]);
        }
    }
}

__device__ __forceinline__ void tma_load_page(void *dst, const CUtensorMap *map, int channel, int token, int head, int page, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(channel), "r"(token), "r"(head), "r"(page) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// (a constant offset is part of the instruction)
template <int OFFSET, bool TRANS>
__device__ __forceinline__ void ldmatrix4_at(uint32_t addr, uint32_t (&r)[4]) {
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4 + %5];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr), "n"(OFFSET) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4 + %5];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr), "n"(OFFSET) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory"); }
// a value whose exponent is all ones (infinite or NaN) among the two
template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t x) {
    constexpr uint32_t e = KvType<T>::kExponents;
    return (x & e & 0xffffu) == (e & 0xffffu) || (x & e & 0xffff0000u) == (e & 0xffff0000u);
}

template <typename T, int D, bool CHOSEN>
__global__ void __launch_bounds__(kAttendThreads, 2) kv_attend_kernel(const KvAttendParams p, const __grid_constant__ KvMaps maps) {
    using G = Geometry<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    AttendShared<D> &sh = *reinterpret_cast<AttendShared<D> *>(ring + G::kStages * G::kStageBytes);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == kConsumers * 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.v) : "memory");
    }
    if (tid == 0) {
        for (int s = 0; s < G::kStages; ++s) { mbar_init(&sh.full[s], 1); mbar_init(&sh.empty[s], kConsumers); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // after a prefix kernel nothing that it writes is read here: this one may run beside it, and what was before it had ended
    // when it let this one begin
    if (CHOSEN || !p.tensor_prefix) asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    __syncthreads();
    Walk<CHOSEN> walk{p};
    int64_t per;
    set_up<CHOSEN>(walk, sh.scratch, per);
    // a prefix kernel before this one must have ended when this one has: the join waits for this one alone
    if (walk.at >= walk.end) {
        if (!CHOSEN && p.tensor_prefix) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    Part w;
    uint32_t n = 0;                                     // tiles since the beginning: stage n % kStages, round n / kStages

    if (warp == kConsumers) {                           // ---- the producer
        const int box = min(kKvTile, 1 << p.page_shift), boxes = kKvTile / box;
        bool ok = true;
        while (walk.next(w)) {
            const int last = walk.last_tile(w);
            int chosen_count = p.budget;
            const int32_t *list = nullptr, *pool = nullptr;
            if constexpr (CHOSEN) {
                const int64_t row = (int64_t(w.first_token) * p.kv_heads + w.h) * p.budget;
                list = p.chosen + row; pool = p.chosen_pool + row;
            }
            for (int tile = w.tile0; tile < last; ++tile, ++n) {
                const int s = n % G::kStages;
                const int64_t key = int64_t(tile) * kKvTile + lane * box;
                const int64_t entry = key >> p.page_shift;
                const int token = int(key & ((1 << p.page_shift) - 1));
                int page = -1, first = kNothing;
                if (lane < boxes) {
                    if constexpr (CHOSEN) {
                        const int logical = entry < chosen_count ? list[entry] : -1;
                        if (logical >= 0) { page = pool[entry]; first = (logical << p.page_shift) + token; }
                    } else if (w.b < 0) {
                        if (entry < p.prefix_width) page = __ldg(p.prefix_pages + entry);
                        first = int(key);
                    } else {
                        if (entry < p.batch.table_width) page = __ldg(p.batch.table + int64_t(w.b) * p.batch.table_stride + entry);
                        first = int(key);
                    }
                }
                const bool good = page >= 0 && page < p.pages;
                if (!good) { page = p.pages; first = kNothing; }      // outside the pool: the copy fills with zeros
                if (ok && n >= G::kStages) ok = mbar_wait(&sh.empty[s], ((n / G::kStages) - 1) & 1, p.timeouts);
                ok = __all_sync(kFullMask, ok);
                if (!ok) break;
                const int of_group = __shfl_sync(kFullMask, first, (lane & 3) * 16 / box);
                if (lane < kConsumers) sh.first_key[s][lane] = of_group == kNothing ? kNothing : of_group + ((lane * 16) & (box - 1));
                __syncwarp();
                if (lane == 0) mbar_arrive_expect_tx(&sh.full[s], G::kStageBytes);
                __syncwarp();
                if (lane < boxes) {
                    uint8_t *k = ring + s * G::kStageBytes + lane * box * 128, *v = k + G::kOperandBytes;
#pragma unroll
                    for (int c = 0; c < D / 64; ++c) {
                        tma_load_page(k + c * G::kHalfBytes, &maps.k, c * 64, token, w.h, page, &sh.full[s]);
                        tma_load_page(v + c * G::kHalfBytes, &maps.v, c * 64, token, w.h, page, &sh.full[s]);
                    }
                }
            }
            if (!ok) break;
        }
        if (!ok)                                        // the copies in flight land before the block ends
            for (uint32_t i = n > G::kStages ? n - G::kStages : 0; i < n; ++i) mbar_wait(&sh.full[i % G::kStages], (i / G::kStages) & 1, p.timeouts);
        if (!CHOSEN && p.tensor_prefix) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }

    // ---- the consumers: 16 keys of every tile each
    bool ok = true;
    const int r0 = lane >> 2, r1 = r0 + 8, c2 = (lane & 3) * 2;
    const uint32_t ring_addr = smem_u32(ring);
    // row of this lane's ldmatrix address, and its 16-byte chunk before the swizzle
    const int k_row = warp * 16 + ((lane >> 4) & 1) * 8 + (lane & 7), k_chunk = (lane >> 3) & 1;
    const int v_row = warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), v_chunk = (lane >> 4) & 1;
    // Piece 2 i + chunk of row r lies at place (2 i + chunk) ^ (r & 7) of its 128 bytes: the place of i = 0, of which 2 i flips bits that no other part
    // of the address has.
    const uint32_t k_at = ring_addr + k_row * 128 + ((k_chunk ^ (k_row & 7)) << 4), v_at = ring_addr + G::kOperandBytes + v_row * 128 + ((v_chunk ^ (v_row & 7)) << 4);
    while (walk.next(w)) {
        const int last = walk.last_tile(w);
        uint32_t qf[D / 16][4];
        // Q through shared memory: every warp needs all of it, and eight 16-byte loads are under way where 32 of 4 bytes were
        for (int i = tid; i < kKvRows * (D / 8); i += kConsumers * 32) {
            const int r = i / (D / 8), c = i % (D / 8), row = w.row0 + r, j = row / p.group;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (r < w.rows)
                x = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.q.data) + int64_t(w.first_token + j) * p.q.token_stride +
                                                     int64_t(w.h * p.group + row - j * p.group) * p.q.head_stride + 8 * c);
            *reinterpret_cast<uint4 *>(&sh.q[r][8 * c]) = x;
        }
        const bool have0 = r0 < w.rows, have1 = r1 < w.rows;
        const int j0 = have0 ? (w.row0 + r0) / p.group : 0, j1 = have1 ? (w.row0 + r1) / p.group : 0;       // tokens of the two rows
        consumers_sync();
#pragma unroll
        for (int i = 0; i < D / 16; ++i) ldmatrix4(smem_u32(&sh.q[((lane >> 3) & 1) * 8 + (lane & 7)][16 * i + ((lane >> 4) & 1) * 8]), qf[i]);
        const int lim0 = have0 ? walk.limit(w, j0) : 0, lim1 = have1 ? walk.limit(w, j1) : 0;
        const int lim_first = walk.limit(w, w.row0 / p.group), lim_last = walk.limit(w, (w.row0 + w.rows - 1) / p.group);
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
        float o[D / 8][4];
#pragma unroll
        for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;

        for (int tile = w.tile0; tile < last; ++tile, ++n) {
            const int s = n % G::kStages;
            if (ok) ok = mbar_wait(&sh.full[s], (n / G::kStages) & 1, p.timeouts);
            const uint32_t k_addr = k_at + s * G::kStageBytes, v_addr = v_at + s * G::kStageBytes;
            const int first = sh.first_key[s][warp];
            // all of K's fragments first, so that their loads overlap; two accumulators to a product halve the chain of MMAs
            uint32_t kf[D / 16][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ldmatrix4_at<0, false>(k_addr ^ (i << 5), kf[i]);
                if constexpr (D == 128) ldmatrix4_at<G::kHalfBytes, false>(k_addr ^ (i << 5), kf[i + 4]);
            }
            float sc[2][4] = {}, sd[2][4] = {};
#pragma unroll
            for (int i = 0; i < D / 16; i += 2) {
                mma16816<T>(sc[0], qf[i], kf[i][0], kf[i][1]);
                mma16816<T>(sc[1], qf[i], kf[i][2], kf[i][3]);
                mma16816<T>(sd[0], qf[i + 1], kf[i + 1][0], kf[i + 1][1]);
                mma16816<T>(sd[1], qf[i + 1], kf[i + 1][2], kf[i + 1][3]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) { sc[0][e] += sd[0][e]; sc[1][e] += sd[1][e]; }
            // logits in powers of two; keys that a row does not see count for nothing, whatever they hold
            const bool border = first + 16 > lim_first;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    sc[j][e] *= p.scale_log2;
                    sc[j][2 + e] *= p.scale_log2;
                    if (border) {
                        const int key = first + 8 * j + c2 + e;
                        if (key >= lim0) sc[j][e] = -INFINITY;
                        if (key >= lim1) sc[j][2 + e] = -INFINITY;
                    }
                }
            float t0 = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1])), t1 = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3]));
            t0 = fmaxf(t0, __shfl_xor_sync(kFullMask, t0, 1)); t1 = fmaxf(t1, __shfl_xor_sync(kFullMask, t1, 1));
            t0 = fmaxf(t0, __shfl_xor_sync(kFullMask, t0, 2)); t1 = fmaxf(t1, __shfl_xor_sync(kFullMask, t1, 2));
            // a base (KvType) that logits are not far above stays
            constexpr float kLift = KvType<T>::kLift, kUpTo = kLift + KvType<T>::kRescaleAt;
            if (__any_sync(kFullMask, t0 > m0 + kUpTo || t1 > m1 + kUpTo)) {
                // (for the rows that need it: what the others give must not depend on their neighbours)
                const float n0 = t0 > m0 + kUpTo ? t0 - kLift : m0, n1 = t1 > m1 + kUpTo ? t1 - kLift : m1;
                const float a0 = n0 == m0 ? 1.0f : kv_exp2(m0 - n0), a1 = n1 == m1 ? 1.0f : kv_exp2(m1 - n1);
                m0 = n0; m1 = n1;
                l0 *= a0; l1 *= a1;
#pragma unroll
                for (int j = 0; j < D / 8; ++j) { o[j][0] *= a0; o[j][1] *= a0; o[j][2] *= a1; o[j][3] *= a1; }
            }
            const float s0 = m0 == -INFINITY ? 0.0f : m0, s1 = m1 == -INFINITY ? 0.0f : m1;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    sc[j][e] = kv_exp2(sc[j][e] - s0);
                    sc[j][2 + e] = kv_exp2(sc[j][2 + e] - s1);
                    l0 += sc[j][e];
                    l1 += sc[j][2 + e];
                }
            // Weights for the second product: rounded to the type, and what that leaves rounded to the type as well, so that they are good to
            // twice its bits and the result is rounded once, at the end (relative error against 64 bits with one rounding of the weights 1.35
            // times this one's; attend_48_ragged 54.0 us with it, 55.9 so).
            uint32_t pf[4], pr[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = sc[i >> 1][2 * (i & 1)], y = sc[i >> 1][2 * (i & 1) + 1];
                pf[i] = KvType<T>::pack(x, y);
                const float2 z = KvType<T>::unpack(pf[i]);
                pr[i] = KvType<T>::pack(x - z.x, y - z.y);
            }
            // values of keys that no row sees: zero, for 0 * NaN is not 0
            auto live_mask = [&](int key, int limit) { return (key < limit ? 0xffffu : 0u) | (key + 1 < limit ? 0xffff0000u : 0u); };
            auto values = [&](int i, uint32_t (&vf)[4]) {
                if (i < 4) ldmatrix4_at<0, true>(v_addr ^ ((i & 3) << 5), vf);
                else ldmatrix4_at<G::kHalfBytes, true>(v_addr ^ ((i & 3) << 5), vf);
            };
            auto product = [&](const uint32_t (&a)[4], const uint32_t (&rest)[4], int limit) {
                const bool all = first + 16 <= limit;
                const uint32_t x0 = all ? ~0u : live_mask(first + c2, limit), x1 = all ? ~0u : live_mask(first + 8 + c2, limit);
#pragma unroll
                for (int i0 = 0; i0 < D / 16; i0 += 4) {
                    uint32_t vf[4][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) values(i0 + i, vf[i]);
#pragma unroll
                    for (int i = 0; i < 4 && !all; ++i) { vf[i][0] &= x0; vf[i][1] &= x1; vf[i][2] &= x0; vf[i][3] &= x1; }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        mma16816<T>(o[2 * (i0 + i)], a, vf[i][0], vf[i][1]);
                        mma16816<T>(o[2 * (i0 + i) + 1], a, vf[i][2], vf[i][3]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        mma16816<T>(o[2 * (i0 + i)], rest, vf[i][0], vf[i][1]);
                        mma16816<T>(o[2 * (i0 + i) + 1], rest, vf[i][2], vf[i][3]);
                    }
                }
            };
            bool apart = false;
            if (!CHOSEN && border && lim_first < lim_last && first < lim_last) {
                // keys that some rows see and others do not: an infinite value there must not reach the others
                bool odd = false;
                const uint32_t x0 = live_mask(first + c2, lim_last), x1 = live_mask(first + 8 + c2, lim_last);
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    uint32_t vf[4];
                    values(i, vf);
                    odd |= not_finite<T>(vf[0] & x0) | not_finite<T>(vf[1] & x1) | not_finite<T>(vf[2] & x0) | not_finite<T>(vf[3] & x1);
                }
                apart = __any_sync(kFullMask, odd);
            }
            if (apart) {
                // They are taken out of the tile, this warp's 16 rows of which nobody else reads, and added where they belong: to the rows that
                // see them they give what they are.  (The sums to add wait where the part's result goes later.)
                for (int i = lane; i < kKvRows * (D + 8); i += 32) (&sh.o[warp][0][0])[i] = 0.0f;
                __syncwarp();
#pragma unroll 1
                for (int r = 0; r < 16; ++r) {
                    const int key = first + r;
                    if (key < lim_first || key >= lim_last) continue;
#pragma unroll 1
                    for (int word = lane; word < D / 2; word += 32) {
                        uint32_t *at = reinterpret_cast<uint32_t *>(ring + s * G::kStageBytes + G::kOperandBytes + (word >> 5) * G::kHalfBytes + (warp * 16 + r) * 128 +
                                                                    ((((word >> 2) & 7) ^ (r & 7)) << 4)) + (word & 3);
                        const uint32_t x = *at;
                        if (!not_finite<T>(x)) continue;
                        const bool low = not_finite<T>(x & 0xffffu), high = not_finite<T>(x & 0xffff0000u);
                        const float2 z = KvType<T>::unpack(x);
                        *at = (low ? 0u : x & 0xffffu) | (high ? 0u : x & 0xffff0000u);
                        for (int row = 0; row < w.rows; ++row) {
                            if (key >= walk.limit(w, (w.row0 + row) / p.group)) continue;
                            if (low) sh.o[warp][row][2 * word] += z.x;
                            if (high) sh.o[warp][row][2 * word + 1] += z.y;
                        }
                    }
                    __syncwarp();
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // before the next copy into the tile
            }
            product(pf, pr, lim_last);
            if (apart) {
#pragma unroll
                for (int j = 0; j < D / 8; ++j) {
                    const float2 x = *reinterpret_cast<const float2 *>(&sh.o[warp][r0][8 * j + c2]), y = *reinterpret_cast<const float2 *>(&sh.o[warp][r1][8 * j + c2]);
                    o[j][0] += x.x; o[j][1] += x.y;
                    o[j][2] += y.x; o[j][3] += y.y;
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.empty[s]);
        }

        // ---- the four warps' results together
        l0 += __shfl_xor_sync(kFullMask, l0, 1); l1 += __shfl_xor_sync(kFullMask, l1, 1);
        l0 += __shfl_xor_sync(kFullMask, l0, 2); l1 += __shfl_xor_sync(kFullMask, l1, 2);
        if ((lane & 3) == 0) { sh.ml[warp][r0] = make_float2(m0, l0); sh.ml[warp][r1] = make_float2(m1, l1); }
        consumers_sync();
        float big0 = -INFINITY, big1 = -INFINITY, sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
        for (int i = 0; i < kConsumers; ++i) { big0 = fmaxf(big0, sh.ml[i][r0].x); big1 = fmaxf(big1, sh.ml[i][r1].x); }
        const float base0 = big0 == -INFINITY ? 0.0f : big0, base1 = big1 == -INFINITY ? 0.0f : big1;
#pragma unroll
        for (int i = 0; i < kConsumers; ++i) {
            sum0 = fmaf(kv_exp2(sh.ml[i][r0].x - base0), sh.ml[i][r0].y, sum0);
            sum1 = fmaf(kv_exp2(sh.ml[i][r1].x - base1), sh.ml[i][r1].y, sum1);
        }
        const float f0 = kv_exp2(m0 - base0), f1 = kv_exp2(m1 - base1);
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
            *reinterpret_cast<float2 *>(&sh.o[warp][r0][8 * j + c2]) = make_float2(o[j][0] * f0, o[j][1] * f0);
            if (w.rows > 8) *reinterpret_cast<float2 *>(&sh.o[warp][r1][8 * j + c2]) = make_float2(o[j][2] * f1, o[j][3] * f1);
        }
        // the sums for the rows, where a lane that writes a row's result finds them
        if (warp == 0 && (lane & 3) == 0) { sh.total[r0] = make_float2(big0, sum0); sh.total[r1] = make_float2(big1, sum1); }
        consumers_sync();
        // row after row: a warp every fourth, a lane D / 32 channels
        const bool whole = w.tile0 == 0 && w.tile1 == w.item_tiles && p.prefix_len == 0;
        const int64_t slot = int64_t(w.item) + blockIdx.x;
        for (int r = warp; r < w.rows; r += kConsumers) {
            constexpr int kPer = D / 32;
            float x[kPer] = {};
#pragma unroll
            for (int i = 0; i < kConsumers; ++i) {
                const float *src = &sh.o[i][r][lane * kPer];
                if constexpr (kPer == 4) { const float4 y = *reinterpret_cast<const float4 *>(src); x[0] += y.x; x[1] += y.y; x[2] += y.z; x[3] += y.w; }
                else { const float2 y = *reinterpret_cast<const float2 *>(src); x[0] += y.x; x[1] += y.y; }
            }
            const float2 total = sh.total[r];
            const int row = w.row0 + r, j = row / p.group;
            const int64_t token = w.first_token + j, head = w.h * p.group + row - j * p.group;
            if (whole) {
                const bool any = total.y > 0.0f || total.y != total.y;
                const float inv = any ? 1.0f / total.y : 0.0f;             // no key: zero
                uint32_t *dst = reinterpret_cast<uint32_t *>(static_cast<T *>(p.out.data) + token * p.out.token_stride + head * p.out.head_stride + lane * kPer);
#pragma unroll
                for (int i = 0; i < kPer / 2; ++i) dst[i] = KvType<T>::pack(x[2 * i] * inv, x[2 * i + 1] * inv);
                if (lane == 0 && p.lse) p.lse[token * p.heads + head] = any ? (total.x + log2f(total.y)) * 0.6931471805599453f : -INFINITY;
            } else if (uint64_t(slot) < uint64_t(p.slots)) {               // (offsets that do not ascend can give more items than there are slots)
                float *dst = p.part_o + (slot * kKvRows + r) * D + lane * kPer;
                if constexpr (kPer == 4) *reinterpret_cast<float4 *>(dst) = make_float4(x[0], x[1], x[2], x[3]);
                else *reinterpret_cast<float2 *>(dst) = make_float2(x[0], x[1]);
                if (lane == 0) p.part_ml[slot * kKvRows + r] = total;
            }
            if (lane == 0 && w.tile0 == 0) {                               // where the parts of the item lie
                const int64_t begin = divide(w.item_start, per), finish_at = divide(w.item_start + w.item_tiles - 1, per);
                const KvPieces pc{(w.item + begin) * kKvRows + r, whole ? 0 : int(finish_at - begin + 1), 0};
                (w.b < 0 ? p.prefix_pieces : p.own_pieces)[token * p.heads + head] = pc;
            }
        }
    }
    if (!CHOSEN && p.tensor_prefix) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Joins the parts of a row (token, head): WARPS warps each take every WARPS-th part.
template <typename T, int D, int WARPS>
__global__ void __launch_bounds__(128) kv_join_kernel(const KvAttendParams p) {
    constexpr int kPer = D / 32;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    __shared__ float4 others[WARPS > 1 ? WARPS - 1 : 1][32];
    __shared__ float2 others_ml[WARPS > 1 ? WARPS - 1 : 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, turn = warp % WARPS;
    const int64_t row = int64_t(blockIdx.x) * (4 / WARPS) + warp / WARPS;
    const int token = int(row / p.heads), head = int(row % p.heads);
    const KvSpan all = kv_span(p.batch.offsets[0], p.batch.offsets[p.batch.sequences], p.tokens);
    if (token < all.first || token >= all.first + all.count) return;       // behind the last sequence: as it was
    const KvPieces own = p.own_pieces[row];
    if (own.count == 0 && p.prefix_len == 0) return;
    // Two lists of parts, n1 of a prefix and n2 of the row's own keys: sums o at step floats, (base, sum of weights) at step / D.
    const float *o1 = nullptr, *o2 = nullptr;
    const float2 *ml1 = nullptr, *ml2 = nullptr;
    int64_t step1 = 0;
    int n1 = 0, n2 = 0;
    auto of_items = [&](const KvPieces &pc, const float *&o, const float2 *&ml) {
        if (pc.first_row < 0 || pc.count < 0 || pc.first_row / kKvRows + pc.count > p.slots) return 0;
        o = p.part_o + pc.first_row * D;
        ml = p.part_ml + pc.first_row;
        return pc.count;
    };
    if (p.tensor_prefix) {
        const int h = head / p.group;                // rows of a key head lie together, token after token
        const int64_t r = int64_t(token - all.first) * p.group + head - h * p.group;
        const KvPrefixPlan &w = p.plan;
        const int first = int(divide(h * w.places, w.per)), count = int(divide(h * w.places + w.tiles - 1, w.per)) - first + 1;
        const int tile = w.paired ? int(uint32_t(r) / uint32_t(w.rows)) : 0, in_tile = int(r) - tile * w.rows;     // r < 2^31: tokens * heads are
        const int64_t at = ((int64_t(h) + first) * w.units * 2 + tile) * kKvPrefixRows + in_tile;
        o1 = p.pre_o + at * D;
        ml1 = p.pre_ml + at;
        step1 = (w.paired ? 2 * int64_t(w.units) : 1) * kKvPrefixRows * D;       // not paired: both streams of a block, one after the other
        n1 = w.paired ? count : 2 * count;
    } else if (p.prefix_len > 0) {
        step1 = int64_t(kKvRows) * D;
        n1 = of_items(p.prefix_pieces[row], o1, ml1);
    }
    n2 = of_items(own, o2, ml2);
    constexpr int64_t kStep2 = int64_t(kKvRows) * D;
    float big = -INFINITY, sum = 0.0f, acc[kPer] = {};
    const int n = (n1 + n2 - turn + WARPS - 1) / WARPS;                         // parts turn, turn + WARPS, ... are this warp's
    for (int k0 = 0; k0 < n; k0 += 32) {
        const int left = min(32, n - k0), mine_at = turn + (k0 + lane) * WARPS;
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (lane < left) ml = mine_at < n1 ? ml1[mine_at * (step1 / D)] : ml2[(mine_at - n1) * (kStep2 / D)];
        float top = ml.x;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, d));
        const float next = fmaxf(big, top), base = next == -INFINITY ? 0.0f : next;
        const float old = kv_exp2(big - base), mine = kv_exp2(ml.x - base);
        float part = mine * ml.y;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) part += __shfl_xor_sync(kFullMask, part, d);
        sum = fmaf(sum, old, part);
        big = next;
#pragma unroll
        for (int j = 0; j < kPer; ++j) acc[j] *= old;
#pragma unroll 8
        for (int k = 0; k < left; ++k) {
            const float f = __shfl_sync(kFullMask, mine, k);
            const int i = turn + (k0 + k) * WARPS;
            const float *src = (i < n1 ? o1 + i * step1 : o2 + (i - n1) * kStep2) + lane * kPer;
            float x[kPer] = {};
            if (f != 0.0f) {                         // a part without keys may have no sums
                if constexpr (kPer == 4) { const float4 y = *reinterpret_cast<const float4 *>(src); x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w; }
                else { const float2 y = *reinterpret_cast<const float2 *>(src); x[0] = y.x; x[1] = y.y; }
            }
#pragma unroll
            for (int j = 0; j < kPer; ++j) acc[j] = fmaf(f, x[j], acc[j]);
        }
    }
    if constexpr (WARPS > 1) {
        static_assert(WARPS == 4, "a block is one row");
        if (turn > 0) {
            float4 y = make_float4(acc[0], acc[1], 0.0f, 0.0f);
            if constexpr (kPer == 4) { y.z = acc[2]; y.w = acc[3]; }
            others[turn - 1][lane] = y;
            if (lane == 0) others_ml[turn - 1] = make_float2(big, sum);
        }
        __syncthreads();
        if (turn > 0) return;
#pragma unroll
        for (int i = 0; i < WARPS - 1; ++i) {
            const float2 ml = others_ml[i];
            const float4 y = others[i][lane];
            const float next = fmaxf(big, ml.x), base = next == -INFINITY ? 0.0f : next;
            const float old = kv_exp2(big - base), f = kv_exp2(ml.x - base);
            const float x[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int j = 0; j < kPer; ++j) acc[j] = fmaf(f, x[j], acc[j] * old);
            sum = fmaf(f, ml.y, sum * old);
            big = next;
        }
    }
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    uint32_t *dst = reinterpret_cast<uint32_t *>(static_cast<T *>(p.out.data) + token * p.out.token_stride + head * p.out.head_stride + lane * kPer);
#pragma unroll
    for (int j = 0; j < kPer / 2; ++j) dst[j] = KvType<T>::pack(acc[2 * j] * inv, acc[2 * j + 1] * inv);
    if (lane == 0 && p.lse) p.lse[row] = sum > 0.0f || sum != sum ? (big + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

template <typename T, int D, bool CHOSEN>
cudaError_t launch(const KvAttendParams &p, const KvMaps &maps, int device, int sm_count, cudaStream_t s) {
    using G = Geometry<D>;
    const size_t smem = size_t(G::kStages) * G::kStageBytes + sizeof(AttendShared<D>) + 1024;
    auto *kern = kv_attend_kernel<T, D, CHOSEN>;
    static std::atomic<uint64_t> allowed{0};
    cudaError_t e = kv_allow_shared(kern, allowed, device);
    if (e != cudaSuccess) return e;
    e = kv_launch(kern, dim3(unsigned(kv_attend_grid(sm_count))), kAttendThreads, smem, s, p, maps);
    if (e != cudaSuccess) return e;
    // Four warps to a row where rows are few and have many parts each (attend_48_ragged, 1,536 rows: 54.5 us a call with four, 56.0 with one;
    // attend_128_prefix_32768, 8,192 rows: 201.4 and 194.7).
    const int64_t rows = int64_t(p.tokens) * p.heads;
    if (rows <= 16 * sm_count) return kv_launch(kv_join_kernel<T, D, 4>, dim3(unsigned(rows)), 128, 0, s, p);
    return kv_launch(kv_join_kernel<T, D, 1>, dim3(unsigned((rows + 3) / 4)), 128, 0, s, p);
}

}  // namespace

int kv_attend_grid(int sm_count) { return 2 * sm_count; }

uint32_t *kv_timeouts_symbol(int device) {
    static std::atomic<void *> known[kKvMaxDevices];
    void *ptr = known[device].load(std::memory_order_relaxed);
    if (ptr == nullptr && cudaGetSymbolAddress(&ptr, g_kv_timeouts) == cudaSuccess) known[device].store(ptr, std::memory_order_relaxed);
    return static_cast<uint32_t *>(ptr);
}

cudaError_t launch_kv_attend(const KvAttendParams &p, const KvMaps &maps, int dtype, int head_dim, bool chosen, int device, int sm_count, cudaStream_t s) {
    if (p.tokens == 0 || p.batch.sequences == 0) return cudaSuccess;
    auto go = [&](auto t, auto d) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        return chosen ? launch<T, D, true>(p, maps, device, sm_count, s) : launch<T, D, false>(p, maps, device, sm_count, s);
    };
    using D64 = std::integral_constant<int, 64>;
    using D128 = std::integral_constant<int, 128>;
    if (dtype == TV_KV_BF16) return head_dim == 128 ? go(__nv_bfloat16(), D128()) : go(__nv_bfloat16(), D64());
    return head_dim == 128 ? go(__half(), D128()) : go(__half(), D64());
}

}  // namespace tv
