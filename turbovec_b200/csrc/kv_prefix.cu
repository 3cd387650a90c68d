// Attention of many query rows over a shared prefix, on the tensor cores (tcgen05, accumulators in tensor memory).
//
// All rows of a batch (tokens x heads of a key head) see all keys of the prefix, so the prefix is read once for 256 rows instead of
// once for every sequence.  S = Q K^T and O += P V are MMAs of 128 rows; four warps turn S into P, a row to a thread: running
// base, weights in powers of two, their sum.  O is rescaled only when a row's logits go well above the base (KvType in kv_cache.cuh).  P
// replaces S in tensor memory and is the A operand of the second MMA.
//
// Weights are rounded to the type once, half a step each, while their sum keeps what is rounded off: with the result's own rounding
// the relative error is 1.4 times that of the latter alone (attend_24_drafts_prefix_8200 and attend_128_prefix_32768 against 64 bits: 2.3e-3,
// with one rounding 1.66e-3).  Carrying the rest of each weight along, as kv_attend.cu does, would be half
// as many MMAs again and twice the stores of P where both are what bounds the kernel.
//
// Two streams keep the tensor cores and the other units busy at once.  With more than one tile of rows the streams are two such tiles
// that share each tile of keys and values; else they are one tile of rows over every other tile of keys.  A stream's S has two
// halves of 64 keys: while the weights of one are computed, P of the other goes through its MMAs and becomes the next logits.
// 128 channels: 256 columns of S and 256 of O fill tensor memory.
//
// Blocks of one unit of rows share the list of (key head, tile) steps evenly; the units of one group of blocks go over the same keys at
// the same time, so that the second and later ones find them in L2.
//
// What bounds it is the weights.  A step (256 rows x 128 keys x 128 channels) is 2,048 cycles of MMAs (2,480 measured: halves of S
// are MMAs of N = 64, which shared memory feeds in 48 cycles and not in 32), and it takes 3,700 (211,000 cycles for 56 steps, beginning and
// end included); when it took 3,800, 3,630 with the MMAs left out and 2,500 with the weights left out.  1,536 cycles of it are the
// exponential unit (8 cycles an instruction; a quarter of the weights go by the multiply-add pipe, 0, 1/8 and 3/8 are 5, 1 and 1 %
// slower), 960 multiply-adds, 770 maxima and conversions, per scheduler, and two warps do not overlap them well.  Tried and slower: tiles of
// 128 keys without halves (3,650 a step, but 8,000 cycles more around the loop), two threads to a row on 16 warps (4,600), one warp for
// all MMAs with halves (4,300).
// attend_128_prefix_32768 (1,024 rows of 8 key heads, 32,768 keys, 137 GFLOP): 129 us from the end of
// the kernel before it to its own end, in a row of calls: 1.06 PFLOP/s.
#include "kv_cache.cuh"
#include "scan_tc_common.cuh"

namespace tv {
namespace {

constexpr int kPrefixThreads = 12 * 32;          // 2 x 4 warps of weights, two of MMAs, one of copies, one that completes the group
constexpr int kWeightRegs = 184, kOtherRegs = 136;   // registers a thread: 256 * 184 + 128 * 136 = 384 * 168, what the block starts with
static_assert(256 * kWeightRegs + 128 * kOtherRegs <= kPrefixThreads * 168, "more registers than the block has");
constexpr int kMmaWarp = 8, kCopyWarp = 10;      // MMAs of stream s: warp kMmaWarp + s
constexpr int kHalfKeys = kKvPrefixTile / 2;
constexpr int kByPolynomial = 2;                 // pairs of weights of every eight

template <int D>
struct PrefixGeometry {
    static constexpr int kHalfBytes = 128 * 128;                 // 128 rows of 64 channels
    static constexpr int kTileBytes = kHalfBytes * (D / 64);
    static constexpr int kSlots = D == 128 ? 5 : 8;              // tiles of keys or values in the ring
    static constexpr int kQBytes = 2 * kTileBytes;
    static constexpr int kOColumns = D;
};
template <int D>
struct alignas(16) PrefixShared {
    uint64_t full[2][PrefixGeometry<D>::kSlots], empty[PrefixGeometry<D>::kSlots];     // [stream; 0 where both use a tile][slot]
    uint64_t s_full[2][2], p_ready[2][2], o_done[2], q_full[2], q_free[2];    // [stream][half of a tile], [stream]
    uint32_t tmem_base;
};

__device__ __forceinline__ void tma_load_page(void *dst, const CUtensorMap *map, int channel, int token, int head, int page, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(channel), "r"(token), "r"(head), "r"(page) : "memory");
}
// 128-byte swizzle, channels (values) or keys... of a row adjacent: the MMA's other dimension is the one that is adjacent in
// memory.  64 adjacent elements by 8 rows are 1,024 bytes; further rows 1,024 apart, further 64 elements `next` bytes apart.
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t next) {
    return umma_desc(addr) & ~(uint64_t(0x3fff) << 16) | uint64_t(next >> 4) << 16;
}
template <typename T>
constexpr uint32_t idesc(int n, bool b_adjacent) {
    return (1u << 4) | (std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u) | (b_adjacent ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (128u >> 4 << 24);
}
// MMAs and commits are executed by the whole warp and issued by its elected lane: no branch, so that descriptors and addresses, which are
// the same in all lanes, stay in uniform registers.  (With a branch around them an MMA took 100 cycles to issue, 64 to execute.)
__device__ __forceinline__ uint32_t elected() {
    uint32_t x;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(x));
    return x;
}
template <bool ACCUMULATE>
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t id) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 q, %4, 0;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(leader), "n"(ACCUMULATE ? 1 : 0) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 q, %4, 0;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(leader), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void commit(uint32_t leader, uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
        ::"r"(smem_u32(bar)), "r"(leader) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
          "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
          "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr) : "memory");
}
// two at a time: twice the rate of the single form
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float2 unpair(uint64_t x) {
    float2 y;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(x));
    return y;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// Largest of three, NaN if one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// 2^y for a pair, -126 <= y < 127, on the multiply-add pipe: y = n + f with n whole and |f| <= 1/2 (adding 1.5 * 2^23 leaves n in the low
// bits), 2^f by a polynomial of degree 4 (fitted to the smallest largest relative error: 2.7e-6, a hundredth of what rounding
// the weight to 11 bits leaves), n added to the exponent.
__device__ __forceinline__ float2 exp2_pair(float2 y) {
    constexpr float kShift = 12582912.0f;
    const uint64_t v = pair(fmaxf(y.x, -126.0f), fmaxf(y.y, -126.0f));
    const uint64_t t = add2(v, pair(kShift, kShift)), n = add2(t, pair(-kShift, -kShift)), f = fma2(n, pair(-1.0f, -1.0f), v);
    uint64_t r = pair(0x1.3997d4p-7f, 0x1.3997d4p-7f);
    r = fma2(r, f, pair(0x1.ca1440p-5f, 0x1.ca1440p-5f));
    r = fma2(r, f, pair(0x1.ec06dap-3f, 0x1.ec06dap-3f));
    r = fma2(r, f, pair(0x1.62e0dcp-1f, 0x1.62e0dcp-1f));
    r = fma2(r, f, pair(0x1.ffffe8p-1f, 0x1.ffffe8p-1f));
    const float2 a = unpair(r), k = unpair(t);
    return make_float2(__uint_as_float(__float_as_uint(a.x) + (__float_as_uint(k.x) << 23)), __uint_as_float(__float_as_uint(a.y) + (__float_as_uint(k.y) << 23)));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_shared_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// a block's steps [at, end) of the (key head, tile) list, a part per key head
struct PrefixPart {
    int h, tile0, count;
};
__device__ __forceinline__ bool next_part(const KvPrefixPlan &plan, int64_t &at, int64_t end, PrefixPart &w) {
    while (at < end) {
        w.h = int(at / plan.places);
        const int64_t begin = int64_t(w.h) * plan.places, stop = min(end, begin + plan.tiles);
        w.tile0 = int(at - begin);
        w.count = int(stop - at);
        at = min(end, begin + plan.places);
        if (w.count > 0) return true;
    }
    return false;
}

template <typename T, int D>
__global__ void __launch_bounds__(kPrefixThreads, 1) kv_prefix_kernel(const KvAttendParams p, const __grid_constant__ KvMaps maps) {
    using G = PrefixGeometry<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *q_smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *ring = q_smem + G::kQBytes;
    PrefixShared<D> &sh = *reinterpret_cast<PrefixShared<D> *>(ring + G::kSlots * G::kTileBytes);
    // the warp's number and the tensor-memory address come from lane 0, so that the compiler knows them to be the same in all lanes and keeps
    // what follows from them (branches, descriptors) in uniform registers
    const int tid = threadIdx.x, warp = __shfl_sync(kFullMask, tid >> 5, 0), lane = tid & 31;
    const KvPrefixPlan plan = p.plan;
    const int unit = blockIdx.x % plan.units, group = blockIdx.x / plan.units;
    if (tid == 0) {
        for (int s = 0; s < G::kSlots; ++s) { mbar_init(&sh.full[0][s], 1); mbar_init(&sh.full[1][s], 1); mbar_init(&sh.empty[s], plan.paired ? 2 : 1); }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&sh.o_done[s], 1);
            mbar_init(&sh.q_full[s], 1); mbar_init(&sh.q_free[s], 10);
            for (int b = 0; b < 2; ++b) { mbar_init(&sh.s_full[s][b], 1); mbar_init(&sh.p_ready[s][b], 4); }
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // rows of a tile that no copy writes
    for (int i = tid; i < 2 * (D / 64) * (kKvPrefixRows - plan.rows) * 8; i += kPrefixThreads) {
        const int half = i / ((kKvPrefixRows - plan.rows) * 8), rest = i % ((kKvPrefixRows - plan.rows) * 8);
        *reinterpret_cast<uint4 *>(q_smem + half * G::kHalfBytes + plan.rows * 128 + rest * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_shared_async();
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(kFullMask, sh.tmem_base, 0);
    // the attention kernel that follows does not wait for this one before it reads: what both read must be there by now
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const KvSpan all = kv_span(p.batch.offsets[0], p.batch.offsets[p.batch.sequences], p.tokens);
    const int q_first = all.first, q_count = all.count;
    const int64_t steps = int64_t(p.kv_heads) * plan.places;
    int64_t at = min(steps, group * plan.per);
    const int64_t end = min(steps, at + plan.per);
    const int lookahead = plan.paired ? 1 : 2;                   // tiles of keys whose logits are under way
    PrefixPart w;
    bool ok = true;

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kCopyWarp) {
        // ---- tiles in the order of their use: the keys `lookahead` tiles ahead of the values
        const int box = min(kKvPrefixTile, 1 << p.page_shift), boxes = kKvPrefixTile / box;
        uint32_t n = 0, armed = 0;                               // a bit per stream and slot: the phase that its next copy completes
        auto load = [&](const PrefixPart &part, int i, const CUtensorMap *map) {
            if (!ok) return;
            // A wait tells a phase from the one before it only, so a barrier's phases are all waited for by those who wait for it: tiles of
            // keys that are dealt to the streams complete barriers of the stream that uses them.
            const int s = n % G::kSlots, owner = plan.paired ? 0 : i & 1;
            const int64_t key = int64_t(part.tile0 + i) * kKvPrefixTile + lane * box;
            const int64_t entry = key >> p.page_shift;
            int page = -1;
            if (lane < boxes && entry < p.prefix_width && key < p.prefix_len) page = __ldg(p.prefix_pages + entry);
            const bool good = page >= 0 && page < p.pages;
            if (!good) page = p.pages;                           // outside the pool: the copy fills with zeros
            if (n >= G::kSlots) ok = mbar_wait(&sh.empty[s], ((n / G::kSlots) - 1) & 1, p.timeouts);
            ok = __all_sync(kFullMask, ok);
            if (!ok) return;
            uint64_t *bar = &sh.full[owner][s];
            armed ^= 1u << (16 * owner + s);
            if (lane == 0) mbar_arrive_expect_tx(bar, G::kTileBytes);
            __syncwarp();
            if (lane < boxes)
#pragma unroll
                for (int c = 0; c < D / 64; ++c)
                    tma_load_page(ring + s * G::kTileBytes + c * G::kHalfBytes + lane * box * 128, map, c * 64, int(key & ((1 << p.page_shift) - 1)), part.h, page, bar);
            ++n;
        };
        uint32_t parts = 0;
        while (next_part(plan, at, end, w)) {
            // rows of Q: whole tokens, plan.rows of them to a tile; those behind the last token are zeros
            for (int s = 0; s < (plan.paired ? 2 : 1); ++s) {
                if (ok && parts > 0) ok = mbar_wait(&sh.q_free[s], (parts - 1) & 1, p.timeouts);
                ok = __all_sync(kFullMask, ok);
                if (!ok) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&sh.q_full[s], uint32_t(plan.rows * 128 * (D / 64)));
                    const int token = q_first + (plan.paired ? 2 * unit + s : unit) * (plan.rows / p.group);
                    for (int c = 0; c < D / 64; ++c)
                        tma_load_page(q_smem + s * G::kTileBytes + c * G::kHalfBytes, &maps.q, c * 64, 0, w.h, token, &sh.q_full[s]);
                }
                __syncwarp();
            }
            ++parts;
            for (int i = 0; i < min(lookahead, w.count); ++i) load(w, i, &maps.k);
            for (int i = 0; i < w.count; ++i) {
                load(w, i, &maps.v);
                if (i + lookahead < w.count) load(w, i + lookahead, &maps.k);
            }
        }
        if (!ok)                                                 // the copies in flight land before the block ends
        {
            for (int i = 0; i < 2 * G::kSlots; ++i) {
                const int owner = i & 1, slot = i >> 1;
                mbar_wait(&sh.full[owner][slot], ((armed >> (16 * owner + slot)) & 1) ^ 1, p.timeouts);
            }
            for (int s = 0; s < (plan.paired ? 2 : 1) && parts > 0; ++s) mbar_wait(&sh.q_full[s], (parts - 1) & 1, p.timeouts);
        }
    } else if (warp < kMmaWarp + 2) {
        // ---- MMAs of stream s.  One warp for both would be what bounds the kernel: waiting for a barrier that has completed takes it some 200
        // cycles, six times a tile, and an MMA 30 to issue (3,000 cycles a step with weights that cost nothing; 2,048 are the MMAs').
        const int s = warp - kMmaWarp, first = plan.paired ? 0 : s, stride = plan.paired ? 1 : 2, qs = plan.paired ? s : 0;    // `first`: its full barriers, too
        uint32_t parts = 0, p_count = 0, base = 0, seen = 0;     // tiles of the ring before this part; a bit per slot: the phase to wait for
        constexpr uint32_t kIdS = idesc<T>(kHalfKeys, false), kIdO = idesc<T>(D, true);
        auto wait = [&](uint64_t *bar, uint32_t parity) {
            if (ok) ok = mbar_wait(bar, parity, p.timeouts);
            fence_after();
        };
        const uint32_t leader = elected();
        const uint64_t q_desc = umma_desc(smem_u32(q_smem) + qs * G::kTileBytes), ring_k = umma_desc(smem_u32(ring)), ring_v = desc_mn(smem_u32(ring), G::kHalfBytes);
        const uint32_t s_tmem = tmem + 128 * s, o_tmem = tmem + 256 + G::kOColumns * s;
        while (next_part(plan, at, end, w)) {
            const int ahead = min(lookahead, w.count);
            // places in the ring: `ahead` tiles of keys, then values and keys in turn
            auto place_v = [&](int i) { return base + uint32_t(ahead + i + min(i, w.count - ahead)); };
            auto place_k = [&](int i) { return i < lookahead ? base + uint32_t(i) : place_v(i - lookahead) + 1; };
            // descriptors of other addresses: 16-byte units added to the address field, which has room for all of shared memory
            auto logits = [&](int b, uint32_t slot) {            // S of half b = Q K^T
                const uint64_t k = ring_k + slot * uint32_t(G::kTileBytes >> 4) + uint32_t(b * (kHalfKeys * 128 >> 4));
                const uint32_t d = s_tmem + kHalfKeys * b;
                mma_ss<false>(leader, d, q_desc, k, kIdS);
#pragma unroll
                for (int c = 1; c < D / 16; ++c) {
                    const uint32_t off = ((c >> 2) * G::kHalfBytes + (c & 3) * 32) >> 4;
                    mma_ss<true>(leader, d, q_desc + off, k + off, kIdS);
                }
                commit(leader, &sh.s_full[s][b]);
            };
            auto tile_of = [&](uint32_t n) {                     // waits for place n of the ring
                const uint32_t slot = n % G::kSlots;
                wait(&sh.full[first][slot], (seen >> slot) & 1);
                seen ^= 1u << slot;
                return slot;
            };
            // Q of the part, also where this stream has no tile of it: a wait tells a phase from the one before it only, so nobody may be
            // more than one behind, and Q is not loaded anew before both streams have seen it
            wait(&sh.q_full[qs], parts & 1);
            if (lane == 0) { mbar_arrive(&sh.q_free[0]); mbar_arrive(&sh.q_free[1]); }
            __syncwarp();
            if (first < w.count) {
                const uint32_t slot = tile_of(place_k(first));
                logits(0, slot);
                logits(1, slot);
                commit(leader, &sh.empty[slot]);
            }
            for (int i = first; i < w.count; i += stride) {
                const uint32_t slot = tile_of(place_v(i));
                const int64_t left = int64_t(p.prefix_len) - int64_t(w.tile0 + i) * kKvPrefixTile;
                if (left < kKvPrefixTile) {                      // places behind the prefix may hold anything, and 0 * NaN is not 0 (the other
                    uint8_t *v = ring + slot * G::kTileBytes;    // stream's warp writes the same zeros)
                    for (int row = int(left); row < kKvPrefixTile; ++row)
                        if (lane < D / 8) *reinterpret_cast<uint4 *>(v + (lane >> 3) * G::kHalfBytes + row * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                    fence_shared_async();
                    __syncwarp();
                }
                const uint64_t v = ring_v + slot * uint32_t(G::kTileBytes >> 4);
                const bool more = i + stride < w.count;
                uint32_t k_slot = 0;
#pragma unroll
                for (int b = 0; b < 2; ++b) {                    // O += P V, and the next logits where this P was
                    wait(&sh.p_ready[s][b], p_count & 1);
#pragma unroll
                    for (int c = 0; c < kHalfKeys / 16; ++c)
                        mma_ts(leader, o_tmem, s_tmem + kHalfKeys * b + 8 * c, v + (4 * b + c) * (2048 >> 4), kIdO, i != first || b + c > 0);
                    commit(leader, &sh.o_done[s]);
                    if (more) {
                        if (b == 0) k_slot = tile_of(place_k(i + stride));
                        logits(b, k_slot);
                    }
                }
                ++p_count;
                commit(leader, &sh.empty[slot]);
                if (more) commit(leader, &sh.empty[k_slot]);
            }
            base += 2 * uint32_t(w.count);
            ++parts;
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWeightRegs));
        // ---- weights: stream `s`, a row to a thread
        const int s = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t quarter = uint32_t((warp & 3) * 32) << 16, s_addr = tmem + 128 * s + quarter, o_addr = tmem + 256 + G::kOColumns * s + quarter;
        uint32_t s_count = 0, o_count = 0, parts = 0;
        const int64_t live = int64_t(q_count) * p.group;
        const int64_t row_base = int64_t(plan.paired ? 2 * unit + s : unit) * plan.rows;
        auto wait = [&](uint64_t *bar, uint32_t parity) {
            if (ok) ok = mbar_wait(bar, parity, p.timeouts);
        };
        while (next_part(plan, at, end, w)) {
            float m = -INFINITY, l = 0.0f;
            int done = 0;                                        // halves of tiles of this stream so far
            // pages outside the pool hold no keys: lane l < 4 looks after keys 16 l .. 16 l + 15 of a half, if the part has any such page
            auto page_is_good = [&](int64_t key) {
                const int64_t entry = key >> p.page_shift;
                const int page = key < p.prefix_len && entry < p.prefix_width ? __ldg(p.prefix_pages + entry) : -1;
                return page >= 0 && page < p.pages;
            };
            bool all_good = true;
            {
                const int64_t from = int64_t(w.tile0) * kKvPrefixTile, to = min(from + int64_t(w.count) * kKvPrefixTile, int64_t(p.prefix_len));
                for (int64_t entry = (from >> p.page_shift) + lane; entry << p.page_shift < to; entry += 32) all_good = all_good && page_is_good(entry << p.page_shift);
                all_good = __all_sync(kFullMask, all_good);
            }
            const int stride = plan.paired ? 1 : 2;
            for (int i = plan.paired ? 0 : s; i < w.count; i += stride, ++s_count)
#pragma unroll 1
            for (int b = 0; b < 2; ++b, ++done) {
                wait(&sh.s_full[s][b], s_count & 1);
                fence_after();
                const uint32_t half_addr = s_addr + kHalfKeys * b;
                uint32_t x[kHalfKeys];
                tmem_ld32(half_addr, reinterpret_cast<uint32_t (&)[32]>(x[0]));
                tmem_ld32(half_addr + 32, reinterpret_cast<uint32_t (&)[32]>(x[32]));
                tmem_wait_ld();
                const int first_key = (w.tile0 + i) * kKvPrefixTile + kHalfKeys * b, left = p.prefix_len - first_key;     // below 2^30 + 128
                if (!all_good || left < kHalfKeys) {
                    const uint32_t good = __ballot_sync(kFullMask, page_is_good(first_key + 16 * (lane & 3)));
#pragma unroll
                    for (int c = 0; c < kHalfKeys; ++c)
                        if (c >= left || !((good >> (c >> 4)) & 1u)) x[c] = 0xff800000u;
                }
                // the weights of columns c0 .. c0 + 31, over the base m, and their sum
                const uint64_t scale2 = pair(p.scale_log2, p.scale_log2);
                auto weights = [&](int c0, uint32_t (&pk)[16], uint64_t (&part)[2]) {
                    const float base = m == -INFINITY ? 0.0f : -m;
                    const uint64_t base2 = pair(base, base);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float2 z = unpair(fma2(pair(__uint_as_float(x[c0 + 2 * j]), __uint_as_float(x[c0 + 2 * j + 1])), scale2, base2));
                        // some of the weights by the multiply-add pipe: the exponential unit gives 4 a cycle to each scheduler and
                        // would take 2,048 cycles a step
                        float2 e;
                        if ((j & 7) < kByPolynomial) e = exp2_pair(z);
                        else e = make_float2(kv_exp2(z.x), kv_exp2(z.y));
                        part[j & 1] = add2(part[j & 1], pair(e.x, e.y));
                        pk[j] = KvType<T>::pack(e.x, e.y);
                    }
                };
                auto largest = [&] {
                    float t8[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) t8[j] = __uint_as_float(x[j]);
#pragma unroll
                    for (int c = 8; c < 56; c += 16)
#pragma unroll
                        for (int j = 0; j < 8; ++j) t8[j] = max3_nan(t8[j], __uint_as_float(x[c + j]), __uint_as_float(x[c + 8 + j]));
#pragma unroll
                    for (int j = 0; j < 8; j += 2) t8[j] = max3_nan(max3_nan(t8[j], t8[j + 1], __uint_as_float(x[56 + j])), __uint_as_float(x[57 + j]), t8[j]);
                    const float top = max3_nan(max3_nan(t8[0], t8[2], t8[4]), t8[6], t8[6]) * p.scale_log2;
                    return top < INFINITY ? top : NAN;           // an infinite logit makes the row NaN, as inf - inf does
                };
                // The weights are computed over the base so far, before it is known whether that still holds: it mostly does, and then
                // looking for the largest logit costs no time of its own.
                constexpr float kLift = KvType<T>::kLift, kUpTo = kLift + KvType<T>::kRescaleAt;
                if (done == 0) m = largest() - kLift;
                uint32_t pk[2][16];
                uint64_t part[2] = {0, 0};
                weights(0, pk[0], part);
                weights(32, pk[1], part);
                if (done > 0) {
                    const float top = largest();
                    if (__any_sync(kFullMask, !(top <= m + kUpTo))) {
                        // For the rows that need it: what the others give must not depend on their neighbours.  (A NaN becomes the maximum: the
                        // polynomial would lose it.)
                        const float next = top <= m + kUpTo ? m : max3_nan(m, top - kLift, top - kLift), f = next == m ? 1.0f : kv_exp2(m - next);
                        m = next;
                        l *= f;
                        wait(&sh.o_done[s], (o_count + done - 1) & 1);      // (the half before that had ended when these logits were there)
                        fence_after();
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            uint32_t y[32];
                            tmem_ld32(o_addr + c, y);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; ++j) y[j] = __float_as_uint(__uint_as_float(y[j]) * f);
                            tmem_st32(o_addr + c, y);
                        }
                        part[0] = part[1] = 0;
                        weights(0, pk[0], part);
                        weights(32, pk[1], part);
                    }
                }
                tmem_st16(half_addr, pk[0]);
                tmem_st16(half_addr + 16, pk[1]);
                const float2 sums = unpair(add2(part[0], part[1]));
                l += sums.x + sums.y;
                tmem_wait_st();
                // A wait tells a phase from the one before it only.  At the end of the part the last half's product is waited for, so the one
                // before must be known to have ended; it has, or is under way, while the last one cannot have begun.
                if (b == 1 && i + stride >= w.count) wait(&sh.o_done[s], (o_count + done - 1) & 1);
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_ready[s][b]);
            }
            // ---- the part's result
            const int64_t block = ((int64_t(w.h) + group) * plan.units + unit) * 2 + s;
            const bool have = r < plan.rows && row_base + r < live;
            if (done > 0) {
                wait(&sh.o_done[s], (o_count + done - 1) & 1);
                fence_after();
                // a row to a thread as it comes from tensor memory, rows of 128 bytes as it goes out: each warp turns its 32 rows in 4 KB of
                // shared memory (stores of 16 bytes in 32 rows at once took 7,000 cycles).  Q has been read by now: its place is used where
                // there is no other; a stream without a tile of rows of its own uses the second tile's.
                uint8_t *stage = (D == 64 ? reinterpret_cast<uint8_t *>(&sh + 1) + s * 16384
                                          : q_smem + (plan.paired ? s * G::kTileBytes : G::kTileBytes + s * 16384)) + (warp & 3) * 4096;
                const int64_t first_row = row_base + (warp & 3) * 32;
                const int rows = int(max(int64_t(0), min(live - first_row, int64_t(min(32, plan.rows - (warp & 3) * 32)))));     // of this warp that are there
                float *dst = p.pre_o + (block * kKvPrefixRows + (warp & 3) * 32) * D;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t y[32];
                    tmem_ld32(o_addr + c, y);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        *reinterpret_cast<uint4 *>(stage + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int row = 4 * j + (lane >> 3), piece = lane & 7;
                        if (row < rows) *reinterpret_cast<uint4 *>(dst + row * D + c + 4 * piece) = *reinterpret_cast<const uint4 *>(stage + row * 128 + ((piece ^ (row & 7)) << 4));
                    }
                    __syncwarp();
                }
                if (D == 128 && plan.paired)                     // the rows of Q's tile that no copy writes are zeros again
                    for (int row = max((warp & 3) * 32, plan.rows); row < (warp & 3) * 32 + 32; ++row)
                        if (lane < 8) *reinterpret_cast<uint4 *>(stage + (row - (warp & 3) * 32) * 128 + lane * 16) = make_uint4(0, 0, 0, 0);
                fence_shared_async();
            } else {
                // no tile of this part (one tile of keys, and it is the other stream's): without this wait the stream could be a part ahead and
                // give Q back twice, in the other one's place
                wait(&sh.q_full[0], parts & 1);
            }
            o_count += done;
            ++parts;
            if (have) p.pre_ml[block * kKvPrefixRows + r] = make_float2(m, l);
            // Q, S and O may be written anew
            fence_before();
            __syncwarp();
            if (lane == 0) { mbar_arrive(&sh.q_free[0]); mbar_arrive(&sh.q_free[1]); }
        }
    }

    fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <typename T, int D>
cudaError_t launch(const KvAttendParams &p, const KvMaps &maps, int device, cudaStream_t s) {
    using G = PrefixGeometry<D>;
    constexpr size_t smem = G::kQBytes + G::kSlots * G::kTileBytes + sizeof(PrefixShared<D>) + (D == 64 ? 32768 : 0) + 1024;
    static_assert(smem <= kBlockSharedBytes, "more shared memory than a block can have");
    auto *kern = kv_prefix_kernel<T, D>;
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = kv_allow_shared(kern, allowed, device);
    if (e != cudaSuccess) return e;
    return kv_launch(kern, dim3(unsigned(p.plan.units * p.plan.groups)), kPrefixThreads, smem, s, p, maps);
}

}  // namespace

cudaError_t launch_kv_prefix(const KvAttendParams &p, const KvMaps &maps, int dtype, int head_dim, int device, cudaStream_t s) {
    if (dtype == TV_KV_BF16) return head_dim == 128 ? launch<__nv_bfloat16, 128>(p, maps, device, s) : launch<__nv_bfloat16, 64>(p, maps, device, s);
    return head_dim == 128 ? launch<__half, 128>(p, maps, device, s) : launch<__half, 64>(p, maps, device, s);
}

}  // namespace tv
