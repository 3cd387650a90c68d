// Appending keys and values to the pages of a cache, with the position rotation and the pages' bounds.
//
// A block takes one page that a sequence's new tokens touch, and one to eight key heads (whole warps each): it rotates the page's new
// keys and the queries of the heads' groups, copies the values, and brings the page's bounds up to date.  A page and head belongs to
// one block, so bounds need no atomics and no order matters.  A thread takes 16 channels of a token: key, value and the group's
// queries, whose angles it reads once.
//
// Bound by memory where there are many tokens (append_prompts_4, 32,818 tokens of 8 + 32 heads of 128 channels, 824 MB: 149 us, 5.5 TB/s),
// by dependent loads where there are few (place in the batch, page, rows: 6.1 us for one token).
//
// Rotation: (y1, y2) = (x1 cos - x2 sin, x2 cos + x1 sin) in 32 bits, each product and sum rounded by itself, then to the type.
// Bounds: for every channel the lowest and highest key of the page, as int8 multiples of one power of two 2^e per page and key head,
// rounded outwards: hi = ceil(max / 2^e), lo = floor(min / 2^e), e the smallest with max |key| <= 127 * 2^e.  Because
// ceil(ceil(x / 2^a) / 2^b) = ceil(x / 2^(a+b)) and rounding is monotone, widening the 8-bit bounds by new keys gives what the
// bounds of all keys together would be: tokens may come in any pieces, and the page is not read again.
#include "kv_cache.cuh"

namespace tv {
namespace {

constexpr int kAppendThreads = 256;

template <typename T>
__device__ __forceinline__ void rotate8(const uint4 &a, const uint4 &b, const float (&c)[8], const float (&s)[8], uint4 &ya, uint4 &yb) {
    const uint32_t *pa = reinterpret_cast<const uint32_t *>(&a), *pb = reinterpret_cast<const uint32_t *>(&b);
    uint32_t *qa = reinterpret_cast<uint32_t *>(&ya), *qb = reinterpret_cast<uint32_t *>(&yb);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x1 = KvType<T>::unpack(pa[i]), x2 = KvType<T>::unpack(pb[i]);
        qa[i] = KvType<T>::pack(__fsub_rn(__fmul_rn(x1.x, c[2 * i]), __fmul_rn(x2.x, s[2 * i])),
                                __fsub_rn(__fmul_rn(x1.y, c[2 * i + 1]), __fmul_rn(x2.y, s[2 * i + 1])));
        qb[i] = KvType<T>::pack(__fadd_rn(__fmul_rn(x2.x, c[2 * i]), __fmul_rn(x1.x, s[2 * i])),
                                __fadd_rn(__fmul_rn(x2.y, c[2 * i + 1]), __fmul_rn(x1.y, s[2 * i + 1])));
    }
}
// pairs of neighbours: the 16 channels of (a, b) are the pairs of angles 0 .. 7
template <typename T>
__device__ __forceinline__ void rotate_pairs(const uint4 &a, const uint4 &b, const float (&c)[8], const float (&s)[8], uint4 &ya, uint4 &yb) {
    const uint32_t *pa = reinterpret_cast<const uint32_t *>(&a), *pb = reinterpret_cast<const uint32_t *>(&b);
    uint32_t *qa = reinterpret_cast<uint32_t *>(&ya), *qb = reinterpret_cast<uint32_t *>(&yb);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 x = KvType<T>::unpack(i < 4 ? pa[i] : pb[i - 4]);
        const uint32_t y = KvType<T>::pack(__fsub_rn(__fmul_rn(x.x, c[i]), __fmul_rn(x.y, s[i])), __fadd_rn(__fmul_rn(x.y, c[i]), __fmul_rn(x.x, s[i])));
        if (i < 4) qa[i] = y; else qb[i - 4] = y;
    }
}

// Channels of unit u of a row: two runs of 8, which the rotation mixes (half-split: i and i + rotary / 2) or which are neighbours.
struct Unit {
    int a, b;
    bool turned;
};
__device__ __forceinline__ Unit unit_of(int u, int rotary, int interleaved) {
    const int turned = rotary >> 4;
    if (u < turned && !interleaved) return {8 * u, (rotary >> 1) + 8 * u, true};
    return {16 * u, 16 * u + 8, u < turned};
}

struct Run16 {
    uint4 a, b;
};
template <typename T>
__device__ __forceinline__ Run16 load_unit(const T *src, const Unit &un) {
    return {*reinterpret_cast<const uint4 *>(src + un.a), *reinterpret_cast<const uint4 *>(src + un.b)};
}
template <typename T>
__device__ __forceinline__ void store_unit(T *dst, const Unit &un, const Run16 &x) {
    *reinterpret_cast<uint4 *>(dst + un.a) = x.a;
    *reinterpret_cast<uint4 *>(dst + un.b) = x.b;
}
template <typename T>
__device__ __forceinline__ Run16 turn(const Run16 &x, const Unit &un, int interleaved, const float (&c)[8], const float (&s)[8]) {
    if (!un.turned) return x;
    Run16 y;
    if (interleaved) rotate_pairs<T>(x.a, x.b, c, s, y.a, y.b);
    else rotate8<T>(x.a, x.b, c, s, y.a, y.b);
    return y;
}
// lowest / highest of two values each; a NaN is left out
__device__ __forceinline__ uint32_t low2(uint32_t x, uint32_t y, __nv_bfloat16) { uint32_t d; asm("min.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y)); return d; }
__device__ __forceinline__ uint32_t high2(uint32_t x, uint32_t y, __nv_bfloat16) { uint32_t d; asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y)); return d; }
__device__ __forceinline__ uint32_t low2(uint32_t x, uint32_t y, __half) { uint32_t d; asm("min.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y)); return d; }
__device__ __forceinline__ uint32_t high2(uint32_t x, uint32_t y, __half) { uint32_t d; asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y)); return d; }

// HEADS key heads to a block: whole warps each.
template <typename T, int D, int HEADS>
__global__ void __launch_bounds__(kAppendThreads, 3) kv_append_kernel(const KvAppendParams p) {
    constexpr int kUnits = D / 16;                          // threads of one row, 16 channels each
    constexpr int kWarps = kAppendThreads / 32;
    constexpr int kWarpsPerHead = kWarps / HEADS;
    constexpr int kLanes = kWarpsPerHead * 32 / kUnits;     // tokens of a head at a time
    __shared__ int64_t scratch[kWarps + 2];
    __shared__ uint32_t lows[kWarps][D / 2], highs[kWarps][D / 2];   // pairs of channels
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, page_size = 1 << p.page_shift;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");

    int b;
    int64_t place;
    auto first_position = [&](int i, const KvSpan &sp) { return int64_t(p.batch.lens[i]) - sp.count; };
    // pages that sequence i's tokens touch; positions before 0 belong to no page
    auto touched = [&](int i) -> int64_t {
        const KvSpan sp = kv_span(p.batch.offsets[i], p.batch.offsets[i + 1], p.tokens);
        const int64_t from = first_position(i, sp), to = from + sp.count;
        if (sp.count == 0 || to <= 0) return 0;
        return ((to - 1) >> p.page_shift) - ((from < 0 ? 0 : from) >> p.page_shift) + 1;
    };
    kv_locate<kAppendThreads>(int64_t(blockIdx.x), p.batch.sequences, touched, scratch, b, place);
    if (b >= p.batch.sequences) return;
    const KvSpan sp = kv_span(p.batch.offsets[b], p.batch.offsets[b + 1], p.tokens);
    const int64_t from = first_position(b, sp), to = from + sp.count;
    const int64_t page_index = ((from < 0 ? 0 : from) >> p.page_shift) + place, page_from = page_index << p.page_shift;
    const int64_t begin = from > page_from ? from : page_from;                                  // positions of this block
    const int64_t end = to < page_from + page_size ? to : page_from + page_size;
    const int64_t page = page_index < p.batch.table_width ? int64_t(p.batch.table[int64_t(b) * p.batch.table_stride + page_index]) : -1;
    const bool stored = page >= 0 && page < p.pages;
    const int count = int(end - begin), row0 = sp.first + int(begin - from), at0 = int(begin - page_from);
    const int half = p.rotary >> 1;
    const int h = blockIdx.y * HEADS + warp / kWarpsPerHead;
    const int in_head = tid % (kWarpsPerHead * 32), u = in_head % kUnits;
    const Unit un = unit_of(u, p.rotary, p.interleaved);
    uint32_t lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { lo[i] = KvType<T>::pack(INFINITY, INFINITY); hi[i] = KvType<T>::pack(-INFINITY, -INFINITY); }
    if (h < p.kv_heads) {
        for (int i = in_head / kUnits; i < count; i += kLanes) {
            // a position outside the tables has no angle: its token is neither stored nor rotated
            const int64_t angle = begin + i + p.position_offset;
            if (p.rotary > 0 && (angle < 0 || angle >= p.positions)) continue;
            const int64_t row = row0 + i;
            Run16 k, v;
            if (stored) {
                k = load_unit(static_cast<const T *>(p.k_new.data) + row * p.k_new.token_stride + int64_t(h) * p.k_new.head_stride, un);
                v = load_unit(static_cast<const T *>(p.v_new.data) + row * p.v_new.token_stride + int64_t(h) * p.v_new.head_stride, un);
            }
            float c[8] = {}, s[8] = {};
            if (un.turned) {
                const float4 *pc = reinterpret_cast<const float4 *>(p.cos + angle * half + 8 * u), *ps = reinterpret_cast<const float4 *>(p.sin + angle * half + 8 * u);
                *reinterpret_cast<float4 *>(c) = pc[0]; *reinterpret_cast<float4 *>(c + 4) = pc[1];
                *reinterpret_cast<float4 *>(s) = ps[0]; *reinterpret_cast<float4 *>(s + 4) = ps[1];
            }
            if (stored) {
                k = turn<T>(k, un, p.interleaved, c, s);
                store_unit(reinterpret_cast<T *>(p.k) + page * p.k_page + int64_t(h) * p.k_head + int64_t(at0 + i) * p.k_token, un, k);
                store_unit(reinterpret_cast<T *>(p.v) + page * p.v_page + int64_t(h) * p.v_head + int64_t(at0 + i) * p.v_token, un, v);
                const uint32_t *w = reinterpret_cast<const uint32_t *>(&k);
#pragma unroll
                for (int j = 0; j < 8; ++j) { lo[j] = low2(lo[j], w[j], T()); hi[j] = high2(hi[j], w[j], T()); }
            }
            if (p.q.data) {                                  // two heads at a time, so that their loads overlap
                const T *src = static_cast<const T *>(p.q.data) + row * p.q.token_stride + int64_t(h) * p.group * p.q.head_stride;
                T *dst = static_cast<T *>(p.q_out.data) + row * p.q_out.token_stride + int64_t(h) * p.group * p.q_out.head_stride;
                int g = 0;
                for (; g + 1 < p.group; g += 2) {
                    const Run16 x = load_unit(src + g * p.q.head_stride, un), y = load_unit(src + (g + 1) * p.q.head_stride, un);
                    store_unit(dst + g * p.q_out.head_stride, un, turn<T>(x, un, p.interleaved, c, s));
                    store_unit(dst + (g + 1) * p.q_out.head_stride, un, turn<T>(y, un, p.interleaved, c, s));
                }
                if (g < p.group) store_unit(dst + g * p.q_out.head_stride, un, turn<T>(load_unit(src + g * p.q.head_stride, un), un, p.interleaved, c, s));
            }
        }
    }
    if (p.bounds == nullptr || !stored) return;
    // places of the page that the tokens with an angle took: without any, the page and its bounds are as they were
    int64_t first_place = at0, last_place = at0 + count - 1;
    if (p.rotary > 0) {
        first_place = max(first_place, -p.position_offset - page_from);
        last_place = min(last_place, p.positions - 1 - p.position_offset - page_from);
    }
    if (first_place > last_place) return;

    // lowest and highest new key of every channel: over the rows of a warp, then over the head's warps
#pragma unroll
    for (int o = kUnits; o < 32; o <<= 1)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            lo[i] = low2(lo[i], __shfl_xor_sync(kFullMask, lo[i], o), T());
            hi[i] = high2(hi[i], __shfl_xor_sync(kFullMask, hi[i], o), T());
        }
    if (lane < kUnits)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = (i < 4 ? un.a : un.b) / 2 + (i & 3);
            lows[warp][at] = lo[i];
            highs[warp][at] = hi[i];
        }
    __syncthreads();
    // one warp per head: a lane takes D / 64 pairs of channels
    const int mine = blockIdx.y * HEADS + warp;
    if (warp >= HEADS || mine >= p.kv_heads) return;
    constexpr int kPairs = D / 64;
    float2 low[kPairs], high[kPairs];
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
        uint32_t l = lows[warp * kWarpsPerHead][lane + 32 * j], g = highs[warp * kWarpsPerHead][lane + 32 * j];
#pragma unroll
        for (int w = 1; w < kWarpsPerHead; ++w) {
            l = low2(l, lows[warp * kWarpsPerHead + w][lane + 32 * j], T());
            g = high2(g, highs[warp * kWarpsPerHead + w][lane + 32 * j], T());
        }
        low[j] = KvType<T>::unpack(l);
        high[j] = KvType<T>::unpack(g);
        if (low[j].x <= high[j].x) top = fmaxf(top, fmaxf(fabsf(low[j].x), fabsf(high[j].x)));
        if (low[j].y <= high[j].y) top = fmaxf(top, fmaxf(fabsf(low[j].y), fabsf(high[j].y)));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
    const int64_t at = page * p.kv_heads + mine;
    const bool widen = first_place > 0;                     // the page holds earlier keys
    const float old_scale = widen ? p.scales[at] : 0.0f;
    const float scale = fmaxf(kv_pow2(kv_exponent(top)), old_scale), ratio = old_scale / scale;
    int8_t *row = p.bounds + at * 2 * D;
    auto low8 = [&](float x, float y, int8_t old) {         // x <= y unless no new key has a value in the channel
        const float q = x > y ? 127.0f : fminf(fmaxf(floorf(x / scale), -127.0f), 127.0f);
        return widen ? fminf(q, floorf(float(old) * ratio)) : x > y ? 0.0f : q;
    };
    auto high8 = [&](float x, float y, int8_t old) {
        const float q = x > y ? -127.0f : fminf(fmaxf(ceilf(y / scale), -127.0f), 127.0f);
        return widen ? fmaxf(q, ceilf(float(old) * ratio)) : x > y ? 0.0f : q;
    };
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
        char2 *pl = reinterpret_cast<char2 *>(row) + lane + 32 * j, *ph = reinterpret_cast<char2 *>(row + D) + lane + 32 * j;
        const char2 ol = widen ? *pl : make_char2(0, 0), oh = widen ? *ph : make_char2(0, 0);
        *pl = make_char2(int8_t(int(low8(low[j].x, high[j].x, ol.x))), int8_t(int(low8(low[j].y, high[j].y, ol.y))));
        *ph = make_char2(int8_t(int(high8(low[j].x, high[j].x, oh.x))), int8_t(int(high8(low[j].y, high[j].y, oh.y))));
    }
    __syncwarp();                                           // every lane has read the old scale
    if (lane == 0) p.scales[at] = scale;
}

template <typename T, int D>
cudaError_t launch(const KvAppendParams &p, cudaStream_t s) {
    // pages touched: at most one per token, and at most two partial ones beside the full ones of a sequence
    const int64_t most = (int64_t(p.tokens) >> p.page_shift) + 2 * int64_t(p.batch.sequences);
    const unsigned blocks = unsigned(most < p.tokens ? most : p.tokens);
    // Several heads to a block, so that finding its page is not most of its work: two where a page gets many tokens (append_prompts_4 with
    // one, two, four: 164, 158, 161 us; append_chunks_9 34.6, 31.9, 33.1), more where it gets few (append_197x1 with one 43 us, with
    // eight 29).
    const int64_t tokens_of_page = p.tokens / blocks;
    const int heads = p.kv_heads == 1 ? 1 : tokens_of_page >= 8 || p.kv_heads == 2 ? 2 : tokens_of_page >= 4 || p.kv_heads <= 4 ? 4 : 8;
    const dim3 grid(blocks, unsigned((p.kv_heads + heads - 1) / heads));
    if (heads == 1) return kv_launch(kv_append_kernel<T, D, 1>, grid, kAppendThreads, 0, s, p);
    if (heads == 2) return kv_launch(kv_append_kernel<T, D, 2>, grid, kAppendThreads, 0, s, p);
    if (heads == 4) return kv_launch(kv_append_kernel<T, D, 4>, grid, kAppendThreads, 0, s, p);
    return kv_launch(kv_append_kernel<T, D, 8>, grid, kAppendThreads, 0, s, p);
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendParams &p, int dtype, int head_dim, cudaStream_t s) {
    if (p.tokens == 0 || p.batch.sequences == 0) return cudaSuccess;
    if (dtype == TV_KV_BF16) return head_dim == 128 ? launch<__nv_bfloat16, 128>(p, s) : launch<__nv_bfloat16, 64>(p, s);
    return head_dim == 128 ? launch<__half, 128>(p, s) : launch<__half, 64>(p, s);
}

}  // namespace tv
