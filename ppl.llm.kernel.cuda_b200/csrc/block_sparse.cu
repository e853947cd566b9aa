// Attention of one new token per sequence over blocks that a cheap score selects: bounds of the keys of complete blocks, the choice, and the attention
// over what was chosen.
#include "paged_attention.cuh"
#include "ptx.cuh"
#include "quotient.cuh"

#include <type_traits>

namespace pplb200 {
namespace {

using ptx::cluster_ctarank;
using ptx::cluster_sync_all;
using ptx::map_to_cta;

// The smallest fp16 of which 127 are no less than amax, at least 2^-24; two roundings upwards are one.
__device__ __forceinline__ half outer_scale(float amax) {
    const uint32_t s = __half_as_ushort(__float2half_ru(__fdiv_ru(amax, 127.0f)));
    return __ushort_as_half((unsigned short)max(s, 1u));
}
__device__ __forceinline__ bool is_finite(half s) { return (__half_as_ushort(s) & 0x7c00u) != 0x7c00u; }

// ---- bounds ------------------------------------------------------------------------------------------------------------
// A CTA looks through a few slots for those that end a block; its warps then take these blocks, a head each: a lane has 16 bytes of a token's row, and eight loads are on
// their way.  The lanes that have the same dimensions of different rows halve them between each other at the end, so that all divide and write.  Nothing is
// shared but these shuffles.
// In fp16 bound by HBM in a long prompt, the keys once (131072 tokens of 8 heads of 128, blocks of 64: 48 us, 5.6 TB/s), int8 by the minima and maxima, which are
// in fp32 as the products are, of three numbers at a time (45 us, groups of 8 49; of two numbers 51 and 58; with eight bytes a lane 53 and 59).  16384 tokens: 7.7, 7.1 and
// 7.9 us; in a decode step look-ups and the launch, 3 us.  Four CTAs share an SM over int8: left to itself the compiler takes up to 164 registers, and heads of 256 in groups of 8 98 us
// instead of 81, of 96 56 instead of 47 (131072 tokens); in fp16, where it takes 80, a bound costs 2 %.
constexpr int BWARPS = 4, BTPB = 32 * BWARPS;
struct BoundsParams {
    pplb200_kv_cache cache;
    int8_t* bounds;
    half* scale;
    const int64_t* slots;
    int64_t tokens;
    int32_t block, per_page, slots_here;
    uint32_t block_magic, block_shift;
};

__device__ __forceinline__ float least(float a, float b, float c) {
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float greatest(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Bytes `at` and at + 1 of four int8 values, times a scale.  A byte without its sign in the last bits of 2^23 is that number more, exactly; conversions have a
// quarter of the rate.
__device__ __forceinline__ float2 products(uint32_t values, int at, float scale) {
    const uint32_t u = values ^ 0x80808080u;
    const float2 whole = ptx::add2(make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540 + at)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7541 + at))),
                                   make_float2(-8388736.0f, -8388736.0f));
    return ptx::mul2(whole, make_float2(scale, scale));
}

template <int D, int KIND>
__global__ void __launch_bounds__(BTPB, KIND == CACHE_F16 ? 0 : 4) key_bounds_kernel(const __grid_constant__ BoundsParams p) {
    constexpr int PER = KIND == CACHE_F16 ? 8 : 16, LANES = D / PER;   // dimensions of a lane, and lanes of a row
    constexpr int ROWS = D == 96 ? 24 / LANES : 32 / LANES, BATCH = 8; // rows at once (a power of two); loads on their way
    constexpr int LEFT = PER / ROWS, GROUPS = KIND == CACHE_I8_GROUPS ? PER / 8 : 1;
    struct Block {
        int64_t page;
        int32_t x;
    };
    __shared__ Block block_of[BTPB];
    __shared__ int32_t found;
    const pplb200_kv_cache& c = p.cache;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) found = 0;
    pdl_wait_prior_grid();
    __syncthreads();
    const int64_t first_slot = (int64_t)blockIdx.x * p.slots_here;
    if (threadIdx.x < p.slots_here && first_slot + threadIdx.x < p.tokens) {
        int64_t page;
        int32_t in_page;
        if (kv_find(p.slots[first_slot + threadIdx.x], c.num_pages, c.page_size, page, in_page)) {
            const int32_t x = (uint32_t)((uint64_t)(uint32_t)in_page * p.block_magic >> p.block_shift);
            if (in_page - x * p.block == p.block - 1) block_of[atomicAdd(&found, 1)] = {page, x};
        }
    }
    __syncthreads();
    const int64_t head = (int64_t)blockIdx.y * BWARPS + warp;
    if (head >= c.kv_heads) return;
    const int row = lane / LANES, part = lane - row * LANES;
    const bool active = row < ROWS; // (heads of 96: 24 lanes)
    for (int i = 0; i < found; ++i) {
        const int64_t page = block_of[i].page;
        const int32_t x = block_of[i].x, token0 = x * p.block + (active ? row : 0);
        const int64_t at = kv_row(page, token0, head, c.page_stride, c.head_stride, c.token_stride) + part * PER;
        const int64_t scale_at = kv_row(page, token0, head, c.scale_page_stride, c.scale_head_stride, c.scale_token_stride) + (KIND == CACHE_I8_GROUPS ? part * GROUPS : 0);
        float lo[PER], hi[PER];
        bool bad = false; // a scale that is infinite or NaN; of fp16 keys, these come through in the bounds
        if constexpr (KIND == CACHE_F16) {
            __half2 l[4], h[4];
#pragma unroll
            for (int d = 0; d < 4; ++d) l[d] = as_h2(0x7c007c00u), h[d] = as_h2(0xfc00fc00u);
            for (int32_t t = 0; t < p.block; t += BATCH * ROWS) { // (ROWS divides 16, and 16 the block)
                uint4 w[BATCH];
#pragma unroll
                for (int k = 0; k < BATCH; ++k)
                    if (t + k * ROWS < p.block) w[k] = ld_global_16((const half*)c.k + at + (t + k * ROWS) * c.token_stride);
#pragma unroll
                for (int k = 0; k < BATCH; ++k)
                    if (t + k * ROWS < p.block) {
                        const uint32_t words[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
                        for (int d = 0; d < 4; ++d) l[d] = __hmin2_nan(l[d], as_h2(words[d])), h[d] = __hmax2_nan(h[d], as_h2(words[d]));
                    }
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const float2 a = __half22float2(l[d]), b = __half22float2(h[d]);
                lo[2 * d] = a.x; lo[2 * d + 1] = a.y;
                hi[2 * d] = b.x; hi[2 * d + 1] = b.y;
            }
#pragma unroll
            for (int d = 0; d < 8; ++d) bad |= !(fabsf(lo[d]) < INFINITY) || !(fabsf(hi[d]) < INFINITY);
        } else {
#pragma unroll
            for (int d = 0; d < PER; ++d) lo[d] = INFINITY, hi[d] = -INFINITY;
            static_assert(16 % (2 * ROWS) == 0); // two rows at a time
            for (int32_t t = 0; t < p.block; t += BATCH * ROWS) {
                uint4 w[BATCH];
                half s[BATCH][GROUPS];
#pragma unroll
                for (int k = 0; k < BATCH; ++k)
                    if (t + k * ROWS < p.block) {
                        w[k] = ld_global_16((const int8_t*)c.k + at + (t + k * ROWS) * c.token_stride);
#pragma unroll
                        for (int x = 0; x < GROUPS; ++x) s[k][x] = ld_global_half((const half*)c.k_scale + scale_at + (t + k * ROWS) * c.scale_token_stride + x);
                    }
#pragma unroll
                for (int k = 0; k < BATCH; k += 2)
                    if (t + k * ROWS < p.block) { // and the next one with it
                        const uint32_t words[2][4] = {{w[k].x, w[k].y, w[k].z, w[k].w}, {w[k + 1].x, w[k + 1].y, w[k + 1].z, w[k + 1].w}};
#pragma unroll
                        for (int x = 0; x < GROUPS; ++x) bad |= !is_finite(s[k][x]) || !is_finite(s[k + 1][x]);
#pragma unroll
                        for (int d = 0; d < PER; d += 2) {
                            const float2 a = products(words[0][d >> 2], d & 2, __half2float(s[k][GROUPS == 1 ? 0 : d / 8]));
                            const float2 b = products(words[1][d >> 2], d & 2, __half2float(s[k + 1][GROUPS == 1 ? 0 : d / 8]));
                            lo[d] = least(lo[d], a.x, b.x);
                            hi[d] = greatest(hi[d], a.x, b.x);
                            lo[d + 1] = least(lo[d + 1], a.y, b.y);
                            hi[d + 1] = greatest(hi[d + 1], a.y, b.y);
                        }
                    }
            }
        }
        // Two rows exchange halves of their dimensions, until each is left with LEFT of them.
        int mine = part * PER;
#pragma unroll
        for (int r = 1, half_of = PER / 2; r < ROWS; r <<= 1, half_of >>= 1) {
            const bool upper = row & r;
            const int other = active ? part + (row ^ r) * LANES : lane;
            mine += upper ? half_of : 0;
#pragma unroll
            for (int d = 0; d < half_of; ++d) {
                const float l = __shfl_sync(0xffffffffu, upper ? lo[d] : lo[d + half_of], other), h = __shfl_sync(0xffffffffu, upper ? hi[d] : hi[d + half_of], other);
                lo[d] = fminf(upper ? lo[d + half_of] : lo[d], l);
                hi[d] = fmaxf(upper ? hi[d + half_of] : hi[d], h);
            }
        }
        const bool lost_key = __any_sync(0xffffffffu, bad && active);
        float amax = 0.0f;
#pragma unroll
        for (int d = 0; d < LEFT; ++d) amax = fmaxf(amax, fmaxf(fabsf(lo[d]), fabsf(hi[d])));
        amax = __uint_as_float(__reduce_max_sync(0xffffffffu, active ? __float_as_uint(amax) : 0u));
        half s = outer_scale(amax);
        const bool lost = lost_key || !is_finite(s);
        if (lost) s = __ushort_as_half(0x7c00);
        const float step = __half2float(s);
        uint64_t l = 0, h = 0;
#pragma unroll
        for (int d = 0; d < LEFT; ++d) {
            const int a = lost ? 0 : (int)floorf(__fdiv_rn(lo[d], step)), b = lost ? 0 : (int)ceilf(__fdiv_rn(hi[d], step));
            l |= (uint64_t)(a & 0xff) << (8 * d);
            h |= (uint64_t)(b & 0xff) << (8 * d);
        }
        if (active) {
            using Piece = std::conditional_t<LEFT == 2, uint16_t, std::conditional_t<LEFT == 4, uint32_t, uint64_t>>;
            static_assert(sizeof(Piece) == LEFT);
            const int64_t of = (page * c.kv_heads + head) * p.per_page + x;
            *reinterpret_cast<Piece*>(p.bounds + of * 2 * D + mine) = (Piece)l;
            *reinterpret_cast<Piece*>(p.bounds + (of * 2 + 1) * D + mine) = (Piece)h;
            if (lane == 0) p.scale[of] = s;
        }
    }
}

struct BoundsReadParams {
    const int8_t* bounds;
    const half* scale;
    const int64_t* blocks;
    float *lo, *hi;
    int64_t count, all_blocks;
    int32_t per_page, kv_heads, head_dim;
};
// A thread has four dimensions of one of the two bounds.
__global__ void __launch_bounds__(BTPB) key_bounds_read_kernel(const __grid_constant__ BoundsReadParams p) {
    pdl_wait_prior_grid();
    const int quads = p.head_dim >> 2, of_head = 2 * quads, all = p.kv_heads * of_head;
    for (int64_t i = blockIdx.x; i < p.count; i += gridDim.x) {
        const int64_t block = p.blocks[i], page = block / p.per_page;
        const bool there = block >= 0 && block < p.all_blocks;
        for (int x = blockIdx.y * BTPB + threadIdx.x; x < all; x += gridDim.y * BTPB) {
            const int head = x / of_head, rest = x - head * of_head, high = rest >= quads, d = (rest - high * quads) * 4;
            float4 v = make_float4(0, 0, 0, 0);
            if (there) {
                const int64_t at = (page * p.kv_heads + head) * p.per_page + (block - page * p.per_page);
                const uint32_t w = ld_global_u32((const uint32_t*)(p.bounds + (at * 2 + high) * p.head_dim + d));
                const half s = ld_global_half(p.scale + at);
                const float f = __half2float(s);
                v = make_float4((float)(int8_t)w * f, (float)(int8_t)(w >> 8) * f, (float)(int8_t)(w >> 16) * f, (float)(int8_t)(w >> 24) * f);
                if (!is_finite(s)) v.x = v.y = v.z = v.w = high ? INFINITY : -INFINITY;
            }
            *reinterpret_cast<float4*>((high ? p.hi : p.lo) + (i * p.kv_heads + head) * p.head_dim + d) = v;
        }
    }
}

// ---- the choice ----------------------------------------------------------------------------------------------------------
// One cluster of CTAs for each sequence and key head.  A CTA scores its share of the blocks, 16 a warp at a time, on int8 mma.sync (16 blocks x 32
// dimensions x 8 query heads; the product is tiny, what counts is that the bounds are read once and wide): sum_d max(q lo, q hi) is the product of q's
// positive part with the greatest and of its negative part with the least.  The scores stay in shared memory as numbers that order alike; a cluster's CTAs tell
// each other theirs, where all have room for them, and then each finds the threshold by itself.  It is found by histograms: of 2048 bins over the range that the scores
// have, then over the bin with the threshold in it, until that holds nothing but scores that are taken, or one value; one to three rounds.  (Digits of the scores
// themselves, whose leading ones hardly differ, put all on a few counters; histograms that a cluster fills together cost two of its barriers a round, 2 us.)  Then
// every CTA writes those of its blocks that are above the threshold, and as many of those at it, from the lowest on, as there is room for.
constexpr int MAX_CLUSTER = 8, BINS = 2048;
constexpr int64_t MAX_BLOCKS = 1 << 18, MAX_TOTAL = 65536, MAX_ITEMS = 1 << 24;
constexpr int MOST_SCORES = MAX_BLOCKS / MAX_CLUSTER; // of a CTA: of its share; gathered, or with the blocks' numbers beside them, half as many and as many again
struct ChoiceParams {
    const half* q;
    int64_t q_stride, pages_stride;
    const int8_t* bounds;
    const half* scale;
    const int32_t *pages, *lengths;
    int32_t* lists;           // [batch, kv_heads, total]: blocks of the cache, or -1
    int32_t* listed_tokens;   // [batch]
    int32_t* optional_blocks; // [batch, kv_heads, total]
    int64_t tokens_in_table, items;
    int32_t kv_heads, shared, block, per_page, num_pages, first, last, top, total;
    uint32_t block_magic, block_shift, page_magic, page_shift; // / block, / per_page
    int32_t share, kept_keys; // blocks of a CTA at most, a multiple of 16; scores that it keeps
    bool gathered, units_kept;
};

__device__ __forceinline__ void mma_s8(int32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Numbers that order as the floats do; 0 is below all of them.
__device__ __forceinline__ uint32_t ordered(float f) {
    const uint32_t b = __float_as_uint(f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ void add_in_cluster(uint32_t addr, uint32_t v) {
    asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void min_in_cluster(uint32_t addr, uint32_t v) {
    asm volatile("red.relaxed.cluster.shared::cluster.min.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void max_in_cluster(uint32_t addr, uint32_t v) {
    asm volatile("red.relaxed.cluster.shared::cluster.max.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint4 ld4_in_cluster(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t ld_in_cluster(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

template <int D, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) choose_blocks_kernel(const __grid_constant__ ChoiceParams p) {
    constexpr int TPB = 32 * WARPS;
    constexpr int KB = D / 4, KP = piece(KB), KN = KB / KP, KW = KP / 4; // a quad's lane has a quarter of a row, in pieces
    constexpr int MMAS = D / 32, TILES = D == 256 ? 1 : 2;               // tiles of 16 blocks that a warp has on their way together
    constexpr int PIECES = (D + TPB - 1) / TPB;                          // of q, eight dimensions each, a thread
    // Scores: of the CTA's share; gathered: of all blocks, each CTA's share in every CTA.  Where there is room, the share's blocks' numbers in the cache.
    extern __shared__ uint32_t keys[];
    int32_t* const units = p.units_kept ? reinterpret_cast<int32_t*>(keys + p.kept_keys) : nullptr;
    __shared__ __align__(16) uint32_t q8[8][D / 4];
    __shared__ uint32_t q_bits[8];
    __shared__ float q_scale[8]; // of a head without a say, or beyond the last: NaN
    // each CTA's own where scores are gathered, else the cluster's first CTA's
    __shared__ __align__(16) uint32_t histogram[BINS];
    __shared__ __align__(16) uint32_t found[4]; // least and greatest of the range; how many of it are taken; whether these are all of it
    __shared__ uint32_t above, at_threshold; // counts of this CTA
    __shared__ uint32_t scan[WARPS][2];
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), g = lane >> 2, t = lane & 3;
    const int32_t ctas = gridDim.x, rank = blockIdx.x; // one cluster along x
    const int64_t item = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
    if (item >= p.items) return; // (the whole cluster)
    const int64_t b = item / p.kv_heads;
    const int32_t kvh = (int32_t)(item - b * p.kv_heads);
    for (int x = threadIdx.x; x < BINS; x += TPB) histogram[x] = 0;
    if (threadIdx.x == 0) found[0] = 0xffffffffu, found[1] = 0, above = at_threshold = 0;
    pdl_wait_prior_grid();
    pdl_launch_dependents();

    // q of up to eight heads, and the length: on their way together
    const half* const q = p.q + b * p.q_stride + (int64_t)kvh * p.shared * D;
    uint4 raw[PIECES];
    auto load_q = [&](int32_t head0) {
        const int heads = min(8, p.shared - head0);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int x = threadIdx.x + i * TPB;
            raw[i] = x < heads * (D / 8) ? ld_global_16(q + (int64_t)head0 * D + x * 8) : make_uint4(0, 0, 0, 0);
        }
    };
    load_q(0);
    const int32_t n = (int32_t)min((int64_t)max(p.lengths[b], 0), p.tokens_in_table);
    const int32_t blocks = (uint32_t)((uint64_t)(uint32_t)(n + p.block - 1) * p.block_magic >> p.block_shift);
    const int32_t* const row_pages = p.pages + b * p.pages_stride;
    int32_t* const list = p.lists + item * p.total;
    int32_t* const told = p.optional_blocks ? p.optional_blocks + item * p.total : nullptr;
    const int32_t count = min(blocks, p.total);
    auto page_index = [&](int32_t block) { return (int32_t)(uint32_t)((uint64_t)(uint32_t)block * p.page_magic >> p.page_shift); };
    auto unit_of = [&](int32_t block, int32_t page) { return (uint32_t)page < (uint32_t)p.num_pages ? page * p.per_page + (block - page_index(block) * p.per_page) : -1; };
    auto put = [&](int32_t at, int32_t block, int32_t unit) {
        list[at] = unit;
        if (told) told[at] = block;
    };
    if (rank == 0 && kvh == 0 && threadIdx.x == 0) p.listed_tokens[b] = count == 0 ? 0 : n - (blocks - count) * p.block;
    if (told)
        for (int32_t i = count + rank * TPB + threadIdx.x; i < p.total; i += ctas * TPB) told[i] = -1;
    if (blocks <= p.total) { // all of them
        for (int32_t i = rank * TPB + threadIdx.x; i < count; i += ctas * TPB) put(i, i, unit_of(i, row_pages[page_index(i)]));
        return;
    }
    // the first and the last ones: their pages are looked up now, by the cluster's last CTA, and used at the end (the first TPB of them)
    const int32_t kept = p.first + p.last;
    auto kept_block = [&](int32_t i) { return i < p.first ? i : blocks - kept + i; };
    const bool keeps = rank == ctas - 1;
    int32_t kept_page = keeps && (int32_t)threadIdx.x < kept ? row_pages[page_index(kept_block(threadIdx.x))] : -1;
    auto put_kept = [&] {
        if (!keeps) return;
        for (int32_t i = threadIdx.x; i < kept; i += TPB) {
            const int32_t block = kept_block(i), page = i < TPB ? kept_page : row_pages[page_index(block)];
            put(i < p.first ? i : p.top + i, block, unit_of(block, page));
        }
    };
    const int32_t between = blocks - kept; // more than p.top
    if (p.top == 0) {
        put_kept();
        return;
    }

    // ---- scores of this CTA's share ------------------------------------------------------------------------------------------
    if (ctas > 1 && p.gathered) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const int32_t share = (between + ctas * 16 - 1) / (ctas * 16) * 16;
    const int32_t begin = min(between, rank * share), mine = min(between, begin + share) - begin;
    uint32_t* const mine_keys = keys + (p.gathered ? begin : 0);
    // A warp has up to TILES * 16 neighbouring blocks at once; lane l looks after block l of them: its page, a round ahead, its place, its scale.
    const int32_t at_once = mine > WARPS * 16 ? TILES * 16 : 16;
    int32_t page_of_mine = -1;
    auto look_up = [&](int32_t tile) {
        const int32_t x = tile + lane;
        page_of_mine = lane < at_once && x < mine ? row_pages[page_index(p.first + begin + x)] : -1;
    };
    // Bounds and scales of a round of blocks.  What is not there reads those of the cache's first block, and
    // comes behind everything.
    uint32_t lo[TILES][2][KN][KW], hi[TILES][2][KN][KW], state = 0; // state: the scale, and above it whether the block is there
    auto load = [&](int32_t tile) {
        const int32_t unit = lane < at_once && tile + lane < mine ? unit_of(p.first + begin + tile + lane, page_of_mine) : -1;
        const int64_t of_mine = unit >= 0 ? ((int64_t)page_of_mine * p.kv_heads + kvh) * p.per_page + (unit - page_of_mine * p.per_page) : 0;
        state = unit >= 0 ? 0x10000u : 0u;
        if (p.num_pages > 0) {
            state |= __half_as_ushort(ld_global_half(p.scale + of_mine));
#pragma unroll
            for (int m = 0; m < TILES; ++m)
                if (m * 16 < at_once) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int64_t at = __shfl_sync(0xffffffffu, of_mine, m * 16 + g + 8 * r);
                        const char* const src = (const char*)p.bounds + at * 2 * D + t * KP;
#pragma unroll
                        for (int i = 0; i < KN; ++i) {
                            load_piece<KP>(lo[m][r][i], src + i * 4 * KP);
                            load_piece<KP>(hi[m][r][i], src + D + i * 4 * KP);
                        }
                    }
                }
        }
        if (units && lane < at_once && tile + lane < mine) units[tile + lane] = unit;
        look_up(tile + WARPS * at_once);
    };
    uint32_t lowest = 0xffffffffu, highest = 0;
    for (int32_t head0 = 0; head0 < p.shared; head0 += 8) {
        const int heads = min(8, p.shared - head0);
        const bool ends = head0 + 8 >= p.shared;
        look_up(warp * at_once);
        if (threadIdx.x < 8) q_bits[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int x = threadIdx.x + i * TPB;
            const uint32_t w[4] = {raw[i].x & 0x7fff7fffu, raw[i].y & 0x7fff7fffu, raw[i].z & 0x7fff7fffu, raw[i].w & 0x7fff7fffu};
            uint32_t m = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) m = max(m, max(w[k] & 0xffffu, w[k] >> 16));
            if constexpr (32 % (D / 8) == 0) { // a head's pieces lie in one warp
#pragma unroll
                for (int k = 1; k < D / 8; k <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, k));
                if (x < heads * (D / 8) && x % (D / 8) == 0) q_bits[x / (D / 8)] = m;
            } else if (x < heads * (D / 8)) {
                atomicMax(&q_bits[x / (D / 8)], m);
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int x = threadIdx.x + i * TPB, h = x / (D / 8);
            if (x >= 8 * (D / 8)) break;
            uint2 o = make_uint2(0, 0);
            float scale = __int_as_float(0x7fffffff);
            if (h < heads && q_bits[h] < 0x7c00u) {
                const half s = outer_scale(__half2float(__ushort_as_half((unsigned short)q_bits[h])));
                scale = __half2float(s);
                Eight e;
                e.raw = raw[i];
                o = Quotient(s).eight(e);
            }
            if (x % (D / 8) == 0) q_scale[h] = scale;
            q8[h][(x - h * (D / 8)) * 2] = o.x;
            q8[h][(x - h * (D / 8)) * 2 + 1] = o.y;
        }
        __syncthreads();
        load(warp * at_once);
        if (!ends) load_q(head0 + 8);
        // a product's dimensions come as the lane has them: words 2 m and 2 m + 1 of its own
        uint32_t plus[MMAS][2], minus[MMAS][2];
#pragma unroll
        for (int m = 0; m < MMAS; ++m)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int word = 2 * m + x, i = word / KW, s = word - i * KW;
                const uint32_t w = q8[g][(i * 4 + t) * KW + s], negative = ((w >> 7) & 0x01010101u) * 255u;
                plus[m][x] = w & ~negative;
                minus[m][x] = w & negative;
            }
        const float qs[2] = {q_scale[2 * t], q_scale[2 * t + 1]}; // of heads 2 t and 2 t + 1
        for (int32_t tile = warp * at_once; tile < mine; tile += WARPS * at_once) {
#pragma unroll
            for (int m = 0; m < TILES; ++m)
                if (m * 16 < at_once) {
                    int32_t c[4] = {}, c2[4] = {};
#pragma unroll
                    for (int k = 0; k < MMAS; ++k) {
                        const int w = 2 * k, i = w / KW, s = w - i * KW;
                        mma_s8(c, lo[m][0][i][s], lo[m][1][i][s], lo[m][0][i][s + 1], lo[m][1][i][s + 1], minus[k][0], minus[k][1]);
                        mma_s8(c2, hi[m][0][i][s], hi[m][1][i][s], hi[m][0][i][s + 1], hi[m][1][i][s + 1], plus[k][0], plus[k][1]);
                    }
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const uint32_t of_row = __shfl_sync(0xffffffffu, state, m * 16 + g + 8 * r);
                        const half scale = __ushort_as_half((unsigned short)of_row);
                        const float f = __half2float(scale);
                        uint32_t key = 0;
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const float score = __fmul_rn((float)(c[2 * r + x] + c2[2 * r + x]), qs[x] * f);
                            if (qs[x] == qs[x]) key = max(key, ordered(score));
                        }
                        key = max(key, __shfl_xor_sync(0xffffffffu, key, 1));
                        key = max(key, __shfl_xor_sync(0xffffffffu, key, 2));
                        if (!is_finite(scale)) key = 0xffffffffu;
                        key = of_row >> 16 ? max(key, 1u) : 0u; // holes come behind everything that is there
                        const int32_t x = tile + m * 16 + g + 8 * r;
                        if (t == 0 && x < mine) {
                            if (head0 > 0) key = max(key, mine_keys[x]);
                            mine_keys[x] = key;
                            if (ends) lowest = min(lowest, key), highest = max(highest, key);
                        }
                    }
                }
            if (tile + WARPS * at_once < mine) load(tile + WARPS * at_once);
        }
    }
    put_kept(); // their pages are there by now

    // ---- the threshold ---------------------------------------------------------------------------------------------------------
    const bool alone = ctas == 1 || p.gathered; // every CTA finds it by itself, with barriers of its own
    auto sync = [&] {
        if (alone) __syncthreads();
        else cluster_sync_all();
    };
    if (ctas > 1 && p.gathered) {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); // all CTAs are there
        __syncthreads();
        for (int32_t r = 0; r < ctas; ++r) {
            if (r == rank) continue;
            const uint32_t there = map_to_cta(ptx::smem_addr(mine_keys), r);
            for (int32_t x = threadIdx.x; x < mine; x += TPB) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there + x * 4), "r"(mine_keys[x]) : "memory");
        }
        cluster_sync_all(); // from here on nobody looks into another CTA
        lowest = 0xffffffffu;
        highest = 0;
        for (int32_t x = threadIdx.x; x < between; x += TPB) lowest = min(lowest, keys[x]), highest = max(highest, keys[x]);
    }
    const int32_t looked_at = ctas > 1 && p.gathered ? between : mine;
    const uint32_t first = alone ? rank : 0, bins0 = map_to_cta(ptx::smem_addr(histogram), first), found0 = map_to_cta(ptx::smem_addr(found), first);
    lowest = __reduce_min_sync(0xffffffffu, lowest);
    highest = __reduce_max_sync(0xffffffffu, highest);
    sync(); // the histogram and the range are there
    if (lane == 0 && lowest <= highest) min_in_cluster(found0, lowest), max_in_cluster(found0 + 4, highest);
    sync();
    uint4 now = ld4_in_cluster(found0);
    uint32_t least = now.x, most = now.y, room = p.top, all = 0; // of the scores in [least, most], `room` are taken
    for (;;) {
        const uint32_t shift = max(0, 21 - __clz((int)(most - least))); // 2048 bins at most
        for (int32_t x = threadIdx.x; x < looked_at; x += TPB)
            if (keys[x] >= least && keys[x] <= most) add_in_cluster(bins0 + ((keys[x] - least) >> shift) * 4, 1);
        sync();
        if (alone || rank == 0) {
            // bins from the highest down: thread x has EACH of them, from BINS - EACH x - 1 on
            constexpr int EACH = BINS / TPB;
            uint32_t n_of[EACH], own = 0;
#pragma unroll
            for (int k = 0; k < EACH; k += 4) {
                uint4* const here = reinterpret_cast<uint4*>(histogram + BINS - EACH * threadIdx.x - 4 - k);
                const uint4 v = *here;
                *here = make_uint4(0, 0, 0, 0);
                n_of[k] = v.w; n_of[k + 1] = v.z; n_of[k + 2] = v.y; n_of[k + 3] = v.x;
                own += v.x + v.y + v.z + v.w;
            }
            uint32_t sum = own;
#pragma unroll
            for (int m = 1; m < 32; m <<= 1) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, sum, m);
                if (lane >= m) sum += v;
            }
            if (lane == 31) scan[warp][0] = sum;
            __syncthreads();
            sum += __reduce_add_sync(0xffffffffu, lane < warp ? scan[lane][0] : 0u);
            uint32_t over = sum - own;
            if (over < room && sum >= room) {
#pragma unroll
                for (int k = 0; k < EACH; ++k) {
                    if (over < room && over + n_of[k] >= room) {
                        const uint32_t bin = BINS - 1 - EACH * threadIdx.x - k;
                        const uint32_t begins = least + (bin << shift), width = (1u << shift) - 1;
                        *reinterpret_cast<uint4*>(found) = make_uint4(begins, most - begins < width ? most : begins + width, room - over, n_of[k] == room - over);
                    }
                    over += n_of[k];
                }
            }
        }
        sync();
        now = ld4_in_cluster(found0);
        least = now.x; most = now.y; room = now.z; all = now.w;
        if (shift == 0 || all) break;
    }

    // ---- what is above the threshold, and the first `room` of those at it, in order ------------------------------------------------
    auto over_it = [&](uint32_t key) { return all ? key >= least : key > least; };
    auto at_it = [&](uint32_t key) { return !all && key == least; };
    uint32_t before[2] = {};
    if (ctas > 1) { // those of the shares before this one
        uint32_t counts[2] = {};
        const int32_t end = p.gathered ? begin : mine;
        for (int32_t x = threadIdx.x; x < end; x += TPB) {
            counts[0] += over_it(keys[x]);
            counts[1] += at_it(keys[x]);
        }
        counts[0] = __reduce_add_sync(0xffffffffu, counts[0]);
        counts[1] = __reduce_add_sync(0xffffffffu, counts[1]);
        if (lane == 0) atomicAdd(&above, counts[0]), atomicAdd(&at_threshold, counts[1]);
        sync();
        if (p.gathered) {
            before[0] = above;
            before[1] = at_threshold;
        } else {
            for (int32_t r = 0; r < rank; ++r) {
                before[0] += ld_in_cluster(map_to_cta(ptx::smem_addr(&above), r));
                before[1] += ld_in_cluster(map_to_cta(ptx::smem_addr(&at_threshold), r));
            }
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); // nothing of another CTA's is read any more
        }
    }
    for (int32_t x0 = 0; x0 < mine; x0 += TPB) {
        const int32_t x = x0 + threadIdx.x, block = p.first + begin + x;
        const uint32_t key = x < mine ? mine_keys[x] : 0u;
        const bool over = x < mine && over_it(key), same = x < mine && at_it(key);
        int32_t unit = -1;
        if (over || same) unit = units ? units[x] : unit_of(block, row_pages[page_index(block)]);
        const uint32_t overs = __ballot_sync(0xffffffffu, over), sames = __ballot_sync(0xffffffffu, same), below = (1u << lane) - 1;
        if (lane == 0) scan[warp][0] = __popc(overs), scan[warp][1] = __popc(sames);
        __syncthreads();
        const uint32_t in_warps[2] = {lane < WARPS ? scan[lane][0] : 0u, lane < WARPS ? scan[lane][1] : 0u};
        const uint32_t o = before[0] + __popc(overs & below) + __reduce_add_sync(0xffffffffu, lane < warp ? in_warps[0] : 0u);
        const uint32_t s = before[1] + __popc(sames & below) + __reduce_add_sync(0xffffffffu, lane < warp ? in_warps[1] : 0u);
        before[0] += __reduce_add_sync(0xffffffffu, in_warps[0]);
        before[1] += __reduce_add_sync(0xffffffffu, in_warps[1]);
        if (over || (same && s < room)) put(p.first + o + min(s, room), block, unit);
        __syncthreads();
    }
    if (!alone) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); // no CTA leaves while another reads its shared memory
}

int32_t check_bounds(const pplb200_kv_cache* c, const pplb200_key_bounds* k) {
    const int32_t rc = check_kv_cache(c);
    if (rc != RC_SUCCESS) return rc;
    if (!k) return fail(RC_INVALID_VALUE, "null bounds");
    if (c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128 && c->head_dim != 256)
        return fail(RC_UNSUPPORTED, "key bounds: head_dim must be 64, 96, 128 or 256, got %d", c->head_dim);
    if (k->block <= 0 || k->block % 16 || c->page_size % k->block)
        return fail(RC_INVALID_VALUE, "a block must be a multiple of 16 tokens that divides a page (%d), got %d", c->page_size, k->block);
    if (k->block > 1 << 30) return fail(RC_UNSUPPORTED, "a block of more than 2^30 tokens");
    if (c->num_pages == 0) return RC_SUCCESS;
    if (!k->bounds || !k->scale || !aligned16(k->bounds) || ((uintptr_t)k->scale & 1)) return fail(RC_INVALID_VALUE, "bounds must be 16-byte, their scales 2-byte aligned pointers");
    if ((__int128)c->num_pages * c->kv_heads * (c->page_size / k->block) * 2 * c->head_dim >> 61) return fail(RC_INVALID_VALUE, "bounds of too many blocks");
    return RC_SUCCESS;
}

int64_t list_bytes(int64_t batch, int32_t kv_heads, int64_t total) { return round_up(batch * kv_heads * total * 4, 256) + round_up(batch * 4, 256); }

template <int D>
void launch_bounds_of(cudaStream_t stream, const BoundsParams& p, dim3 grid) {
    if (p.cache.quant_group == 0) launch_ex(key_bounds_kernel<D, CACHE_F16>, grid, dim3(BTPB), stream, true, p);
    else if (p.cache.quant_group == 8) launch_ex(key_bounds_kernel<D, CACHE_I8_GROUPS>, grid, dim3(BTPB), stream, true, p);
    else launch_ex(key_bounds_kernel<D, CACHE_I8_ROWS>, grid, dim3(BTPB), stream, true, p);
}

template <int D, int WARPS>
int32_t launch_choice(cudaStream_t stream, const ChoiceParams& p, int32_t cluster) {
    const int64_t y = std::min<int64_t>(p.items, 32768);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)cluster, (unsigned)y, (unsigned)((p.items + y - 1) / y));
    cfg.blockDim = dim3(32 * WARPS);
    cfg.dynamicSmemBytes = (size_t)(p.kept_keys + (p.units_kept ? p.share : 0)) * 4;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (cfg.dynamicSmemBytes > 32768) { // beyond what a kernel has without being asked for, its static 11 KB included: always the same, since another thread may be about to launch
        const cudaError_t e = cudaFuncSetAttribute(choose_blocks_kernel<D, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_SCORES * 4);
        if (e != cudaSuccess) return fail(RC_DEVICE_RUNTIME_ERROR, "choice of blocks: %s", cudaGetErrorString(e));
    }
    cudaLaunchKernelEx(&cfg, choose_blocks_kernel<D, WARPS>, p);
    return check_launch("choice of blocks");
}

} // namespace
} // namespace pplb200

using namespace pplb200;

extern "C" {

int32_t pplb200_key_bounds_update(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_key_bounds* bounds, const int64_t* slots, int64_t tokens) {
    const int32_t rc = check_bounds(cache, bounds);
    if (rc != RC_SUCCESS) return rc;
    if (tokens < 0) return fail(RC_INVALID_VALUE, "negative extent");
    if (tokens > 0x7fffffffLL) return fail(RC_UNSUPPORTED, "more than 2^31 - 1 tokens");
    if (tokens == 0) return RC_SUCCESS;
    if (!slots || ((uintptr_t)slots & 7)) return fail(RC_INVALID_VALUE, "slots must be an 8-byte aligned pointer");
    if (cache->num_pages == 0) return RC_SUCCESS;
    BoundsParams p = {};
    p.cache = *cache;
    p.bounds = (int8_t*)bounds->bounds; p.scale = (half*)bounds->scale;
    p.slots = slots; p.tokens = tokens;
    p.block = bounds->block; p.per_page = cache->page_size / bounds->block;
    small_division(p.block, p.block_magic, p.block_shift);
    // one slot a CTA while that makes no more than eight CTAs an SM, then more of them, and in a long prompt as many as a block has, so that each CTA has one block (16384
    // tokens of 8 heads, blocks of 64, int8 rows: 7.1 us; with 27 slots, which makes eight CTAs an SM, most of them idle, 9.0; with 8 12.5)
    const int64_t heads = (cache->kv_heads + BWARPS - 1) / BWARPS;
    const int64_t share = tokens * heads / (8 * kSms), whole = std::min(p.block, BTPB);
    p.slots_here = (int32_t)(share >= 16 ? whole : std::min(whole, std::max<int64_t>(1, share)));
    const dim3 grid((unsigned)((tokens + p.slots_here - 1) / p.slots_here), (unsigned)heads);
    if (cache->head_dim == 64) launch_bounds_of<64>((cudaStream_t)stream, p, grid);
    else if (cache->head_dim == 96) launch_bounds_of<96>((cudaStream_t)stream, p, grid);
    else if (cache->head_dim == 128) launch_bounds_of<128>((cudaStream_t)stream, p, grid);
    else launch_bounds_of<256>((cudaStream_t)stream, p, grid);
    return check_launch("key bounds");
}

int32_t pplb200_key_bounds_read(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_key_bounds* bounds, const int64_t* blocks, int64_t count,
                                float* lo, float* hi) {
    const int32_t rc = check_bounds(cache, bounds);
    if (rc != RC_SUCCESS) return rc;
    if (count < 0) return fail(RC_INVALID_VALUE, "negative extent");
    if (count == 0) return RC_SUCCESS;
    if (!blocks || ((uintptr_t)blocks & 7)) return fail(RC_INVALID_VALUE, "blocks must be an 8-byte aligned pointer");
    if (!lo || !hi || !aligned16(lo) || !aligned16(hi)) return fail(RC_INVALID_VALUE, "lo and hi must be 16-byte aligned pointers");
    if (count > (1LL << 38) / (cache->kv_heads * (int64_t)cache->head_dim)) return fail(RC_UNSUPPORTED, "too many elements");
    BoundsReadParams p = {};
    p.bounds = (const int8_t*)bounds->bounds; p.scale = (const half*)bounds->scale;
    p.blocks = blocks; p.lo = lo; p.hi = hi; p.count = count;
    p.per_page = cache->page_size / bounds->block; p.kv_heads = cache->kv_heads; p.head_dim = cache->head_dim;
    p.all_blocks = cache->num_pages * p.per_page;
    const int64_t shares = ((int64_t)p.kv_heads * p.head_dim / 2 + BTPB - 1) / BTPB;
    launch_ex(key_bounds_read_kernel, dim3((unsigned)std::min<int64_t>(count, 1 << 20), (unsigned)std::min<int64_t>(shares, 65535)), dim3(BTPB), (cudaStream_t)stream, true, p);
    return check_launch("key bounds read");
}

int64_t pplb200_block_sparse_attention_workspace_bytes(int64_t batch, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t attended_blocks) {
    if (batch < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || head_dim <= 0 || attended_blocks < 0 || batch > MAX_ITEMS / kv_heads) return -1;
    return workspace_bytes(q_heads / kv_heads, head_dim) + list_bytes(batch, kv_heads, attended_blocks);
}

int32_t pplb200_block_sparse_attention_fp16(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_key_bounds* bounds,
                                            const pplb200_paged_attention_args* a, const pplb200_block_choice* choice) {
    AttentionParams own = {};
    int32_t rc = take_call(cache, a, own);
    if (rc != RC_SUCCESS) return rc;
    if ((rc = check_bounds(cache, bounds)) != RC_SUCCESS) return rc;
    if (!choice) return fail(RC_INVALID_VALUE, "null choice");
    if (a->window) return fail(RC_UNSUPPORTED, "chosen blocks are not seen through a window");
    if (choice->first < 0 || choice->last < 1 || choice->top < 0) return fail(RC_INVALID_VALUE, "first and top must not be negative, last at least 1");
    const int64_t total = (int64_t)choice->first + choice->last + choice->top;
    const int64_t per_page = cache->page_size / bounds->block, in_table = a->pages_per_sequence * per_page;
    if (total > MAX_TOTAL || total * bounds->block > (1LL << 30)) return fail(RC_UNSUPPORTED, "too many blocks to attend: %lld", (long long)total);
    if (in_table > MAX_BLOCKS) return fail(RC_UNSUPPORTED, "a page table of more than 2^18 blocks");
    if ((__int128)cache->num_pages * per_page > 0x7fffffff) return fail(RC_UNSUPPORTED, "a cache of 2^31 blocks");
    if (a->batch > MAX_ITEMS / cache->kv_heads) return fail(RC_UNSUPPORTED, "more than 2^24 choices");
    if ((uintptr_t)choice->optional_blocks & 3) return fail(RC_INVALID_VALUE, "the chosen blocks must be 4-byte aligned");
    if (a->batch == 0) return RC_SUCCESS;
    const int64_t need = pplb200_block_sparse_attention_workspace_bytes(a->batch, a->q_heads, cache->kv_heads, cache->head_dim, (int32_t)total);
    if (!a->ws || a->ws_bytes < need || ((uintptr_t)a->ws & 255))
        return fail(RC_INVALID_VALUE, "workspace of %lld bytes (256-byte aligned) needed, got %lld", (long long)need, (long long)a->ws_bytes);
    int32_t* const lists = (int32_t*)((char*)a->ws + need - list_bytes(a->batch, cache->kv_heads, total));
    ChoiceParams p = {};
    p.q = own.q; p.q_stride = own.q_stride; p.pages = own.pages; p.pages_stride = own.pages_stride; p.lengths = own.lengths;
    p.bounds = (const int8_t*)bounds->bounds; p.scale = (const half*)bounds->scale;
    p.lists = lists;
    p.listed_tokens = (int32_t*)((char*)lists + round_up(a->batch * cache->kv_heads * total * 4, 256));
    p.optional_blocks = choice->optional_blocks;
    p.tokens_in_table = own.tokens_in_table;
    p.items = a->batch * cache->kv_heads;
    p.kv_heads = cache->kv_heads; p.shared = a->q_heads / cache->kv_heads;
    p.block = bounds->block; p.per_page = (int32_t)per_page; p.num_pages = own.num_pages;
    p.first = choice->first; p.last = choice->last; p.top = choice->top; p.total = (int32_t)total;
    small_division(p.block, p.block_magic, p.block_shift);
    small_division(p.per_page, p.page_magic, p.page_shift);
    // Sixteen warps a CTA where there are few choices, which then take 512 blocks in one round of loads (whole calls, one sequence, 8 key heads: 1024 blocks 26 us, with four
    // warps 33; 16 sequences, 375 blocks 36, 40); four for many or short ones, so that several share an SM (64 sequences, 250 blocks 91, with sixteen 96; 16 of 63
    // 29, 35).  Clusters, whose barriers cost a microsecond each, only where a CTA would have more rounds to go (32 choices of 257 blocks 17 us, by four CTAs each 21; 8 of 2048
    // by one CTA each 34, by eight 27), and for room for the scores (128 KB).
    const bool wide = p.items <= kSms && in_table > 128;
    int32_t cluster = 1;
    while (cluster < MAX_CLUSTER && ((p.items * cluster * 2 <= kSms && in_table > 512 && in_table > cluster * 128) || in_table > cluster * 32768LL)) cluster *= 2;
    p.share = (int32_t)std::max<int64_t>(16, (in_table + cluster * 16 - 1) / (cluster * 16) * 16);
    p.gathered = cluster > 1 && (int64_t)p.share * cluster <= MOST_SCORES / 2;
    p.kept_keys = p.gathered ? p.share * cluster : p.share;
    p.units_kept = p.share <= MOST_SCORES / 2;
    const cudaStream_t s = (cudaStream_t)stream;
    const auto launch_dims = [&](auto warps) {
        constexpr int W = decltype(warps)::value;
        if (cache->head_dim == 64) return launch_choice<64, W>(s, p, cluster);
        if (cache->head_dim == 96) return launch_choice<96, W>(s, p, cluster);
        if (cache->head_dim == 128) return launch_choice<128, W>(s, p, cluster);
        return launch_choice<256, W>(s, p, cluster);
    };
    rc = wide ? launch_dims(std::integral_constant<int, 16>()) : launch_dims(std::integral_constant<int, 4>());
    if (rc != RC_SUCCESS) return rc;
    own.pages = lists;
    own.pages_stride = cache->kv_heads * total;
    own.pages_head_stride = total;
    own.lengths = p.listed_tokens;
    own.tokens_in_table = total * bounds->block;
    own.unit_tokens = bounds->block;
    own.units_per_page = (int32_t)per_page;
    own.num_units = (int32_t)(own.num_pages * per_page);
    own.rows_per_head = p.shared;
    lay_out(own, a->ws, p.shared);
    return launch_general(s, own);
}

} // extern "C"
