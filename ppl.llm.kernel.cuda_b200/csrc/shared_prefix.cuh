// The prefix that a batch shares, for many rows of q at once: scores and weighted sums on tcgen05, statistics in registers.
//
// A row is a query head of one sequence; the rows that ask one key head are a matrix, and so this is a product of it with the keys, a softmax by rows that is
// never whole in one place, and a product with the values.  A CTA has up to 256 rows of a key head in two tiles of 128 and goes through a part of the
// prefix in blocks of NB tokens; its sums and reference exponents are left as one of `splits` parts, which are joined where the output is written.
//
//   warps 0 - 3, 4 - 7   softmax of one tile each, a thread a row (tensor memory's lanes): scores in, weights out, in place
//   warps 8 - 11         keys from the pages into shared memory; int8 ones are widened on the way
//   warps 12 - 15        values
//   warp 16              issues all products, and owns the tensor memory
//
// The two tiles' products and softmaxes alternate, so that the tensor cores work on one while the exponentials of the other are computed.  Where a CTA has one
// tile only, the two softmax groups take turns at the blocks of it, each with a sum of its own (heads of 256: one group, whose sum alone fills
// half of the tensor memory, over two buffers of scores).
//
// Bound by the tensor cores and the exponentials: a block of 128 tokens of two tiles of heads of 128 is 2048 clocks of either.  64 sequences of 64 heads over 8 with 100
// tokens each behind 32768: fp16 88 us, 780 TFLOP/s (1270 for the 20000 tokens from 12345 on; with the products alone the call took 71 us, then of 93), int8 rows 128
// and groups of 8 160: there the loading warps widen every element, for each tile or pair of tiles, the weights are two operands, and groups' keys too.  What a call takes besides,
// 10 to 30 us, is the start, q, the parts' sums (64 KB a tile and part) and their joining, and own tokens that do not fit beside it.
// Tried on fp16 and left, since none changed a block's time: two softmax groups a tile, half of the exponentials as polynomials of degree 3 to 5, looking whether the reference
// exponent has to move after the weights instead of before them.
// Weights are fp16 of 2^-24 to 2^14, over an fp16 cache 11 bits, off by at most 2^-11 of themselves, as much as the output's own rounding; their sum is of what they were.  (In two
// operands, 22 bits, as over int8: 85 us would be 99, the relative error 0.00021 instead of 0.00024, 2-norm, of which the output's rounding is 0.00021.)  v of groups of 8 is
// rounded to fp16 itself, and the two errors came to half as much again as the output's: over int8 caches the weights are two operands, 22 bits.  v of rows is whole numbers, and
// its scales are in the weights, so that any finite scale is taken, as by decode attention, and nothing but the output is rounded to fp16 (relative error 0.00021, 2-norm).
// The code of the softmax is long: where a form of it is only there for rare blocks, it is a loop (unrolled four times, the whole call took 2.7 us longer, in fetching instructions).
#pragma once

#include "paged_attention.cuh"
#include "ptx.cuh"

#include <type_traits>

namespace pplb200 {
namespace prefix {

using namespace paged;

// How long the warp that issues the products waits for the values of task i.  (Tests of what is left behind a wait that gives up build the kernel with another limit.)
__device__ __forceinline__ long long value_wait(int32_t i, int32_t tasks) {
#ifdef PPLB200_IMPATIENT_PREFIX
    return i >= tasks - 2 ? -1 : ptx::kWaitCycleLimit;
#else
    return ptx::kWaitCycleLimit;
#endif
}

__device__ unsigned int g_status = 0; // codes of waits that gave up
__device__ uint4 g_nothing[32]; // zeros: what a token that is not there reads
constexpr float kAbove = 4.0f; // where a reference exponent goes above the score that moved it
constexpr unsigned ST_LOAD = 1u, ST_MMA = 2u, ST_SOFTMAX = 4u;

template <int D_, int KIND_>
struct Tile {
    static constexpr int D = D_, KIND = KIND_, ES = KIND == CACHE_F16 ? 2 : 1;
    static constexpr int DP = (D + 63) / 64 * 64, ATOMS = DP / 64; // a row of shared memory is 128 bytes, 64 dimensions
    static constexpr bool LOW = KIND == CACHE_I8_GROUPS;           // keys: value x scale rounded to fp16, and what that left
    static constexpr bool FINE = KIND != CACHE_F16;                // weights: likewise two operands, 22 bits, each 32 tokens' where their scores were
    static constexpr int NB = D == 256 ? 64 : 128;                 // tokens of a block
    static constexpr int STREAMS = D == 256 ? 1 : 2;
    static constexpr int TILES = D == 256 || (LOW && D > 64) ? 1 : 2; // of rows, at most
    static constexpr int KS = D == 64 ? (LOW ? 3 : 4) : LOW && D == 256 ? 1 : 2, VS = D == 64 ? (LOW ? 3 : 4) : LOW && D < 256 ? 1 : 2; // stages of keys and of values
    static constexpr int Q_BYTES = 128 * DP * 2, V_BYTES = NB * DP * 2, K_BYTES = V_BYTES * (LOW ? 2 : 1);
    static constexpr int RING = TILES * Q_BYTES, V_RING = RING + KS * K_BYTES, INFO = V_RING + VS * V_BYTES;
    static constexpr int INFOS = 8; // blocks whose masks and scales are kept: more than stages of values
    static constexpr int SCALES = KIND == CACHE_I8_ROWS ? INFOS * NB * 6 : 0; // of keys, in 32 bits, and of values
    // What is read back of the sums lies over the rings and q, behind the sums that the two groups of one tile exchange (tiles' sums and these are not there at
    // the same time, and one tile's are half as long).
    static constexpr int STAGED_BYTES = STREAMS * 128 * (D + 4) * 4, EXCHANGE = STREAMS == 2 ? D * 512 : 0, ONE_TILE = EXCHANGE + 128 * (D + 4) * 4;
    static constexpr int BODY = INFO + SCALES, LEAST = STAGED_BYTES > ONE_TILE ? STAGED_BYTES : ONE_TILE;
    static constexpr int SMEM = (BODY > LEAST ? BODY : LEAST) + 1024; // the base is rounded up to 1024
    static constexpr int CH = D * ES / 16, LOADS = CH * NB / 128; // pieces of 16 bytes: of a row, and of a block for a thread
    static_assert(CH * NB % 128 == 0 && VS < INFOS);
    static constexpr int THREADS = 640;
    // Registers of softmax, loading and issuing threads: what 640 threads are launched with, 96 each.  (int8 rows of 256: with 152 and 72 its loading warps spill, 64 sequences of 32 heads over 8
    // behind 32768 tokens 139 us, 125 with 160 and 64; of 128 the other way round, 105 and 109.)
    static constexpr bool LEAN = KIND == CACHE_I8_ROWS && D == 256;
    static constexpr int R_SOFTMAX = KIND == CACHE_F16 ? 176 : LEAN ? 160 : 152, R_LOAD = KIND == CACHE_F16 ? 48 : LEAN ? 64 : 72, R_ISSUE = 32;
    static constexpr int KEPT = KIND == CACHE_F16 ? NB : NB / 2; // scores of a row that a softmax thread keeps
    static_assert(2 * R_SOFTMAX + 2 * R_LOAD + R_ISSUE <= 5 * 96);
    static constexpr uint32_t O_COLUMN = 256; // scores: columns 0 and 128
};

struct PrefixParams {
    CUtensorMap kmap, vmap; // box_rows > 0: fp16 pages as [pages, heads, tokens, dimensions]
    int32_t box_rows;       // tokens of a box: a power of two, 16 at least, that divides a page
    const half* q;
    int64_t q_stride;
    const int32_t *pages, *length;
    int64_t tokens_in_table;
    int32_t num_pages, rows, tiles; // rows of a key head, and tiles of rows that a CTA takes at once (1 or 2)
    int32_t items, splits;          // items: groups of rows of a key head
    int32_t rows_per_head, q_heads;
    uint32_t rows_magic, rows_shift, page_magic, page_shift;
    float scale_log2;
    pplb200_kv_cache cache;
    uint32_t* ahead; // what is said to the kernel for the own tokens
    int64_t part_rows;
    float2* part_tops;
    float* part_sums;
};

// Descriptors of rows of 128 bytes with the 128-byte swizzle: K-major (ptx::desc_lo_sw128), or MN-major, 64 dimensions wide, the next 64 `apart` bytes on.
__device__ __forceinline__ uint32_t mn_desc_lo(uint32_t addr, uint32_t apart) { return ((addr & 0x3ffffu) >> 4) | (apart >> 4 << 16); }

// How large a scale is: less than 2^size, -24 to 16.  (An infinite one: as large as a finite one can be.)
__device__ __forceinline__ int32_t size_of(float scale) { return max(-24, min(16, (int32_t)(__float_as_uint(scale) >> 23 & 0xffu) - 126)); }
// 16 bytes of int8 as fp16, whole numbers, in order
__device__ __forceinline__ void whole_numbers(const uint4& raw, uint32_t (&o)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t f = w[i] ^ 0x80808080u;
        o[2 * i] = less_1152(__byte_perm(f, 0x64646464u, 0x4140));
        o[2 * i + 1] = less_1152(__byte_perm(f, 0x64646464u, 0x4342));
    }
}

template <class T>
__global__ void __launch_bounds__(T::THREADS, 1) prefix_tile_kernel(const __grid_constant__ PrefixParams p) {
    extern __shared__ uint8_t raw_smem[];
    __shared__ __align__(8) uint64_t full_k[T::KS], empty_k[T::KS], full_v[T::VS], empty_v[T::VS], info_full[T::INFOS], score_full[2], weight_half[2], weight_full[2], sum_done[2], q_full, all_done, tail_full;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t products_lost; // a wait of the warp that issues them has given up
    __shared__ __align__(16) uint32_t masks[T::INFOS][4]; // (blocks of 64 tokens: two, and two that say that all is there)
    struct __align__(16) Row { // where a token's row and its scales begin
        const char *at, *scale;
    };
    __shared__ Row row_at[2][4][T::NB]; // keys and values, of four blocks
    __shared__ float2 joint[128];
    __shared__ __align__(16) int2 sizes[T::KIND == CACHE_I8_ROWS ? T::INFOS : 1][T::NB / 32]; // of the scales of 32 values: the largest and the least
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t smem = (ptx::smem_addr(raw_smem) + 1023u) & ~1023u;
    auto bar = [](uint64_t& b) { return ptx::smem_addr(&b); };
    auto report = [&](uint32_t b) { // a warp's threads have done their part: one arrival
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(b);
    };
    const bool boxes = T::KIND == CACHE_F16 && p.box_rows > 0; // whole boxes by the TMA unit: one thread reports
    if (threadIdx.x == 0) {
        for (int i = 0; i < T::KS; ++i) ptx::mbar_init(bar(full_k[i]), boxes ? 1 : 4), ptx::mbar_init(bar(empty_k[i]), 1);
        for (int i = 0; i < T::VS; ++i) ptx::mbar_init(bar(full_v[i]), boxes ? 1 : 4), ptx::mbar_init(bar(empty_v[i]), 1);
        for (int i = 0; i < T::INFOS; ++i) ptx::mbar_init(bar(info_full[i]), boxes ? 1 : 4);
        ptx::mbar_init(bar(tail_full), 1);
        for (int i = 0; i < 2; ++i) ptx::mbar_init(bar(score_full[i]), 1), ptx::mbar_init(bar(weight_half[i]), 4), ptx::mbar_init(bar(weight_full[i]), 4), ptx::mbar_init(bar(sum_done[i]), 1);
        ptx::mbar_init(bar(q_full), 8);
        ptx::mbar_init(bar(all_done), 2);
        products_lost = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 16) {
        ptx::tmem_alloc(ptx::smem_addr(&tmem_slot), 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait_prior_grid();
    if (blockIdx.x == 0 && threadIdx.x == 0) let_go_ahead(p.ahead);
    pdl_launch_dependents(); // behind the allocation, so that no later kernel has this SM's tensor memory

    const int32_t item = blockIdx.x / p.splits, split = blockIdx.x - item * p.splits;
    const int32_t per_head = p.items / p.cache.kv_heads, kvh = item / per_head;
    const int32_t row0 = (item - kvh * per_head) * p.tiles * 128;
    const int32_t tiles = p.tiles == 2 && p.rows - row0 > 128 ? 2 : 1;
    const int32_t n = p.num_pages > 0 ? (int32_t)min((int64_t)max(*(const volatile int32_t*)p.length, 0), p.tokens_in_table) : 0;
    const int32_t all_blocks = (n + T::NB - 1) / T::NB;
    const int32_t block0 = (int32_t)((int64_t)all_blocks * split / p.splits), blocks = (int32_t)((int64_t)all_blocks * (split + 1) / p.splits) - block0;
    const int32_t tasks = tiles * blocks; // task i: buffer i & 1, block i / tiles; with two streams also stream i & 1
    const int32_t shift = tiles - 1;

    if (warp >= 16) {
        ptx::registers_down<T::R_ISSUE>();
        if (warp == 16 && tasks > 0) {
            // ---- products, by one lane of a warp that does the same in all -------------------------------------------------------------------------------------------------
            constexpr uint32_t QK = ptx::make_f16_idesc(128, T::NB, false), PV = ptx::make_f16_idesc(128, T::D, true);
            const uint32_t leads = ptx::elect_one();
            bool ok = __all_sync(0xffffffffu, ptx::mbar_wait(bar(q_full), 0, &g_status, ST_MMA));
            auto scores = [&](int32_t i) {
                const int32_t j = i >> shift, stage = j % T::KS;
                if (!(ok = ok && __all_sync(0xffffffffu, ptx::mbar_wait(bar(full_k[stage]), (j / T::KS) & 1, &g_status, ST_MMA)))) return;
                ptx::tc_fence_after();
                const uint32_t q = ptx::desc_lo_sw128(smem + (tiles == 2 ? (i & 1) * T::Q_BYTES : 0)), k = ptx::desc_lo_sw128(smem + T::RING + stage * T::K_BYTES);
                const uint32_t d = tmem + (i & 1) * 128;
#pragma unroll
                for (int s = 0; s < T::D / 16; ++s) {
                    const uint32_t a = q + ((s / 4) * (128 * 128) + (s % 4) * 32) / 16, b = k + ((s / 4) * (T::NB * 128) + (s % 4) * 32) / 16;
                    ptx::mma_f16(d, ptx::desc_from_lo(a), ptx::desc_from_lo(b), QK, s > 0, leads);
                    if constexpr (T::LOW) ptx::mma_f16(d, ptx::desc_from_lo(a), ptx::desc_from_lo(b + T::V_BYTES / 16), QK, 1, leads);
                }
                ptx::mma_commit_by(bar(score_full[i & 1]), leads);
                if (tiles == 1 || (i & 1)) ptx::mma_commit_by(bar(empty_k[stage]), leads);
            };
            scores(0);
            if (tasks > 1) scores(1);
            for (int32_t i = 0; i < tasks && ok; ++i) {
                const int32_t j = i >> shift, stage = j % T::VS;
                if (!(ok = __all_sync(0xffffffffu, ptx::mbar_wait(bar(full_v[stage]), (j / T::VS) & 1, &g_status, ST_MMA, value_wait(i, tasks))))) break;
                const uint32_t v = mn_desc_lo(smem + T::V_RING + stage * T::V_BYTES, T::NB * 128);
                const uint32_t d = tmem + T::O_COLUMN + (T::STREAMS == 2 ? (i & 1) * T::DP : 0), w = tmem + (i & 1) * 128;
                // the weights of the block's first half are worked with while the others are computed
#pragma unroll
                for (int half = 0; half < 2 && ok; ++half) {
                    if (!(ok = __all_sync(0xffffffffu, ptx::mbar_wait(bar(half ? weight_full[i & 1] : weight_half[i & 1]), (i >> 1) & 1, &g_status, ST_MMA)))) break;
                    ptx::tc_fence_after();
#pragma unroll
                    for (int s = half * T::NB / 32; s < (half + 1) * T::NB / 32; ++s) {
                        const uint32_t a = T::FINE ? w + (s >> 1) * 32 + (s & 1) * 8 : w + s * 8;
                        ptx::mma_f16_tmem(d, a, ptx::desc_from_lo(v + s * (2048 / 16)), PV, (T::STREAMS == 2 ? i > 1 : i > 0) || s > 0, leads);
                        if constexpr (T::FINE) ptx::mma_f16_tmem(d, a + 16, ptx::desc_from_lo(v + s * (2048 / 16)), PV, 1, leads);
                    }
                }
                ptx::mma_commit_by(bar(sum_done[i & 1]), leads);
                if (tiles == 1 || (i & 1)) ptx::mma_commit_by(bar(empty_v[stage]), leads);
                if (i + 2 < tasks) scores(i + 2);
            }
            // All that was issued, and whether that is all there is: the softmax has scores, and no more to wait for, where only the last tasks' values are missing.
            if (leads) {
                if (!ok) products_lost = 1;
                ptx::mbar_arrive(bar(all_done));
            }
            __syncwarp();
            ptx::mma_commit_by(bar(all_done), leads);
        }
    } else if (warp >= 8) {
        ptx::registers_down<T::R_LOAD>();
        // ---- keys and values ---------------------------------------------------------------------------------------------------
        const int id = threadIdx.x & 127;
        const bool values = warp >= 12;
        const int stages = values ? T::VS : T::KS, stage_bytes = values ? T::V_BYTES : T::K_BYTES;
        const uint32_t ring = smem + (values ? T::V_RING : T::RING);
        const char* const base = (const char*)(values ? p.cache.v : p.cache.k) + (int64_t)kvh * p.cache.head_stride * T::ES;
        const char* const sbase = (const char*)(values ? p.cache.v_scale : p.cache.k_scale) + (int64_t)kvh * p.cache.scale_head_stride * 2;
        auto full = [&](int stage) { return values ? bar(full_v[stage]) : bar(full_k[stage]); };
        auto empty = [&](int stage) { return values ? bar(empty_v[stage]) : bar(empty_k[stage]); };
        // Where a block's tokens lie, which of them are there, and (rows) the keys' scales: thread id looks after token id, its page three blocks ahead, its row
        // two, and what the softmax has to know is published one ahead.
        int32_t page = -1;
        bool there = false;
        uint32_t scale = 0, value_scale = 0; // fp16
        auto request = [&](int32_t j) {
            const int32_t token = (block0 + j) * T::NB + id;
            page = -1;
            if (j < blocks && id < T::NB && token < n) page = p.pages[(uint32_t)((uint64_t)(uint32_t)token * p.page_magic >> p.page_shift)];
        };
        auto locate = [&](int32_t j) {
            const int32_t token = (block0 + j) * T::NB + id;
            there = j < blocks && (uint32_t)page < (uint32_t)p.num_pages;
            const int32_t in_page = token - (int32_t)((uint32_t)((uint64_t)(uint32_t)token * p.page_magic >> p.page_shift)) * p.cache.page_size;
            Row to = {reinterpret_cast<const char*>(g_nothing), reinterpret_cast<const char*>(g_nothing)};
            if (there) {
                to.at = base + kv_row(page, in_page, 0, p.cache.page_stride, 0, p.cache.token_stride) * T::ES;
                if constexpr (T::KIND != CACHE_F16) to.scale = sbase + kv_row(page, in_page, 0, p.cache.scale_page_stride, 0, p.cache.scale_token_stride) * 2;
            }
            if (id < T::NB) row_at[values][j & 3][id] = to;
            if constexpr (T::KIND == CACHE_I8_ROWS)
                if (!values) {
                    scale = load_scales<1>(to.scale);
                    value_scale = load_scales<1>(there ? to.scale + ((const char*)p.cache.v_scale - (const char*)p.cache.k_scale) : to.scale); // (strides are those of the keys')
                }
        };
        auto publish = [&](int32_t j) { // to the softmax: by the keys' threads
            const int slot = j % T::INFOS;
            const uint32_t mask = __ballot_sync(0xffffffffu, there);
            if (values) return;
            if (lane == 0) masks[slot][id >> 5] = id < T::NB ? mask : 0xffffffffu;
            if constexpr (T::KIND == CACHE_I8_ROWS)
                if (id < T::NB) {
                    uint8_t* const to = raw_smem + (smem - ptx::smem_addr(raw_smem)) + T::INFO + slot * 6 * T::NB;
                    reinterpret_cast<float*>(to)[id] = __half2float(__ushort_as_half((unsigned short)scale)) * p.scale_log2;
                    reinterpret_cast<uint16_t*>(to + 4 * T::NB)[id] = (uint16_t)value_scale;
                    const int32_t size = size_of(__half2float(__ushort_as_half((unsigned short)value_scale)));
                    const int32_t most = __reduce_max_sync(0xffffffffu, there ? size : -24), least = __reduce_min_sync(0xffffffffu, there ? size : 16);
                    if (lane == 0) sizes[slot][id >> 5] = make_int2(most, least);
                }
            report(bar(info_full[slot]));
        };
        const int barrier_id = values ? 3 : 1;
        // Blocks 0 and 1 are located before the first is loaded; then, with every block, the next one is published, the one behind it located and the third's
        // pages requested.
        auto begin = [&] {
            request(0);
            locate(0);
            request(1);
            publish(0);
            locate(1);
            request(2);
            ptx::named_barrier(barrier_id, 128);
        };
        auto go_on = [&](int32_t j) {
            if (j + 1 < blocks) publish(j + 1);
            locate(j + 2);
            request(j + 3);
            ptx::named_barrier(barrier_id, 128);
        };
        // piece i of this thread: of which token, and which of its row (CH divides 128 but for heads of 96)
        constexpr bool even = 128 % T::CH == 0;
        const uint32_t id_token = (uint32_t)id / T::CH, id_piece = (uint32_t)id % T::CH;
        auto token_of = [&](int i) { return even ? id_token + i * (128 / T::CH) : (uint32_t)(id + 128 * i) / T::CH; };
        auto piece_of = [&](int i) { return even ? id_piece : (uint32_t)(id + 128 * i) % T::CH; };
        // where 16 bytes of fp16 (dimensions 8 c on) of a token lie in a tile
        auto place = [](uint32_t token, uint32_t c) { return (c >> 3) * (T::NB * 128) + token * 128 + (((c & 7) ^ (token & 7)) << 4); };
        bool ok = true;
        if constexpr (T::KIND == CACHE_F16) {
            if (boxes) {
                // Warp 8 brings keys, warp 12 values: lane i the box of tokens from i * box_rows on; a box that is not there lies on the page behind the last
                // and reads as zeros.  Tokens behind the prefix's last in a box that is there are what the page holds: masked as keys, as values overwritten with zeros.
                if ((warp & 3) == 0) {
                    const int groups = T::NB / p.box_rows;
                    const CUtensorMap* const map = values ? &p.vmap : &p.kmap;
                    if (lane == 0) ptx::prefetch_tensormap(map);
                    order_before_tma();
                    auto page_of = [&](int32_t j) {
                        const int32_t token = (block0 + j) * T::NB + lane * p.box_rows;
                        return j < blocks && lane < groups && token < n ? p.pages[(uint32_t)((uint64_t)(uint32_t)token * p.page_magic >> p.page_shift)] : -1;
                    };
                    int32_t next = page_of(0), issued = 0; // blocks whose barrier `full` tells when they are there
                    for (int32_t j = 0; j < blocks; ++j) {
                        const int32_t now = next, first = (block0 + j) * T::NB, token = first + lane * p.box_rows;
                        next = page_of(j + 1);
                        const bool here = (uint32_t)now < (uint32_t)p.num_pages;
                        const uint32_t present = __ballot_sync(0xffffffffu, here);
                        const int stage = j % stages;
                        ok = __all_sync(0xffffffffu, ptx::mbar_wait(empty(stage), ((j / stages) & 1) ^ 1, &g_status, ST_LOAD));
                        if (!ok) break;
                        if (!values) { // the scores' masks: bit x of word w is token 32 w + x
                            if (lane >= T::NB / 32 && lane < 4) masks[j % T::INFOS][lane] = 0xffffffffu;
                            if (lane < T::NB / 32) {
                                const uint32_t half0 = present >> (lane * 32 / p.box_rows) & 1, half1 = present >> ((lane * 32 + 16) / p.box_rows) & 1;
                                const int32_t left = n - first - lane * 32;
                                masks[j % T::INFOS][lane] = (half0 * 0xffffu | half1 * 0xffff0000u) & (left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1);
                            }
                            __syncwarp();
                            if (lane == 0) ptx::mbar_arrive(bar(info_full[j % T::INFOS]));
                        }
                        const bool tail = values && first + T::NB > n;
                        const uint32_t landed = tail ? bar(tail_full) : full(stage);
                        if (lane == 0) ptx::mbar_arrive_expect_tx(landed, T::V_BYTES);
                        __syncwarp();
                        if (lane < groups) {
                            const int32_t in_page = token - (int32_t)((uint32_t)((uint64_t)(uint32_t)token * p.page_magic >> p.page_shift)) * p.cache.page_size;
#pragma unroll
                            for (int a = 0; a < T::ATOMS; ++a)
                                ptx::tma_load_4d(ring + stage * T::V_BYTES + a * (T::NB * 128) + lane * p.box_rows * 128, map, landed, a * 64, here ? in_page : 0, kvh, here ? now : p.num_pages);
                        }
                        if (tail) { // the last block
                            ok = __all_sync(0xffffffffu, ptx::mbar_wait(landed, 0, &g_status, ST_LOAD));
                            if (!ok) break;
                            for (int32_t x = (n - first) * 8 + lane; x < T::NB * 8; x += 32)
#pragma unroll
                                for (int a = 0; a < T::ATOMS; ++a) ptx::st_shared_v4(ring + stage * T::V_BYTES + a * (T::NB * 128) + x * 16, make_uint4(0, 0, 0, 0));
                            ptx::fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0) ptx::mbar_arrive(full(stage));
                        }
                        issued = j + 1;
                    }
                    // no copy is under way when the CTA leaves, although nobody may have waited for it
                    for (int32_t j = max(0, issued - stages); j < issued; ++j)
                        if (!__all_sync(0xffffffffu, ptx::mbar_wait(full(j % stages), (j / stages) & 1, &g_status, ST_LOAD))) break;
                }
            } else {
                // one block's pieces on their way while the next one's are issued
                int32_t arrived = 0;
                auto settle = [&](int32_t issued) { // what is issued has landed
                    ptx::cp_async_wait<0>();
                    for (; arrived < issued; ++arrived) {
                        ptx::fence_proxy_async_smem();
                        report(full(arrived % stages));
                    }
                };
                if (blocks > 0) begin();
                for (int32_t j = 0; j < blocks; ++j) {
                    go_on(j);
                    const int stage = j % stages;
                    const uint32_t parity = ((j / stages) & 1) ^ 1;
                    if (ok && !__all_sync(0xffffffffu, ptx::mbar_try_wait(empty(stage), parity))) { // what is on its way may be what the place waits for
                        settle(j);
                        ok = __all_sync(0xffffffffu, ptx::mbar_wait(empty(stage), parity, &g_status, ST_LOAD));
                    }
                    if (!ok) continue; // (every thread comes to every barrier and ballot)
#pragma unroll
                    for (int i = 0; i < T::LOADS; ++i) {
                        ptx::cp_async_16(ring + stage * stage_bytes + place(token_of(i), piece_of(i)), row_at[values][j & 3][token_of(i)].at + piece_of(i) * 16);
                    }
                    ptx::cp_async_commit();
                    if (j > arrived) {
                        ptx::cp_async_wait<1>();
                        ptx::fence_proxy_async_smem();
                        report(full(arrived % stages));
                        ++arrived;
                    }
                }
                if (ok) settle(blocks);
                ptx::cp_async_wait<0>();
            }
        } else {
            uint4 w[T::LOADS];
            uint32_t scales[T::LOADS]; // CACHE_I8_GROUPS
            auto fetch = [&](int32_t j, int i) {
                const Row row = row_at[values][j & 3][token_of(i)];
                w[i] = ld_global_16(row.at + piece_of(i) * 16);
                if constexpr (T::KIND == CACHE_I8_GROUPS) scales[i] = load_scales<2>(row.scale + piece_of(i) * 4);
            };
            // into its place, and each piece's successor of the next block is requested
            auto put = [&](uint32_t dst, int32_t next) {
#pragma unroll
                for (int i = 0; i < T::LOADS; ++i) {
                    uint32_t o[8], r[8] = {};
                    whole_numbers(w[i], o);
                    if constexpr (T::KIND == CACHE_I8_GROUPS) {
                        const uint32_t s = scales[i];
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            const __half2 f = as_h2(__byte_perm(s, 0, x < 4 ? 0x1010 : 0x3232));
                            const __half2 h = __hmul2(as_h2(o[x]), f);
                            r[x] = h2(__hfma2(as_h2(o[x]), f, __hneg2(h)));
                            o[x] = h2(h);
                        }
                    } // (rows' scales go into the scores and the weights)
                    // (eight threads meet the banks twice; a store the other way round for every second 64 dimensions costs more instructions than that time)
                    const uint32_t c = 2 * piece_of(i), a = dst + place(token_of(i), c), b = dst + place(token_of(i), c + 1);
                    ptx::st_shared_v4(a, make_uint4(o[0], o[1], o[2], o[3]));
                    ptx::st_shared_v4(b, make_uint4(o[4], o[5], o[6], o[7]));
                    if (T::LOW && !values) {
                        ptx::st_shared_v4(a + T::V_BYTES, make_uint4(r[0], r[1], r[2], r[3]));
                        ptx::st_shared_v4(b + T::V_BYTES, make_uint4(r[4], r[5], r[6], r[7]));
                    }
                    if (next < blocks) fetch(next, i);
                }
                ptx::fence_proxy_async_smem();
            };
            if (blocks > 0) {
                begin();
#pragma unroll
                for (int i = 0; i < T::LOADS; ++i) fetch(0, i);
            }
            for (int32_t j = 0; j < blocks; ++j) {
                go_on(j);
                const int stage = j % stages;
                // (after a wait that ran out nothing is stored any more, but every thread comes to every barrier and ballot)
                ok = ok && __all_sync(0xffffffffu, ptx::mbar_wait(empty(stage), ((j / stages) & 1) ^ 1, &g_status, ST_LOAD));
                if (ok) {
                    put(ring + stage * stage_bytes, j + 1);
                    report(full(stage));
                }
            }
        }
    } else {
        ptx::registers_up<T::R_SOFTMAX>();
        // ---- softmax ---------------------------------------------------------------------------------------------------------------
        const int stream = warp >> 2, r = threadIdx.x & 127;
        // the rows of q: a tile at a time, requested together
        for (int t = 0; t < tiles; ++t) {
            constexpr int PIECES = 128 * (T::D / 8) / 256;
            uint4 v[PIECES];
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int x = threadIdx.x + 256 * i, row = x / (T::D / 8), c = x - row * (T::D / 8), of = row0 + t * 128 + row;
                const int32_t sequence = (uint32_t)((uint64_t)(uint32_t)of * p.rows_magic >> p.rows_shift);
                v[i] = of < p.rows ? ld_global_16(p.q + sequence * p.q_stride + (int64_t)(kvh * p.rows_per_head + of - sequence * p.rows_per_head) * T::D + c * 8) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int x = threadIdx.x + 256 * i, row = x / (T::D / 8), c = x - row * (T::D / 8);
                ptx::st_shared_v4(smem + t * T::Q_BYTES + (c >> 3) * (128 * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4), v[i]);
            }
        }
        ptx::fence_proxy_async_smem();
        report(bar(q_full));

        const uint32_t lanes = (uint32_t)(warp & 3) << 21; // 32 (warp & 3) in the address's upper half
        const uint32_t sum_at = tmem + lanes + T::O_COLUMN + (T::STREAMS == 2 ? stream * T::DP : 0);
        float top = kNothingSeen, sum = 0.0f;
        bool met = false, ok = true;
        if (T::STREAMS == 2 || stream == 0) {
            for (int32_t i = T::STREAMS == 2 ? stream : 0; i < tasks && ok; i += T::STREAMS) {
                const int32_t j = i >> shift;
                const int slot = j % T::INFOS;
                ok = ok && ptx::mbar_wait(bar(info_full[slot]), (j / T::INFOS) & 1, &g_status, ST_SOFTMAX) && ptx::mbar_wait(bar(score_full[i & 1]), (i >> 1) & 1, &g_status, ST_SOFTMAX);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                ptx::tc_fence_after();
                const uint32_t at = tmem + lanes + (i & 1) * 128;
                // Where registers hold half of the scores (KEPT), the others are looked at for the largest and loaded again when the first half's weights are on their way.
                constexpr int HALF = T::NB / 2, KEPT = T::KEPT, ROLL = T::KIND == CACHE_I8_ROWS ? 1 : 2;
                const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
                // CACHE_I8_ROWS: keys' scales times scale_log2 in 32 bits, values' as they are (with both as they are, 64 x 32768 tokens took 137 us; 128 so).
                const uint8_t* const scales_at = raw_smem + (smem - ptx::smem_addr(raw_smem)) + T::INFO + slot * 6 * T::NB;
                auto scales_of = [&](int c, auto use) { // of values c to c + 31
                    const uint4* const from = reinterpret_cast<const uint4*>(scales_at + 4 * T::NB + c * 2);
#pragma unroll
                    for (int k = 0; k < 32; k += 8) {
                        const uint4 f = from[k / 8];
                        const uint32_t f4[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                        for (int y = 0; y < 4; ++y) use(k + 2 * y, __half22float2(as_h2(f4[y])));
                    }
                };
                const uint4 mask4 = *reinterpret_cast<const uint4*>(masks[slot]);
                met |= (mask4.x | mask4.y | (T::NB == 128 ? mask4.z | mask4.w : 0u)) != 0;
                const bool whole = (mask4.x & mask4.y & mask4.z & mask4.w) == 0xffffffffu;
                // Of tokens c to c + 31, rounded to 32 bits here: fused with the reference exponent's subtraction below, which takes half an instruction less, scores from 2^27 on
                // would differ from the largest, which is rounded, by more than a weight has room for.
                auto score = [&](const uint32_t (&bits)[32], float (&x)[32], int c) {
                    if constexpr (T::KIND == CACHE_I8_ROWS) {
                        const float4* const from = reinterpret_cast<const float4*>(scales_at + c * 4);
#pragma unroll
                        for (int k = 0; k < 32; k += 4) {
                            const float4 f = from[k / 4];
                            const float2 u = ptx::mul2(make_float2(__uint_as_float(bits[k]), __uint_as_float(bits[k + 1])), make_float2(f.x, f.y));
                            const float2 v = ptx::mul2(make_float2(__uint_as_float(bits[k + 2]), __uint_as_float(bits[k + 3])), make_float2(f.z, f.w));
                            x[k] = u.x; x[k + 1] = u.y; x[k + 2] = v.x; x[k + 3] = v.y;
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; k += 2) {
                            const float2 u = ptx::mul2(make_float2(__uint_as_float(bits[k]), __uint_as_float(bits[k + 1])), scale2);
                            x[k] = u.x; x[k + 1] = u.y;
                        }
                    }
                    if (!whole) {
                        const uint32_t mask = c == 0 ? mask4.x : c == 32 ? mask4.y : c == 64 ? mask4.z : mask4.w;
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (!(mask >> k & 1)) x[k] = -INFINITY;
                    }
                };
                float high[8];
#pragma unroll
                for (int y = 0; y < 8; ++y) high[y] = -INFINITY;
                // CACHE_I8_ROWS: a value's scale goes into its weight (the sum of the weights is without it), and its size into what decides about the reference exponent.  Where the block's
                // scales are much alike, the largest size stands for all; else each counts for itself, so that a large scale takes no bits from what weighs more.
                int32_t most = 0;
                bool alike = true;
                if constexpr (T::KIND == CACHE_I8_ROWS) {
                    int32_t least = 16;
                    most = -24;
#pragma unroll
                    for (int w = 0; w < T::NB / 32; ++w) {
                        const int2 of = sizes[slot][w];
                        most = max(most, of.x);
                        least = min(least, of.y);
                    }
                    alike = most - least <= 4;
                }
                auto look = [&](const float (&x)[32]) {
#pragma unroll
                    for (int k = 0; k < 32; k += 16)
#pragma unroll
                        for (int y = 0; y < 8; ++y) high[y] = fmaxf(high[y], fmaxf(x[k + y], x[k + 8 + y]));
                };
#pragma unroll ROLL
                for (int c = KEPT; c < T::NB; c += 32) {
                    uint32_t bits[32];
                    float x[32];
                    ptx::tmem_ld_32x32(at + c, bits);
                    ptx::tmem_ld_wait();
                    score(bits, x, c);
                    look(x);
                }
                float s[KEPT / 32][32];
                {
                    uint32_t bits[KEPT / 32][32];
#pragma unroll
                    for (int c = 0; c < KEPT; c += 32) ptx::tmem_ld_32x32(at + c, bits[c / 32]);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < KEPT; c += 32) {
                        score(bits[c / 32], s[c / 32], c);
                        look(s[c / 32]);
                    }
                }
                if (T::KIND == CACHE_I8_ROWS && !alike) {
#pragma unroll
                    for (int y = 0; y < 8; ++y) high[y] = -INFINITY;
#pragma unroll 1
                    for (int c = 0; c < T::NB; c += 32) {
                        uint32_t bits[32];
                        float x[32];
                        ptx::tmem_ld_32x32(at + c, bits);
                        ptx::tmem_ld_wait();
                        score(bits, x, c);
                        scales_of(c, [&](int k, float2 f) { x[k] += (float)size_of(f.x), x[k + 1] += (float)size_of(f.y); });
                        look(x);
                    }
                }
#pragma unroll
                for (int y = 4; y > 0; y >>= 1)
#pragma unroll
                    for (int k = 0; k < y; ++k) high[k] = fmaxf(high[k], high[k + y]);
                const float m = high[0] + (T::KIND == CACHE_I8_ROWS && alike ? (float)most : 0.0f);
                // The reference exponent moves when a weight would pass 2^14, each row's for itself, and then to kAbove above the largest score: some row of 32 meets a score
                // 2^6 times as heavy again and again where keys have a few large dimensions.  The largest weight is 2^4 at least; those below 2^-18 of it lose bits.
                const bool higher = m - top > 6.0f; // (top + 6 may be rounded to top + 8)
                if (__any_sync(0xffffffffu, higher)) {
                    const float to = higher ? m + kAbove : top, keep = exp2_fast(top - to);
                    top = to;
                    sum *= keep;
                    const int32_t before = T::STREAMS == 2 ? i - 2 : i - 1; // the last task that has added to these sums
                    if (before >= 0) {
                        ok = ptx::mbar_wait(bar(sum_done[before & 1]), (before >> 1) & 1, &g_status, ST_SOFTMAX);
                        if (!(ok = __all_sync(0xffffffffu, ok))) break;
                        ptx::tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < T::D; c += 32) {
                            uint32_t o[32];
                            ptx::tmem_ld_32x32(sum_at + c, o);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * keep);
                            ptx::tmem_st_32x16(sum_at + c, o);
                            ptx::tmem_st_32x16(sum_at + c + 16, o + 16);
                        }
                    }
                }
                const float less = __fadd_rd(8.0f, -top); // down: of numbers 16 apart the next one would make a weight 2^16
                const float2 reference = make_float2(less, less);
                float2 sums[2] = {};
                auto weigh = [&](const float (&x)[32], int c) { // weights of tokens c to c + 31 into their place
                    uint32_t w[16], low[T::FINE ? 16 : 1];
                    auto pair = [&](int k, float2 f) {
                        float2 e = ptx::add2(make_float2(x[k], x[k + 1]), reference);
                        e.x = exp2_fast(e.x);
                        e.y = exp2_fast(e.y);
                        sums[k >> 1 & 1] = ptx::add2(sums[k >> 1 & 1], e);
                        if constexpr (T::KIND == CACHE_I8_ROWS) e = ptx::mul2(e, f);
                        w[k / 2] = h2(__floats2half2_rn(e.x, e.y));
                        if constexpr (T::FINE) {
                            const float2 high = __half22float2(as_h2(w[k / 2]));
                            low[k / 2] = h2(__floats2half2_rn(e.x - high.x, e.y - high.y));
                        }
                    };
                    if constexpr (T::KIND == CACHE_I8_ROWS) {
                        scales_of(c, pair);
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; k += 2) pair(k, float2());
                    }
                    ptx::tmem_st_32x16(T::FINE ? at + c : at + c / 2, w);
                    if constexpr (T::FINE) ptx::tmem_st_32x16(at + c + 16, low);
                };
#pragma unroll
                for (int c = 0; c < KEPT; c += 32) {
                    weigh(s[c / 32], c);
                    if (c + 32 == HALF) {
                        ptx::tmem_st_wait();
                        ptx::tc_fence_before();
                        report(bar(weight_half[i & 1]));
                    }
                }
#pragma unroll ROLL
                for (int c = KEPT; c < T::NB; c += 32) {
                    uint32_t bits[32];
                    float x[32];
                    ptx::tmem_ld_32x32(at + c, bits);
                    ptx::tmem_ld_wait();
                    score(bits, x, c);
                    weigh(x, c);
                }
                sum += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
                ptx::tmem_st_wait();
                ptx::tc_fence_before();
                report(bar(weight_full[i & 1]));
            }
        }
        // ---- the sums ---------------------------------------------------------------------------------------------------------------
        if (tasks > 0) ok = __all_sync(0xffffffffu, ptx::mbar_wait(bar(all_done), 0, &g_status, ST_SOFTMAX)) && ok && !products_lost;
        ptx::tc_fence_after();
        if (met) top = fmaxf(top, kLowest);
        if (!ok) top = sum = __int_as_float(0x7fffffff); // a wait ran out: not a number rather than a wrong one
        float own = 1.0f, other = 0.0f;
        const bool mine = T::STREAMS == 2 ? (tiles == 2 || stream == 0) : stream == 0; // whether this group writes a tile
        float* const exchange = reinterpret_cast<float*>(raw_smem + (smem - ptx::smem_addr(raw_smem))); // [D][128]: the rings and q are idle
        const bool joined = T::STREAMS == 2 && tiles == 1 && tasks > 1; // two groups' sums of one tile
        if (joined) {
            if (stream == 1) {
                joint[r] = make_float2(top, sum);
#pragma unroll 1
                for (int c = 0; c < T::D; c += 32) {
                    uint32_t o[32];
                    ptx::tmem_ld_32x32(sum_at + c, o);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int x = 0; x < 32; ++x) exchange[(c + x) * 128 + r] = __uint_as_float(o[x]);
                }
            }
            ptx::named_barrier(2, 256);
            if (stream == 0) {
                const float2 s = joint[r];
                const float up = fmaxf(top, s.x);
                own = exp2_fast(top - up);
                other = exp2_fast(s.x - up);
                if (top != top || s.x != s.x) own = other = __int_as_float(0x7fffffff);
                sum = sum * own + s.y * other;
                top = up;
            }
        }
        const int32_t of = row0 + (T::STREAMS == 2 && tiles == 2 ? stream * 128 : 0) + r;
        const int32_t sequence = (uint32_t)((uint64_t)(uint32_t)of * p.rows_magic >> p.rows_shift);
        const int64_t at = (int64_t)sequence * p.q_heads + kvh * p.rows_per_head + (of - sequence * p.rows_per_head) + split * p.part_rows;
        const bool there = mine && of < p.rows;
        if (there) __stcg(&p.part_tops[at], make_float2(top, sum));
        if (mine && tasks > 0) {
            // by way of shared memory, so that a row leaves in whole lines: 32 rows of a warp, which it alone writes and reads
            constexpr int PITCH = T::D + 4;
            float* const rows = reinterpret_cast<float*>(raw_smem + (smem - ptx::smem_addr(raw_smem)) + (joined ? T::EXCHANGE : 0)) + (threadIdx.x >> 5) * 32 * PITCH;
#pragma unroll 1
            for (int c = 0; c < T::D; c += 32) {
                uint32_t o[32];
                ptx::tmem_ld_32x32(sum_at + c, o);
                ptx::tmem_ld_wait();
                float v[32];
#pragma unroll
                for (int x = 0; x < 32; ++x) {
                    v[x] = __uint_as_float(o[x]);
                    if (joined) v[x] = v[x] * own + exchange[(c + x) * 128 + r] * other;
                }
#pragma unroll
                for (int x = 0; x < 32; x += 4) *reinterpret_cast<float4*>(rows + lane * PITCH + c + x) = make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
            }
            __syncwarp();
            const int64_t mine_at = there ? at : -1;
#pragma unroll 4
            for (int x = 0; x < 32; ++x) {
                const int64_t row = __shfl_sync(0xffffffffu, mine_at, x);
                if (row >= 0)
                    for (int c = lane * 4; c < T::D; c += 128) __stcg(reinterpret_cast<float4*>(p.part_sums + row * T::D + c), *reinterpret_cast<const float4*>(rows + x * PITCH + c));
            }
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 16) ptx::tmem_dealloc(tmem, 512);
}

} // namespace prefix
} // namespace pplb200
