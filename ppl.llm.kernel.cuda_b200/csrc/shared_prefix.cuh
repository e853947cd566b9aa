// The prefix that a batch shares, for many rows of q at once: scores and weighted sums on tcgen05, statistics in registers.
//
// A row is a query head of one sequence; the rows that ask one key head are a matrix, and so this is a product of it with the keys, a softmax by rows that is
// never whole in one place, and a product with the values.  A CTA has up to 256 rows of a key head in two tiles of 128 and goes through a part of the
// prefix in blocks of NB tokens; its sums and reference exponents are left as one of `splits` parts, which are joined where the output is written.
//
//   warps 0 - 3, 4 - 7   softmax of one tile each, a thread a row (tensor memory's lanes): scores in, weights of 11 bits out, in place
//   warps 8 - 11         keys and values from the pages into shared memory; int8 ones are widened on the way
//   warp 12              one thread issues all products; the warp owns the tensor memory
//
// The two tiles' products and softmaxes alternate, so that the tensor cores work on one while the exponentials of the other are computed.  Where a CTA has one
// tile only, the two softmax groups take turns at the blocks of it, each with a sum of its own (heads of 256: one group, whose sum alone fills
// half of the tensor memory, over two buffers of scores).
// Bound by both: a block of 128 tokens of two tiles of heads of 128 is 2048 clocks of the tensor cores and 2048 of the exponentials.
#pragma once

#include "paged_attention.cuh"
#include "ptx.cuh"

namespace pplb200 {
namespace prefix {

using namespace paged;

__device__ unsigned int g_status = 0;
constexpr unsigned ST_LOAD = 1u, ST_MMA = 2u, ST_SOFTMAX = 4u;

template <int D_, int KIND_>
struct Tile {
    static constexpr int D = D_, KIND = KIND_, ES = KIND == CACHE_F16 ? 2 : 1;
    static constexpr int DP = (D + 63) / 64 * 64, ATOMS = DP / 64; // a row of shared memory is 128 bytes, 64 dimensions
    static constexpr bool LOW = KIND == CACHE_I8_GROUPS;           // keys: value x scale rounded to fp16, and what that left
    static constexpr int NB = D == 256 ? 64 : 128;                 // tokens of a block
    static constexpr int STREAMS = D == 256 ? 1 : 2;
    static constexpr int TILES = D == 256 || (LOW && D > 64) ? 1 : 2; // of rows, at most
    static constexpr int KS = D == 64 ? (LOW ? 3 : 4) : LOW && D == 256 ? 1 : 2, VS = D == 64 ? (LOW ? 3 : 4) : LOW && D < 256 ? 1 : 2; // stages of keys and of values
    static constexpr int Q_BYTES = 128 * DP * 2, V_BYTES = NB * DP * 2, K_BYTES = V_BYTES * (LOW ? 2 : 1);
    static constexpr int RING = TILES * Q_BYTES, V_RING = RING + KS * K_BYTES, INFO = V_RING + VS * V_BYTES;
    static constexpr int INFOS = 8; // blocks whose masks and scales are kept: more than stages of values
    static constexpr int SCALES = KIND == CACHE_I8_ROWS ? INFOS * NB * 8 : 0;
    static constexpr int SMEM = INFO + SCALES + 1024; // the base is rounded up to 1024
    static constexpr int CH = D * ES / 16, LOADS = CH * NB / 128; // pieces of 16 bytes: of a row, and of a block for a thread
    static_assert(CH * NB % 128 == 0 && VS < INFOS);
    static constexpr int THREADS = 512;
    static constexpr uint32_t O_COLUMN = 256; // scores: columns 0 and 128
};

struct PrefixParams {
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
    int64_t part_rows;
    float2* part_tops;
    float* part_sums;
};

// Descriptors of rows of 128 bytes with the 128-byte swizzle: K-major (ptx::desc_lo_sw128), or MN-major, 64 dimensions wide, the next 64 `apart` bytes on.
__device__ __forceinline__ uint32_t mn_desc_lo(uint32_t addr, uint32_t apart) { return ((addr & 0x3ffffu) >> 4) | (apart >> 4 << 16); }

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
    __shared__ __align__(8) uint64_t full_k[T::KS], empty_k[T::KS], full_v[T::VS], empty_v[T::VS], info_full[T::INFOS], score_full[2], weight_full[2], sum_done[2], q_full, all_done;
    __shared__ uint32_t tmem_slot;
    __shared__ uint32_t masks[T::INFOS][4];
    __shared__ float sizes[T::INFOS][4];
    __shared__ int64_t row_at[2][T::NB], scale_at[2][T::KIND == CACHE_F16 ? 1 : T::NB];
    __shared__ float2 joint[128];
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t smem = (ptx::smem_addr(raw_smem) + 1023u) & ~1023u;
    auto bar = [](uint64_t& b) { return ptx::smem_addr(&b); };
    if (threadIdx.x == 0) {
        for (int i = 0; i < T::KS; ++i) ptx::mbar_init(bar(full_k[i]), 128), ptx::mbar_init(bar(empty_k[i]), 1);
        for (int i = 0; i < T::VS; ++i) ptx::mbar_init(bar(full_v[i]), 128), ptx::mbar_init(bar(empty_v[i]), 1);
        for (int i = 0; i < T::INFOS; ++i) ptx::mbar_init(bar(info_full[i]), 128);
        for (int i = 0; i < 2; ++i) ptx::mbar_init(bar(score_full[i]), 1), ptx::mbar_init(bar(weight_full[i]), 128), ptx::mbar_init(bar(sum_done[i]), 1);
        ptx::mbar_init(bar(q_full), 256);
        ptx::mbar_init(bar(all_done), 1);
        ptx::fence_mbar_init();
    }
    if (warp == 12) {
        ptx::tmem_alloc(ptx::smem_addr(&tmem_slot), 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait_prior_grid();
    pdl_launch_dependents(); // behind the allocation, so that no later kernel has this SM's tensor memory

    const int32_t item = blockIdx.x / p.splits, split = blockIdx.x - item * p.splits;
    const int32_t per_head = p.items / p.cache.kv_heads, kvh = item / per_head;
    const int32_t row0 = (item - kvh * per_head) * p.tiles * 128;
    const int32_t tiles = p.tiles == 2 && p.rows - row0 > 128 ? 2 : 1;
    const int32_t n = (int32_t)min((int64_t)max(*(const volatile int32_t*)p.length, 0), p.tokens_in_table);
    const int32_t all_blocks = (n + T::NB - 1) / T::NB;
    const int32_t block0 = (int32_t)((int64_t)all_blocks * split / p.splits), blocks = (int32_t)((int64_t)all_blocks * (split + 1) / p.splits) - block0;
    const int32_t tasks = tiles * blocks; // task i: buffer i & 1, block i / tiles; with two streams also stream i & 1
    const int32_t shift = tiles - 1;

    if (warp >= 12) {
        ptx::registers_down<40>();
        if (warp == 12 && lane == 0 && tasks > 0) {
            // ---- products --------------------------------------------------------------------------------------------------
            constexpr uint32_t QK = ptx::make_f16_idesc(128, T::NB, false), PV = ptx::make_f16_idesc(128, T::D, true);
            bool ok = ptx::mbar_wait(bar(q_full), 0, &g_status, ST_MMA);
            auto scores = [&](int32_t i) {
                const int32_t j = i >> shift, stage = j % T::KS;
                if (!(ok = ok && ptx::mbar_wait(bar(full_k[stage]), (j / T::KS) & 1, &g_status, ST_MMA))) return;
                ptx::tc_fence_after();
                const uint32_t q = ptx::desc_lo_sw128(smem + (tiles == 2 ? (i & 1) * T::Q_BYTES : 0)), k = ptx::desc_lo_sw128(smem + T::RING + stage * T::K_BYTES);
                const uint32_t d = tmem + (i & 1) * 128;
#pragma unroll
                for (int s = 0; s < T::D / 16; ++s) {
                    const uint32_t a = q + ((s / 4) * (128 * 128) + (s % 4) * 32) / 16, b = k + ((s / 4) * (T::NB * 128) + (s % 4) * 32) / 16;
                    ptx::mma_f16(d, ptx::desc_from_lo(a), ptx::desc_from_lo(b), QK, s > 0);
                    if constexpr (T::LOW) ptx::mma_f16(d, ptx::desc_from_lo(a), ptx::desc_from_lo(b + T::V_BYTES / 16), QK, 1);
                }
                ptx::mma_commit(bar(score_full[i & 1]));
                if (tiles == 1 || (i & 1)) ptx::mma_commit(bar(empty_k[stage]));
            };
            scores(0);
            if (tasks > 1) scores(1);
            for (int32_t i = 0; i < tasks && ok; ++i) {
                const int32_t j = i >> shift, stage = j % T::VS;
                if (!(ok = ptx::mbar_wait(bar(full_v[stage]), (j / T::VS) & 1, &g_status, ST_MMA) && ptx::mbar_wait(bar(weight_full[i & 1]), (i >> 1) & 1, &g_status, ST_MMA))) break;
                ptx::tc_fence_after();
                const uint32_t v = mn_desc_lo(smem + T::V_RING + stage * T::V_BYTES, T::NB * 128);
                const uint32_t d = tmem + T::O_COLUMN + (T::STREAMS == 2 ? (i & 1) * T::DP : 0), w = tmem + (i & 1) * 128;
#pragma unroll
                for (int s = 0; s < T::NB / 16; ++s) ptx::mma_f16_tmem(d, w + s * 8, ptx::desc_from_lo(v + s * (2048 / 16)), PV, (T::STREAMS == 2 ? i > 1 : i > 0) || s > 0);
                ptx::mma_commit(bar(sum_done[i & 1]));
                if (tiles == 1 || (i & 1)) ptx::mma_commit(bar(empty_v[stage]));
                if (i + 2 < tasks) scores(i + 2);
            }
            ptx::mma_commit(bar(all_done)); // all that was issued
        }
    } else if (warp >= 8) {
        ptx::registers_down<120>();
        // ---- keys and values ---------------------------------------------------------------------------------------------------
        const int id = threadIdx.x - 256;
        const char *const kbase = (const char*)p.cache.k + (int64_t)kvh * p.cache.head_stride * T::ES, *const vbase = (const char*)p.cache.v + (int64_t)kvh * p.cache.head_stride * T::ES;
        const char *const ksbase = (const char*)p.cache.k_scale + (int64_t)kvh * p.cache.scale_head_stride * 2, *const vsbase = (const char*)p.cache.v_scale + (int64_t)kvh * p.cache.scale_head_stride * 2;
        // where block j's tokens lie, which of them are there, and (rows) their scales
        auto locate = [&](int32_t j) {
            const int32_t token = (block0 + j) * T::NB + id;
            bool there = false;
            int64_t row = -1, scale_row = 0;
            if (id < T::NB && token < n) {
                const uint32_t index = (uint32_t)((uint64_t)(uint32_t)token * p.page_magic >> p.page_shift);
                const int32_t page = p.pages[index], in_page = token - index * p.cache.page_size;
                there = (uint32_t)page < (uint32_t)p.num_pages;
                if (there) {
                    row = kv_row(page, in_page, 0, p.cache.page_stride, 0, p.cache.token_stride) * T::ES;
                    if constexpr (T::KIND != CACHE_F16) scale_row = kv_row(page, in_page, 0, p.cache.scale_page_stride, 0, p.cache.scale_token_stride) * 2;
                }
            }
            const int slot = j % T::INFOS;
            if (id < T::NB) {
                row_at[j & 1][id] = row;
                if constexpr (T::KIND != CACHE_F16) scale_at[j & 1][id] = scale_row;
            }
            const uint32_t mask = __ballot_sync(0xffffffffu, there);
            if (lane == 0) masks[slot][id >> 5] = mask;
            if constexpr (T::KIND == CACHE_I8_ROWS) {
                const float ks = there ? __half2float(__ushort_as_half((unsigned short)load_scales<1>(ksbase + scale_row))) : 0.0f;
                const float vs = there ? __half2float(__ushort_as_half((unsigned short)load_scales<1>(vsbase + scale_row))) : 0.0f;
                // a value's scale goes into its weight, its logarithm into what decides about the reference exponent, as far as a finite one could
                float size = fminf(fmaxf(log2_fast(fabsf(vs)), -24.0f), 16.0f);
#pragma unroll
                for (int m = 16; m > 0; m >>= 1) size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, m));
                if (lane == 0) sizes[slot][id >> 5] = id < T::NB ? size : -24.0f;
                if (id < T::NB) {
                    float* const scales = reinterpret_cast<float*>(raw_smem + (smem - ptx::smem_addr(raw_smem)) + T::INFO) + slot * T::NB * 2;
                    scales[id] = ks * p.scale_log2;
                    scales[T::NB + id] = vs;
                }
            }
            ptx::mbar_arrive(bar(info_full[slot]));
            ptx::named_barrier(1, 128);
        };
        // piece i of this thread: of token (id + 128 i) / CH
        auto token_of = [&](int i) { return (id + 128 * i) / T::CH; };
        auto piece_of = [&](int i) { return (id + 128 * i) % T::CH; };
        // where 16 bytes of fp16 (dimensions 8 c on) of a token lie in a tile
        auto place = [](int token, int c) { return (uint32_t)((c >> 3) * (T::NB * 128) + token * 128 + (((c & 7) ^ (token & 7)) << 4)); };
        bool ok = true;
        if constexpr (T::KIND == CACHE_F16) {
            // loads 2 j (keys) and 2 j + 1 (values); up to three are on their way when the next is issued
            int32_t arrived = 0, issued = 0;
            auto arrive = [&] {
                ptx::fence_proxy_async_smem();
                ptx::mbar_arrive(arrived & 1 ? bar(full_v[(arrived >> 1) % T::VS]) : bar(full_k[(arrived >> 1) % T::KS]));
                ++arrived;
            };
            auto settle = [&] {
                ptx::cp_async_wait<0>();
                while (arrived < issued) arrive();
            };
            for (int32_t j = 0; j < blocks; ++j) {
                locate(j);
#pragma unroll
                for (int values = 0; values < 2; ++values) {
                    const int stages = values ? T::VS : T::KS, stage = j % stages;
                    const uint32_t empty = values ? bar(empty_v[stage]) : bar(empty_k[stage]), parity = ((j / stages) & 1) ^ 1;
                    if (ok && !ptx::mbar_try_wait(empty, parity)) { // what is on its way may be what the place waits for
                        settle();
                        ok = ptx::mbar_wait(empty, parity, &g_status, ST_LOAD);
                    }
                    if (!ok) continue; // (every thread comes to every barrier of locate)
                    const uint32_t dst = smem + (values ? T::V_RING + stage * T::V_BYTES : T::RING + stage * T::K_BYTES);
                    const char* const base = values ? vbase : kbase;
#pragma unroll
                    for (int i = 0; i < T::LOADS; ++i) {
                        const int token = token_of(i), c = piece_of(i);
                        const int64_t at = row_at[j & 1][token];
                        ptx::cp_async_16(dst + place(token, c), base + (at < 0 ? 0 : at) + c * 16, at >= 0);
                    }
                    ptx::cp_async_commit();
                    ++issued;
                    if (issued - arrived > 3) {
                        ptx::cp_async_wait<3>();
                        arrive();
                    }
                }
            }
            settle();
        } else {
            uint4 kw[T::LOADS], vw[T::LOADS];
            uint32_t ks[T::LOADS], vs[T::LOADS];
            auto fetch = [&](int32_t j, uint4 (&w)[T::LOADS], uint32_t (&s)[T::LOADS], const char* base, const char* sbase) {
#pragma unroll
                for (int i = 0; i < T::LOADS; ++i) {
                    const int token = token_of(i), c = piece_of(i);
                    const int64_t at = row_at[j & 1][token];
                    w[i] = at >= 0 ? ld_global_16(base + at + c * 16) : make_uint4(0, 0, 0, 0);
                    if constexpr (T::KIND == CACHE_I8_GROUPS) s[i] = at >= 0 ? load_scales<2>(sbase + scale_at[j & 1][token] + c * 4) : 0u;
                }
            };
            auto put = [&](uint32_t dst, const uint4 (&w)[T::LOADS], const uint32_t (&s)[T::LOADS], bool keys) {
#pragma unroll
                for (int i = 0; i < T::LOADS; ++i) {
                    const int token = token_of(i), c = 2 * piece_of(i);
                    uint32_t o[8], r[8] = {};
                    whole_numbers(w[i], o);
                    if constexpr (T::KIND == CACHE_I8_GROUPS) {
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            const __half2 f = as_h2(__byte_perm(s[i], 0, x < 4 ? 0x1010 : 0x3232));
                            const __half2 h = __hmul2(as_h2(o[x]), f);
                            if (keys) r[x] = h2(__hfma2(as_h2(o[x]), f, __hneg2(h)));
                            o[x] = h2(h);
                        }
                    }
                    const uint32_t a = dst + place(token, c), b = dst + place(token, c + 1);
                    ptx::st_shared_v4(a, make_uint4(o[0], o[1], o[2], o[3]));
                    ptx::st_shared_v4(b, make_uint4(o[4], o[5], o[6], o[7]));
                    if (T::LOW && keys) {
                        ptx::st_shared_v4(a + T::V_BYTES, make_uint4(r[0], r[1], r[2], r[3]));
                        ptx::st_shared_v4(b + T::V_BYTES, make_uint4(r[4], r[5], r[6], r[7]));
                    }
                }
                ptx::fence_proxy_async_smem();
            };
            if (blocks > 0) {
                locate(0);
                fetch(0, kw, ks, kbase, ksbase);
            }
            for (int32_t j = 0; j < blocks; ++j) {
                fetch(j, vw, vs, vbase, vsbase);
                const int kstage = j % T::KS, vstage = j % T::VS;
                // (after a wait that ran out nothing is stored any more, but every thread comes to every barrier of locate)
                ok = ok && ptx::mbar_wait(bar(empty_k[kstage]), ((j / T::KS) & 1) ^ 1, &g_status, ST_LOAD);
                if (ok) {
                    put(smem + T::RING + kstage * T::K_BYTES, kw, ks, true);
                    ptx::mbar_arrive(bar(full_k[kstage]));
                }
                ok = ok && ptx::mbar_wait(bar(empty_v[vstage]), ((j / T::VS) & 1) ^ 1, &g_status, ST_LOAD);
                if (j + 1 < blocks) {
                    locate(j + 1);
                    fetch(j + 1, kw, ks, kbase, ksbase);
                }
                if (ok) {
                    put(smem + T::V_RING + vstage * T::V_BYTES, vw, vs, false);
                    ptx::mbar_arrive(bar(full_v[vstage]));
                }
            }
        }
    } else {
        ptx::registers_up<176>();
        // ---- softmax ---------------------------------------------------------------------------------------------------------------
        const int stream = warp >> 2, r = threadIdx.x & 127;
        for (int t = 0; t < tiles; ++t)
            for (int x = threadIdx.x; x < 128 * (T::D / 8); x += 256) {
                const int row = x / (T::D / 8), c = x - row * (T::D / 8), of = row0 + t * 128 + row;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (of < p.rows) {
                    const int32_t sequence = (uint32_t)((uint64_t)(uint32_t)of * p.rows_magic >> p.rows_shift);
                    v = ld_global_16(p.q + sequence * p.q_stride + (int64_t)(kvh * p.rows_per_head + of - sequence * p.rows_per_head) * T::D + c * 8);
                }
                ptx::st_shared_v4(smem + t * T::Q_BYTES + (c >> 3) * (128 * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4), v);
            }
        ptx::fence_proxy_async_smem();
        ptx::mbar_arrive(bar(q_full));

        const uint32_t lanes = (uint32_t)(warp & 3) << 21; // 32 (warp & 3) in the address's upper half
        const uint32_t sum_at = tmem + lanes + T::O_COLUMN + (T::STREAMS == 2 ? stream * T::DP : 0);
        float top = kNothingSeen, sum = 0.0f;
        bool met = false, ok = true;
        if (T::STREAMS == 2 || stream == 0) {
            for (int32_t i = T::STREAMS == 2 ? stream : 0; i < tasks && ok; i += T::STREAMS) {
                const int32_t j = i >> shift;
                const int slot = j % T::INFOS;
                ok = ptx::mbar_wait(bar(info_full[slot]), (j / T::INFOS) & 1, &g_status, ST_SOFTMAX) && ptx::mbar_wait(bar(score_full[i & 1]), (i >> 1) & 1, &g_status, ST_SOFTMAX);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                ptx::tc_fence_after();
                const uint32_t at = tmem + lanes + (i & 1) * 128;
                uint32_t bits[T::NB];
#pragma unroll
                for (int c = 0; c < T::NB; c += 32) ptx::tmem_ld_32x32(at + c, reinterpret_cast<uint32_t(&)[32]>(bits[c]));
                ptx::tmem_ld_wait();
                float s[T::NB];
#pragma unroll
                for (int c = 0; c < T::NB; ++c) s[c] = __uint_as_float(bits[c]);
                const float4* const ks = reinterpret_cast<const float4*>(raw_smem + (smem - ptx::smem_addr(raw_smem)) + T::INFO) + slot * T::NB / 2;
#pragma unroll
                for (int c = 0; c < T::NB; c += 4) {
                    if constexpr (T::KIND == CACHE_I8_ROWS) {
                        const float4 f = ks[c / 4];
                        s[c] *= f.x; s[c + 1] *= f.y; s[c + 2] *= f.z; s[c + 3] *= f.w;
                    } else {
#pragma unroll
                        for (int x = 0; x < 4; ++x) s[c + x] *= p.scale_log2;
                    }
                }
                uint32_t any = 0;
#pragma unroll
                for (int c = 0; c < T::NB; c += 32) {
                    const uint32_t mask = masks[slot][c / 32];
                    any |= mask;
                    if (mask != 0xffffffffu) {
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (!(mask >> x & 1)) s[c + x] = -INFINITY;
                    }
                }
                met |= any != 0;
                float high[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int c = 4; c < T::NB; c += 4)
#pragma unroll
                    for (int x = 0; x < 4; ++x) high[x] = fmaxf(high[x], s[c + x]);
                float m = fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3]));
                if constexpr (T::KIND == CACHE_I8_ROWS) m += fmaxf(fmaxf(sizes[slot][0], sizes[slot][1]), fmaxf(sizes[slot][2], sizes[slot][3]));
                // the reference exponent moves when a weight would pass 2^14, each row's for itself
                const bool higher = m > top + 6.0f;
                if (__any_sync(0xffffffffu, higher)) {
                    const float keep = higher ? exp2_fast(top - m) : 1.0f;
                    if (higher) top = m;
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
                const float reference = top - 8.0f;
                float sums[4] = {};
#pragma unroll
                for (int c = 0; c < T::NB; c += 32) {
                    uint32_t w[16];
#pragma unroll
                    for (int x = 0; x < 32; x += 4) {
                        float e[4];
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            e[y] = exp2_fast(s[c + x + y] - reference);
                            sums[y] += e[y];
                        }
                        if constexpr (T::KIND == CACHE_I8_ROWS) {
                            const float4 f = ks[T::NB / 4 + (c + x) / 4];
                            e[0] *= f.x; e[1] *= f.y; e[2] *= f.z; e[3] *= f.w;
                        }
                        w[x / 2] = h2(__floats2half2_rn(e[0], e[1]));
                        w[x / 2 + 1] = h2(__floats2half2_rn(e[2], e[3]));
                    }
                    ptx::tmem_st_32x16(at + c / 2, w);
                }
                sum += (sums[0] + sums[1]) + (sums[2] + sums[3]);
                ptx::tmem_st_wait();
                ptx::tc_fence_before();
                ptx::mbar_arrive(bar(weight_full[i & 1]));
            }
        }
        // ---- the sums ---------------------------------------------------------------------------------------------------------------
        if (tasks > 0) ok = __all_sync(0xffffffffu, ptx::mbar_wait(bar(all_done), 0, &g_status, ST_SOFTMAX)) && ok;
        ptx::tc_fence_after();
        if (met) top = fmaxf(top, kLowest);
        if (!ok) top = sum = __int_as_float(0x7fffffff); // a wait ran out: not a number rather than a wrong one
        float own = 1.0f, other = 0.0f;
        const bool mine = T::STREAMS == 2 ? (tiles == 2 || stream == 0) : stream == 0; // whether this group writes a tile
        float* const exchange = reinterpret_cast<float*>(raw_smem + (smem - ptx::smem_addr(raw_smem)) + T::RING); // [D][128]: the rings are idle
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
                if (there)
#pragma unroll
                    for (int x = 0; x < 32; x += 4) __stcg(reinterpret_cast<float4*>(p.part_sums + at * T::D + c + x), make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]));
            }
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 12) ptx::tmem_dealloc(tmem, 512);
}

} // namespace prefix
} // namespace pplb200
