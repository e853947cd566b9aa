// Attention of one new token per sequence over the paged key-value cache, split over the tokens and joined.
//
// What bounds it is the cache: every key and value is read once, for a few multiply-adds per element.  So the work is laid out for
// loads: tiles of CT tokens of one head, numbered over all sequences and heads, are dealt out evenly to as many CTAs as the device holds
// at once, whatever the sequences' lengths; a CTA whose share begins or ends inside a sequence leaves its sums in the workspace
// and a second kernel joins them.  A warp takes 16 tokens at a time and brings them into a ring of its own: every lane copies exactly the
// bytes it will use (the dimensions of a product may be taken in any order), so that the ring needs no barrier, no swizzle and no
// second look at an address.  Scores are computed transposed, keys [16 tokens x dimensions] x queries [dimensions x 8 heads]: the eight
// columns hold the query heads that share the key head, and the weights turn into the operand of the second product, values^T x
// weights^T, by transposing 8 x 8 blocks between registers.
#include "kv_cache.cuh"

#include <algorithm>
#include <cmath>

namespace pplb200 {
namespace paged {

constexpr int WARPS = 4, ATPB = 32 * WARPS, WT = 16, CT = WARPS * WT;
constexpr int kSms = 148;
enum : int { CACHE_F16 = 0, CACHE_I8_GROUPS = 1, CACHE_I8_ROWS = 2 };

constexpr int piece(int bytes) { return bytes % 16 == 0 ? 16 : bytes % 8 == 0 ? 8 : 4; }

// Sizes of one variant: D dimensions, KIND of cache, NT blocks of eight query heads.
template <int D_, int KIND_, int NT_>
struct Shape {
    static constexpr int D = D_, KIND = KIND_, NT = NT_, HEADS = 8 * NT;
    static constexpr int ES = KIND == CACHE_F16 ? 2 : 1;
    // a quad's lane holds a quarter of the dimensions of two keys, an eighth of those of four values
    static constexpr int KB = D * ES / 4, KP = piece(KB), KN = KB / KP;
    static constexpr int VB = D * ES / 8, VP = piece(VB), VN = VB / VP;
    static constexpr int SB = D / 4, SP = piece(SB), SN = SB / SP; // CACHE_I8_GROUPS: a row's scales
    static constexpr int K_BYTES = WT * D * ES, V_BYTES = K_BYTES;
    static constexpr int SCALE_BYTES = KIND == CACHE_I8_GROUPS ? 2 * WT * SB : KIND == CACHE_I8_ROWS ? WT * 8 : 0;
    static constexpr int STAGE = K_BYTES + V_BYTES + SCALE_BYTES + 16;
    static constexpr int BUDGET = 17408; // of shared memory per warp, for three CTAs of four warps on an SM
    static constexpr int STAGES = STAGE * 4 <= BUDGET ? 4 : STAGE * 3 <= BUDGET ? 3 : 2;
    static constexpr int CTAS = STAGES * STAGE * WARPS * 3 <= 225 * 1024 ? 3 : STAGES * STAGE * WARPS * 2 <= 225 * 1024 ? 2 : 1;
    static constexpr int ROW = D + 4; // of the sums that the warps exchange
    static constexpr int EXCHANGE = WARPS * HEADS * (ROW + 2) * 4;
    static constexpr int SMEM = STAGES * STAGE * WARPS > EXCHANGE ? STAGES * STAGE * WARPS : EXCHANGE;
    static constexpr int STEPS = D / 16; // of 16 dimensions in the first product, and blocks of 16 in the second
};

} // namespace paged

namespace {

using namespace paged;

struct AttentionParams {
    const half* q;
    half* out;
    float* lse;
    const int32_t *pages, *lengths;
    int64_t q_stride, out_stride, pages_stride, tokens_in_table, batch;
    int32_t q_heads, shared, tiles; // query heads per key-value head, and how many blocks of HEADS these make
    int32_t window;
    float scale_log2;
    int32_t unit; // log2 of the bytes in which offsets of rows are counted
    pplb200_kv_cache cache;
    // workspace
    float* sums;       // [2 * CTAs][HEADS][D]
    float2* tops;      // [2 * CTAs][HEADS]: reference exponent and sum of weights
    int32_t* items;    // [CTAs][2]: the item that the CTA began and did not end (or -1), and what its share began with
};
enum : int { TAIL_NONE = 0, TAIL_MORE = 1, TAIL_END = 2 };

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? BYTES : 0; // the rest of the destination is filled with zeros
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int BYTES>
__device__ __forceinline__ void load_words(uint32_t (&w)[BYTES / 4], uint32_t at) {
    if constexpr (BYTES == 16) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
    else if constexpr (BYTES == 8) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
    else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t h2(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// A half whose bits are 0x6400 + u is 1024 + u: with the byte's sign bit flipped, u = value + 128, and 1152 taken off leaves the value.
constexpr uint32_t k1152 = 0x64806480u;
__device__ __forceinline__ uint32_t less_1152(uint32_t v) { return h2(__hsub2(as_h2(v), as_h2(k1152))); }

// Bytes 0, 2 and bytes 1, 3 of a word as pairs of halves (the first product takes dimensions in any order).
__device__ __forceinline__ void widen(uint32_t w, uint32_t& even, uint32_t& odd) {
    even = less_1152((w & 0x00ff00ffu) ^ k1152);
    odd = less_1152(((w >> 8) & 0x00ff00ffu) ^ k1152);
}
// The four bytes of the words of two tokens as pairs (token a, token b).
__device__ __forceinline__ void widen_pairs(uint32_t a, uint32_t b, uint32_t (&o)[4]) {
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    const uint32_t lo = __byte_perm(a, b, 0x5140), hi = __byte_perm(a, b, 0x7362);
    o[0] = less_1152(__byte_perm(lo, 0x64646464u, 0x4140));
    o[1] = less_1152(__byte_perm(lo, 0x64646464u, 0x4342));
    o[2] = less_1152(__byte_perm(hi, 0x64646464u, 0x4140));
    o[3] = less_1152(__byte_perm(hi, 0x64646464u, 0x4342));
}

// Tokens of a sequence that are looked at: [first, n).
__device__ __forceinline__ void visible(const AttentionParams& p, int64_t b, int32_t& first, int32_t& n) {
    n = (int32_t)min((int64_t)max(p.lengths[b], 0), p.tokens_in_table);
    first = p.window > 0 ? max(0, n - p.window) : 0;
}
// Tiles of a sequence and head; an empty sequence has one too, so that its output is written.
__device__ __forceinline__ int32_t tiles_of(const AttentionParams& p, int64_t b) {
    int32_t first, n;
    visible(p, b, first, n);
    return max(1, (n - first + CT - 1) / CT);
}

struct Share { // where a CTA's share begins or ends
    int64_t b;
    int32_t head, tile, tiles; // item of sequence b, tile of it, tiles it has
};

// Moves a cut to a multiple of `quantum` tiles from its item's beginning (or to its end), so that no piece is shorter than half of that.
__device__ __forceinline__ void snap(Share& s, int32_t quantum) {
    const int32_t t = (s.tile + quantum / 2) / quantum * quantum;
    s.tile = t > 0 && s.tiles - t <= quantum / 2 ? s.tiles : t;
}

template <class S>
__global__ void __launch_bounds__(ATPB, S::CTAS) paged_attention_kernel(const __grid_constant__ AttentionParams p) {
    extern __shared__ __align__(128) char smem[];
    __shared__ int64_t scan[WARPS], ends[2][2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int heads_per_sequence = p.cache.kv_heads * p.tiles;
    pdl_wait_prior_grid();
    pdl_launch_dependents();

    // ---- this CTA's share: tiles [c, c + 1) * total / CTAs, in the order sequence, head, tile --------------------------
    Share from, to;
    {
        const int64_t per_thread = (p.batch + ATPB - 1) / ATPB, b0 = min(p.batch, threadIdx.x * per_thread), b1 = min(p.batch, b0 + per_thread);
        int64_t mine = 0;
        for (int64_t b = b0; b < b1; ++b) mine += tiles_of(p, b);
        int64_t before = mine;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, before, m);
            if (lane >= m) before += v;
        }
        if (lane == 31) scan[warp] = before;
        __syncthreads();
        int64_t total = 0;
        before -= mine;
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) before += scan[w];
            total += scan[w];
        }
        // a cut at tile x lies in sequence b where the tiles of one head up to b are at most x / heads
        const int64_t all = total * heads_per_sequence;
        int64_t cut[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            cut[e] = (int64_t)(blockIdx.x + e) * all / gridDim.x;
            const int64_t y = cut[e] / heads_per_sequence;
            if (y >= before && y < before + mine) {
                int64_t b = b0, at = before;
                for (;; ++b) {
                    const int32_t n = tiles_of(p, b);
                    if (y < at + n) break;
                    at += n;
                }
                ends[e][0] = b;
                ends[e][1] = at;
            }
            if (threadIdx.x == 0 && cut[e] == all) ends[e][0] = p.batch, ends[e][1] = total;
        }
        __syncthreads();
        // With few tiles a CTA, pieces of a tile or two cost more to join than they spare.
        const int32_t quantum = all >= 16 * (int64_t)gridDim.x ? 1 : 4;
        Share* const end[2] = {&from, &to};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            Share& s = *end[e];
            s.b = ends[e][0];
            s.head = s.tile = s.tiles = 0;
            if (s.b < p.batch) {
                s.tiles = tiles_of(p, s.b);
                const int64_t in = cut[e] - ends[e][1] * heads_per_sequence;
                s.head = (int32_t)(in / s.tiles);
                s.tile = (int32_t)(in - (int64_t)s.head * s.tiles);
                snap(s, quantum);
            }
        }
    }
    auto item_of = [&](const Share& s) { return s.b * heads_per_sequence + s.head; };
    const int64_t last_item = item_of(to); // nothing of it if to.tile == 0

    int32_t begun = -1, began_with = TAIL_NONE;
    int64_t b = from.b;
    int32_t hh = from.head, tile0 = from.tile;
    const uint32_t ring = smem_of(smem) + warp * S::STAGES * S::STAGE;

    for (; b < p.batch; tile0 = 0) {
        const int64_t item = b * heads_per_sequence + hh;
        int32_t first, n;
        visible(p, b, first, n);
        const int32_t tiles = max(1, (n - first + CT - 1) / CT);
        if (item > last_item || (item == last_item && to.tile <= tile0)) break;
        const int32_t tile1 = item == last_item ? to.tile : tiles;
        if (tile0 < tile1) {
            const int kvh = hh / p.tiles, q_first = (hh - kvh * p.tiles) * S::HEADS;
            const int q_count = min(S::HEADS, p.shared - q_first);
            const char* const kbase = (const char*)p.cache.k + (int64_t)kvh * p.cache.head_stride * S::ES;
            const char* const vbase = (const char*)p.cache.v + (int64_t)kvh * p.cache.head_stride * S::ES;
            const half* const ksbase = (const half*)p.cache.k_scale + (int64_t)kvh * p.cache.scale_head_stride;
            const half* const vsbase = (const half*)p.cache.v_scale + (int64_t)kvh * p.cache.scale_head_stride;
            const int32_t* const row_pages = p.pages + b * p.pages_stride;

            // ---- queries: column g of block nt, the dimensions of quad lane t --------------------------------------------
            uint32_t q[S::NT][S::STEPS][2];
#pragma unroll
            for (int nt = 0; nt < S::NT; ++nt) {
                const int h = nt * 8 + g;
                const half* src = p.q + b * p.q_stride + (int64_t)(kvh * p.shared + q_first + h) * S::D;
                constexpr int EP = S::KP / S::ES; // dimensions of a piece, EP / 4 steps
#pragma unroll
                for (int i = 0; i < S::KN; ++i)
#pragma unroll
                    for (int s = 0; s < EP / 4; ++s) {
                        uint2 w = make_uint2(0, 0);
                        if (h < q_count) w = *reinterpret_cast<const uint2*>(src + (i * 4 + t) * EP + s * 4);
                        q[nt][i * (EP / 4) + s][0] = S::ES == 2 ? w.x : __byte_perm(w.x, w.y, 0x5410);
                        q[nt][i * (EP / 4) + s][1] = S::ES == 2 ? w.y : __byte_perm(w.x, w.y, 0x7632);
                    }
            }

            float o[S::NT][S::STEPS][4] = {}, top[S::NT][2], sum[S::NT][2] = {};
#pragma unroll
            for (int nt = 0; nt < S::NT; ++nt) top[nt][0] = top[nt][1] = -1e30f;

            // ---- the ring --------------------------------------------------------------------------------------------------
            // Lane l looks after token l % 16 of a tile: its page, then the offset of its row.
            auto token_of = [&](int32_t tile) { return first + tile * CT + warp * WT + (lane & 15); };
            auto page_of = [&](int32_t tile) {
                const int32_t token = token_of(tile);
                return tile < tile1 && token < n ? row_pages[token / p.cache.page_size] : -1;
            };
            // CACHE_I8_ROWS: the key's scale (lanes 0 to 15) or the value's of the lane's token.  Two bytes are too few for the copy engine:
            // they come through a register, and are put into their stage when the next one is requested.
            auto request = [&](int32_t tile, int32_t page, uint32_t stage, float& scale_ahead) {
                const int32_t token = token_of(tile);
                const bool ok = page >= 0 && page < p.cache.num_pages;
                const int32_t in_page = token - token / p.cache.page_size * p.cache.page_size;
                const uint32_t seen = __ballot_sync(0xffffffffu, ok) & 0xffffu;
                const uint32_t off = ok ? (uint32_t)((((int64_t)page * p.cache.page_stride + (int64_t)in_page * p.cache.token_stride) * S::ES) >> p.unit) : 0u;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int row = g + 8 * r;
                    const char* src = kbase + ((uint64_t)__shfl_sync(0xffffffffu, off, row) << p.unit) + t * S::KP;
#pragma unroll
                    for (int i = 0; i < S::KN; ++i)
                        copy_async<S::KP>(stage + ((r * S::KN + i) * 32 + lane) * S::KP, src + i * 4 * S::KP, seen >> row & 1);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int row = 2 * t + (j & 1) + 8 * (j >> 1);
                    const char* src = vbase + ((uint64_t)__shfl_sync(0xffffffffu, off, row) << p.unit) + g * S::VP;
#pragma unroll
                    for (int i = 0; i < S::VN; ++i)
                        copy_async<S::VP>(stage + S::K_BYTES + ((j * S::VN + i) * 32 + lane) * S::VP, src + i * 8 * S::VP, seen >> row & 1);
                }
                if constexpr (S::KIND != CACHE_F16) {
                    const int64_t at = ok ? (int64_t)page * p.cache.scale_page_stride + (int64_t)in_page * p.cache.scale_token_stride : 0;
                    if constexpr (S::KIND == CACHE_I8_ROWS) {
                        scale_ahead = ok ? __half2float(ld_global_half((lane < 16 ? ksbase : vsbase) + at)) : 0.0f;
                    } else {
#pragma unroll
                        for (int i = 0; i < WT * S::SN; i += 32) {
                            const int row = (i + lane) / S::SN, part = (i + lane) - row * S::SN;
                            const int64_t from_row = __shfl_sync(0xffffffffu, at, row & 15);
                            if (i + lane < WT * S::SN) {
                                const bool there = seen >> row & 1;
                                const uint32_t dst = stage + S::K_BYTES + S::V_BYTES + (i + lane) * S::SP;
                                copy_async<S::SP>(dst, ksbase + from_row + part * (S::SP / 2), there);
                                copy_async<S::SP>(dst + WT * S::SB, vsbase + from_row + part * (S::SP / 2), there);
                            }
                        }
                    }
                }
                if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(stage + S::STAGE - 16), "r"(seen) : "memory");
                copy_commit();
            };
            auto put_scale = [&](uint32_t stage, float scale) {
                if constexpr (S::KIND == CACHE_I8_ROWS)
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(stage + S::K_BYTES + S::V_BYTES + (lane & 15) * 8 + (lane >> 4) * 4), "f"(scale) : "memory");
            };

            float scale_ahead = 0.0f;
            uint32_t scale_stage = ring;
            {
                int32_t pages[S::STAGES];
                float scales[S::STAGES] = {};
#pragma unroll
                for (int s = 0; s < S::STAGES; ++s) pages[s] = page_of(tile0 + s);
#pragma unroll
                for (int s = 0; s < S::STAGES; ++s) request(tile0 + s, pages[s], ring + s * S::STAGE, scales[s]);
#pragma unroll
                for (int s = 0; s < S::STAGES; ++s) put_scale(ring + s * S::STAGE, scales[s]);
                scale_ahead = scales[0];
            }
            int32_t page_ahead = page_of(tile0 + S::STAGES);
            uint32_t stage = ring;
            for (int32_t tile = tile0; tile < tile1; ++tile) {
                put_scale(scale_stage, scale_ahead);
                copy_wait<S::STAGES - 1>();
                __syncwarp();
                uint32_t seen;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(seen) : "r"(stage + S::STAGE - 16) : "memory");
                if (seen != 0) {
                    // ---- scores [16 tokens x 8 heads] ----------------------------------------------------------------------
                    float c[S::NT][4] = {};
                    constexpr int KW = S::KP / 4;
#pragma unroll
                    for (int i = 0; i < S::KN; ++i) {
                        uint32_t w0[KW], w1[KW];
                        load_words<S::KP>(w0, stage + (i * 32 + lane) * S::KP);
                        load_words<S::KP>(w1, stage + ((S::KN + i) * 32 + lane) * S::KP);
                        if constexpr (S::ES == 2) {
#pragma unroll
                            for (int s = 0; s < KW / 2; ++s)
#pragma unroll
                                for (int nt = 0; nt < S::NT; ++nt) {
                                    const auto& b = q[nt][i * (KW / 2) + s];
                                    mma(c[nt], w0[2 * s], w1[2 * s], w0[2 * s + 1], w1[2 * s + 1], b[0], b[1]);
                                }
                        } else {
                            // scales of this piece's dimensions for keys g and g + 8
                            constexpr int GROUPS = S::KP >= 8 ? S::KP / 8 : 1;
                            uint32_t s0[GROUPS], s1[GROUPS];
                            if constexpr (S::KIND == CACHE_I8_GROUPS) {
#pragma unroll
                                for (int j = 0; j < GROUPS; ++j) {
                                    const uint32_t at = stage + S::K_BYTES + S::V_BYTES + ((i * 4 + t) * GROUPS + j) * 2;
                                    uint16_t x, y;
                                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(at + g * S::SB) : "memory");
                                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(y) : "r"(at + (g + 8) * S::SB) : "memory");
                                    s0[j] = x * 0x10001u;
                                    s1[j] = y * 0x10001u;
                                }
                            }
#pragma unroll
                            for (int s = 0; s < KW; ++s) {
                                uint32_t a0, a1, a2, a3;
                                widen(w0[s], a0, a2);
                                widen(w1[s], a1, a3);
                                if constexpr (S::KIND == CACHE_I8_GROUPS) {
                                    // value x scale has up to 18 bits: its rounding to fp16, and what that left, as a second operand
                                    const __half2 f0 = as_h2(s0[s / 2]), f1 = as_h2(s1[s / 2]);
                                    const __half2 h0 = __hmul2(as_h2(a0), f0), h1 = __hmul2(as_h2(a1), f1), h2_ = __hmul2(as_h2(a2), f0), h3 = __hmul2(as_h2(a3), f1);
                                    const uint32_t r0 = h2(__hfma2(as_h2(a0), f0, __hneg2(h0))), r1 = h2(__hfma2(as_h2(a1), f1, __hneg2(h1)));
                                    const uint32_t r2 = h2(__hfma2(as_h2(a2), f0, __hneg2(h2_))), r3 = h2(__hfma2(as_h2(a3), f1, __hneg2(h3)));
#pragma unroll
                                    for (int nt = 0; nt < S::NT; ++nt) {
                                        const auto& b = q[nt][i * KW + s];
                                        mma(c[nt], h2(h0), h2(h1), h2(h2_), h2(h3), b[0], b[1]);
                                        mma(c[nt], r0, r1, r2, r3, b[0], b[1]);
                                    }
                                } else {
#pragma unroll
                                    for (int nt = 0; nt < S::NT; ++nt) mma(c[nt], a0, a1, a2, a3, q[nt][i * KW + s][0], q[nt][i * KW + s][1]);
                                }
                            }
                        }
                    }

                    // ---- weights: 2^(score - top + 8) ----------------------------------------------------------------------
                    float f0 = p.scale_log2, f1 = p.scale_log2, v0 = 1.0f, v1 = 1.0f, e0 = 0.0f, e1 = 0.0f;
                    if constexpr (S::KIND == CACHE_I8_ROWS) {
                        const uint32_t at = stage + S::K_BYTES + S::V_BYTES;
                        float k0, k1;
                        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(k0), "=f"(v0) : "r"(at + g * 8) : "memory");
                        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(k1), "=f"(v1) : "r"(at + (g + 8) * 8) : "memory");
                        f0 *= k0;
                        f1 *= k1;
                        // the value's scale goes into the weight; 2^e is above it
                        e0 = (float)max((int)(__float_as_uint(v0) >> 23) - 126, -24);
                        e1 = (float)max((int)(__float_as_uint(v1) >> 23) - 126, -24);
                    }
                    bool higher = false;
#pragma unroll
                    for (int nt = 0; nt < S::NT; ++nt) {
                        c[nt][0] *= f0; c[nt][1] *= f0;
                        c[nt][2] *= f1; c[nt][3] *= f1;
                    }
                    if (seen != 0xffffu) {
#pragma unroll
                        for (int nt = 0; nt < S::NT; ++nt) {
                            if (!(seen >> g & 1)) c[nt][0] = c[nt][1] = -INFINITY;
                            if (!(seen >> (g + 8) & 1)) c[nt][2] = c[nt][3] = -INFINITY;
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < S::NT; ++nt) {
                        higher |= fmaxf(c[nt][0] + e0, c[nt][2] + e1) > top[nt][0] + 6.0f;
                        higher |= fmaxf(c[nt][1] + e0, c[nt][3] + e1) > top[nt][1] + 6.0f;
                    }
                    // The reference exponent need not be the maximum: it moves when a weight would pass 2^14, which after the first tiles is rare.
                    if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
                        for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                float m = fmaxf(c[nt][k] + e0, c[nt][2 + k] + e1);
#pragma unroll
                                for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
                                m = fmaxf(m, top[nt][k]);
                                const float keep = exp2_fast(top[nt][k] - m);
                                top[nt][k] = m;
                                sum[nt][k] *= keep;
#pragma unroll
                                for (int j = 0; j < S::STEPS; ++j) {
                                    o[nt][j][k] *= keep;
                                    o[nt][j][2 + k] *= keep;
                                }
                            }
                    }
                    uint32_t wh[S::NT][2], wl[S::NT][2]; // weights in fp16, and what the rounding left: together 22 bits
#pragma unroll
                    for (int nt = 0; nt < S::NT; ++nt) {
                        const float a = exp2_fast(c[nt][0] - (top[nt][0] - 8.0f)), b2 = exp2_fast(c[nt][1] - (top[nt][1] - 8.0f));
                        const float a1 = exp2_fast(c[nt][2] - (top[nt][0] - 8.0f)), b1 = exp2_fast(c[nt][3] - (top[nt][1] - 8.0f));
                        sum[nt][0] += a + a1;
                        sum[nt][1] += b2 + b1;
                        const __half2 x = __floats2half2_rn(a * v0, b2 * v0), y = __floats2half2_rn(a1 * v1, b1 * v1);
                        const float2 xf = __half22float2(x), yf = __half22float2(y);
                        wh[nt][0] = transpose8x8(h2(x));
                        wh[nt][1] = transpose8x8(h2(y));
                        wl[nt][0] = transpose8x8(h2(__floats2half2_rn(a * v0 - xf.x, b2 * v0 - xf.y)));
                        wl[nt][1] = transpose8x8(h2(__floats2half2_rn(a1 * v1 - yf.x, b1 * v1 - yf.y)));
                    }

                    // ---- values^T x weights^T ------------------------------------------------------------------------------
                    constexpr int VW = S::VP / 4, EP = S::VP / S::ES; // words and dimensions of a piece
#pragma unroll
                    for (int i = 0; i < S::VN; ++i) {
                        uint32_t w[4][VW];
#pragma unroll
                        for (int j = 0; j < 4; ++j) load_words<S::VP>(w[j], stage + S::K_BYTES + ((j * S::VN + i) * 32 + lane) * S::VP);
                        if constexpr (S::ES == 2) {
#pragma unroll
                            for (int x = 0; x < VW; ++x) {
                                const uint32_t a0 = __byte_perm(w[0][x], w[1][x], 0x5410), a1 = __byte_perm(w[0][x], w[1][x], 0x7632);
                                const uint32_t a2 = __byte_perm(w[2][x], w[3][x], 0x5410), a3 = __byte_perm(w[2][x], w[3][x], 0x7632);
#pragma unroll
                                for (int nt = 0; nt < S::NT; ++nt) {
                                    mma(o[nt][i * EP / 2 + x], a0, a1, a2, a3, wh[nt][0], wh[nt][1]);
                                    mma(o[nt][i * EP / 2 + x], a0, a1, a2, a3, wl[nt][0], wl[nt][1]);
                                }
                            }
                        } else {
#pragma unroll
                            for (int x = 0; x < VW; ++x) {
                                uint32_t u[4], v[4];
                                widen_pairs(w[0][x], w[1][x], u);
                                widen_pairs(w[2][x], w[3][x], v);
                                if constexpr (S::KIND == CACHE_I8_GROUPS) {
                                    // the group of these four dimensions; value x scale is rounded to fp16, as it is when it is read back
                                    const int group = ((i * 8 + g) * EP + x * 4) / 8;
                                    const uint32_t at = stage + S::K_BYTES + S::V_BYTES + WT * S::SB + group * 2;
                                    uint16_t s[4];
#pragma unroll
                                    for (int j = 0; j < 4; ++j)
                                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(s[j]) : "r"(at + (2 * t + (j & 1) + 8 * (j >> 1)) * S::SB) : "memory");
                                    const __half2 fu = as_h2(s[0] | (uint32_t)s[1] << 16), fv = as_h2(s[2] | (uint32_t)s[3] << 16);
#pragma unroll
                                    for (int y = 0; y < 4; ++y) {
                                        u[y] = h2(__hmul2(as_h2(u[y]), fu));
                                        v[y] = h2(__hmul2(as_h2(v[y]), fv));
                                    }
                                }
#pragma unroll
                                for (int y = 0; y < 2; ++y)
#pragma unroll
                                    for (int nt = 0; nt < S::NT; ++nt) {
                                        mma(o[nt][i * EP / 2 + 2 * x + y], u[2 * y], u[2 * y + 1], v[2 * y], v[2 * y + 1], wh[nt][0], wh[nt][1]);
                                        mma(o[nt][i * EP / 2 + 2 * x + y], u[2 * y], u[2 * y + 1], v[2 * y], v[2 * y + 1], wl[nt][0], wl[nt][1]);
                                    }
                            }
                        }
                    }
                }
                __syncwarp();
                request(tile + S::STAGES, page_ahead, stage, scale_ahead);
                scale_stage = stage;
                page_ahead = page_of(tile + S::STAGES + 1);
                stage = stage == ring + (S::STAGES - 1) * S::STAGE ? ring : stage + S::STAGE;
            }
            copy_wait<0>();
            __syncthreads();

            // ---- the four warps' sums --------------------------------------------------------------------------------------
            float* const part = reinterpret_cast<float*>(smem);                 // [warp][head][ROW]
            float* const tops = part + WARPS * S::HEADS * S::ROW;               // [warp][head][2]
#pragma unroll
            for (int nt = 0; nt < S::NT; ++nt) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float s = sum[nt][k];
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
                    const int h = nt * 8 + 2 * t + k;
                    if (g == 0) {
                        tops[(warp * S::HEADS + h) * 2] = top[nt][k];
                        tops[(warp * S::HEADS + h) * 2 + 1] = s;
                    }
                    constexpr int EP = S::VP / S::ES;
#pragma unroll
                    for (int i = 0; i < S::VN; ++i)
#pragma unroll
                        for (int x = 0; x < EP; x += 4)
                            *reinterpret_cast<float4*>(&part[(warp * S::HEADS + h) * S::ROW + (i * 8 + g) * EP + x]) =
                                make_float4(o[nt][(i * EP + x) / 2][k], o[nt][(i * EP + x) / 2][2 + k], o[nt][(i * EP + x) / 2 + 1][k], o[nt][(i * EP + x) / 2 + 1][2 + k]);
                }
            }
            __syncthreads();
            const bool whole = tile0 == 0 && tile1 == tiles;
            const int64_t slot = 2 * (int64_t)blockIdx.x + (tile0 == 0 ? 1 : 0);
            for (int x = threadIdx.x; x < q_count * (S::D / 4); x += ATPB) {
                const int h = x / (S::D / 4), d = (x - h * (S::D / 4)) * 4;
                float m = -1e30f, l = 0.0f;
                float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
                for (int w = 0; w < WARPS; ++w) m = fmaxf(m, tops[(w * S::HEADS + h) * 2]);
#pragma unroll
                for (int w = 0; w < WARPS; ++w) {
                    const float f = exp2_fast(tops[(w * S::HEADS + h) * 2] - m);
                    const float4 a = *reinterpret_cast<const float4*>(&part[(w * S::HEADS + h) * S::ROW + d]);
                    l += f * tops[(w * S::HEADS + h) * 2 + 1];
                    v.x += f * a.x; v.y += f * a.y; v.z += f * a.z; v.w += f * a.w;
                }
                if (whole) {
                    const int head = kvh * p.shared + q_first + h;
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    const uint2 r = make_uint2(h2(__floats2half2_rn(v.x * inv, v.y * inv)), h2(__floats2half2_rn(v.z * inv, v.w * inv)));
                    *reinterpret_cast<uint2*>(p.out + b * p.out_stride + (int64_t)head * S::D + d) = r;
                    if (p.lse && d == 0) p.lse[b * p.q_heads + head] = l == 0.0f ? -INFINITY : (m - 8.0f + log2f(l)) * 0.69314718055994531f;
                } else {
                    *reinterpret_cast<float4*>(p.sums + (slot * S::HEADS + h) * S::D + d) = v;
                    if (d == 0) p.tops[slot * S::HEADS + h] = make_float2(m, l);
                }
            }
            __syncthreads();
            if (tile0 != 0) began_with = tile1 == tiles ? TAIL_END : TAIL_MORE;
            else if (!whole) begun = (int32_t)item;
        }
        if (++hh == heads_per_sequence) hh = 0, ++b;
    }
    if (threadIdx.x == 0 && p.items) *reinterpret_cast<int2*>(p.items + 2 * blockIdx.x) = make_int2(begun, began_with);
}

// Joins the pieces of the item that CTA blockIdx.x began and others went on with, in the order of the tokens: a warp per query head.
template <int D, int HEADS>
__global__ void __launch_bounds__(ATPB) paged_attention_join_kernel(const __grid_constant__ AttentionParams p, int32_t ctas) {
    constexpr int V = D / 32;
    pdl_wait_prior_grid();
    const int lane = threadIdx.x & 31, h = blockIdx.y * WARPS + (threadIdx.x >> 5);
    const int32_t item = p.items[2 * blockIdx.x];
    if (item < 0) return;
    const int heads_per_sequence = p.cache.kv_heads * p.tiles;
    const int64_t b = item / heads_per_sequence;
    const int hh = (int)(item - b * heads_per_sequence), kvh = hh / p.tiles, q_first = (hh - kvh * p.tiles) * HEADS;
    if (h >= min(HEADS, p.shared - q_first)) return;
    float m = -1e30f, l = 0.0f, o[V] = {};
    auto add = [&](int64_t slot, float w) {
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] += w * p.sums[(slot * HEADS + h) * D + i * 32 + lane];
    };
    {
        const int64_t slot = 2 * (int64_t)blockIdx.x + 1;
        const float2 s = p.tops[slot * HEADS + h];
        m = s.x;
        l = s.y;
        add(slot, 1.0f);
    }
    for (int32_t c0 = blockIdx.x + 1; c0 < ctas; c0 += 32) {
        const int32_t c = c0 + lane;
        int32_t kind = c < ctas ? p.items[2 * c + 1] : TAIL_NONE;
        const uint32_t end = __ballot_sync(0xffffffffu, kind == TAIL_END);
        const uint32_t upto = end ? (end & (0u - end)) * 2u - 1u : 0xffffffffu; // lanes up to the one that ends the item
        if (!(upto >> lane & 1)) kind = TAIL_NONE;
        const float2 s = kind != TAIL_NONE ? p.tops[2 * (int64_t)c * HEADS + h] : make_float2(-1e30f, 0.0f);
        float top = s.x;
#pragma unroll
        for (int x = 16; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        top = fmaxf(top, m);
        const float keep = exp2_fast(m - top), w = kind != TAIL_NONE ? exp2_fast(s.x - top) : 0.0f;
        m = top;
        float part = w * s.y;
#pragma unroll
        for (int x = 16; x >= 1; x >>= 1) part += __shfl_xor_sync(0xffffffffu, part, x);
        l = l * keep + part;
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] *= keep;
        uint32_t todo = __ballot_sync(0xffffffffu, kind != TAIL_NONE);
        while (todo) {
            const int x = __ffs(todo) - 1;
            todo &= todo - 1;
            add(2 * (int64_t)(c0 + x), __shfl_sync(0xffffffffu, w, x));
        }
        if (end) break;
    }
    const int head = kvh * p.shared + q_first + h;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < V; ++i) p.out[b * p.out_stride + (int64_t)head * D + i * 32 + lane] = __float2half_rn(o[i] * inv);
    if (p.lse && lane == 0) p.lse[b * p.q_heads + head] = l == 0.0f ? -INFINITY : (m - 8.0f + log2f(l)) * 0.69314718055994531f;
}

// Query heads that a CTA takes at once: two blocks of eight where that many share a key-value head and registers allow.
int heads_at_once(int32_t head_dim, int32_t shared) { return shared > 8 && head_dim <= 128 ? 16 : 8; }
constexpr int kMostCtas = 3 * kSms;

template <class S>
int32_t launch(cudaStream_t stream, AttentionParams& p, int64_t tokens) {
    static_assert(S::CTAS * kSms <= kMostCtas, "workspace");
    if (cudaFuncSetAttribute(paged_attention_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM) != cudaSuccess)
        return fail(RC_DEVICE_RUNTIME_ERROR, "shared memory of the attention kernel: %s", cudaGetErrorString(cudaGetLastError()));
    const int64_t tiles = (tokens + CT - 1) / CT;
    const int64_t items = p.batch * p.cache.kv_heads * p.tiles;
    const int64_t most = S::CTAS * kSms;
    const int64_t ctas = tiles > most || items > most ? most : std::min(most, items * std::max<int64_t>(1, tiles));
    launch_ex(paged_attention_kernel<S>, dim3((unsigned)ctas), dim3(ATPB), (size_t)S::SMEM, stream, true, p);
    int32_t rc = check_launch("paged attention");
    if (rc != RC_SUCCESS) return rc;
    // no cut falls inside an item of one tile, nor, where cuts are moved by four tiles (see `quantum`), of six
    if (tiles <= 1 || (tiles <= 6 && items * tiles < 16 * ctas)) return RC_SUCCESS;
    launch_ex(paged_attention_join_kernel<S::D, S::HEADS>, dim3((unsigned)ctas, S::HEADS / WARPS), dim3(ATPB), stream, true, p, (int32_t)ctas);
    return check_launch("joining of attention");
}

template <int D>
int32_t launch_kind(cudaStream_t stream, AttentionParams& p, int64_t tokens) {
    const int kind = p.cache.quant_group == 0 ? CACHE_F16 : p.cache.quant_group == 8 ? CACHE_I8_GROUPS : CACHE_I8_ROWS;
    if constexpr (D <= 128) {
        if (heads_at_once(D, p.shared) == 16) {
            if (kind == CACHE_F16) return launch<Shape<D, CACHE_F16, 2>>(stream, p, tokens);
            if (kind == CACHE_I8_GROUPS) return launch<Shape<D, CACHE_I8_GROUPS, 2>>(stream, p, tokens);
            return launch<Shape<D, CACHE_I8_ROWS, 2>>(stream, p, tokens);
        }
    }
    if (kind == CACHE_F16) return launch<Shape<D, CACHE_F16, 1>>(stream, p, tokens);
    if (kind == CACHE_I8_GROUPS) return launch<Shape<D, CACHE_I8_GROUPS, 1>>(stream, p, tokens);
    return launch<Shape<D, CACHE_I8_ROWS, 1>>(stream, p, tokens);
}

} // namespace
} // namespace pplb200

using namespace pplb200;

extern "C" {

int64_t pplb200_paged_decode_attention_workspace_bytes(int64_t batch, int64_t max_tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
    if (batch < 0 || max_tokens < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || head_dim <= 0) return -1;
    // two pieces a CTA at most
    const int heads = heads_at_once(head_dim, q_heads / kv_heads);
    return round_up(kMostCtas * 8, 256) + round_up(2 * kMostCtas * heads * 8, 256) + 2LL * kMostCtas * heads * head_dim * 4;
}

int32_t pplb200_paged_decode_attention_fp16(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_paged_attention_args* a) {
    const int32_t rc = check_kv_cache(cache);
    if (rc != RC_SUCCESS) return rc;
    if (!a) return fail(RC_INVALID_VALUE, "null arguments");
    const int64_t D = cache->head_dim;
    if (D != 64 && D != 96 && D != 128 && D != 256) return fail(RC_UNSUPPORTED, "attention: head_dim must be 64, 96, 128 or 256, got %lld", (long long)D);
    if (a->batch < 0 || a->pages_per_sequence < 0) return fail(RC_INVALID_VALUE, "negative extent");
    if (a->batch > 65535) return fail(RC_UNSUPPORTED, "more than 65535 sequences");
    if (a->q_heads <= 0 || a->q_heads > 65535 || a->q_heads % cache->kv_heads)
        return fail(RC_INVALID_VALUE, "q_heads (%d) must be a multiple of the cache's heads (%d)", a->q_heads, cache->kv_heads);
    if (!std::isfinite(a->scale)) return fail(RC_INVALID_VALUE, "the scale must be finite");
    if (a->batch == 0) return RC_SUCCESS;
    if (!a->q || !a->out || !aligned16(a->q) || !aligned16(a->out)) return fail(RC_INVALID_VALUE, "q and out must be 16-byte aligned pointers");
    if (a->q_stride % 8 || a->out_stride % 8 || (a->batch > 1 && (a->q_stride < a->q_heads * D || a->out_stride < a->q_heads * D)))
        return fail(RC_INVALID_VALUE, "q / out: sequences must be a multiple of 8 elements apart, and no closer than their heads are long");
    if (!a->lengths || (a->pages_per_sequence > 0 && !a->pages)) return fail(RC_INVALID_VALUE, "null lengths or pages");
    if ((((uintptr_t)a->lengths | (uintptr_t)a->pages | (uintptr_t)a->optional_lse) & 3) != 0) return fail(RC_INVALID_VALUE, "lengths, pages and lse must be 4-byte aligned");
    if (a->batch > 1 && a->pages_stride < a->pages_per_sequence) return fail(RC_INVALID_VALUE, "rows of the page table overlap");
    // token numbers are 32-bit, and go a few tiles beyond the last one
    if (a->pages_per_sequence > (1LL << 30) / cache->page_size) return fail(RC_UNSUPPORTED, "a page table of more than 2^30 tokens");
    const int64_t need = pplb200_paged_decode_attention_workspace_bytes(a->batch, a->pages_per_sequence * cache->page_size, a->q_heads, cache->kv_heads, cache->head_dim);
    if (!a->ws || a->ws_bytes < need || ((uintptr_t)a->ws & 255))
        return fail(RC_INVALID_VALUE, "workspace of %lld bytes (256-byte aligned) needed, got %lld", (long long)need, (long long)a->ws_bytes);
    AttentionParams p = {};
    if (cache->quant_group == 8) {
        const int64_t unit = D == 96 ? 4 : 8;
        if ((((uintptr_t)cache->k_scale | (uintptr_t)cache->v_scale) & (2 * unit - 1)) || cache->scale_page_stride % unit || cache->scale_head_stride % unit || cache->scale_token_stride % unit)
            return fail(RC_INVALID_VALUE, "attention: scales of groups of 8 must be aligned to, and their strides multiples of, %lld bytes", (long long)(2 * unit));
    }
    // Offsets of rows travel between lanes as 32-bit numbers of the largest power of two of bytes that divides the strides.
    const int64_t es = cache->quant_group ? 1 : 2;
    const uint64_t strides = (uint64_t)(cache->page_stride | cache->token_stride) * es;
    p.unit = strides ? __builtin_ctzll(strides) : 4;
    if (cache->num_pages > 0) {
        const __int128 last = ((__int128)(cache->num_pages - 1) * cache->page_stride + (__int128)(cache->page_size - 1) * cache->token_stride) * es;
        if ((last >> p.unit) >= ((__int128)1 << 32)) return fail(RC_UNSUPPORTED, "attention: a cache whose rows lie further apart than 2^32 times their alignment");
    }
    p.q = (const half*)a->q; p.out = (half*)a->out; p.lse = a->optional_lse;
    p.pages = a->pages; p.lengths = a->lengths;
    p.q_stride = a->q_stride; p.out_stride = a->out_stride;
    p.pages_stride = a->pages_stride; p.tokens_in_table = a->pages_per_sequence * cache->page_size; p.batch = a->batch;
    p.q_heads = a->q_heads; p.shared = a->q_heads / cache->kv_heads;
    const int heads = heads_at_once(cache->head_dim, p.shared);
    p.tiles = (p.shared + heads - 1) / heads;
    p.window = a->window; p.scale_log2 = a->scale * 1.4426950408889634f;
    p.cache = *cache;
    p.items = (int32_t*)a->ws;
    p.tops = (float2*)((char*)a->ws + round_up(kMostCtas * 8, 256));
    p.sums = (float*)((char*)p.tops + round_up(2 * kMostCtas * heads * 8, 256));
    if (a->batch * (int64_t)cache->kv_heads * p.tiles > 0x7fffffffLL) return fail(RC_UNSUPPORTED, "too many sequences and heads");
    const cudaStream_t s = (cudaStream_t)stream;
    if (D == 64) return launch_kind<64>(s, p, p.tokens_in_table);
    if (D == 96) return launch_kind<96>(s, p, p.tokens_in_table);
    if (D == 128) return launch_kind<128>(s, p, p.tokens_in_table);
    return launch_kind<256>(s, p, p.tokens_in_table);
}

} // extern "C"
