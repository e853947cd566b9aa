// Attention of one new token per sequence over the paged key-value cache, split over the tokens and joined.
//
// What bounds it is the cache: every key and value is read once, for a few multiply-adds per element.  So the work is laid out for
// loads: tiles of CT tokens of one head, numbered over all sequences and heads, are dealt out evenly to as many CTAs as the device holds
// at once, whatever the sequences' lengths; a CTA whose share begins or ends inside a sequence leaves its sums in the workspace
// and a second kernel joins them.  A warp takes 16 tokens at a time, and while it works on these the next ones are on their way into
// its registers: a lane loads exactly the bytes that it will use (the dimensions of a product may be taken in any order), so that
// nothing passes through shared memory.  Scores are computed transposed, keys [16 tokens x dimensions] x queries [dimensions x 8
// heads]: the eight columns hold the query heads that share the key head, and the weights turn into the operand of the second
// product, values^T x weights^T, by transposing 8 x 8 blocks between registers.
#include "kv_cache.cuh"

#include <algorithm>
#include <cmath>

namespace pplb200 {
namespace paged {

constexpr int WARPS = 4, ATPB = 32 * WARPS, WT = 16, CT = WARPS * WT;
constexpr int kSms = 148, kMostCtas = 4 * kSms;
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
    static constexpr int KG = KP >= 8 ? KP / 8 : 1, VG = VP >= 8 ? VP / 8 : 1; // CACHE_I8_GROUPS: scales of a piece
    // CTAs on an SM, by the registers a thread needs: sums, queries and a tile on its way
    static constexpr int REGS = NT * D / 4 + NT * D / 8 + D * ES / 4;
    static constexpr int CTAS = REGS <= 80 ? 4 : REGS <= 128 ? 3 : 2;
    static constexpr int ROW = D + 4; // of the sums that the warps exchange
    static constexpr int EXCHANGE = WARPS * HEADS * (ROW + 2) * 4;
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
    int32_t num_pages;
    // Offsets of rows and scales within a head, which travel between lanes, are 32-bit numbers of `unit` and `scale_unit` bytes.
    uint32_t unit, page_units, token_units, scale_unit, scale_page_units, scale_token_units;
    uint32_t page_magic, page_shift; // token / page_size = token * page_magic >> page_shift
    pplb200_kv_cache cache;
    // workspace
    float* sums;       // [2 * CTAs][HEADS][D]
    float2* tops;      // [2 * CTAs][HEADS]: reference exponent and sum of weights
    int32_t* items;    // [CTAs][2]: the item that the CTA began and did not end (or -1), and what its share began with
};
enum : int { TAIL_NONE = 0, TAIL_MORE = 1, TAIL_END = 2 };

// A piece of a row, read once: kept out of L1.  volatile: loads stay where they are put, ahead of the work on the tile before.
template <int BYTES>
__device__ __forceinline__ void load_piece(uint32_t (&w)[BYTES / 4], const char* p) {
    if constexpr (BYTES == 16) asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
    else if constexpr (BYTES == 8) asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    else asm volatile("ld.global.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
}
// N neighbouring scales of two bytes, in one word
template <int N>
__device__ __forceinline__ uint32_t load_scales(const char* p) {
    uint32_t w;
    if constexpr (N == 2) {
        asm volatile("ld.global.u32 %0, [%1];" : "=r"(w) : "l"(p));
    } else {
        uint16_t x;
        asm volatile("ld.global.u16 %0, [%1];" : "=h"(x) : "l"(p));
        w = x;
    }
    return w;
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
    __shared__ __align__(16) float part[WARPS * S::HEADS * S::ROW], tops[WARPS * S::HEADS * 2];
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
            const char* const ksbase = (const char*)p.cache.k_scale + (int64_t)kvh * p.cache.scale_head_stride * 2;
            const char* const vsbase = (const char*)p.cache.v_scale + (int64_t)kvh * p.cache.scale_head_stride * 2;
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

            // ---- tiles on their way ----------------------------------------------------------------------------------------
            // Lane l looks after token l % 16 of a tile: its page, two tiles ahead, then where its row lies, one tile ahead.
            struct Place {
                int32_t page;
                uint32_t in_page;
            };
            auto find = [&](int32_t tile) {
                const int32_t token = first + tile * CT + warp * WT + (lane & 15);
                const uint32_t index = (uint32_t)((uint64_t)(uint32_t)token * p.page_magic >> p.page_shift);
                Place at;
                at.page = tile < tile1 && token < n ? row_pages[index] : -1;
                at.in_page = token - index * p.cache.page_size;
                return at;
            };
            uint32_t row = 0, scale_row = 0, coming = 0; // of the tile that is loaded next: offsets, and which tokens there are
            auto locate = [&](const Place& at) {
                const bool ok = (uint32_t)at.page < (uint32_t)p.num_pages;
                coming = __ballot_sync(0xffffffffu, ok) & 0xffffu;
                row = ok ? at.page * p.page_units + at.in_page * p.token_units : 0u;
                if constexpr (S::KIND != CACHE_F16) scale_row = ok ? at.page * p.scale_page_units + at.in_page * p.scale_token_units : 0u;
            };
            uint32_t kw[2][S::KN][S::KP / 4] = {}, vw[4][S::VN][S::VP / 4] = {};
            uint32_t ks[2][S::KN] = {}, vs[4][S::VN] = {}; // CACHE_I8_GROUPS
            uint32_t scale_bits = 0;                       // CACHE_I8_ROWS: key scale of a token in lanes 0 to 15, value scale in the others
            auto load_keys = [&](bool all) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int token = g + 8 * r;
                    const char* src = kbase + (uint64_t)__shfl_sync(0xffffffffu, row, token) * p.unit + t * S::KP;
                    const char* scales = ksbase;
                    if constexpr (S::KIND == CACHE_I8_GROUPS) scales += (uint64_t)__shfl_sync(0xffffffffu, scale_row, token) * p.scale_unit + t * S::KG * 2;
                    const bool there = all || (coming >> token & 1);
#pragma unroll
                    for (int i = 0; i < S::KN; ++i) {
                        if (there) {
                            load_piece<S::KP>(kw[r][i], src + i * 4 * S::KP);
                            if constexpr (S::KIND == CACHE_I8_GROUPS) ks[r][i] = load_scales<S::KG>(scales + i * 4 * S::KG * 2);
                        } else { // zeros: what lies there may be anything
#pragma unroll
                            for (int x = 0; x < S::KP / 4; ++x) kw[r][i][x] = 0;
                            ks[r][i] = 0;
                        }
                    }
                }
            };
            auto load_values = [&](bool all) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int token = 2 * t + (j & 1) + 8 * (j >> 1);
                    const char* src = vbase + (uint64_t)__shfl_sync(0xffffffffu, row, token) * p.unit + g * S::VP;
                    const char* scales = vsbase;
                    if constexpr (S::KIND == CACHE_I8_GROUPS) scales += (uint64_t)__shfl_sync(0xffffffffu, scale_row, token) * p.scale_unit;
                    const bool there = all || (coming >> token & 1);
#pragma unroll
                    for (int i = 0; i < S::VN; ++i) {
                        constexpr int EP = S::VP / S::ES;
                        if (there) {
                            load_piece<S::VP>(vw[j][i], src + i * 8 * S::VP);
                            if constexpr (S::KIND == CACHE_I8_GROUPS) vs[j][i] = load_scales<S::VG>(scales + (i * 8 + g) * EP / 8 * 2);
                        } else {
#pragma unroll
                            for (int x = 0; x < S::VP / 4; ++x) vw[j][i][x] = 0;
                            vs[j][i] = 0;
                        }
                    }
                }
                if constexpr (S::KIND == CACHE_I8_ROWS)
                    scale_bits = (coming >> (lane & 15) & 1) ? load_scales<1>((lane < 16 ? ksbase : vsbase) + (uint64_t)scale_row * p.scale_unit) : 0u;
            };

            Place ahead = find(tile0);
            {
                const Place second = find(tile0 + 1);
                locate(ahead);
                ahead = second;
            }
            uint32_t seen = coming;
            if (seen == 0xffffu) load_keys(true), load_values(true);
            else if (seen) load_keys(false), load_values(false);
            locate(ahead);
            ahead = find(tile0 + 2);

            for (int32_t tile = tile0; tile < tile1; ++tile) {
                float c[S::NT][4] = {};
                if (seen != 0) {
                    // ---- scores [16 tokens x 8 heads], in two chains -----------------------------------------------------------
                    float c2[S::NT][4] = {};
                    constexpr int KW = S::KP / 4;
#pragma unroll
                    for (int i = 0; i < S::KN; ++i) {
                        if constexpr (S::ES == 2) {
#pragma unroll
                            for (int s = 0; s < KW / 2; ++s)
#pragma unroll
                                for (int nt = 0; nt < S::NT; ++nt) {
                                    const auto& qs = q[nt][i * (KW / 2) + s];
                                    mma(s & 1 ? c2[nt] : c[nt], kw[0][i][2 * s], kw[1][i][2 * s], kw[0][i][2 * s + 1], kw[1][i][2 * s + 1], qs[0], qs[1]);
                                }
                        } else {
#pragma unroll
                            for (int s = 0; s < KW; ++s) {
                                uint32_t a0, a1, a2, a3;
                                widen(kw[0][i][s], a0, a2);
                                widen(kw[1][i][s], a1, a3);
                                if constexpr (S::KIND == CACHE_I8_GROUPS) {
                                    // value x scale has up to 18 bits: its rounding to fp16, and what that left, as a second operand
                                    const __half2 f0 = as_h2(__byte_perm(ks[0][i], 0, s < 2 ? 0x1010 : 0x3232)), f1 = as_h2(__byte_perm(ks[1][i], 0, s < 2 ? 0x1010 : 0x3232));
                                    const __half2 h0 = __hmul2(as_h2(a0), f0), h1 = __hmul2(as_h2(a1), f1), h2_ = __hmul2(as_h2(a2), f0), h3 = __hmul2(as_h2(a3), f1);
                                    const uint32_t r0 = h2(__hfma2(as_h2(a0), f0, __hneg2(h0))), r1 = h2(__hfma2(as_h2(a1), f1, __hneg2(h1)));
                                    const uint32_t r2 = h2(__hfma2(as_h2(a2), f0, __hneg2(h2_))), r3 = h2(__hfma2(as_h2(a3), f1, __hneg2(h3)));
#pragma unroll
                                    for (int nt = 0; nt < S::NT; ++nt) {
                                        const auto& qs = q[nt][i * KW + s];
                                        mma(c[nt], h2(h0), h2(h1), h2(h2_), h2(h3), qs[0], qs[1]);
                                        mma(c2[nt], r0, r1, r2, r3, qs[0], qs[1]);
                                    }
                                } else {
#pragma unroll
                                    for (int nt = 0; nt < S::NT; ++nt) mma(s & 1 ? c2[nt] : c[nt], a0, a1, a2, a3, q[nt][i * KW + s][0], q[nt][i * KW + s][1]);
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
                        for (int x = 0; x < 4; ++x) c[nt][x] += c2[nt][x];
                }
                if (coming == 0xffffu) load_keys(true);
                else if (coming) load_keys(false);

                if (seen != 0) {
                    // ---- weights: 2^(score - top + 8) ----------------------------------------------------------------------
                    float f0 = p.scale_log2, f1 = p.scale_log2, v0 = 1.0f, v1 = 1.0f, e0 = 0.0f, e1 = 0.0f;
                    if constexpr (S::KIND == CACHE_I8_ROWS) {
                        const float mine = __half2float(__ushort_as_half((unsigned short)scale_bits));
                        f0 *= __shfl_sync(0xffffffffu, mine, g);
                        f1 *= __shfl_sync(0xffffffffu, mine, g + 8);
                        v0 = __shfl_sync(0xffffffffu, mine, g + 16);
                        v1 = __shfl_sync(0xffffffffu, mine, g + 24);
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
                        if constexpr (S::ES == 2) {
#pragma unroll
                            for (int x = 0; x < VW; ++x) {
                                const uint32_t a0 = __byte_perm(vw[0][i][x], vw[1][i][x], 0x5410), a1 = __byte_perm(vw[0][i][x], vw[1][i][x], 0x7632);
                                const uint32_t a2 = __byte_perm(vw[2][i][x], vw[3][i][x], 0x5410), a3 = __byte_perm(vw[2][i][x], vw[3][i][x], 0x7632);
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
                                widen_pairs(vw[0][i][x], vw[1][i][x], u);
                                widen_pairs(vw[2][i][x], vw[3][i][x], v);
                                if constexpr (S::KIND == CACHE_I8_GROUPS) {
                                    // these four dimensions are of one group; value x scale is rounded to fp16, as it is when it is read back
                                    const __half2 fu = as_h2(__byte_perm(vs[0][i], vs[1][i], x < 2 ? 0x5410 : 0x7632));
                                    const __half2 fv = as_h2(__byte_perm(vs[2][i], vs[3][i], x < 2 ? 0x5410 : 0x7632));
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
                if (coming == 0xffffu) load_values(true);
                else if (coming) load_values(false);
                seen = coming;
                locate(ahead);
                ahead = find(tile + 3);
            }

            // ---- the four warps' sums --------------------------------------------------------------------------------------
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

// Joins the pieces of the item that CTA blockIdx.x began and others went on with: four warps for each of two query heads, every fourth
// piece to a warp, in an order that does not change.
constexpr int JTPB = 256, JWARPS = 4;
template <int D, int HEADS>
__global__ void __launch_bounds__(JTPB) paged_attention_join_kernel(const __grid_constant__ AttentionParams p, int32_t ctas) {
    constexpr int V = D / 32;
    __shared__ int32_t slots[kMostCtas];
    __shared__ float weights[2][kMostCtas], part[2][JWARPS][D], total[2];
    __shared__ int32_t count;
    pdl_wait_prior_grid();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, side = warp / JWARPS, w = warp - side * JWARPS;
    const int32_t item = p.items[2 * blockIdx.x];
    if (item < 0) return;
    const int heads_per_sequence = p.cache.kv_heads * p.tiles;
    const int64_t b = item / heads_per_sequence;
    const int hh = (int)(item - b * heads_per_sequence), kvh = hh / p.tiles, q_first = (hh - kvh * p.tiles) * HEADS;
    const int heads = min(HEADS, p.shared - q_first), h = blockIdx.y * 2 + side;
    if ((int)blockIdx.y * 2 >= heads) return;

    // the pieces: this CTA's own, then those with which the next CTAs' shares begin, up to the one that ends the item
    if (warp == 0) {
        int32_t found = 1;
        if (lane == 0) slots[0] = 2 * blockIdx.x + 1;
        for (int32_t c0 = blockIdx.x + 1; c0 < ctas; c0 += 32) {
            const int32_t c = c0 + lane, kind = c < ctas ? p.items[2 * c + 1] : TAIL_NONE;
            const uint32_t end = __ballot_sync(0xffffffffu, kind == TAIL_END);
            const uint32_t upto = end ? (end & (0u - end)) * 2u - 1u : 0xffffffffu;
            const uint32_t has = __ballot_sync(0xffffffffu, kind != TAIL_NONE) & upto;
            if (has >> lane & 1) slots[found + __popc(has & ((1u << lane) - 1))] = 2 * c;
            found += __popc(has);
            if (end) break;
        }
        if (lane == 0) count = found;
    }
    __syncthreads();
    const int32_t pieces = count;
    // their factors, by the first warp of each head
    float m = -1e30f;
    if (w == 0 && h < heads) {
        for (int i = lane; i < pieces; i += 32) m = fmaxf(m, p.tops[(int64_t)slots[i] * HEADS + h].x);
#pragma unroll
        for (int x = 16; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
        float l = 0.0f;
        for (int i = lane; i < pieces; i += 32) {
            const float2 s = p.tops[(int64_t)slots[i] * HEADS + h];
            const float f = exp2_fast(s.x - m);
            weights[side][i] = f;
            l += f * s.y;
        }
#pragma unroll
        for (int x = 16; x >= 1; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
        if (lane == 0) total[side] = l;
    }
    __syncthreads();
    float o[V] = {};
    if (h < heads) {
        for (int i0 = w; i0 < pieces; i0 += 4 * JWARPS) {
            float v[4][V];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int x = 0; x < V; ++x) v[u][x] = i0 + u * JWARPS < pieces ? p.sums[((int64_t)slots[i0 + u * JWARPS] * HEADS + h) * D + x * 32 + lane] : 0.0f;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int x = 0; x < V; ++x)
                    if (i0 + u * JWARPS < pieces) o[x] += weights[side][i0 + u * JWARPS] * v[u][x];
        }
    }
#pragma unroll
    for (int x = 0; x < V; ++x) part[side][w][x * 32 + lane] = o[x];
    __syncthreads();
    if (h >= heads) return;
    const int head = kvh * p.shared + q_first + h;
    const float l = total[side], inv = l == 0.0f ? 0.0f : 1.0f / l;
    for (int d = w * 32 + lane; d < D; d += JWARPS * 32) {
        float v = 0.0f;
#pragma unroll
        for (int x = 0; x < JWARPS; ++x) v += part[side][x][d];
        p.out[b * p.out_stride + (int64_t)head * D + d] = __float2half_rn(v * inv);
    }
    if (p.lse && w == 0 && lane == 0) p.lse[b * p.q_heads + head] = l == 0.0f ? -INFINITY : (m - 8.0f + log2f(l)) * 0.69314718055994531f;
}

// Strides in bytes -> in units of the largest power of two that divides them; false where an offset would not fit 32 bits.
bool row_units(int64_t pages, int64_t page_size, int64_t page_bytes, int64_t token_bytes, uint32_t& unit, uint32_t& page_units, uint32_t& token_units) {
    const int64_t strides = (pages > 1 ? page_bytes : 0) | (page_size > 1 ? token_bytes : 0);
    const int shift = strides ? std::min(__builtin_ctzll((uint64_t)strides), 30) : 0;
    const __int128 last = pages > 0 ? (__int128)(pages - 1) * page_bytes + (__int128)(page_size - 1) * token_bytes : 0;
    unit = 1u << shift;
    page_units = (uint32_t)(pages > 1 ? page_bytes >> shift : 0);
    token_units = (uint32_t)(page_size > 1 ? token_bytes >> shift : 0);
    return (last >> shift) < ((__int128)1 << 32);
}

// token / d = token * magic >> shift for all tokens below 2^31: with 2^(s - 1) < d <= 2^s and magic = ceil(2^(31 + s) / d), magic * d
// exceeds 2^(31 + s) by less than d <= 2^s, which token < 2^31 keeps below 1 / d of the quotient.
void page_division(uint32_t d, uint32_t& magic, uint32_t& shift) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    shift = 31 + s;
    magic = (uint32_t)(((1ull << shift) + d - 1) / d);
}

// Query heads that a CTA takes at once: two blocks of eight where that many share a key-value head and registers allow.
int heads_at_once(int32_t head_dim, int32_t shared) { return shared > 8 && head_dim <= 128 ? 16 : 8; }
template <class S>
int32_t launch(cudaStream_t stream, AttentionParams& p, int64_t tokens) {
    static_assert(S::CTAS * kSms <= kMostCtas, "workspace");
    const int64_t tiles = (tokens + CT - 1) / CT;
    const int64_t items = p.batch * p.cache.kv_heads * p.tiles;
    const int64_t most = S::CTAS * kSms;
    const int64_t ctas = tiles > most || items > most ? most : std::min(most, items * std::max<int64_t>(1, tiles));
    launch_ex(paged_attention_kernel<S>, dim3((unsigned)ctas), dim3(ATPB), stream, true, p);
    int32_t rc = check_launch("paged attention");
    if (rc != RC_SUCCESS) return rc;
    // no cut falls inside an item of one tile, nor, where cuts are moved by four tiles (see `quantum`), of six
    if (tiles <= 1 || (tiles <= 6 && items * tiles < 16 * ctas)) return RC_SUCCESS;
    launch_ex(paged_attention_join_kernel<S::D, S::HEADS>, dim3((unsigned)ctas, S::HEADS / 2), dim3(JTPB), stream, true, p, (int32_t)ctas);
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
    if (cache->quant_group == 8 && ((((uintptr_t)cache->k_scale | (uintptr_t)cache->v_scale) & 3) ||
                                    ((cache->scale_page_stride | cache->scale_head_stride | cache->scale_token_stride) & 1)))
        return fail(RC_INVALID_VALUE, "attention: scales of groups of 8 must be 4-byte aligned, and their strides even");
    if (!row_units(cache->num_pages, cache->page_size, cache->page_stride * (cache->quant_group ? 1 : 2), cache->token_stride * (cache->quant_group ? 1 : 2),
                   p.unit, p.page_units, p.token_units) ||
        (cache->quant_group && !row_units(cache->num_pages, cache->page_size, cache->scale_page_stride * 2, cache->scale_token_stride * 2, p.scale_unit,
                                          p.scale_page_units, p.scale_token_units)))
        return fail(RC_UNSUPPORTED, "attention: the rows of a head lie further apart than 2^32 times their alignment");
    page_division(cache->page_size, p.page_magic, p.page_shift);
    p.num_pages = (int32_t)std::min<int64_t>(cache->num_pages, 0x7fffffff); // a table's entry is no larger
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
