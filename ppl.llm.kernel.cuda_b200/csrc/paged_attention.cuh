// Attention of one new token per sequence over the paged key-value cache, split over the tokens and joined.
//
// out = sum_t w_t v_t / sum_t w_t with w_t = 2^(scale log2(e) q . k_t - top), in one pass: `top` is a reference exponent that moves only when
// a weight would leave fp16's range, and then rescales what was summed.
//
// What bounds it is the cache: every key and value is read once, for a few multiply-adds per element.  So the work is laid out for
// loads: steps of 16 or 32 tokens of one head, numbered over all sequences and heads, are dealt out evenly to as many CTAs as the device
// holds at once, whatever the sequences' lengths; a CTA whose share begins or ends inside a sequence leaves its sums in the workspace
// and the CTA that is last to do so joins them, where they are many in groups and then the groups.  While a warp works on its step the next one
// is on its way into its registers, each part requested as soon as its registers are free: a lane loads exactly the bytes that it will
// use (the dimensions of a product may be taken in any order), so that nothing passes through shared memory.  Tried instead: rings in shared memory
// filled by cp.async, whose 64- and 128-byte row parts end at 4.2 TB/s, and by bulk copies of whole runs of rows (65 us instead of what were then
// 68 with groups of 8, but 149 instead of 121 with int8 rows and 103 instead of 91 in fp16: values are then read with bank conflicts); bringing the step
// after the next into L2 (then 66 -> 69, 116 -> 119, 88 -> 93).
//
// Scores are computed transposed, keys [16 tokens x dimensions] x queries [dimensions x 8 heads]: the eight columns hold the query heads that
// share the key head, and the weights turn into the operand of the second product, values^T x weights^T, by transposing 8 x 8 blocks
// between registers.  mma.sync, because an operand of tcgen05.mma would first have to be widened into shared memory, and the tensor pipe is
// busy for a quarter of the time.
//
// Heads of 128 in one graph, caches larger than L2, against the bytes at a copy's 6.55 TB/s: 64 sequences of up to 8192 tokens, 64 query
// heads over 8, int8 rows 118 us (86 %; 135 over seconds, at the power limit and 1.67 GHz); one of 131072, fp16, 89 us (92 %); 16 of up to 4096, 32
// heads of their own, groups of 8, 67 us (71 %: 575 instructions for 16 tokens, issue slots 55 % busy at 16 warps an SM).  Short
// ones consist of look-ups that wait for each other, lengths, pages, rows, and of the join: one of 333 tokens 9 us.
#pragma once

#include "kv_cache.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>

namespace pplb200 {
namespace paged {

constexpr int kSms = 148, kCtas = 4 * kSms;
enum : int { CACHE_F16 = 0, CACHE_I8_GROUPS = 1, CACHE_I8_ROWS = 2 };

constexpr int piece(int bytes) { return bytes % 16 == 0 ? 16 : bytes % 8 == 0 ? 8 : 4; }

// Sizes of one variant: D dimensions, KIND of cache, NT blocks of eight query heads.  PACKED: a page has a multiple of 16 tokens, whose
// rows follow each other, so that 16 tokens are one address and offsets that the instructions hold.  Other pages (of 8 or 24 tokens) take 4 to 7 %
// longer over int8 caches, tokens ahead of heads or pages of one token 10 to 12 %, over fp16 ones nothing (16 x 2048 groups 64.7, 67, 71 us;
// 32 x 4096 rows 51, 55, 57; 16 x 4096 fp16 46).
//
// GENERAL: what attention over a shared prefix and over chosen blocks ask for besides.  The page table may differ from key head to key
// head, and its entries be blocks, several to a page; the query rows of an item may be those of several sequences; the sums may be left for a
// later call in place of the output, or be joined with those that an earlier call has left.  Threads and CTAs an SM are those of the plain forms, for which they were measured;
// what there is besides takes registers that these do not leave, so that 27 of the 42 forms spill 4 to 260 bytes (of the plain ones 14, up to 72): groups of 8, heads of 128, eight query heads,
// 80, int8 rows of 64 and 96, sixteen, 244 and 260.
template <int D_, int KIND_, int NT_, bool PACKED_, bool GENERAL_ = false>
struct Shape {
    static constexpr int D = D_, KIND = KIND_, NT = NT_, HEADS = 8 * NT;
    static constexpr bool PACKED = PACKED_, GENERAL = GENERAL_;
    static constexpr int ES = KIND == CACHE_F16 ? 2 : 1;
    // Tokens of a step: 32 where that leaves a form for eight query heads room for twelve warps on an SM (64 x 8192, int8 rows: 118 us with 32,
    // 129 with 16; groups, whose scales take registers too: 16 x 4096 68.2 us with 32, 66.7 with 16).  Forms for sixteen take as many tokens as
    // those for eight, although int8 rows of 128 then leave room for eight warps only; 16 tokens have not been measured there.
    static constexpr int SUBS = D * ES <= 64 || (D * ES <= 128 && KIND == CACHE_I8_ROWS) ? 2 : 1, TOKENS = 16 * SUBS;
    // of 16 tokens a quad's lane holds a quarter of the dimensions of two keys, an eighth of those of four values
    static constexpr int KB = D * ES / 4, KP = piece(KB), KN = KB / KP;
    static constexpr int VB = D * ES / 8, VP = piece(VB), VN = VB / VP;
    static constexpr int KG = KP >= 8 ? KP / 8 : 1, VG = VP >= 8 ? VP / 8 : 1; // CACHE_I8_GROUPS: scales of a piece
    static constexpr int STEPS = D / 16; // of 16 dimensions in the first product, and blocks of 16 in the second
    // Registers for the sums, the queries and the tokens on their way decide how many CTAs share an SM (groups of 8, 128 dimensions: 66 us
    // with four, 69 with three).
    static constexpr int WORDS = NT * D / 4 + NT * D / 8 + SUBS * (D * ES / 4 + (KIND == CACHE_I8_GROUPS ? 2 * KN + 4 * VN : 0));
    static constexpr int ROW = D + 4; // of the sums that the warps exchange
    static constexpr int WARPS = 4, THREADS = 32 * WARPS, CTAS = WORDS <= 88 ? 4 : WORDS <= 128 ? 3 : 2;
};

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
    uint32_t page_magic, page_shift; // token / page_size = token * page_magic >> page_shift (GENERAL: / unit_tokens)
    pplb200_kv_cache cache;
    uint32_t flip_1024; // what spread() flips: in a register, since an instruction holds one constant
    // workspace
    uint64_t call;     // number of the call, counted by the process
    uint64_t* arrived; // [CTAs]: pieces, or groups of them, of the item that the CTA began; then [2 * CTAs]: pieces of a group
    float2* tops;      // [2 * CTAs][HEADS]: reference exponent and sum of weights
    float* sums;       // [2 * CTAs][HEADS][D]
    // GENERAL
    int64_t pages_head_stride;                 // between the tables of a sequence's key heads
    int32_t unit_tokens, units_per_page;       // an entry of a table is unit_tokens tokens, units_per_page of them a page
    int32_t num_units;                         // of the cache
    uint32_t unit_magic, unit_shift;           // entry / units_per_page
    int32_t rows_per_head;                     // query heads of one sequence that share a key head: row r of an item is of sequence b + r / rows_per_head
    uint32_t rows_magic, rows_shift;
    int32_t parts;                             // sums of earlier calls that are joined
    bool keep_parts;                           // leave the sums, as part 0
    bool late_wait;                            // go ahead of the wait for the grid before, if *ahead says so
    uint32_t* ahead;                           // of the workspace: 1 from when the grid before is behind its own wait until this one is behind it, else 0
    bool whole_items;                          // as many CTAs as items, one each
    int64_t whole_tokens;                      // for items of no more
    int64_t part_rows;                         // rows of a part: query heads of all sequences
    float2* part_tops;                         // [parts][part_rows]
    float* part_sums;                          // [parts][part_rows][D]
};

// Query heads that a CTA takes at once: two blocks of eight where that many share a key-value head and registers allow.  16 sequences of up to
// 4096 tokens, 128 heads over 8: heads of 128 in fp16 50 us (79 if eight at a time), int8 rows 44 (52), groups of 8 52 (64); of 64 in fp16 31 (40), of
// 96 43 (59).
inline int heads_at_once(int32_t head_dim, int64_t shared) { return shared > 8 && head_dim <= 128 ? 16 : 8; }

// A workspace begins with what has to be zero between calls, in one place for all forms of attention and all sizes, so that one workspace serves them in turn: three counters a CTA and (kAhead) the
// word by which a kernel goes ahead of its wait; then counters once more, of the decode kernel where it goes through a shared prefix while another goes through own tokens.
constexpr int64_t kAhead = 3 * kCtas * 8, kCounters = (kAhead + 4 + 255) / 256 * 256, kZeros = 2 * kCounters;
// Bytes of the attention kernel's workspace: behind the zeros, two pieces a CTA at most.
inline int64_t workspace_bytes(int64_t shared, int32_t head_dim) {
    const int heads = heads_at_once(head_dim, shared);
    return kZeros + round_up(2 * kCtas * heads * 8, 256) + 2LL * kCtas * heads * head_dim * 4;
}

// What is wrong with a call's cache and block (the workspace aside), or RC_SUCCESS with the parameters that all forms have in common.
int32_t take_call(const pplb200_kv_cache* cache, const pplb200_paged_attention_args* a, AttentionParams& p);
// The workspace's parts, for `shared` query rows a key head.
void lay_out(AttentionParams& p, void* ws, int64_t shared);

// GENERAL: p with its tables of units and its rows set.
int32_t launch_general(cudaStream_t stream, AttentionParams& p);
// How many SMs all its CTAs fill.
int32_t sms_of_general(AttentionParams& p);

} // namespace paged

namespace {

using namespace paged;

// Going ahead of a wait.  What a grid may read behind its wait for the grid before it (lengths, pages, q, the cache) is not promised to be visible to the one after it, which has not
// waited yet, although that one starts only when all CTAs of the grid between are behind their waits.  So that grid says that it is, with a release, and the one after it looks,
// with an acquire: what it then finds ordered before that, all that the grid between had waited for, is visible to it too.  Where it does not find the word set, it waits as any other.
__device__ __forceinline__ void let_go_ahead(uint32_t* word) { asm volatile("st.release.gpu.global.u32 [%0], 1;" ::"l"(word) : "memory"); }
__device__ __forceinline__ bool may_go_ahead(const uint32_t* word) {
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(word) : "memory");
    return v == 1;
}

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
__device__ __forceinline__ float log2_fast(float x) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t h2(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// Bytes 0, 2 or (of w >> 8) bytes 1, 3 of a word as two halves' bits: u = value + 128, a byte with its sign bit flipped, beneath the
// exponent that `flip` brings: with 0x64 above it, 1024 + u.
__device__ __forceinline__ uint32_t spread(uint32_t w, uint32_t flip) {
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x00ff00ff, %2, 0x6a;" : "=r"(r) : "r"(w), "r"(flip)); // (w & 0x00ff00ff) ^ flip
    return r;
}
__device__ __forceinline__ uint32_t less_1152(uint32_t v) { return h2(__hsub2(as_h2(v), as_h2(0x64806480u))); }

// The four bytes of a word as halves, 0, 2 and 1, 3 (a product's dimensions may come in any order): the whole numbers themselves.  Keys of rows
// as u * 2^-24, subnormal numbers that need no subtraction, would leave 128 times the sum of a query's elements to be taken off the score,
// which is hundreds of times the score where a row's scale comes from a dimension that the query does not see, and cost the score as many of
// its 24 bits (64 x 8192 tokens: 109 us so, 111 with whole numbers).
__device__ __forceinline__ void widen(const AttentionParams& p, uint32_t w, uint32_t& even, uint32_t& odd) {
    even = less_1152(spread(w, p.flip_1024));
    odd = less_1152(spread(w >> 8, p.flip_1024));
}
// The four bytes of the words of two tokens as pairs (token a, token b).
__device__ __forceinline__ void widen_pairs(const AttentionParams& p, uint32_t a, uint32_t b, uint32_t (&o)[4]) {
    widen(p, __byte_perm(a, b, 0x5410), o[0], o[1]);
    widen(p, __byte_perm(a, b, 0x7632), o[2], o[3]);
}

// Tokens of a sequence that are looked at: [first, n).  Steps begin at a multiple of 16.
__device__ __forceinline__ void visible(const AttentionParams& p, int64_t b, int32_t& first, int32_t& n) {
    n = (int32_t)min((int64_t)max(p.lengths[b], 0), p.tokens_in_table);
    first = p.window > 0 ? max(0, n - p.window) : 0;
}
// Steps of a sequence and head; an empty sequence has one too, so that its output is written.
template <int TOKENS>
__device__ __forceinline__ int32_t steps_of(const AttentionParams& p, int64_t b) {
    int32_t first, n;
    visible(p, b, first, n);
    return max(1, (n - (first & ~15) + TOKENS - 1) / TOKENS);
}

// What beginning a head of a sequence costs, in steps: a chain of look-ups before the first step, the joining of the warps' sums behind
// the last, while the other CTAs of the SM go on.  Without it the heads of empty and short sequences, which cost time but no steps, pile up on one CTA.
template <class S>
constexpr int32_t kBeginning = 2 * S::WARPS;

struct Share { // where a CTA's share begins or ends: a step of a head of a sequence
    int64_t b;
    int32_t head, step;
};

// The reference exponent of a head before its first token.  Where there was one, it ends above that, even if all scores were minus infinity: their
// quotient is NaN, while nothing at all gives zeros.
constexpr float kNothingSeen = -1e30f, kLowest = -0.5e30f;

// Output of one query head, dimensions d to d + 3, from sums in units of 2^top.
__device__ __forceinline__ void write_out(const AttentionParams& p, int64_t b, int32_t head, int32_t dims, int32_t d, const float4& v, float top, float sum) {
    const float inv = sum != 0.0f ? 1.0f / sum : top > kNothingSeen ? __int_as_float(0x7fffffff) : 0.0f;
    const uint2 r = make_uint2(h2(__floats2half2_rn(v.x * inv, v.y * inv)), h2(__floats2half2_rn(v.z * inv, v.w * inv)));
    *reinterpret_cast<uint2*>(p.out + b * p.out_stride + (int64_t)head * dims + d) = r;
    if (p.lse && d == 0) p.lse[b * p.q_heads + head] = sum == 0.0f ? -INFINITY : (top - 8.0f + log2f(sum)) * 0.69314718055994531f;
}
// Row `row` (GENERAL: of those that the item's key head is asked by) of key head kvh.
template <class S>
__device__ __forceinline__ void finish(const AttentionParams& p, int64_t b, int32_t kvh, int32_t row, int32_t d, float4 v, float top, float sum) {
    static_assert(S::GENERAL);
    const int32_t beyond = (uint32_t)((uint64_t)(uint32_t)row * p.rows_magic >> p.rows_shift);
    const int64_t sequence = b + beyond;
    const int32_t head = kvh * p.rows_per_head + (row - beyond * p.rows_per_head);
    const int64_t at = sequence * p.q_heads + head;
    if (p.keep_parts) {
        __stcg(reinterpret_cast<float4*>(p.part_sums + at * S::D + d), v);
        if (d == 0) __stcg(&p.part_tops[at], make_float2(top, sum));
        return;
    }
    if (p.parts > 0) {
        if (p.lengths[sequence] < 0) { // not a sequence
            v = make_float4(0, 0, 0, 0);
            top = kNothingSeen;
            sum = 0.0f;
        } else {
            // eight parts at once, sixteen loads on their way
            constexpr int BATCH = 8;
            for (int32_t i = 0; i < p.parts; i += BATCH) {
                float2 s[BATCH];
                float4 a[BATCH];
                float up = top;
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    const int64_t from = min(i + j, p.parts - 1) * p.part_rows + at;
                    s[j] = __ldcg(&p.part_tops[from]);
                    a[j] = __ldcg(reinterpret_cast<const float4*>(p.part_sums + from * S::D + d));
                }
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    if (i + j >= p.parts) s[j] = make_float2(kNothingSeen, 0.0f);
                    up = fmaxf(up, s[j].x);
                }
                const float keep = exp2_fast(top - up);
                top = up;
                sum *= keep;
                v.x *= keep; v.y *= keep; v.z *= keep; v.w *= keep;
#pragma unroll
                for (int j = 0; j < BATCH; ++j)
                    if (s[j].x != kNothingSeen) { // else its sums need not have been written
                        const float f = exp2_fast(s[j].x - up);
                        sum += s[j].y * f;
                        v.x += a[j].x * f; v.y += a[j].y * f; v.z += a[j].z * f; v.w += a[j].w * f;
                    }
            }
        }
    }
    write_out(p, sequence, head, S::D, d, v, top, sum);
}

template <class S>
__global__ void __launch_bounds__(S::THREADS, S::CTAS) paged_attention_kernel(const __grid_constant__ AttentionParams p) {
    constexpr int WARPS = S::WARPS, PAD = kBeginning<S>;
    __shared__ __align__(16) float part[WARPS * S::HEADS * S::ROW];
    __shared__ float2 tops[WARPS * S::HEADS];
    __shared__ int64_t scan[WARPS], ends[2][2];
    __shared__ volatile struct { int64_t all, last_item; int32_t ctas, to_step; } share; // kept out of the registers
    __shared__ int32_t longest[WARPS], is_last;
    __shared__ bool begun;
    // the warp's number from a shuffle, so that the compiler knows that it is the same in all lanes
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), g = lane >> 2, t = lane & 3;
    const int heads_per_sequence = p.cache.kv_heads * p.tiles;
    // late_wait: the grid before this one belongs to the same call, and only the sums that it leaves are needed from it: where an item's output is written.
    bool late = false;
    if constexpr (S::GENERAL) {
        if (p.late_wait) {
            if (threadIdx.x == 0) begun = may_go_ahead(p.ahead);
            __syncthreads();
            late = begun;
        }
    }
    if (!late) pdl_wait_prior_grid();
    if constexpr (S::GENERAL) {
        if (p.ahead && !p.late_wait && blockIdx.x == 0 && threadIdx.x == 0) let_go_ahead(p.ahead);
    }
    pdl_launch_dependents();

    // ---- this CTA's share -----------------------------------------------------------------------------------------------
    // Steps are numbered in the order sequence, head, step, PAD numbers ahead of every head's first step standing for what its
    // beginning costs.  CTA c takes the steps from c * all / ctas to (c + 1) * all / ctas; or, where no sequence is so long that splitting
    // it would pay for the joining, item c and no other.
    Share from, to;
    int64_t all;
    int32_t ctas;
    if (S::GENERAL && p.whole_items) { // known without the lengths
        all = ctas = gridDim.x;
        from.b = blockIdx.x / heads_per_sequence;
        from.head = blockIdx.x - (int32_t)from.b * heads_per_sequence;
        to.b = (blockIdx.x + 1) / heads_per_sequence;
        to.head = blockIdx.x + 1 - (int32_t)to.b * heads_per_sequence;
        from.step = to.step = 0;
    } else {
        const int64_t per_thread = (p.batch + S::THREADS - 1) / S::THREADS, b0 = min(p.batch, threadIdx.x * per_thread), b1 = min(p.batch, b0 + per_thread);
        int64_t mine = 0;
        int32_t most = 0;
        for (int64_t b = b0; b < b1; ++b) {
            const int32_t n = steps_of<S::TOKENS>(p, b) + PAD;
            mine += n;
            most = max(most, n);
        }
        int64_t before = mine;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, before, m);
            if (lane >= m) before += v;
        }
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 31) scan[warp] = before, longest[warp] = most;
        __syncthreads();
        int64_t total = 0;
        before -= mine;
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) before += scan[w];
            total += scan[w];
            most = max(most, longest[w]);
        }
        all = total * heads_per_sequence;
        const int64_t items = p.batch * heads_per_sequence;
        ctas = (int32_t)min((int64_t)gridDim.x, max((int64_t)1, all / WARPS)); // a step a warp at least
        // Joining takes about as long as three rounds of steps.
        const bool whole_items = items <= gridDim.x && most <= all / ctas + 3 * WARPS;
        if (whole_items) ctas = (int32_t)items;
        if (blockIdx.x >= ctas) {
            if (late) pdl_wait_prior_grid();
            return; // (not CTA 0)
        }
        if (whole_items) {
            from.b = blockIdx.x / heads_per_sequence;
            from.head = blockIdx.x - (int32_t)from.b * heads_per_sequence;
            to.b = (blockIdx.x + 1) / heads_per_sequence;
            to.head = blockIdx.x + 1 - (int32_t)to.b * heads_per_sequence;
            from.step = to.step = 0;
        } else {
            // a cut at step x lies in sequence b where the steps of one head up to b are at most x / heads
            int64_t cut[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                cut[e] = (int64_t)(blockIdx.x + e) * all / ctas;
                const int64_t y = cut[e] / heads_per_sequence;
                if (y >= before && y < before + mine) {
                    int64_t b = b0, at = before;
                    for (;; ++b) {
                        const int32_t n = steps_of<S::TOKENS>(p, b) + PAD;
                        if (y < at + n) break;
                        at += n;
                    }
                    ends[e][0] = b;
                    ends[e][1] = at;
                }
                if (threadIdx.x == 0 && cut[e] == all) ends[e][0] = p.batch, ends[e][1] = total;
            }
            __syncthreads();
            auto place = [&](int e, Share& s) {
                s.b = ends[e][0];
                s.head = s.step = 0;
                if (s.b < p.batch) {
                    const int32_t n = steps_of<S::TOKENS>(p, s.b) + PAD;
                    const int64_t in = cut[e] - ends[e][1] * heads_per_sequence;
                    s.head = (int32_t)(in / n);
                    s.step = max(0, (int32_t)(in - (int64_t)s.head * n) - PAD);
                }
            };
            place(0, from);
            place(1, to);
        }
    }
    if (threadIdx.x == 0) {
        share.all = all;
        share.ctas = ctas;
        share.last_item = to.b * heads_per_sequence + to.head; // nothing of it if to_step == 0
        share.to_step = to.step;
    }
    __syncthreads();
    int64_t b = from.b;
    int32_t hh = from.head, step0 = from.step;

    for (; b < p.batch; step0 = 0) {
        const int64_t item = b * heads_per_sequence + hh;
        if (item > share.last_item || (item == share.last_item && share.to_step <= step0)) break;
        int32_t first, n;
        visible(p, b, first, n);
        const int32_t start = first & ~15, steps = max(1, (n - start + S::TOKENS - 1) / S::TOKENS);
        const int32_t step1 = item == share.last_item ? share.to_step : steps;
        const int kvh = hh / p.tiles, q_first = (hh - kvh * p.tiles) * S::HEADS;
        const int q_count = min(S::HEADS, p.shared - q_first);
        const char* const kbase = (const char*)p.cache.k + (int64_t)kvh * p.cache.head_stride * S::ES + t * S::KP + (S::PACKED ? g * (S::D * S::ES) : 0);
        const char* const vbase = (const char*)p.cache.v + (int64_t)kvh * p.cache.head_stride * S::ES + g * S::VP + (S::PACKED ? 2 * t * (S::D * S::ES) : 0);
        // scales: of the lane's groups, or of the lane's token
        const int64_t scale_bytes = S::KIND == CACHE_I8_ROWS && S::PACKED ? (lane & 15) * p.cache.scale_token_stride * 2 : 0;
        const char* const ksbase = (const char*)p.cache.k_scale + (int64_t)kvh * p.cache.scale_head_stride * 2 + scale_bytes +
                                   (S::KIND == CACHE_I8_GROUPS ? t * S::KG * 2 + (S::PACKED ? g * (S::D / 4) : 0) : 0);
        const char* const vsbase = (const char*)p.cache.v_scale + (int64_t)kvh * p.cache.scale_head_stride * 2 + scale_bytes +
                                   (S::KIND == CACHE_I8_GROUPS ? g * (S::VP / S::ES) / 8 * 2 + (S::PACKED ? 2 * t * (S::D / 4) : 0) : 0);
        const int32_t* const row_pages = p.pages + b * p.pages_stride + (S::GENERAL ? kvh * p.pages_head_stride : 0);

        // ---- tokens on their way -----------------------------------------------------------------------------------------
        // Of the step that is loaded next: which tokens there are, and where their rows lie.  Lane l looks after token l of a step (of l %
        // 16): its page, two steps ahead, then its row, one step ahead; PACKED: all lanes look after the first of every 16.
        constexpr uint32_t EVERY = S::SUBS == 2 ? 0xffffffffu : 0xffffu;
        constexpr int PLACES = S::PACKED ? S::SUBS : 1;
        struct Place {
            int32_t page[PLACES];
            uint32_t in_page[PLACES];
        };
        uint32_t row[PLACES] = {}, scale_row[PLACES] = {}, coming = 0;
        uint64_t off[PLACES], scale_off[PLACES]; // PACKED: of every 16 tokens, in bytes
        auto find = [&](int32_t step) {
            Place at;
#pragma unroll
            for (int i = 0; i < PLACES; ++i) {
                const int32_t token = start + step * S::TOKENS + (S::PACKED ? 16 * i : lane & (S::TOKENS - 1));
                const uint32_t index = (uint32_t)((uint64_t)(uint32_t)token * p.page_magic >> p.page_shift);
                at.page[i] = step < step1 && token < n && (S::PACKED || token >= first) ? row_pages[index] : -1;
                at.in_page[i] = token - index * (S::GENERAL ? p.unit_tokens : p.cache.page_size);
            }
            return at;
        };
        auto locate = [&](const Place& at, int32_t step) {
            if constexpr (S::PACKED) coming = 0;
#pragma unroll
            for (int i = 0; i < PLACES; ++i) {
                const bool ok = (uint32_t)at.page[i] < (uint32_t)(S::GENERAL ? p.num_units : p.num_pages);
                if constexpr (S::GENERAL) { // (a number of 31 bits, or not taken)
                    const uint32_t unit = at.page[i], page = (uint32_t)((uint64_t)unit * p.unit_magic >> p.unit_shift);
                    const uint32_t in_page = at.in_page[i] + (unit - page * p.units_per_page) * p.unit_tokens;
                    row[i] = ok ? page * p.page_units + in_page * p.token_units : 0u;
                    if constexpr (S::KIND != CACHE_F16) scale_row[i] = ok ? page * p.scale_page_units + in_page * p.scale_token_units : 0u;
                } else {
                    row[i] = ok ? at.page[i] * p.page_units + at.in_page[i] * p.token_units : 0u;
                    if constexpr (S::KIND != CACHE_F16) scale_row[i] = ok ? at.page[i] * p.scale_page_units + at.in_page[i] * p.scale_token_units : 0u;
                }
                if constexpr (S::PACKED) {
                    off[i] = (uint64_t)row[i] * p.unit;
                    scale_off[i] = (uint64_t)scale_row[i] * p.scale_unit;
                    const int32_t token = start + step * S::TOKENS + 16 * i; // bits of tokens from `first` and below n
                    if (ok) coming |= ((0xffffu >> max(0, 16 - (n - token))) & (0xffffu << max(0, first - token)) & 0xffffu) << (16 * i);
                } else {
                    coming = __ballot_sync(0xffffffffu, ok) & EVERY;
                }
            }
        };
        auto offset_of = [&](int token) { return (uint64_t)__shfl_sync(0xffffffffu, row[0], token) * p.unit; };
        auto scale_offset_of = [&](int token) { return (uint64_t)__shfl_sync(0xffffffffu, scale_row[0], token) * p.scale_unit; };
        uint32_t kw[S::SUBS][2][S::KN][S::KP / 4] = {}, vw[S::SUBS][4][S::VN][S::VP / 4] = {};
        uint32_t ks[S::SUBS][2][S::KN] = {}, vs[S::SUBS][4][S::VN] = {}; // CACHE_I8_GROUPS
        uint32_t k_scale = 0, v_scale = 0;                               // CACHE_I8_ROWS: of the lane's token
        auto load_keys = [&](int sub) {
            auto load = [&](bool every) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int token = 16 * sub + g + 8 * r;
                    const char *src, *scales = nullptr;
                    if constexpr (S::PACKED) {
                        src = kbase + off[sub] + 8 * r * (S::D * S::ES);
                        scales = ksbase + scale_off[sub] + 8 * r * (S::D / 4);
                    } else {
                        src = kbase + offset_of(token);
                        if constexpr (S::KIND == CACHE_I8_GROUPS) scales = ksbase + scale_offset_of(token);
                    }
                    const bool there = every || (coming >> token & 1);
#pragma unroll
                    for (int i = 0; i < S::KN; ++i) {
                        if (there) {
                            load_piece<S::KP>(kw[sub][r][i], src + i * 4 * S::KP);
                            if constexpr (S::KIND == CACHE_I8_GROUPS) ks[sub][r][i] = load_scales<S::KG>(scales + i * 4 * S::KG * 2);
                        } else { // zeros: what lies there may be anything
#pragma unroll
                            for (int x = 0; x < S::KP / 4; ++x) kw[sub][r][i][x] = 0;
                            ks[sub][r][i] = 0;
                        }
                    }
                }
            };
            if (coming == EVERY) load(true);
            else if (coming) load(false);
        };
        auto load_values = [&](int sub) {
            auto load = [&](bool every) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int token = 16 * sub + 2 * t + (j & 1) + 8 * (j >> 1);
                    const int in_lane = (j & 1) + 8 * (j >> 1); // tokens behind the lane's first
                    const char *src, *scales = nullptr;
                    if constexpr (S::PACKED) {
                        src = vbase + off[sub] + in_lane * (S::D * S::ES);
                        scales = vsbase + scale_off[sub] + in_lane * (S::D / 4);
                    } else {
                        src = vbase + offset_of(token);
                        if constexpr (S::KIND == CACHE_I8_GROUPS) scales = vsbase + scale_offset_of(token);
                    }
                    const bool there = every || (coming >> token & 1);
#pragma unroll
                    for (int i = 0; i < S::VN; ++i) {
                        constexpr int EP = S::VP / S::ES;
                        if (there) {
                            load_piece<S::VP>(vw[sub][j][i], src + i * 8 * S::VP);
                            if constexpr (S::KIND == CACHE_I8_GROUPS) vs[sub][j][i] = load_scales<S::VG>(scales + i * 8 * EP / 8 * 2);
                        } else {
#pragma unroll
                            for (int x = 0; x < S::VP / 4; ++x) vw[sub][j][i][x] = 0;
                            vs[sub][j][i] = 0;
                        }
                    }
                }
            };
            if (coming == EVERY) load(true);
            else if (coming) load(false);
        };
        // CACHE_I8_ROWS: the scales of the lane's token
        auto load_scale = [&](uint32_t& scale, bool values) {
            if constexpr (S::KIND == CACHE_I8_ROWS) {
                const char* at = values ? vsbase : ksbase;
                if constexpr (S::PACKED) at += lane >= 16 ? scale_off[PLACES - 1] : scale_off[0];
                else at += (uint64_t)scale_row[0] * p.scale_unit;
                scale = (coming >> (lane & (S::TOKENS - 1)) & 1) ? load_scales<1>(at) : 0u;
            }
        };

        Place ahead = find(step0 + warp);
        const Place second = find(step0 + warp + WARPS);
        // the queries, while the pages are looked up: column g of block nt, the dimensions of quad lane t
        uint32_t q[S::NT][S::STEPS][2];
#pragma unroll
        for (int nt = 0; nt < S::NT; ++nt) {
            const int h = nt * 8 + g;
            const half* src;
            if constexpr (S::GENERAL) {
                const uint32_t r = q_first + h, beyond = (uint32_t)((uint64_t)r * p.rows_magic >> p.rows_shift);
                src = p.q + (b + beyond) * p.q_stride + (int64_t)(kvh * p.rows_per_head + (int32_t)(r - beyond * p.rows_per_head)) * S::D;
            } else {
                src = p.q + b * p.q_stride + (int64_t)(kvh * p.shared + q_first + h) * S::D;
            }
            constexpr int EP = S::KP / S::ES; // dimensions of a piece
#pragma unroll
            for (int i = 0; i < S::KN; ++i)
#pragma unroll
                for (int s = 0; s < EP / 4; ++s) {
                    uint2 w = make_uint2(0, 0);
                    if (h < q_count) w = *reinterpret_cast<const uint2*>(src + (i * 4 + t) * EP + s * 4);
                    const bool apart = S::ES == 1; // dimensions 0, 2 and 1, 3, as they come out of a word of bytes
                    q[nt][i * (EP / 4) + s][0] = apart ? __byte_perm(w.x, w.y, 0x5410) : w.x;
                    q[nt][i * (EP / 4) + s][1] = apart ? __byte_perm(w.x, w.y, 0x7632) : w.y;
                }
        }
        locate(ahead, step0 + warp);
        ahead = second;
        uint32_t seen = coming;
#pragma unroll
        for (int sub = 0; sub < S::SUBS; ++sub) load_keys(sub);
        load_scale(k_scale, false);
#pragma unroll
        for (int sub = 0; sub < S::SUBS; ++sub) load_values(sub);
        load_scale(v_scale, true);
        locate(ahead, step0 + warp + WARPS);
        ahead = find(step0 + warp + 2 * WARPS);

        float o[S::NT][S::STEPS][4] = {}, top[S::NT][2], sum[S::NT][2] = {};
#pragma unroll
        for (int nt = 0; nt < S::NT; ++nt) top[nt][0] = top[nt][1] = kNothingSeen;

        for (int32_t step = step0 + warp; step < step1; step += WARPS) {
            float c[S::SUBS][S::NT][4];
            // Each part of the next step is requested as soon as its registers are free.
            const uint32_t k_scale_now = k_scale;
            if (seen != 0) {
                // ---- scores [16 tokens x 8 heads] ------------------------------------------------------------------------
                constexpr int KW = S::KP / 4;
#pragma unroll
                for (int sub = 0; sub < S::SUBS; ++sub) {
                    {
                        float c2[S::NT][4] = {}; // a second chain
#pragma unroll
                        for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
                            for (int x = 0; x < 4; ++x) c[sub][nt][x] = 0.0f;
#pragma unroll
                        for (int i = 0; i < S::KN; ++i) {
                            if constexpr (S::KIND == CACHE_F16) {
#pragma unroll
                                for (int s = 0; s < KW / 2; ++s)
#pragma unroll
                                    for (int nt = 0; nt < S::NT; ++nt) {
                                        const auto& qs = q[nt][i * (KW / 2) + s];
                                        mma(s & 1 ? c2[nt] : c[sub][nt], kw[sub][0][i][2 * s], kw[sub][1][i][2 * s], kw[sub][0][i][2 * s + 1], kw[sub][1][i][2 * s + 1], qs[0], qs[1]);
                                    }
                            } else if constexpr (S::KIND == CACHE_I8_ROWS) {
#pragma unroll
                                for (int s = 0; s < KW; ++s) {
                                    uint32_t a0, a1, a2, a3;
                                    widen(p, kw[sub][0][i][s], a0, a2);
                                    widen(p, kw[sub][1][i][s], a1, a3);
#pragma unroll
                                    for (int nt = 0; nt < S::NT; ++nt) mma(s & 1 ? c2[nt] : c[sub][nt], a0, a1, a2, a3, q[nt][i * KW + s][0], q[nt][i * KW + s][1]);
                                }
                            } else {
#pragma unroll
                                for (int s = 0; s < KW; ++s) {
                                    uint32_t a0, a1, a2, a3;
                                    widen(p, kw[sub][0][i][s], a0, a2);
                                    widen(p, kw[sub][1][i][s], a1, a3);
                                    // value x scale has up to 18 bits: its rounding to fp16, and what that left, as a second operand (beyond fp16's range, inf
                                    // and -inf: NaN, not a wrong score)
                                    const __half2 f0 = as_h2(__byte_perm(ks[sub][0][i], 0, s < 2 ? 0x1010 : 0x3232)), f1 = as_h2(__byte_perm(ks[sub][1][i], 0, s < 2 ? 0x1010 : 0x3232));
                                    const __half2 h0 = __hmul2(as_h2(a0), f0), h1 = __hmul2(as_h2(a1), f1), h2_ = __hmul2(as_h2(a2), f0), h3 = __hmul2(as_h2(a3), f1);
                                    const uint32_t r0 = h2(__hfma2(as_h2(a0), f0, __hneg2(h0))), r1 = h2(__hfma2(as_h2(a1), f1, __hneg2(h1)));
                                    const uint32_t r2 = h2(__hfma2(as_h2(a2), f0, __hneg2(h2_))), r3 = h2(__hfma2(as_h2(a3), f1, __hneg2(h3)));
#pragma unroll
                                    for (int nt = 0; nt < S::NT; ++nt) {
                                        const auto& qs = q[nt][i * KW + s];
                                        mma(c[sub][nt], h2(h0), h2(h1), h2(h2_), h2(h3), qs[0], qs[1]);
                                        mma(c2[nt], r0, r1, r2, r3, qs[0], qs[1]);
                                    }
                                }
                            }
                        }
#pragma unroll
                        for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
                            for (int x = 0; x < 4; ++x) c[sub][nt][x] += c2[nt][x];
                        if constexpr (S::KIND == CACHE_I8_ROWS) {
                            const float mine = __half2float(__ushort_as_half((unsigned short)k_scale_now)) * p.scale_log2;
                            const float k0 = __shfl_sync(0xffffffffu, mine, 16 * sub + g), k1 = __shfl_sync(0xffffffffu, mine, 16 * sub + g + 8);
#pragma unroll
                            for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
                                for (int x = 0; x < 4; ++x) c[sub][nt][x] *= x < 2 ? k0 : k1;
                        } else {
#pragma unroll
                            for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
                                for (int x = 0; x < 4; ++x) c[sub][nt][x] *= p.scale_log2;
                        }
                    }
                    load_keys(sub);
                }
                load_scale(k_scale, false);


                // ---- weights: 2^(score - top + 8) --------------------------------------------------------------------------
                float v0[S::SUBS], v1[S::SUBS], e0[S::SUBS] = {}, e1[S::SUBS] = {};
                if constexpr (S::KIND == CACHE_I8_ROWS) {
                    // a value's scale goes into its weight, the scale's logarithm into what decides about the reference exponent; an infinite one only as
                    // far as a finite one could: the sum of the weights, of which the lse is made, is no affair of the values
                    const float mine = __half2float(__ushort_as_half((unsigned short)v_scale)), size = fminf(fmaxf(log2_fast(fabsf(mine)), -24.0f), 16.0f);
#pragma unroll
                    for (int sub = 0; sub < S::SUBS; ++sub) {
                        v0[sub] = __shfl_sync(0xffffffffu, mine, 16 * sub + g);
                        v1[sub] = __shfl_sync(0xffffffffu, mine, 16 * sub + g + 8);
                        e0[sub] = __shfl_sync(0xffffffffu, size, 16 * sub + g);
                        e1[sub] = __shfl_sync(0xffffffffu, size, 16 * sub + g + 8);
                    }
                }
                if (seen != EVERY) {
#pragma unroll
                    for (int sub = 0; sub < S::SUBS; ++sub)
#pragma unroll
                        for (int nt = 0; nt < S::NT; ++nt) {
                            if (!(seen >> (16 * sub + g) & 1)) c[sub][nt][0] = c[sub][nt][1] = -INFINITY;
                            if (!(seen >> (16 * sub + g + 8) & 1)) c[sub][nt][2] = c[sub][nt][3] = -INFINITY;
                        }
                }
                float high[S::NT][2];
                bool higher = false;
#pragma unroll
                for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        high[nt][k] = fmaxf(c[0][nt][k] + e0[0], c[0][nt][2 + k] + e1[0]);
                        if constexpr (S::SUBS == 2) high[nt][k] = fmaxf(high[nt][k], fmaxf(c[S::SUBS - 1][nt][k] + e0[S::SUBS - 1], c[S::SUBS - 1][nt][2 + k] + e1[S::SUBS - 1]));
                        higher |= high[nt][k] - top[nt][k] > 6.0f; // (top + 6 may be rounded to top + 8)
                    }
                // The reference exponent need not be the maximum: it moves when a weight would pass 2^14, which after the first steps is rare.
                if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
                    for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            float m = high[nt][k];
#pragma unroll
                            for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
                            m = fmaxf(m, top[nt][k]);
                            if constexpr (S::GENERAL) // rows of other sequences: what one needs leaves the others' bits alone
                                if (!(m - top[nt][k] > 6.0f)) m = top[nt][k];
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
#pragma unroll
                for (int sub = 0; sub < S::SUBS; ++sub) {
                    // Weights in fp16 and, as a second operand, what that rounding left: 22 bits.  The second operand costs int8 rows, where the rest
                    // draws the most power, 5 % (64 x 8192 tokens 111 us without it, 116 with it), the other caches 2 % at most.
                    uint32_t wh[S::NT][2], wl[S::NT][2];
#pragma unroll
                    for (int nt = 0; nt < S::NT; ++nt) {
                        float w[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) w[x] = exp2_fast(c[sub][nt][x] - __fadd_ru(top[nt][x & 1], -8.0f)); // up: of scores 16 apart the one below would make a weight 2^16
                        sum[nt][0] += w[0] + w[2];
                        sum[nt][1] += w[1] + w[3];
                        if constexpr (S::KIND == CACHE_I8_ROWS) {
                            w[0] *= v0[sub]; w[1] *= v0[sub];
                            w[2] *= v1[sub]; w[3] *= v1[sub];
                        }
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const __half2 x = __floats2half2_rn(w[2 * r], w[2 * r + 1]);
                            wh[nt][r] = transpose8x8(h2(x));
                            const float2 f = __half22float2(x);
                            wl[nt][r] = transpose8x8(h2(__floats2half2_rn(w[2 * r] - f.x, w[2 * r + 1] - f.y)));
                        }
                    }

                    // ---- values^T x weights^T ----------------------------------------------------------------------------------
                    constexpr int VW = S::VP / 4, EP = S::VP / S::ES; // words and dimensions of a piece
#pragma unroll
                    for (int i = 0; i < S::VN; ++i) {
                        const auto& w = vw[sub];
#pragma unroll
                        for (int x = 0; x < VW; ++x) {
                            if constexpr (S::ES == 2) {
                                const uint32_t a0 = __byte_perm(w[0][i][x], w[1][i][x], 0x5410), a1 = __byte_perm(w[0][i][x], w[1][i][x], 0x7632);
                                const uint32_t a2 = __byte_perm(w[2][i][x], w[3][i][x], 0x5410), a3 = __byte_perm(w[2][i][x], w[3][i][x], 0x7632);
#pragma unroll
                                for (int nt = 0; nt < S::NT; ++nt) {
                                    mma(o[nt][i * EP / 2 + x], a0, a1, a2, a3, wh[nt][0], wh[nt][1]);
                                    mma(o[nt][i * EP / 2 + x], a0, a1, a2, a3, wl[nt][0], wl[nt][1]);
                                }
                            } else {
                                uint32_t u[4], v[4];
                                widen_pairs(p, w[0][i][x], w[1][i][x], u);
                                widen_pairs(p, w[2][i][x], w[3][i][x], v);
                                if constexpr (S::KIND == CACHE_I8_GROUPS) {
                                    // These four dimensions are of one group; value x scale is rounded to fp16, as it is when it is read back.  What that
                                    // leaves, in a third product, would take 17 % more time (16 x 4096 tokens 64 -> 75 us) for an error of 0.00021 instead
                                    // of 0.00029 (2-norm; the output's own rounding alone 0.00020).
                                    const __half2 fu = as_h2(__byte_perm(vs[sub][0][i], vs[sub][1][i], x < 2 ? 0x5410 : 0x7632));
                                    const __half2 fv = as_h2(__byte_perm(vs[sub][2][i], vs[sub][3][i], x < 2 ? 0x5410 : 0x7632));
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
                    load_values(sub);
                }
                load_scale(v_scale, true);
            } else { // nothing of this step was there
#pragma unroll
                for (int sub = 0; sub < S::SUBS; ++sub) load_keys(sub), load_values(sub);
                load_scale(k_scale, false);
                load_scale(v_scale, true);
            }
            seen = coming;
            locate(ahead, step + 2 * WARPS);
            ahead = find(step + 3 * WARPS);
        }

        // ---- the warps' sums -------------------------------------------------------------------------------------------------
        bool none = false, met = false; // no weight at all: were there tokens?  Looked up again, since a register for it in the loop costs 1 %
#pragma unroll
        for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) sum[nt][k] += __shfl_xor_sync(0xffffffffu, sum[nt][k], x);
                none |= sum[nt][k] == 0.0f;
            }
        if (__any_sync(0xffffffffu, none))
            for (int32_t step = step0 + warp; step < step1 && !met; step += WARPS) {
                locate(find(step), step);
                met = coming != 0;
            }
#pragma unroll
        for (int nt = 0; nt < S::NT; ++nt) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int h = nt * 8 + 2 * t + k;
                if (g == 0) tops[warp * S::HEADS + h] = make_float2(met ? fmaxf(top[nt][k], kLowest) : top[nt][k], sum[nt][k]);
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
        if (late) pdl_wait_prior_grid();
        const bool whole = step0 == 0 && step1 == steps;
        const int64_t slot = 2 * (int64_t)blockIdx.x + (step0 == 0 ? 1 : 0);
        const int head0 = kvh * p.shared + q_first;
        for (int x = threadIdx.x; x < q_count * (S::D / 4); x += S::THREADS) {
            const int h = x / (S::D / 4), d = (x - h * (S::D / 4)) * 4;
            float m = kNothingSeen, l = 0.0f;
            float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) m = fmaxf(m, tops[w * S::HEADS + h].x);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float2 s = tops[w * S::HEADS + h];
                const float f = exp2_fast(s.x - m);
                const float4 a = *reinterpret_cast<const float4*>(&part[(w * S::HEADS + h) * S::ROW + d]);
                l += f * s.y;
                v.x += f * a.x; v.y += f * a.y; v.z += f * a.z; v.w += f * a.w;
            }
            if (whole) {
                if constexpr (S::GENERAL) finish<S>(p, b, kvh, q_first + h, d, v, m, l);
                else write_out(p, b, head0 + h, S::D, d, v, m, l);
            } else {
                __stcg(reinterpret_cast<float4*>(p.sums + (slot * S::HEADS + h) * S::D + d), v);
                if (d == 0) __stcg(&p.tops[slot * S::HEADS + h], make_float2(m, l));
            }
        }

        // ---- an item in pieces: the CTA that is last to have its sums in the workspace joins them, in the order of the tokens ----
        if (!whole) {
            // CTAs whose shares begin inside the item: c with begin < c * all / ctas < end, rounded down
            const int64_t all = share.all, ctas = share.ctas;
            const int64_t begin = step1 < steps ? (int64_t)(blockIdx.x + 1) * all / ctas - step1 : (int64_t)blockIdx.x * all / ctas - step0;
            const int64_t end = begin + steps;
            const int32_t c0 = (int32_t)(((begin + 1) * ctas + all - 1) / all) - 1; // began the item
            const int32_t pieces = (int32_t)((end * ctas + all - 1) / all) - c0;
            // The barrier puts the other threads' sums ahead of this thread's release, and its acquire ahead of their reads.  A counter is
            // the call's number above 16 bits of arrivals, none between calls; the maximum throws out what earlier calls that ran at the same time
            // on this workspace, against the rules, have left.  A captured call keeps the number of its capture, so that its replays get rid only of
            // what calls before the capture have left.
            auto last_of = [&](uint64_t* counter, int32_t number) {
                __syncthreads();
                if (threadIdx.x == 0) {
                    uint64_t before;
                    asm volatile("red.relaxed.gpu.global.max.u64 [%0], %1;" ::"l"(counter), "l"(p.call << 16) : "memory");
                    asm volatile("atom.add.acq_rel.gpu.global.u64 %0, [%1], 1;" : "=l"(before) : "l"(counter) : "memory");
                    is_last = (before & 0xffffu) == (uint32_t)(number - 1);
                    if (is_last) *counter = before & ~0xffffull;
                }
                __syncthreads();
                return is_last;
            };
            auto slot_of = [&](int32_t piece) { return 2 * (int64_t)(c0 + piece) + (piece == 0 ? 1 : 0); };
            // 16 loads a thread at once: ITEMS places of the output times BATCH pieces
            constexpr int ITEMS = (S::HEADS * S::D / 4 + S::THREADS - 1) / S::THREADS, BATCH = ITEMS >= 4 ? 4 : 16 / ITEMS;
            float4 v[ITEMS];
            float m[ITEMS], l[ITEMS];
            int h[ITEMS], d[ITEMS];
#pragma unroll
            for (int x = 0; x < ITEMS; ++x) {
                const int at = min((int)threadIdx.x + x * S::THREADS, q_count * (S::D / 4) - 1); // some do the last one again
                h[x] = at / (S::D / 4);
                d[x] = (at - h[x] * (S::D / 4)) * 4;
            }
            auto join = [&](int32_t piece, int32_t number, int32_t apart) {
#pragma unroll
                for (int x = 0; x < ITEMS; ++x) {
                    v[x] = make_float4(0, 0, 0, 0);
                    m[x] = kNothingSeen;
                    l[x] = 0.0f;
                }
                for (int32_t i = 0; i < number; i += BATCH) {
                    float2 s[BATCH][ITEMS];
                    float4 a[BATCH][ITEMS];
#pragma unroll
                    for (int j = 0; j < BATCH; ++j) {
                        const int64_t slot = slot_of(piece + min(i + j, number - 1) * apart) * S::HEADS;
#pragma unroll
                        for (int x = 0; x < ITEMS; ++x) {
                            s[j][x] = __ldcg(&p.tops[slot + h[x]]);
                            a[j][x] = __ldcg(reinterpret_cast<const float4*>(p.sums + (slot + h[x]) * S::D + d[x]));
                            if (i + j >= number) s[j][x].x = -INFINITY; // the last piece once more, without weight
                        }
                    }
#pragma unroll
                    for (int x = 0; x < ITEMS; ++x) {
                        float up = m[x];
#pragma unroll
                        for (int j = 0; j < BATCH; ++j) up = fmaxf(up, s[j][x].x);
                        const float keep = exp2_fast(m[x] - up);
                        m[x] = up;
                        l[x] *= keep;
                        v[x].x *= keep; v[x].y *= keep; v[x].z *= keep; v[x].w *= keep;
#pragma unroll
                        for (int j = 0; j < BATCH; ++j)
                            if (i + j < number) {
                                const float f = exp2_fast(s[j][x].x - up);
                                l[x] += f * s[j][x].y;
                                v[x].x += f * a[j][x].x; v[x].y += f * a[j][x].y; v[x].z += f * a[j][x].z; v[x].w += f * a[j][x].w;
                            }
                    }
                }
            };
            // Many pieces are joined in groups, whose sums take the place of their first piece's, and then the groups: one CTA alone took 8 us
            // for 55 pieces and 50 for 500 (8 heads over one, 131072 tokens: 74 -> 22 us).
            const int32_t first_of_mine = (int32_t)blockIdx.x - c0;
            int32_t per_group = 1;
            bool ends = true;
            if (pieces > 2 * BATCH) {
                for (per_group = BATCH; per_group * per_group < pieces;) per_group += BATCH;
                const int32_t piece = first_of_mine / per_group * per_group, number = min(per_group, pieces - piece);
                const int64_t at = slot_of(piece);
                ends = last_of(p.arrived + kCtas + at, number);
                if (ends) {
                    join(piece, number, 1);
                    __syncthreads(); // all have read what is now replaced
#pragma unroll
                    for (int x = 0; x < ITEMS; ++x) {
                        __stcg(reinterpret_cast<float4*>(p.sums + (at * S::HEADS + h[x]) * S::D + d[x]), v[x]);
                        if (d[x] == 0) __stcg(&p.tops[at * S::HEADS + h[x]], make_float2(m[x], l[x]));
                    }
                }
            }
            const int32_t groups = (pieces + per_group - 1) / per_group;
            if (ends && last_of(p.arrived + c0, groups)) {
                join(0, groups, per_group);
#pragma unroll
                for (int x = 0; x < ITEMS; ++x) {
                    if constexpr (S::GENERAL) finish<S>(p, b, kvh, q_first + h[x], d[x], v[x], m[x], l[x]);
                    else write_out(p, b, head0 + h[x], S::D, d[x], v[x], m[x], l[x]);
                }
            }
        }
        __syncthreads();
        if (++hh == heads_per_sequence) hh = 0, ++b;
    }
    if (late) pdl_wait_prior_grid();
    if constexpr (S::GENERAL) {
        if (p.late_wait && blockIdx.x == 0 && threadIdx.x == 0) *(volatile uint32_t*)p.ahead = 0; // CTAs that begin from here on wait first, which takes them no time any more
    }
}

template <class S>
int32_t launch(cudaStream_t stream, AttentionParams& p, int64_t tokens, int32_t* sms) {
    // No more CTAs than there can be work for: the lengths are known on the device only.
    const int64_t steps = std::max<int64_t>(1, (tokens + S::TOKENS - 1) / S::TOKENS), items = p.batch * p.cache.kv_heads * p.tiles;
    const int64_t most = S::CTAS * kSms, ctas = items >= most ? most : std::min(most, std::max(items, items * (steps + kBeginning<S>) / S::WARPS));
    // Items that are short whatever their lengths: a CTA each, of which there may be more than the device holds at once, without looking through the lengths first; so short
    // that the kernel would find the same, or up to 512 tokens where they fill a quarter of the device (16 sequences of 8 heads, 512 chosen tokens 20.4 us, 22.8 if shared
    // out; with 1024 29.3 and 26.4), or more of them where they are many.  In fp16, heads of 128, behind 1000 tokens: 64 sequences of 8 heads with 100 tokens each 25.7
    // and 31.2; 600 of one head with 500 49 and 59; 256 of 8 with up to 1500 217 and 223; but 64 of 8 with up to 1500 78 and 67.  (int8 rows,
    // 1024 tokens: 32 of 8 behind 12345 62 and 64.)  whole_tokens: what pays beside another kernel.
    const int64_t worth = std::max(items, 4 * items >= most ? most : 0);
    p.whole_items = S::GENERAL && (steps + kBeginning<S> <= 4 * S::WARPS || steps * (p.late_wait ? 1 : S::SUBS) * most <= 8 * S::WARPS * worth || tokens <= p.whole_tokens);
    const int64_t grid = p.whole_items ? items : ctas;
    if (sms) {
        *sms = (int32_t)((grid + S::CTAS - 1) / S::CTAS);
        return RC_SUCCESS;
    }
    launch_ex(paged_attention_kernel<S>, dim3((unsigned)grid), dim3(S::THREADS), stream, true, p);
    return check_launch("paged attention");
}

template <int D, int NT, bool PACKED, bool GENERAL>
int32_t launch_kind(cudaStream_t stream, AttentionParams& p, int64_t tokens, int32_t* sms) {
    if (p.cache.quant_group == 0) return launch<Shape<D, CACHE_F16, NT, PACKED, GENERAL>>(stream, p, tokens, sms);
    if (p.cache.quant_group == 8) return launch<Shape<D, CACHE_I8_GROUPS, NT, PACKED, GENERAL>>(stream, p, tokens, sms);
    return launch<Shape<D, CACHE_I8_ROWS, NT, PACKED, GENERAL>>(stream, p, tokens, sms);
}
template <int D, bool PACKED, bool GENERAL>
int32_t launch_heads(cudaStream_t stream, AttentionParams& p, int64_t tokens, int32_t* sms) {
    if constexpr (D <= 128)
        if (heads_at_once(D, p.shared) == 16) return launch_kind<D, 2, PACKED, GENERAL>(stream, p, tokens, sms);
    return launch_kind<D, 1, PACKED, GENERAL>(stream, p, tokens, sms);
}
template <int D, bool GENERAL>
int32_t launch_dim(cudaStream_t stream, AttentionParams& p, int64_t tokens, bool packed, int32_t* sms) {
    return packed ? launch_heads<D, true, GENERAL>(stream, p, tokens, sms) : launch_heads<D, false, GENERAL>(stream, p, tokens, sms);
}

template <bool GENERAL>
int32_t launch_attention(cudaStream_t s, AttentionParams& p, int32_t* sms = nullptr) {
    const int32_t D = p.cache.head_dim;
    const bool packed = p.cache.page_size % 16 == 0 && p.cache.token_stride == D && (p.cache.quant_group != 8 || p.cache.scale_token_stride == D / 8);
    if (D == 64) return launch_dim<64, GENERAL>(s, p, p.tokens_in_table, packed, sms);
    if (D == 96) return launch_dim<96, GENERAL>(s, p, p.tokens_in_table, packed, sms);
    if (D == 128) return launch_dim<128, GENERAL>(s, p, p.tokens_in_table, packed, sms);
    return launch_dim<256, GENERAL>(s, p, p.tokens_in_table, packed, sms);
}

} // namespace
} // namespace pplb200
