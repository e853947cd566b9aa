/*
 * C ABI of what lies between a quantized layer's fused QKV projection and its output projection: rotary positions, the
 * paged key-value cache (fp16, or int8 with fp16 scales) and attention of one new token per sequence over that cache.
 *
 * Same rules as pplb200_i8i8.h: every entry point is stream-ordered and asynchronous, allocates nothing and returns a
 * ppl.common RetCode value; pointers are device pointers of the current device unless a comment says otherwise; the
 * argument blocks and the cache description are HOST memory, read before the call returns.  Activations are fp16.
 */
#ifndef PPLB200_ATTENTION_H
#define PPLB200_ATTENTION_H

#include "pplb200_i8i8.h"

#ifdef __cplusplus
extern "C" {
#endif
#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

/*
 * Rotary frequencies.  Plane i of rotary_dim / 2 turns by f_i radians a position,
 *   NONE        f_i = base ^ (-2 i / rotary_dim)
 *   LINEAR      f_i / factor: positions are divided by it
 *   NTK         the base times factor ^ (rotary_dim / (rotary_dim - 2)): the slowest plane is divided by factor, the fastest kept
 *   YARN        f_i for planes that turn at least keep_turns times within original_length positions, f_i / factor for those
 *               that turn at most stretch_turns times, a blend that is linear in the plane's index between them (the two
 *               limits rounded outwards to whole planes, and to 0 and rotary_dim - 1 where they lie beyond these); rotated
 *               values times 0.1 ln(factor) + 1
 *   WAVELENGTH  the same limits, the blend linear in the number of turns; no factor on the values
 * turns_host[i] (HOST, rotary_dim / 2 words) receives f_i / (2 pi) as a fraction of a turn in units of 2^-64, within four of them (where
 * long double has 64 bits or more); position * turns_host[i] modulo 2^64, which is taken without a rounding, is the angle, within |position| *
 * 2^-62 turns: 2^-22 of a turn at a position of 2^40.  magnitude_host (HOST) receives the factor on the values.
 * To be called once; the caller keeps a copy of turns_host on the device.
 */
enum {
    PPLB200_ROTARY_NONE = 0,
    PPLB200_ROTARY_LINEAR = 1,
    PPLB200_ROTARY_NTK = 2,
    PPLB200_ROTARY_YARN = 3,
    PPLB200_ROTARY_WAVELENGTH = 4
};
int32_t pplb200_rotary_frequencies(int32_t rotary_dim, double base, int32_t scaling, double factor, double original_length,
                                   double keep_turns, double stretch_turns, uint64_t* turns_host, float* magnitude_host);

/*
 * Rotation of query and key heads: (a, b) -> ((a cos - b sin) magnitude, (b cos + a sin) magnitude), where (a, b) are dimensions
 * (i, i + rotary_dim / 2) of a head, or (2 i, 2 i + 1) with `interleaved`; dimensions from rotary_dim on are copied.  In 32 bits,
 * rounded once to fp16.
 * q fp16 [tokens, q_heads, head_dim], k fp16 [tokens, k_heads, head_dim]: *_stride elements between tokens, a token's heads
 * contiguous, so that slices of the fused projection's rows can be given.  Either of q and k may have 0 heads.  q_out may be q and
 * k_out may be k (with the same stride); no other overlap.  positions int64 [tokens], any sign.
 * head_dim and rotary_dim multiples of 16, rotary_dim <= head_dim <= 256, strides multiples of 8, 16-byte aligned q, k, q_out, k_out.
 */
typedef struct pplb200_rotary_args {
    const void *q, *k;
    void *q_out, *k_out;
    const int64_t* positions;
    const uint64_t* turns;
    int64_t tokens, q_stride, k_stride, q_out_stride, k_out_stride;
    int32_t q_heads, k_heads, head_dim, rotary_dim, interleaved;
    float magnitude;
} pplb200_rotary_args;
int32_t pplb200_rotary_fp16(pplb200_stream_t stream, const pplb200_rotary_args* args);

/*
 * A paged key-value cache of one layer.  Token `slot` lies on page slot / page_size, at slot % page_size of it; its keys of head h
 * are the head_dim elements from k + page * page_stride + h * head_stride + (slot % page_size) * token_stride, its values the same
 * from v.  Both orders of heads and a page's tokens are a matter of the strides.  Strides are in elements (scales: in scales), not
 * negative, those of k and v multiples of 16 bytes; k and v 16-byte aligned.  Rows may overlap (a stride of 0) where nothing is written.
 * quant_group 0: k and v are fp16.  quant_group 8 or head_dim: int8, and every quant_group dimensions share an fp16 scale,
 * head_dim / quant_group contiguous scales for a token and head.  head_dim a multiple of 16, at most 256; at most 65535 heads; the last
 * element, and the last scale, less than 2^61 from the first.
 */
typedef struct pplb200_kv_cache {
    void *k, *v, *k_scale, *v_scale;
    int64_t num_pages, page_stride, head_stride, token_stride, scale_page_stride, scale_head_stride, scale_token_stride;
    int32_t page_size, kv_heads, head_dim, quant_group;
} pplb200_kv_cache;

/*
 * Stores `tokens` new tokens: k, v fp16 [tokens, kv_heads, head_dim] with their strides as above, slots int64 [tokens].  With
 * rotary_dim > 0 the same call rotates q and k first, as pplb200_rotary_fp16 does (k is rounded to fp16 before it is quantized, so
 * that the result is that of the two calls), and writes q_out; with rotary_dim 0 q, q_out, positions and turns are not used.
 * A group's scale is its largest magnitude / 127, rounded up to fp16, at least 2^-24 and at most 515.5 (so that no finite value
 * reads back as infinity); elements are divided by that scale and rounded to nearest even, which puts them within +-127.
 * A group that contains an infinity or a NaN gets an infinite or NaN scale and reads back as NaN.
 * A token whose slot is negative or beyond the cache's last page is not stored (its q is rotated all the same).  No two tokens of a
 * call may have the same slot.
 */
typedef struct pplb200_kv_write_args {
    const void *q, *k, *v;
    void* q_out;
    const int64_t *positions, *slots;
    const uint64_t* turns;
    int64_t tokens, q_stride, k_stride, v_stride, q_out_stride;
    int32_t q_heads, rotary_dim, interleaved;
    float magnitude;
} pplb200_kv_write_args;
int32_t pplb200_kv_cache_write_fp16(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_kv_write_args* args);

/*
 * Reads tokens back: k_out, v_out fp16 [tokens, kv_heads, head_dim], contiguous, 16-byte aligned = the stored values, or value x
 * scale rounded to fp16.  A slot that is negative or beyond the last page gives zeros; a slot may be asked for several times.
 */
int32_t pplb200_kv_cache_read_fp16(pplb200_stream_t stream, const pplb200_kv_cache* cache, const int64_t* slots, int64_t tokens,
                                   void* k_out, void* v_out);

/*
 * Attention of one new token per sequence: out[b, h] = sum_t softmax_t(scale q[b, h] . k_t) v_t over the tokens t of sequence b in
 * head h / (q_heads / kv_heads) of the cache: the stored values, or values x scales, which are not rounded to fp16 in between, except
 * v with groups of 8, which is.  With groups of 8 a value x scale beyond fp16's range, which no scale up to 515.5 reaches (the writer's largest), is
 * infinite as v and makes its token's score NaN as k; rows that share a scale a head take any finite one.  Scores, sums and statistics are held in 32 bits; the softmax's weights enter their product with v
 * with 22 bits.
 * q, out fp16 [batch, q_heads, head_dim], *_stride elements between sequences, heads contiguous; lengths int32 [batch]: tokens in the
 * cache, the new one among them (at most pages_per_sequence * page_size are looked at); pages int32 [batch, pages_per_sequence] with
 * pages_stride between rows: the page of token t is pages[b, t / page_size].  A page that is negative or not below num_pages is a
 * hole: its tokens take no part.  window > 0: only the last `window` tokens do.  What lies in the cache beyond a sequence's
 * tokens has no influence, whatever it is.  A sequence of which nothing is seen has zeros for its output and -inf for its lse; one whose
 * tokens are seen, but have scores of -inf only, NaN and -inf.
 * optional_lse fp32 [batch, q_heads], contiguous: log(sum_t exp(scale q . k_t)), for joining results over parts of a context.
 * head_dim 64, 96, 128 or 256 (with quant_group 8: scales 4-byte aligned, their strides even); q_heads a multiple of kv_heads; strides
 * multiples of 8; q and out 16-byte aligned; out may be q; scale within 2^50 of zero; at most 2^30 tokens a row of the table, 65535
 * sequences and 65535 query heads; rows of one head of the cache, and their scales, less than 2^32 times the largest power of two (up to
 * 2^30 bytes) that divides their distances apart.
 * ws: pplb200_paged_decode_attention_workspace_bytes(), 256-byte aligned, zeroed before its first use (every call leaves it fit for the
 * next, of whatever sizes), not shared by calls that may run at the same time (two captured graphs that are replayed at once need
 * one each).  Where calls have overlapped all the same, their results are void, and the workspace is to be zeroed before a captured call is
 * replayed on it again.
 * The result does not depend on what else is in the batch's other rows beyond the order in which a sequence's parts are summed,
 * and is the same for the same call, run after run.
 */
typedef struct pplb200_paged_attention_args {
    const void* q;
    void* out;
    float* optional_lse;
    const int32_t *pages, *lengths;
    void* ws;
    int64_t ws_bytes, batch, pages_per_sequence, pages_stride, q_stride, out_stride;
    int32_t q_heads, window;
    float scale;
    int32_t reserved;
} pplb200_paged_attention_args;
int64_t pplb200_paged_decode_attention_workspace_bytes(int64_t batch, int64_t max_tokens, int32_t q_heads, int32_t kv_heads,
                                                       int32_t head_dim);
int32_t pplb200_paged_decode_attention_fp16(pplb200_stream_t stream, const pplb200_kv_cache* cache,
                                            const pplb200_paged_attention_args* args);

/*
 * Host-only: offset in elements of head `head` of a slot from cache->k, as the kernels that write and read the cache compute it, and as
 * attention's does, which has arithmetic of its own; -1 where the slot is not in the cache, or the cache is refused.
 */
int64_t pplb200_kv_cache_offset(const pplb200_kv_cache* cache, int64_t slot, int32_t head);
int64_t pplb200_paged_attention_offset(const pplb200_kv_cache* cache, int64_t slot, int32_t head);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#ifdef __cplusplus
}
#endif
#endif
