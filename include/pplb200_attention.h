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
 * Rotary positions with several axes, as tokens of images and videos have them (time, height, width): every plane belongs to one of
 * up to four axes and is turned by the token's position on that axis.
 * pplb200_rotary_axes_frequencies: planes_host[a] (HOST, `axes` numbers, not negative, rotary_dim / 2 together) planes belong to axis a: one axis behind the
 * other, or, with `alternating`, dealt out in turn (axis 0, 1, ..., 0, 1, ...), an axis that has all its planes being passed over.  The planes' frequencies are those of
 * pplb200_rotary_frequencies; with `restart` the n planes of each axis have those of a rotary_dim of 2 n, in order, instead.  axis_of_plane_host (HOST,
 * rotary_dim / 2 bytes) receives the axes; the caller keeps a copy on the device, as of turns_host.
 * The calls: as those with one axis, but positions int64 [axes, tokens], axis_stride elements between axes: `tokens` or more, or 0 where all axes have the same positions.  axis_of_plane (device, 4-byte aligned): the
 * two lowest bits are looked at, and a number beyond the axes stands for the last one.
 */
enum { PPLB200_ROTARY_MAX_AXES = 4 };
typedef struct pplb200_rotary_axes {
    const uint8_t* axis_of_plane;
    int64_t axis_stride;
    int32_t axes, reserved;
} pplb200_rotary_axes;
int32_t pplb200_rotary_axes_frequencies(int32_t rotary_dim, double base, int32_t scaling, double factor, double original_length,
                                        double keep_turns, double stretch_turns, int32_t axes, const int32_t* planes_host, int32_t alternating,
                                        int32_t restart, uint64_t* turns_host, uint8_t* axis_of_plane_host, float* magnitude_host);
int32_t pplb200_rotary_axes_fp16(pplb200_stream_t stream, const pplb200_rotary_args* args, const pplb200_rotary_axes* axes);

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
/* The same with positions of several axes (rotary_dim > 0). */
int32_t pplb200_kv_cache_write_axes_fp16(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_kv_write_args* args,
                                         const pplb200_rotary_axes* axes);

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
 * next, of whatever sizes, over a shared prefix or chosen blocks (below) too), not shared by calls that may run at the same time (two captured graphs that are replayed at once need
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
 * Attention of one new token per sequence for a batch whose sequences begin with the same tokens, which lie in the cache once: out[b, h] as
 * above over the prefix's tokens and sequence b's own, of which `lengths` counts and `pages` lists only the latter.  The prefix is read once for the
 * batch.  prefix->pages int32 [prefix->num_pages], prefix->length int32 [1], both on the device: how many tokens (at most num_pages * page_size are
 * looked at); pages that are not in the cache are holes.  A sequence with a length of 0 sees the prefix alone; a negative length stands for a row that is
 * no sequence: zeros and -inf, whatever its q.  As above otherwise, but window has to be 0, at most 2^24 rows of q (batch * q_heads), and over the prefix
 * the softmax's weights enter their product with v with 11 bits over an fp16 cache (22 over int8 ones).
 * ws: pplb200_shared_prefix_attention_workspace_bytes(), which holds for smaller batches too, with the rules above.
 */
typedef struct pplb200_shared_prefix {
    const int32_t *pages, *length;
    int64_t num_pages;
} pplb200_shared_prefix;
int64_t pplb200_shared_prefix_attention_workspace_bytes(int64_t batch, int32_t q_heads, int32_t kv_heads, int32_t head_dim);
int32_t pplb200_shared_prefix_attention_fp16(pplb200_stream_t stream, const pplb200_kv_cache* cache,
                                             const pplb200_paged_attention_args* args, const pplb200_shared_prefix* prefix);
/*
 * Health word of the kernel that takes a prefix through tensor memory, as pplb200_i8i8_gemm_status is the GEMM's: a wait in it that gives up leaves NaN in
 * the rows that it was for and a code here.  0 if none has on the current device since the last call with reset != 0; -1 where it cannot be read.  Not to be called
 * while a stream is being captured; synchronise the streams you launched on first.
 */
int32_t pplb200_shared_prefix_attention_status(int32_t reset);

/*
 * Bounds of the keys of blocks of tokens, for choosing among them.  A page has page_size / block blocks, block a multiple of 16 up to 2^30; block x of page p is block
 * number p * (page_size / block) + x of the cache.  bounds int8 [num_pages, kv_heads, page_size / block, 2, head_dim], contiguous, 16-byte aligned: in every
 * dimension the least and the greatest of the block's keys (as they are stored: fp16, or values x scales), divided by the block's scale and rounded outwards
 * to whole numbers; scale fp16 [num_pages, kv_heads, page_size / block], contiguous: the largest of the magnitudes / 127, rounded up to fp16, at least 2^-24.
 * A block with a key that is infinite or NaN, or whose scale would be beyond fp16's range, has zeros and an infinite scale.  head_dim as for attention.
 * pplb200_key_bounds_update: slots int64 [tokens], those that have been written: every block whose LAST token is among them is taken to be complete, and
 * its bounds are computed from what the cache then holds.  Slots that are not in the cache are passed over; no slot comes twice.
 * pplb200_key_bounds_read: blocks int64 [count], block numbers -> lo, hi fp32 [count, kv_heads, head_dim], contiguous, 16-byte aligned: whole numbers x scale
 * (-inf and inf for a block with an infinite scale; zeros for a number that is not in the cache).
 */
typedef struct pplb200_key_bounds {
    void *bounds, *scale;
    int32_t block, reserved;
} pplb200_key_bounds;
int32_t pplb200_key_bounds_update(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_key_bounds* bounds, const int64_t* slots,
                                  int64_t tokens);
int32_t pplb200_key_bounds_read(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_key_bounds* bounds, const int64_t* blocks,
                                int64_t count, float* lo, float* hi);

/*
 * Attention of one new token per sequence over some of its blocks.  A sequence of n tokens has ceil(n / block) blocks in order, the last of which may be
 * begun only.  The first choice->first and the last choice->last of them are attended, and of those between the choice->top with the highest scores,
 * each key head choosing its own; all, where there are no more.  The score of a block is the largest over the key head's query heads of
 *   sum_d max(q8_d lo_d, q8_d hi_d), the whole numbers of the bounds, times (q's scale x the block's scale), rounded once to fp32,
 * where q8 is q of that head quantized to int8: divided by its scale (the head's largest magnitude / 127, rounded up to fp16, at least 2^-24) and rounded to
 * nearest even.  Whole numbers throughout, so that the same blocks are chosen everywhere; among equal scores the lowest block.  The score is an upper bound of
 * q . k for the block's keys, up to the rounding of q.  A block with an infinite scale comes before all others; a block on a page that is not in the
 * cache comes behind all others (it is a hole, chosen or not); a query head with an infinity or a NaN has no say.
 * Then as pplb200_paged_decode_attention_fp16 over the chosen blocks' tokens, which are joined in order; args->window has to be 0.  Bounds are looked at for blocks between
 * the first and the last ones only: with choice->last >= 1 these are complete.
 * optional_blocks int32 [batch, kv_heads, first + last + top], contiguous: receives the chosen blocks of the sequence in ascending order, then -1.
 * first, last, top not negative, last at least 1, first + last + top at most 65536; at most 2^18 blocks a row of the page table; num_pages * (page_size / block) below 2^31; batch * kv_heads at most 2^24.
 * ws: pplb200_block_sparse_attention_workspace_bytes(), with the rules above.
 */
typedef struct pplb200_block_choice {
    int32_t first, last, top, reserved;
    int32_t* optional_blocks;
} pplb200_block_choice;
int64_t pplb200_block_sparse_attention_workspace_bytes(int64_t batch, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t attended_blocks);
int32_t pplb200_block_sparse_attention_fp16(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_key_bounds* bounds,
                                            const pplb200_paged_attention_args* args, const pplb200_block_choice* choice);

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
