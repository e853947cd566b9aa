// Attention of one new token per sequence: the call's checks, and the forms that one page table a sequence and one output a call need.
#include "paged_attention.cuh"

namespace pplb200 {
namespace {

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

// Units of the rows, and of the scales, of a cache that has been checked.
bool cache_units(const pplb200_kv_cache* c, AttentionParams& p) {
    const int bytes = c->quant_group ? 1 : 2;
    return row_units(c->num_pages, c->page_size, c->page_stride * bytes, c->token_stride * bytes, p.unit, p.page_units, p.token_units) &&
           (!c->quant_group || row_units(c->num_pages, c->page_size, c->scale_page_stride * 2, c->scale_token_stride * 2, p.scale_unit, p.scale_page_units, p.scale_token_units));
}

} // namespace

namespace paged {

int32_t take_call(const pplb200_kv_cache* cache, const pplb200_paged_attention_args* a, AttentionParams& p) {
    const int32_t rc = check_kv_cache(cache);
    if (rc != RC_SUCCESS) return rc;
    if (!a) return fail(RC_INVALID_VALUE, "null arguments");
    const int64_t D = cache->head_dim;
    if (D != 64 && D != 96 && D != 128 && D != 256) return fail(RC_UNSUPPORTED, "attention: head_dim must be 64, 96, 128 or 256, got %lld", (long long)D);
    if (a->batch < 0 || a->pages_per_sequence < 0) return fail(RC_INVALID_VALUE, "negative extent");
    if (a->batch > 65535) return fail(RC_UNSUPPORTED, "more than 65535 sequences");
    if (a->q_heads <= 0 || a->q_heads > 65535 || a->q_heads % cache->kv_heads)
        return fail(RC_INVALID_VALUE, "q_heads (%d) must be a multiple of the cache's heads (%d)", a->q_heads, cache->kv_heads);
    // up to here no score is as low as -1e30, the reference exponent of a sequence before its first token
    if (!(std::fabs(a->scale) <= 0x1p50f)) return fail(RC_INVALID_VALUE, "the scale must be within 2^50 of zero");
    if (a->batch == 0) return RC_SUCCESS; // the pointers are not looked at
    if (!a->q || !a->out || !aligned16(a->q) || !aligned16(a->out)) return fail(RC_INVALID_VALUE, "q and out must be 16-byte aligned pointers");
    if (a->q_stride % 8 || a->out_stride % 8 || (a->batch > 1 && (a->q_stride < a->q_heads * D || a->out_stride < a->q_heads * D)))
        return fail(RC_INVALID_VALUE, "q / out: sequences must be a multiple of 8 elements apart, and no closer than their heads are long");
    if (!a->lengths || (a->pages_per_sequence > 0 && !a->pages)) return fail(RC_INVALID_VALUE, "null lengths or pages");
    if ((((uintptr_t)a->lengths | (uintptr_t)a->pages | (uintptr_t)a->optional_lse) & 3) != 0) return fail(RC_INVALID_VALUE, "lengths, pages and lse must be 4-byte aligned");
    if (a->batch > 1 && a->pages_stride < a->pages_per_sequence) return fail(RC_INVALID_VALUE, "rows of the page table overlap");
    // token numbers are 32-bit, and go a few tiles beyond the last one
    if (a->pages_per_sequence > (1LL << 30) / cache->page_size) return fail(RC_UNSUPPORTED, "a page table of more than 2^30 tokens");
    if (cache->quant_group == 8 && ((((uintptr_t)cache->k_scale | (uintptr_t)cache->v_scale) & 3) ||
                                    ((cache->scale_page_stride | cache->scale_head_stride | cache->scale_token_stride) & 1)))
        return fail(RC_INVALID_VALUE, "attention: scales of groups of 8 must be 4-byte aligned, and their strides even");
    if (!cache_units(cache, p))
        return fail(RC_UNSUPPORTED, "attention: the rows of a head lie further apart than 2^32 times their alignment");
    small_division(cache->page_size, p.page_magic, p.page_shift);
    p.num_pages = (int32_t)std::min<int64_t>(cache->num_pages, 0x7fffffff); // a table's entry is no larger
    p.q = (const half*)a->q; p.out = (half*)a->out; p.lse = a->optional_lse;
    p.pages = a->pages; p.lengths = a->lengths;
    p.q_stride = a->q_stride; p.out_stride = a->out_stride;
    p.pages_stride = a->pages_stride; p.tokens_in_table = a->pages_per_sequence * cache->page_size; p.batch = a->batch;
    p.q_heads = a->q_heads; p.shared = a->q_heads / cache->kv_heads;
    p.window = a->window; p.scale_log2 = a->scale * 1.4426950408889634f;
    p.cache = *cache;
    p.flip_1024 = 0x64806480u;
    return RC_SUCCESS;
}

void lay_out(AttentionParams& p, void* ws, int64_t shared) {
    const int heads = heads_at_once(p.cache.head_dim, shared);
    static std::atomic<uint64_t> calls{0};
    p.shared = (int32_t)shared;
    p.tiles = (int32_t)((shared + heads - 1) / heads);
    p.call = ++calls;
    p.arrived = (uint64_t*)ws;
    p.tops = (float2*)((char*)ws + kZeros);
    p.sums = (float*)((char*)p.tops + round_up(2 * kCtas * heads * 8, 256));
}

} // namespace paged
} // namespace pplb200

using namespace pplb200;

extern "C" {

int64_t pplb200_paged_decode_attention_workspace_bytes(int64_t batch, int64_t max_tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
    if (batch < 0 || max_tokens < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || head_dim <= 0) return -1;
    return workspace_bytes(q_heads / kv_heads, head_dim);
}

int32_t pplb200_paged_decode_attention_fp16(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_paged_attention_args* a) {
    AttentionParams p = {};
    const int32_t rc = take_call(cache, a, p);
    if (rc != RC_SUCCESS || a->batch == 0) return rc;
    const int64_t need = pplb200_paged_decode_attention_workspace_bytes(a->batch, a->pages_per_sequence * cache->page_size, a->q_heads, cache->kv_heads, cache->head_dim);
    if (!a->ws || a->ws_bytes < need || ((uintptr_t)a->ws & 255))
        return fail(RC_INVALID_VALUE, "workspace of %lld bytes (256-byte aligned) needed, got %lld", (long long)need, (long long)a->ws_bytes);
    lay_out(p, a->ws, a->q_heads / cache->kv_heads);
    return launch_attention<false>((cudaStream_t)stream, p);
}

int64_t pplb200_paged_attention_offset(const pplb200_kv_cache* c, int64_t slot, int32_t head) {
    AttentionParams p = {};
    int64_t page;
    int32_t in_page;
    if (check_kv_cache(c) != RC_SUCCESS || !cache_units(c, p) || head < 0 || head >= c->kv_heads || !kv_find(slot, c->num_pages, c->page_size, page, in_page)) return -1;
    const uint32_t row = (uint32_t)page * p.page_units + (uint32_t)in_page * p.token_units;
    return head * c->head_stride + (int64_t)((uint64_t)row * p.unit / (c->quant_group ? 1 : 2));
}

} // extern "C"
