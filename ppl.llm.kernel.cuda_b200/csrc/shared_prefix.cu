// Attention of one new token per sequence for a batch that shares a prefix: the prefix for the rows of all sequences at once, then each sequence's
// own tokens, whose sums are joined with the prefix's where the output is written.
#include "paged_attention.cuh"

namespace pplb200 {
namespace {

constexpr int64_t kMaxRows = 1 << 24;

// Sums over the prefix: reference exponents and sums of weights, then sums of values.
int64_t part_bytes(int64_t rows, int32_t head_dim) { return round_up(rows * 8, 256) + round_up(rows * head_dim * 4, 256); }

} // namespace
} // namespace pplb200

using namespace pplb200;

extern "C" {

int64_t pplb200_shared_prefix_attention_workspace_bytes(int64_t batch, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
    if (batch < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || head_dim <= 0 || batch > kMaxRows / q_heads) return -1;
    const int32_t shared = q_heads / kv_heads;
    return std::max(workspace_bytes(shared, head_dim), workspace_bytes(batch * shared, head_dim)) + part_bytes(batch * q_heads, head_dim);
}

int32_t pplb200_shared_prefix_attention_fp16(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_paged_attention_args* a,
                                             const pplb200_shared_prefix* prefix) {
    AttentionParams own = {};
    const int32_t rc = take_call(cache, a, own);
    if (rc != RC_SUCCESS) return rc;
    if (!prefix || prefix->num_pages < 0) return fail(RC_INVALID_VALUE, "no prefix");
    if (a->window) return fail(RC_UNSUPPORTED, "a shared prefix is not seen through a window");
    if (a->batch > kMaxRows / a->q_heads) return fail(RC_UNSUPPORTED, "more than 2^24 rows of q");
    if (a->batch == 0) return RC_SUCCESS;
    if (!prefix->length || (prefix->num_pages > 0 && !prefix->pages)) return fail(RC_INVALID_VALUE, "null prefix length or pages");
    if ((((uintptr_t)prefix->length | (uintptr_t)prefix->pages) & 3) != 0) return fail(RC_INVALID_VALUE, "prefix length and pages must be 4-byte aligned");
    if (prefix->num_pages > (1LL << 30) / cache->page_size) return fail(RC_UNSUPPORTED, "a prefix of more than 2^30 tokens");
    const int64_t need = pplb200_shared_prefix_attention_workspace_bytes(a->batch, a->q_heads, cache->kv_heads, cache->head_dim);
    if (!a->ws || a->ws_bytes < need || ((uintptr_t)a->ws & 255))
        return fail(RC_INVALID_VALUE, "workspace of %lld bytes (256-byte aligned) needed, got %lld", (long long)need, (long long)a->ws_bytes);
    const int32_t shared = a->q_heads / cache->kv_heads;
    const int64_t rows = a->batch * a->q_heads;
    own.unit_tokens = cache->page_size;
    own.units_per_page = 1;
    own.num_units = own.num_pages;
    own.rows_per_head = shared;
    own.part_rows = rows;
    own.part_tops = (float2*)((char*)a->ws + need - part_bytes(rows, cache->head_dim));
    own.part_sums = (float*)((char*)own.part_tops + round_up(rows * 8, 256));
    // the prefix: one sequence, whose key heads are asked by the rows of all
    AttentionParams first = own;
    first.batch = 1;
    first.pages = prefix->pages;
    first.lengths = prefix->length;
    first.pages_stride = prefix->num_pages;
    first.tokens_in_table = prefix->num_pages * cache->page_size;
    first.keep_parts = true;
    lay_out(first, a->ws, a->batch * shared);
    const int32_t done = launch_general((cudaStream_t)stream, first);
    if (done != RC_SUCCESS) return done;
    own.parts = 1;
    lay_out(own, a->ws, shared);
    return launch_general((cudaStream_t)stream, own);
}

} // extern "C"
