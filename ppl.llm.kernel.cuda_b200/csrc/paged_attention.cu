// Attention of one new token per sequence over the paged key-value cache.
#include "kv_cache.cuh"

#include <cmath>

namespace pplb200 {
namespace {

constexpr int ATPB = 128;

struct AttentionParams {
    const half* q;
    half* out;
    float* lse;
    const int32_t *pages, *lengths;
    int64_t q_stride, out_stride, pages_stride, pages_per_sequence;
    int32_t q_heads, shared; // query heads that share a key-value head
    int32_t window;
    float scale;
    pplb200_kv_cache cache;
};

__device__ __forceinline__ float cached(const pplb200_kv_cache& c, const void* data, const void* scale, int64_t at, int64_t sat, int d) {
    if (c.quant_group == 0) return __half2float(((const half*)data)[at + d]);
    const half s = ((const half*)scale)[sat + (c.quant_group == 8 ? d >> 3 : 0)];
    return __half2float(__float2half_rn((float)((const int8_t*)data)[at + d] * __half2float(s)));
}

// One CTA per sequence and query head; a warp takes every fourth token, a lane DPL of its dimensions.
template <int DPL>
__global__ void __launch_bounds__(ATPB) paged_attention_kernel(const AttentionParams p) {
    constexpr int D = 32 * DPL, WARPS = ATPB / 32;
    __shared__ float part[WARPS][D], top[WARPS], total[WARPS];
    pdl_wait_prior_grid();
    const int h = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t b = blockIdx.y;
    const int kvh = h / p.shared;
    const int64_t n = min((int64_t)p.lengths[b], p.pages_per_sequence * p.cache.page_size);
    const int64_t first = p.window > 0 && n > p.window ? n - p.window : 0;
    float q[DPL], o[DPL] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) q[i] = __half2float(p.q[b * p.q_stride + (int64_t)h * D + i * 32 + lane]);
    for (int64_t t = first + warp; t < n; t += WARPS) {
        const int64_t page = p.pages[b * p.pages_stride + t / p.cache.page_size];
        if (page < 0 || page >= p.cache.num_pages) continue;
        const int64_t in_page = t % p.cache.page_size;
        const int64_t at = kv_row(page, in_page, kvh, p.cache.page_stride, p.cache.head_stride, p.cache.token_stride);
        const int64_t sat = kv_row(page, in_page, kvh, p.cache.scale_page_stride, p.cache.scale_head_stride, p.cache.scale_token_stride);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < DPL; ++i) s += q[i] * cached(p.cache, p.cache.k, p.cache.k_scale, at, sat, i * 32 + lane);
#pragma unroll
        for (int x = 16; x >= 1; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= p.scale;
        const float up = fmaxf(m, s), keep = m == up ? 1.0f : __expf(m - up), w = __expf(s - up);
        m = up;
        l = l * keep + w;
#pragma unroll
        for (int i = 0; i < DPL; ++i) o[i] = o[i] * keep + w * cached(p.cache, p.cache.v, p.cache.v_scale, at, sat, i * 32 + lane);
    }
#pragma unroll
    for (int i = 0; i < DPL; ++i) part[warp][i * 32 + lane] = o[i];
    if (lane == 0) { top[warp] = m; total[warp] = l; }
    __syncthreads();
    float mm = -INFINITY, ll = 0.0f;
    for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, top[w]);
    for (int w = 0; w < WARPS; ++w) ll += total[w] > 0.0f ? total[w] * __expf(top[w] - mm) : 0.0f;
    for (int d = threadIdx.x; d < D; d += ATPB) {
        float v = 0.0f;
        for (int w = 0; w < WARPS; ++w) v += total[w] > 0.0f ? part[w][d] * __expf(top[w] - mm) : 0.0f;
        p.out[b * p.out_stride + (int64_t)h * D + d] = __float2half_rn(ll > 0.0f ? v / ll : 0.0f);
    }
    if (p.lse && threadIdx.x == 0) p.lse[b * p.q_heads + h] = ll > 0.0f ? mm + __logf(ll) : -INFINITY;
}

} // namespace
} // namespace pplb200

using namespace pplb200;

extern "C" {

int64_t pplb200_paged_decode_attention_workspace_bytes(int64_t batch, int64_t max_tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
    if (batch < 0 || max_tokens < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || head_dim <= 0) return -1;
    return 256;
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
    if (a->pages_per_sequence > (1LL << 31) / cache->page_size) return fail(RC_UNSUPPORTED, "a page table of more than 2^31 tokens");
    const int64_t need = pplb200_paged_decode_attention_workspace_bytes(a->batch, a->pages_per_sequence * cache->page_size, a->q_heads, cache->kv_heads, cache->head_dim);
    if (!a->ws || a->ws_bytes < need || ((uintptr_t)a->ws & 255))
        return fail(RC_INVALID_VALUE, "workspace of %lld bytes (256-byte aligned) needed, got %lld", (long long)need, (long long)a->ws_bytes);
    AttentionParams p = {};
    p.q = (const half*)a->q; p.out = (half*)a->out; p.lse = a->optional_lse;
    p.pages = a->pages; p.lengths = a->lengths;
    p.q_stride = a->q_stride; p.out_stride = a->out_stride;
    p.pages_stride = a->pages_stride; p.pages_per_sequence = a->pages_per_sequence;
    p.q_heads = a->q_heads; p.shared = a->q_heads / cache->kv_heads;
    p.window = a->window; p.scale = a->scale;
    p.cache = *cache;
    const dim3 grid((unsigned)a->q_heads, (unsigned)a->batch);
    const cudaStream_t s = (cudaStream_t)stream;
    if (D == 64) launch_ex(paged_attention_kernel<2>, grid, dim3(ATPB), s, true, p);
    else if (D == 96) launch_ex(paged_attention_kernel<3>, grid, dim3(ATPB), s, true, p);
    else if (D == 128) launch_ex(paged_attention_kernel<4>, grid, dim3(ATPB), s, true, p);
    else launch_ex(paged_attention_kernel<8>, grid, dim3(ATPB), s, true, p);
    return check_launch("paged attention");
}

} // extern "C"
