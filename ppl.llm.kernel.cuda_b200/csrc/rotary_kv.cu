// Rotary positions, and the paged key-value cache written and read back.
#include "kv_cache.cuh"

#include <cmath>

namespace pplb200 {

int32_t check_kv_cache(const pplb200_kv_cache* c) {
    if (!c) return fail(RC_INVALID_VALUE, "null cache");
    if (c->num_pages < 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->kv_heads > 65535)
        return fail(RC_INVALID_VALUE, "bad cache: %lld pages of %d tokens, %d heads", (long long)c->num_pages, c->page_size, c->kv_heads);
    if (c->head_dim <= 0 || c->head_dim % 16 || c->head_dim > kMaxHeadDim)
        return fail(RC_UNSUPPORTED, "head_dim must be a multiple of 16 up to %d, got %d", kMaxHeadDim, c->head_dim);
    if (c->quant_group != 0 && c->quant_group != 8 && c->quant_group != c->head_dim)
        return fail(RC_UNSUPPORTED, "quant_group must be 0 (fp16), 8 or head_dim, got %d", c->quant_group);
    if (c->num_pages == 0) return RC_SUCCESS;
    if (!c->k || !c->v || (c->quant_group && (!c->k_scale || !c->v_scale))) return fail(RC_INVALID_VALUE, "null cache pointer");
    if (!aligned16(c->k) || !aligned16(c->v)) return fail(RC_INVALID_VALUE, "cache k and v must be 16-byte aligned");
    const int64_t unit = c->quant_group ? 16 : 8;
    if (c->page_stride < 0 || c->head_stride < 0 || c->token_stride < 0 || c->page_stride % unit || c->head_stride % unit ||
        c->token_stride % unit)
        return fail(RC_INVALID_VALUE, "cache strides must be multiples of 16 bytes and not negative");
    if (c->quant_group) {
        if (c->scale_page_stride < 0 || c->scale_head_stride < 0 || c->scale_token_stride < 0)
            return fail(RC_INVALID_VALUE, "negative scale stride");
        if (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 1) return fail(RC_INVALID_VALUE, "scales must be 2-byte aligned");
    }
    return RC_SUCCESS;
}

namespace {

constexpr int TPB = 256;

struct RotaryKvParams {
    const half *q, *k, *v;
    half *q_out, *k_out;
    const int64_t *positions, *slots;
    const uint64_t* turns;
    int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
    int32_t q_heads, k_heads, v_heads, head_dim, rotary_dim, interleaved;
    float magnitude;
    int32_t store; // keys go to the cache instead of k_out, values too
    pplb200_kv_cache cache;
};

union Eight {
    uint4 raw;
    __half2 h[4];
};

// Largest magnitude of eight halves as fp16 bits.  Compared as integers: a NaN is above infinity, so that it comes through.
__device__ __forceinline__ uint32_t absmax_bits(const uint4& a) {
    const uint32_t m = __vmaxu2(__vmaxu2(a.x & 0x7fff7fffu, a.y & 0x7fff7fffu), __vmaxu2(a.z & 0x7fff7fffu, a.w & 0x7fff7fffu));
    return max(m & 0xffffu, m >> 16);
}

// The scale of a group: amax / 127 rounded up to fp16 -- fp16 so that what is divided by is what is stored, up so that no quotient is
// beyond 127 steps, among the subnormal scales of very small groups too -- at least the smallest fp16 above zero, and for finite
// groups at most 515.5: with 516, 127 steps would read back as infinity.
__device__ __forceinline__ half group_scale(uint32_t amax) {
    const uint32_t s = __half_as_ushort(__float2half_ru(__fdiv_rn(__half2float(__ushort_as_half((unsigned short)amax)), 127.0f)));
    return __ushort_as_half((unsigned short)(amax < 0x7c00u ? min(max(s, 1u), 0x6007u) : s));
}

// The quotient in 32 bits, rounded to nearest even.  Its magnitude is at most 127.07 (65504 / 515.5); NaN, in a group with an infinity
// or a NaN in it, becomes 0, and is NaN again when it is multiplied by that group's scale.
__device__ __forceinline__ uint32_t quantize_one(float v, float scale) {
    return (uint32_t)__float2int_rn(__fdiv_rn(v, scale)) & 0xffu;
}
__device__ __forceinline__ uint2 quantize_eight(const Eight& e, float scale) {
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(e.h[i]);
        b[2 * i] = quantize_one(f.x, scale);
        b[2 * i + 1] = quantize_one(f.y, scale);
    }
    return make_uint2(b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24, b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24);
}

// One CTA turns the rows (heads of q, k and v) of one token, LANES threads a row, 16 dimensions a thread: two runs of eight that
// are rotated against each other (half layout: rotary_dim / 2 apart), so that nothing crosses threads but the scale of a whole head.
template <int LANES>
__global__ void __launch_bounds__(TPB) rotary_kv_kernel(const RotaryKvParams p) {
    __shared__ float2 turn[kMaxHeadDim / 2];
    pdl_wait_prior_grid();
    const int64_t token = blockIdx.x;
    const int planes = p.rotary_dim >> 1;
    if (planes > 0) {
        const uint64_t at = (uint64_t)p.positions[token];
        for (int i = threadIdx.x; i < planes; i += TPB) {
            // the angle modulo one turn, exactly, as a signed fraction; half turns for sincospi
            const float half_turns = (float)(int64_t)(at * p.turns[i]) * 0x1p-63f;
            float s, c;
            sincospif(half_turns, &s, &c);
            turn[i] = make_float2(c * p.magnitude, s * p.magnitude);
        }
        __syncthreads();
    }
    int64_t page = 0;
    int32_t in_page = 0;
    const bool stored = p.store && kv_find(p.slots[token], p.cache.num_pages, p.cache.page_size, page, in_page);

    const int u = threadIdx.x & (LANES - 1);
    const int rows = p.q_heads + p.k_heads + p.v_heads;
    const int per_cta = TPB / LANES;
    for (int row = blockIdx.y * per_cta + threadIdx.x / LANES; row < rows; row += gridDim.y * per_cta) {
        const bool is_q = row < p.q_heads, is_v = row >= p.q_heads + p.k_heads;
        const int head = is_q ? row : is_v ? row - p.q_heads - p.k_heads : row - p.q_heads;
        const half* src = is_q ? p.q + token * p.q_stride : is_v ? p.v + token * p.v_stride : p.k + token * p.k_stride;
        src += (int64_t)head * p.head_dim;
        const bool turned = !is_v && 16 * u < p.rotary_dim;
        const int da = turned && !p.interleaved ? 8 * u : 16 * u;
        const int db = turned && !p.interleaved ? planes + 8 * u : 16 * u + 8;
        const bool active = 16 * u < p.head_dim;
        Eight a = {}, b = {};
        if (active) {
            a.raw = ld_global_16(src + da);
            b.raw = ld_global_16(src + db);
        }
        if (turned) {
            if (!p.interleaved) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 x = __half22float2(a.h[i]), y = __half22float2(b.h[i]);
                    const float2 r0 = turn[8 * u + 2 * i], r1 = turn[8 * u + 2 * i + 1];
                    a.h[i] = __floats2half2_rn(x.x * r0.x - y.x * r0.y, x.y * r1.x - y.y * r1.y);
                    b.h[i] = __floats2half2_rn(y.x * r0.x + x.x * r0.y, y.y * r1.x + x.y * r1.y);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 x = __half22float2(a.h[i]), y = __half22float2(b.h[i]);
                    const float2 r0 = turn[8 * u + i], r1 = turn[8 * u + 4 + i];
                    a.h[i] = __floats2half2_rn(x.x * r0.x - x.y * r0.y, x.y * r0.x + x.x * r0.y);
                    b.h[i] = __floats2half2_rn(y.x * r1.x - y.y * r1.y, y.y * r1.x + y.x * r1.y);
                }
            }
        }
        if (is_q || !p.store) {
            half* dst = (is_q ? p.q_out + token * p.q_out_stride : p.k_out + token * p.k_out_stride) + (int64_t)head * p.head_dim;
            if (active) {
                *reinterpret_cast<uint4*>(dst + da) = a.raw;
                *reinterpret_cast<uint4*>(dst + db) = b.raw;
            }
            continue;
        }
        const int64_t at = kv_row(page, in_page, head, p.cache.page_stride, p.cache.head_stride, p.cache.token_stride);
        if (p.cache.quant_group == 0) {
            half* dst = (half*)(is_v ? p.cache.v : p.cache.k) + at;
            if (active && stored) {
                *reinterpret_cast<uint4*>(dst + da) = a.raw;
                *reinterpret_cast<uint4*>(dst + db) = b.raw;
            }
            continue;
        }
        uint32_t ma = absmax_bits(a.raw), mb = absmax_bits(b.raw);
        if (p.cache.quant_group != 8) {
            ma = max(ma, mb);
            const uint32_t row_mask = (LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1)) << (threadIdx.x & 31 & ~(LANES - 1));
#pragma unroll
            for (int m = LANES / 2; m >= 1; m >>= 1) ma = max(ma, __shfl_xor_sync(row_mask, ma, m));
            mb = ma;
        }
        if (active && stored) {
            const half sa = group_scale(ma), sb = group_scale(mb);
            int8_t* dst = (int8_t*)(is_v ? p.cache.v : p.cache.k) + at;
            *reinterpret_cast<uint2*>(dst + da) = quantize_eight(a, __half2float(sa));
            *reinterpret_cast<uint2*>(dst + db) = quantize_eight(b, __half2float(sb));
            half* scale = (half*)(is_v ? p.cache.v_scale : p.cache.k_scale) +
                          kv_row(page, in_page, head, p.cache.scale_page_stride, p.cache.scale_head_stride, p.cache.scale_token_stride);
            if (p.cache.quant_group == 8) {
                scale[da >> 3] = sa;
                scale[db >> 3] = sb;
            } else if (u == 0) {
                scale[0] = sa;
            }
        }
    }
}

int32_t launch_rotary_kv(cudaStream_t stream, int64_t tokens, const RotaryKvParams& p) {
    const int rows = p.q_heads + p.k_heads + p.v_heads;
    if (tokens == 0 || rows == 0) return RC_SUCCESS;
    const int lanes = p.head_dim <= 64 ? 4 : p.head_dim <= 128 ? 8 : 16;
    const int passes = (rows * lanes + TPB - 1) / TPB;
    // few tokens: every CTA makes one pass, so that the rows spread over more SMs
    const dim3 grid((unsigned)tokens, (unsigned)(tokens < 1024 ? passes : 1));
    if (lanes == 4) launch_ex(rotary_kv_kernel<4>, grid, dim3(TPB), stream, true, p);
    else if (lanes == 8) launch_ex(rotary_kv_kernel<8>, grid, dim3(TPB), stream, true, p);
    else launch_ex(rotary_kv_kernel<16>, grid, dim3(TPB), stream, true, p);
    return check_launch("rotary / cache write");
}

// One thread per eight dimensions of a key or value row.
__global__ void __launch_bounds__(TPB) kv_read_kernel(const pplb200_kv_cache c, const int64_t* slots, int64_t units, half* k_out, half* v_out) {
    pdl_wait_prior_grid();
    const int per_head = c.head_dim >> 3;
    const int64_t n = (int64_t)blockIdx.x * TPB + threadIdx.x;
    if (n >= units) return;
    const int64_t row = n / per_head;
    const int d = (int)(n - row * per_head) * 8;
    const int64_t token = row / c.kv_heads;
    const int head = (int)(row - token * c.kv_heads);
    int64_t page = 0;
    int32_t in_page = 0;
    const bool found = kv_find(slots[token], c.num_pages, c.page_size, page, in_page);
    const int64_t at = kv_row(page, in_page, head, c.page_stride, c.head_stride, c.token_stride) + d;
    const int64_t sat = kv_row(page, in_page, head, c.scale_page_stride, c.scale_head_stride, c.scale_token_stride) + (c.quant_group == 8 ? d >> 3 : 0);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        Eight e = {};
        if (found) {
            if (c.quant_group == 0) {
                e.raw = ld_global_16((const half*)(kv ? c.v : c.k) + at);
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>((const int8_t*)(kv ? c.v : c.k) + at);
                const float s = __half2float(ld_global_half((const half*)(kv ? c.v_scale : c.k_scale) + sat));
                const int8_t* b = reinterpret_cast<const int8_t*>(&w);
#pragma unroll
                for (int i = 0; i < 4; ++i) e.h[i] = __floats2half2_rn((float)b[2 * i] * s, (float)b[2 * i + 1] * s);
            }
        }
        *reinterpret_cast<uint4*>((kv ? v_out : k_out) + n * 8) = e.raw;
    }
}

int32_t check_rotary(int32_t rotary_dim, int32_t head_dim, const void* turns, const void* positions) {
    if (rotary_dim < 0 || rotary_dim % 16 || rotary_dim > head_dim)
        return fail(RC_INVALID_VALUE, "rotary_dim must be a multiple of 16 up to head_dim, got %d of %d", rotary_dim, head_dim);
    if (rotary_dim && (!turns || !positions)) return fail(RC_INVALID_VALUE, "null turns or positions");
    if ((((uintptr_t)turns | (uintptr_t)positions) & 7) != 0) return fail(RC_INVALID_VALUE, "turns and positions must be 8-byte aligned");
    return RC_SUCCESS;
}

// Rows of a [tokens, heads, head_dim] tensor; nothing is asked of one without heads.
int32_t check_rows(const char* name, const void* p, int64_t stride, int64_t heads, int64_t head_dim, int64_t tokens) {
    if (heads < 0 || heads > 65535) return fail(RC_INVALID_VALUE, "%s: bad number of heads: %lld", name, (long long)heads);
    if (heads == 0) return RC_SUCCESS;
    if (!p || !aligned16(p)) return fail(RC_INVALID_VALUE, "%s must be a 16-byte aligned pointer", name);
    if (stride % 8 || stride < 0 || (tokens > 1 && stride < heads * head_dim))
        return fail(RC_INVALID_VALUE, "%s: tokens must be a multiple of 8 elements apart, and no closer than a token is long (%lld)", name, (long long)stride);
    return RC_SUCCESS;
}

} // namespace
} // namespace pplb200

using namespace pplb200;

extern "C" {

int32_t pplb200_rotary_frequencies(int32_t rotary_dim, double base, int32_t scaling, double factor, double original_length,
                                   double keep_turns, double stretch_turns, uint64_t* turns_host, float* magnitude_host) {
    if (rotary_dim <= 0 || rotary_dim % 16 || rotary_dim > kMaxHeadDim)
        return fail(RC_INVALID_VALUE, "rotary_dim must be a multiple of 16 up to %d, got %d", kMaxHeadDim, rotary_dim);
    if (scaling < PPLB200_ROTARY_NONE || scaling > PPLB200_ROTARY_WAVELENGTH) return fail(RC_UNSUPPORTED, "unknown rotary scaling %d", scaling);
    if (!turns_host || !magnitude_host) return fail(RC_INVALID_VALUE, "null pointer");
    if (!(base > 1.0) || !std::isfinite(base)) return fail(RC_INVALID_VALUE, "the base must be above 1");
    if (scaling != PPLB200_ROTARY_NONE && (!(factor >= 1.0) || !std::isfinite(factor))) return fail(RC_INVALID_VALUE, "the factor must be at least 1");
    const bool blend = scaling == PPLB200_ROTARY_YARN || scaling == PPLB200_ROTARY_WAVELENGTH;
    if (blend && (!(original_length > 0.0) || !std::isfinite(original_length) || !(stretch_turns > 0.0) || !(keep_turns > stretch_turns) || !std::isfinite(keep_turns)))
        return fail(RC_INVALID_VALUE, "a blend needs original_length > 0 and keep_turns > stretch_turns > 0");
    const double two_pi = 6.283185307179586476925286766559;
    const double rd = rotary_dim;
    const double b = scaling == PPLB200_ROTARY_NTK ? base * std::pow(factor, rd / (rd - 2.0)) : base;
    // planes between which YARN blends: those that turn keep_turns and stretch_turns times within the original length
    double first = 0.0, last = 0.0;
    if (scaling == PPLB200_ROTARY_YARN) {
        first = std::fmax(std::floor(rd * std::log(original_length / (keep_turns * two_pi)) / (2.0 * std::log(base))), 0.0);
        last = std::fmin(std::ceil(rd * std::log(original_length / (stretch_turns * two_pi)) / (2.0 * std::log(base))), rd - 1.0);
    }
    for (int32_t i = 0; i < rotary_dim / 2; ++i) {
        double f = std::pow(b, -2.0 * i / rd);
        if (scaling == PPLB200_ROTARY_LINEAR) f /= factor;
        if (blend) {
            const double keep = scaling == PPLB200_ROTARY_YARN ? 1.0 - (i - first) / std::fmax(last - first, 0.001)
                                                               : (original_length * f / two_pi - stretch_turns) / (keep_turns - stretch_turns);
            const double part = std::fmin(std::fmax(keep, 0.0), 1.0);
            f = f * part + f / factor * (1.0 - part);
        }
        turns_host[i] = (uint64_t)std::floor(f / two_pi * 0x1p64 + 0.5); // f <= 1: below 2^62
    }
    *magnitude_host = scaling == PPLB200_ROTARY_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return RC_SUCCESS;
}

int32_t pplb200_rotary_fp16(pplb200_stream_t stream, const pplb200_rotary_args* a) {
    if (!a) return fail(RC_INVALID_VALUE, "null arguments");
    if (a->tokens < 0) return fail(RC_INVALID_VALUE, "negative extent");
    if (a->tokens > 0x7fffffffLL) return fail(RC_UNSUPPORTED, "more than 2^31 - 1 tokens");
    if (a->head_dim <= 0 || a->head_dim % 16 || a->head_dim > kMaxHeadDim)
        return fail(RC_UNSUPPORTED, "head_dim must be a multiple of 16 up to %d, got %d", kMaxHeadDim, a->head_dim);
    if (a->tokens == 0) return RC_SUCCESS;
    int32_t rc = check_rotary(a->rotary_dim, a->head_dim, a->turns, a->positions);
    if (rc == RC_SUCCESS) rc = check_rows("q", a->q, a->q_stride, a->q_heads, a->head_dim, a->tokens);
    if (rc == RC_SUCCESS) rc = check_rows("k", a->k, a->k_stride, a->k_heads, a->head_dim, a->tokens);
    if (rc == RC_SUCCESS) rc = check_rows("q_out", a->q_out, a->q_out_stride, a->q_heads, a->head_dim, a->tokens);
    if (rc == RC_SUCCESS) rc = check_rows("k_out", a->k_out, a->k_out_stride, a->k_heads, a->head_dim, a->tokens);
    if (rc != RC_SUCCESS) return rc;
    RotaryKvParams p = {};
    p.q = (const half*)a->q; p.k = (const half*)a->k;
    p.q_out = (half*)a->q_out; p.k_out = (half*)a->k_out;
    p.positions = a->positions; p.turns = a->turns;
    p.q_stride = a->q_stride; p.k_stride = a->k_stride;
    p.q_out_stride = a->q_out_stride; p.k_out_stride = a->k_out_stride;
    p.q_heads = a->q_heads; p.k_heads = a->k_heads;
    p.head_dim = a->head_dim; p.rotary_dim = a->rotary_dim; p.interleaved = a->interleaved;
    p.magnitude = a->magnitude;
    return launch_rotary_kv((cudaStream_t)stream, a->tokens, p);
}

int32_t pplb200_kv_cache_write_fp16(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_kv_write_args* a) {
    int32_t rc = check_kv_cache(cache);
    if (rc != RC_SUCCESS) return rc;
    if (!a) return fail(RC_INVALID_VALUE, "null arguments");
    if (a->tokens < 0) return fail(RC_INVALID_VALUE, "negative extent");
    if (a->tokens > 0x7fffffffLL) return fail(RC_UNSUPPORTED, "more than 2^31 - 1 tokens");
    if (a->tokens == 0) return RC_SUCCESS;
    if (!a->slots || ((uintptr_t)a->slots & 7)) return fail(RC_INVALID_VALUE, "slots must be an 8-byte aligned pointer");
    rc = check_rotary(a->rotary_dim, cache->head_dim, a->turns, a->positions);
    const int32_t q_heads = a->rotary_dim ? a->q_heads : 0;
    if (rc == RC_SUCCESS) rc = check_rows("q", a->q, a->q_stride, q_heads, cache->head_dim, a->tokens);
    if (rc == RC_SUCCESS) rc = check_rows("q_out", a->q_out, a->q_out_stride, q_heads, cache->head_dim, a->tokens);
    if (rc == RC_SUCCESS) rc = check_rows("k", a->k, a->k_stride, cache->kv_heads, cache->head_dim, a->tokens);
    if (rc == RC_SUCCESS) rc = check_rows("v", a->v, a->v_stride, cache->kv_heads, cache->head_dim, a->tokens);
    if (rc != RC_SUCCESS) return rc;
    RotaryKvParams p = {};
    p.q = (const half*)a->q; p.k = (const half*)a->k; p.v = (const half*)a->v;
    p.q_out = (half*)a->q_out;
    p.positions = a->positions; p.slots = a->slots; p.turns = a->turns;
    p.q_stride = a->q_stride; p.k_stride = a->k_stride; p.v_stride = a->v_stride; p.q_out_stride = a->q_out_stride;
    p.q_heads = q_heads; p.k_heads = p.v_heads = cache->kv_heads;
    p.head_dim = cache->head_dim; p.rotary_dim = a->rotary_dim; p.interleaved = a->interleaved;
    p.magnitude = a->magnitude;
    p.store = 1;
    p.cache = *cache;
    return launch_rotary_kv((cudaStream_t)stream, a->tokens, p);
}

int32_t pplb200_kv_cache_read_fp16(pplb200_stream_t stream, const pplb200_kv_cache* cache, const int64_t* slots, int64_t tokens,
                                   void* k_out, void* v_out) {
    const int32_t rc = check_kv_cache(cache);
    if (rc != RC_SUCCESS) return rc;
    if (tokens < 0) return fail(RC_INVALID_VALUE, "negative extent");
    if (tokens == 0) return RC_SUCCESS;
    if (!slots || ((uintptr_t)slots & 7)) return fail(RC_INVALID_VALUE, "slots must be an 8-byte aligned pointer");
    if (!k_out || !v_out || !aligned16(k_out) || !aligned16(v_out)) return fail(RC_INVALID_VALUE, "k_out and v_out must be 16-byte aligned pointers");
    if (tokens > (1LL << 38) / (cache->kv_heads * (int64_t)cache->head_dim)) return fail(RC_UNSUPPORTED, "too many elements");
    const int64_t units = tokens * cache->kv_heads * (cache->head_dim / 8);
    launch_ex(kv_read_kernel, dim3((unsigned)((units + TPB - 1) / TPB)), dim3(TPB), (cudaStream_t)stream, true, *cache, slots, units, (half*)k_out, (half*)v_out);
    return check_launch("cache read");
}

int64_t pplb200_kv_cache_offset(const pplb200_kv_cache* c, int64_t slot, int32_t head) {
    int64_t page;
    int32_t in_page;
    if (check_kv_cache(c) != RC_SUCCESS || head < 0 || head >= c->kv_heads || !kv_find(slot, c->num_pages, c->page_size, page, in_page)) return -1;
    return kv_row(page, in_page, head, c->page_stride, c->head_stride, c->token_stride);
}

} // extern "C"
