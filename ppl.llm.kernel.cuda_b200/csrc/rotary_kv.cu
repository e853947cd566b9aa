// Rotary positions, and the paged key-value cache written and read back.
#include "kv_cache.cuh"
#include "quotient.cuh"

#include <algorithm>
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
    // offsets, in bytes too, fit 64 bits
    const auto last = [&](int64_t page, int64_t head, int64_t token) {
        return (__int128)(c->num_pages - 1) * page + (__int128)(c->kv_heads - 1) * head + (__int128)(c->page_size - 1) * token + c->head_dim;
    };
    if (last(c->page_stride, c->head_stride, c->token_stride) >> 61 ||
        (c->quant_group && last(c->scale_page_stride, c->scale_head_stride, c->scale_token_stride) >> 61))
        return fail(RC_INVALID_VALUE, "a cache whose elements lie 2^61 apart");
    return RC_SUCCESS;
}

namespace {

constexpr int TPB = 256; // reading back

enum : int { Q = 0, K = 1, V = 2 };

struct RotaryKvParams {
    const half* src[3];
    half* dst[2];
    int64_t src_stride[3], dst_stride[2];
    int32_t heads[3], turns_of[3]; // rows of a token, and how many of them a thread takes at most
    const int64_t *positions, *slots;
    const uint64_t* turns;
    const uint8_t* axis_of_plane; // axes > 0: positions of several axes, axis_stride apart
    int64_t axis_stride;
    int64_t tokens;
    int32_t head_dim, rotary_dim, interleaved, axes;
    float magnitude;
    int32_t store; // keys go to the cache instead of dst[K], values too
    int32_t groups;                    // threads that share a token's rows, for each 16 dimensions
    uint32_t group_magic, group_shift; // n / groups = n * group_magic >> group_shift
    pplb200_kv_cache cache;
};

// Largest magnitude of eight halves as fp16 bits; a NaN comes through.
__device__ __forceinline__ uint32_t absmax_bits(const Eight& e) {
    const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(e.h[0]), __habs2(e.h[1])), __hmax2_nan(__habs2(e.h[2]), __habs2(e.h[3])));
    const uint32_t bits = *reinterpret_cast<const uint32_t*>(&m);
    return max(bits & 0xffffu, bits >> 16);
}

// The scale of a group: amax / 127 rounded up to fp16 -- fp16 so that what is divided by is what is stored, up so that no quotient is
// beyond 127 steps, among the subnormal scales of very small groups too -- at least the smallest fp16 above zero, and for finite
// groups at most 515.5: with 516, 127 steps would read back as infinity.
// The quotient: a product with the reciprocal, corrected by what it leaves of amax.  That is exact where amax / 127 is an fp16, and
// off by less than 2^-22 otherwise, when amax / 127 lies 2^-18 or more of its size from any fp16 (amax has 11 bits, 127 times an fp16 18).
__device__ __forceinline__ half group_scale(uint32_t amax) {
    const float a = __half2float(__ushort_as_half((unsigned short)amax)), guess = a * (1.0f / 127.0f);
    const float step = __fmaf_rn(__fmaf_rn(-127.0f, guess, a), 1.0f / 127.0f, guess);
    const uint32_t s = __half_as_ushort(__float2half_ru(step));
    return __ushort_as_half((unsigned short)(amax < 0x7c00u ? min(max(s, 1u), 0x6007u) : amax));
}

// Cosines and sines (times the magnitude) of four and four planes: the angle modulo one turn, exactly, as a signed fraction, in half turns.
struct Turns {
    float c[8], s[8];
};
__device__ __forceinline__ void turns_at(Turns& t, uint64_t position, const uint64_t* first, const uint64_t* second, float magnitude) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        sincospif((float)(int64_t)(position * (i < 4 ? first[i] : second[i - 4])) * 0x1p-63f, &t.s[i], &t.c[i]);
        t.c[i] *= magnitude;
        t.s[i] *= magnitude;
    }
}
// The same where each plane has an axis, and the token a position on each, which lie in shared memory: a plane's is one load (chosen by selections
// among registers, 8192 tokens of 64 heads took 49 us where they take 43 with one axis).
struct AxisPositions {
    const uint64_t* at;     // [PPLB200_ROTARY_MAX_AXES]
    uint32_t first, second; // axes of four and four planes
    __device__ __forceinline__ uint64_t of(int i) const { return at[(i < 4 ? first : second) >> (8 * (i & 3)) & 3u]; }
};
__device__ __forceinline__ void turns_at(Turns& t, const AxisPositions& position, const uint64_t* first, const uint64_t* second, float magnitude) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        sincospif((float)(int64_t)(position.of(i) * (i < 4 ? first[i] : second[i - 4])) * 0x1p-63f, &t.s[i], &t.c[i]);
        t.c[i] *= magnitude;
        t.s[i] *= magnitude;
    }
}
// a and b against each other, or (interleaved) neighbours within a and within b.
__device__ __forceinline__ void rotate(Eight& a, Eight& b, const Turns& t, bool interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = __half22float2(a.h[i]), y = __half22float2(b.h[i]);
        if (!interleaved) {
            a.h[i] = __floats2half2_rn(x.x * t.c[2 * i] - y.x * t.s[2 * i], x.y * t.c[2 * i + 1] - y.y * t.s[2 * i + 1]);
            b.h[i] = __floats2half2_rn(y.x * t.c[2 * i] + x.x * t.s[2 * i], y.y * t.c[2 * i + 1] + x.y * t.s[2 * i + 1]);
        } else {
            a.h[i] = __floats2half2_rn(x.x * t.c[i] - x.y * t.s[i], x.y * t.c[i] + x.x * t.s[i]);
            b.h[i] = __floats2half2_rn(y.x * t.c[4 + i] - y.y * t.s[4 + i], y.y * t.c[4 + i] + y.x * t.s[4 + i]);
        }
    }
}

// A thread has 16 dimensions of a token: two runs of eight that are rotated against each other (half layout) or each in itself, so that
// nothing crosses threads but the scale of a whole head; neighbouring threads have neighbouring runs, so that loads and stores fill lines.  It computes their eight sines and cosines once, while its
// first rows are on their way, and takes every groups-th head of q, k and v with them; LANES threads side by side make a row.
// Threads without dimensions or tokens of their own, and turns without a head, read another's row and store nothing: no load waits for
// a branch.
constexpr int RTPB = 128;
enum : int { AS_IS = 0, HALVES = 1, INTERLEAVED = 2 }; // what is rotated against what; AS_IS keeps sixteen registers free
enum : int { NO_STORE = 0, STORE_F16 = 1, STORE_I8_GROUPS = 2, STORE_I8_ROWS = 3 };
template <int LANES, int LAYOUT, int STORE, bool AXES>
struct RotaryKv {
    struct Row {
        Eight a, b;
    };
    const RotaryKvParams& p;
    int64_t token;
    int u, da, db; // the thread's number in its row, and where its runs begin
    bool active, turned; // whether the thread has dimensions, and whether they are rotated
    Turns turns;
    int64_t at, scale_at; // in the cache; at < 0: not stored

    template <int KIND>
    __device__ __forceinline__ void fetch(int head, Row& x) const {
        const half* src = p.src[KIND] + token * p.src_stride[KIND] + (int64_t)min(head, p.heads[KIND] - 1) * p.head_dim;
        x.a.raw = ld_global_16(src + da);
        x.b.raw = ld_global_16(src + db);
    }
    // Called by all threads of a warp.
    template <int KIND>
    __device__ __forceinline__ void finish(int head, Row& x) const {
        if (KIND != V && LAYOUT != AS_IS && turned) rotate(x.a, x.b, turns, LAYOUT == INTERLEAVED);
        const bool there = active && head < p.heads[KIND];
        if constexpr (STORE == NO_STORE || KIND == Q) {
            half* dst = p.dst[KIND] + token * p.dst_stride[KIND] + (int64_t)head * p.head_dim;
            if (there) {
                *reinterpret_cast<uint4*>(dst + da) = x.a.raw;
                *reinterpret_cast<uint4*>(dst + db) = x.b.raw;
            }
        } else {
            const int64_t row = at + (int64_t)head * p.cache.head_stride;
            void* const data = KIND == V ? p.cache.v : p.cache.k;
            const bool stored = there && at >= 0;
            if constexpr (STORE == STORE_F16) {
                if (stored) {
                    *reinterpret_cast<uint4*>((half*)data + row + da) = x.a.raw;
                    *reinterpret_cast<uint4*>((half*)data + row + db) = x.b.raw;
                }
            } else {
                int8_t* const dst = (int8_t*)data + row;
                half* const scale = (half*)(KIND == V ? p.cache.v_scale : p.cache.k_scale) + scale_at + (int64_t)head * p.cache.scale_head_stride;
                uint32_t ma = absmax_bits(x.a), mb = absmax_bits(x.b);
                if constexpr (STORE == STORE_I8_ROWS) {
                    ma = active ? max(ma, mb) : 0u;
#pragma unroll
                    for (int m = LANES / 2; m >= 1; m >>= 1) ma = max(ma, __shfl_xor_sync(0xffffffffu, ma, m));
                    const half s = group_scale(ma);
                    const Quotient by(s);
                    const uint2 qa = by.eight(x.a), qb = by.eight(x.b);
                    if (stored) {
                        *reinterpret_cast<uint2*>(dst + da) = qa;
                        *reinterpret_cast<uint2*>(dst + db) = qb;
                        if (u == 0) scale[0] = s;
                    }
                } else {
                    const half sa = group_scale(ma), sb = group_scale(mb);
                    const uint2 qa = Quotient(sa).eight(x.a), qb = Quotient(sb).eight(x.b);
                    if (stored) {
                        *reinterpret_cast<uint2*>(dst + da) = qa;
                        *reinterpret_cast<uint2*>(dst + db) = qb;
                        scale[da >> 3] = sa;
                        scale[db >> 3] = sb;
                    }
                }
            }
        }
    }
    // Rows behind the first, two at a time: of one tensor, or, where there is no q to go through, a key's and the value's beside it.
    template <int KIND>
    __device__ __forceinline__ void others(int group) const {
        for (int i = 1; i < p.turns_of[KIND]; i += 2) {
            Row x, y;
            fetch<KIND>(group + i * p.groups, x);
            fetch<KIND>(group + (i + 1) * p.groups, y);
            finish<KIND>(group + i * p.groups, x);
            if (i + 1 < p.turns_of[KIND]) finish<KIND>(group + (i + 1) * p.groups, y);
        }
    }
    __device__ __forceinline__ void other_pairs(int group) const {
        for (int i = 1; i < p.turns_of[K]; ++i) {
            Row x, y;
            fetch<K>(group + i * p.groups, x);
            fetch<V>(group + i * p.groups, y);
            finish<K>(group + i * p.groups, x);
            finish<V>(group + i * p.groups, y);
        }
    }
};

// Bound by HBM where nothing is quantized: 8192 tokens of 64 + 8 heads of 128 rotated 47 us, 97 % of a copy's rate; stored as fp16 too, 57 us,
// 91 %.  Quantizing costs some 200 instructions for 16 elements of 32 lanes, which shows: 16384 tokens of 8 + 8 heads 22.4 us, 69 % (29 with
// branches around the loads, keys and values one after the other and a run-time choice of the cache's type).  CTAs that share an
// SM were tried from 5 to 10 (at the bounds taken, the forms that store int8 rows spill 8 to 16 bytes): unrotated, 10 spill more (24.4 us), 6 take as long as 8 but 8.9 instead of 8.2 us for 4096 tokens in groups of 8; rotated, into groups of 8,
// 2048 tokens of 32 + 32 heads, 22.6 us with 7, 24 with 6.
template <int LANES, int LAYOUT, int STORE, bool AXES>
__global__ void __launch_bounds__(RTPB, LAYOUT == AS_IS ? 8 : 7) rotary_kv_kernel(const __grid_constant__ RotaryKvParams p) {
    pdl_wait_prior_grid();
    const uint32_t n = blockIdx.x * (RTPB / LANES) + threadIdx.x / LANES;
    RotaryKv<LANES, LAYOUT, STORE, AXES> r{p};
    r.token = (uint32_t)((uint64_t)n * p.group_magic >> p.group_shift);
    const int group = n - (uint32_t)r.token * p.groups;
    const bool valid = r.token < p.tokens;
    if (!valid) r.token = 0;
    r.u = threadIdx.x & (LANES - 1);
    r.active = valid && 16 * r.u < p.head_dim;
    r.turned = valid && 16 * r.u < p.rotary_dim;
    // runs of the rotated part lie half of it apart, those behind it half of the rest
    const int behind = r.u - (p.rotary_dim >> 4);
    r.da = behind < 0 ? 8 * r.u : p.rotary_dim + 8 * behind;
    r.db = r.da + ((behind < 0 ? p.rotary_dim : p.head_dim - p.rotary_dim) >> 1);
    if (!r.active) r.da = 0, r.db = 0;
    typename RotaryKv<LANES, LAYOUT, STORE, AXES>::Row q, k, v;
    if (p.turns_of[Q] > 0) r.template fetch<Q>(group, q);
    if (p.turns_of[K] > 0) r.template fetch<K>(group, k);
    if (STORE) r.template fetch<V>(group, v);
    __shared__ uint64_t axis_positions[AXES ? RTPB / LANES : 1][PPLB200_ROTARY_MAX_AXES];
    if constexpr (AXES) { // the LANES threads of a row, which lie in one warp, bring a position each
        static_assert(LANES >= PPLB200_ROTARY_MAX_AXES);
        if (r.u < PPLB200_ROTARY_MAX_AXES) axis_positions[threadIdx.x / LANES][r.u] = (uint64_t)p.positions[min(r.u, p.axes - 1) * p.axis_stride + r.token];
        __syncwarp();
    }
    if (LAYOUT != AS_IS && r.turned) {
        const uint64_t* first = p.turns + (LAYOUT == INTERLEAVED ? 4 : 8) * r.u; // planes of the runs: eight of both, or four of each
        const int apart = LAYOUT == INTERLEAVED ? p.rotary_dim >> 2 : 4;
        if constexpr (AXES) {
            const uint8_t* axis = p.axis_of_plane + (first - p.turns);
            const AxisPositions at = {axis_positions[threadIdx.x / LANES], *reinterpret_cast<const uint32_t*>(axis), *reinterpret_cast<const uint32_t*>(axis + apart)};
            turns_at(r.turns, at, first, first + apart, p.magnitude);
        } else {
            turns_at(r.turns, (uint64_t)p.positions[r.token], first, first + apart, p.magnitude);
        }
    }
    r.at = -1;
    r.scale_at = 0;
    if (STORE && valid) {
        int64_t page;
        int32_t in_page;
        if (kv_find(p.slots[r.token], p.cache.num_pages, p.cache.page_size, page, in_page)) {
            r.at = kv_row(page, in_page, 0, p.cache.page_stride, 0, p.cache.token_stride);
            r.scale_at = kv_row(page, in_page, 0, p.cache.scale_page_stride, 0, p.cache.scale_token_stride);
        }
    }
    if (p.turns_of[Q] > 0) r.template finish<Q>(group, q);
    if (p.turns_of[K] > 0) r.template finish<K>(group, k);
    if (STORE) r.template finish<V>(group, v);
    r.template others<Q>(group);
    if (LAYOUT == AS_IS) {
        r.other_pairs(group);
    } else {
        r.template others<K>(group);
        if (STORE) r.template others<V>(group);
    }
}

template <int LANES, int STORE>
void launch_stored(cudaStream_t stream, const RotaryKvParams& p, dim3 grid) {
    if (p.rotary_dim == 0 && STORE != NO_STORE) launch_ex(rotary_kv_kernel<LANES, STORE != NO_STORE ? AS_IS : HALVES, STORE, false>, grid, dim3(RTPB), stream, true, p);
    else if (p.interleaved) launch_ex(p.axes ? rotary_kv_kernel<LANES, INTERLEAVED, STORE, true> : rotary_kv_kernel<LANES, INTERLEAVED, STORE, false>, grid, dim3(RTPB), stream, true, p);
    else launch_ex(p.axes ? rotary_kv_kernel<LANES, HALVES, STORE, true> : rotary_kv_kernel<LANES, HALVES, STORE, false>, grid, dim3(RTPB), stream, true, p);
}
template <int LANES>
int32_t launch_lanes(cudaStream_t stream, RotaryKvParams& p) {
    // Heads a thread: as many as spread the sines over enough of them, while the device stays full.
    const int32_t most = std::max(p.heads[Q], std::max(p.heads[K], p.heads[V]));
    int64_t heads = std::min<int64_t>(4, std::max<int64_t>(1, p.tokens * most * LANES / (148LL * 1024 * 2)));
    if (heads > 2 && most % heads && most % (heads - 1) == 0) --heads; // no turns without a head
    p.groups = (int32_t)std::min<int64_t>((most + heads - 1) / heads, std::max<int64_t>(1, 0x7fff0000LL / p.tokens));
    for (int k = 0; k < 3; ++k) p.turns_of[k] = (p.heads[k] + p.groups - 1) / p.groups;
    small_division(p.groups, p.group_magic, p.group_shift);
    const dim3 grid((unsigned)((p.tokens * p.groups + RTPB / LANES - 1) / (RTPB / LANES)));
    if (!p.store) launch_stored<LANES, NO_STORE>(stream, p, grid);
    else if (p.cache.quant_group == 0) launch_stored<LANES, STORE_F16>(stream, p, grid);
    else if (p.cache.quant_group == 8) launch_stored<LANES, STORE_I8_GROUPS>(stream, p, grid);
    else launch_stored<LANES, STORE_I8_ROWS>(stream, p, grid);
    return check_launch("rotary / cache write");
}
int32_t launch_rotary_kv(cudaStream_t stream, RotaryKvParams& p) {
    if (p.tokens == 0 || p.heads[Q] + p.heads[K] + p.heads[V] == 0) return RC_SUCCESS;
    return p.head_dim <= 64 ? launch_lanes<4>(stream, p) : p.head_dim <= 128 ? launch_lanes<8>(stream, p) : launch_lanes<16>(stream, p);
}

// Eight dimensions of a key and of the value beside it are a unit, so that a warp's stores fill whole lines.  A block looks up once
// where its tokens lie (look-ups by every thread: 207 instructions a unit, 32768 tokens 42 us) and then goes through their units.
// Bound by HBM: 32768 tokens of 8 + 8 heads of 128 from int8 with a scale for every 8, scattered over pages of 16, 38.3 us, 87 % of a copy's rate.
constexpr int UNITS = 4; // a thread
struct KvReadParams {
    pplb200_kv_cache cache;
    const int64_t* slots;
    half *k_out, *v_out;
    int64_t tokens;
    int32_t units, tokens_here; // units of a token, tokens of a block
    uint32_t units_magic, units_shift, head_magic, head_shift;
};
// Bytes 0 to 3 of a word times a scale: whole numbers as halves (a byte with its sign flipped beneath 0x64 is 1152 + value), one rounding.
__device__ __forceinline__ void scaled(uint32_t w, __half2 s, __half2& lo, __half2& hi) {
    w ^= 0x80808080u;
    const __half2 offset = __float2half2_rn(1152.0f);
    uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    lo = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&a), offset), s);
    hi = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&b), offset), s);
}
__device__ __forceinline__ uint2 ld_global_8(const void* p) {
    uint2 v;
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
template <bool INT8>
__global__ void __launch_bounds__(TPB) kv_read_kernel(const __grid_constant__ KvReadParams p) {
    struct Row {
        int64_t at, scale_at; // at < 0: not in the cache
    };
    __shared__ Row where[TPB];
    const pplb200_kv_cache& c = p.cache;
    pdl_wait_prior_grid();
    const int64_t token0 = (int64_t)blockIdx.x * p.tokens_here;
    const int tokens = (int)min((int64_t)p.tokens_here, p.tokens - token0), all = tokens * p.units, per_head = c.head_dim >> 3;
    if (threadIdx.x < tokens) {
        Row w = {-1, 0};
        int64_t page;
        int32_t in_page;
        if (kv_find(p.slots[token0 + threadIdx.x], c.num_pages, c.page_size, page, in_page)) {
            w.at = kv_row(page, in_page, 0, c.page_stride, 0, c.token_stride);
            w.scale_at = kv_row(page, in_page, 0, c.scale_page_stride, 0, c.scale_token_stride);
        }
        where[threadIdx.x] = w;
    }
    __syncthreads();
#pragma unroll 2
    for (int n = blockIdx.y * TPB + threadIdx.x; n < all; n += gridDim.y * TPB) {
        const uint32_t local = (uint32_t)((uint64_t)(uint32_t)n * p.units_magic >> p.units_shift), unit = n - local * p.units;
        const uint32_t head = (uint32_t)((uint64_t)unit * p.head_magic >> p.head_shift), d = (unit - head * per_head) * 8;
        const Row w = where[local];
        const bool found = w.at >= 0;
        const int64_t at = w.at + head * c.head_stride + d, scale_at = w.scale_at + head * c.scale_head_stride + (c.quant_group == 8 ? d >> 3 : 0);
        Eight o[2];
        uint2 q[2];
        half s[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            if constexpr (INT8) {
                q[x] = found ? ld_global_8((const int8_t*)(x ? c.v : c.k) + at) : make_uint2(0, 0);
                s[x] = found ? ld_global_half((const half*)(x ? c.v_scale : c.k_scale) + scale_at) : __ushort_as_half(0);
            } else {
                o[x].raw = found ? ld_global_16((const half*)(x ? c.v : c.k) + at) : make_uint4(0, 0, 0, 0);
            }
        }
        const int64_t out = (token0 * p.units + n) * 8;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            if constexpr (INT8) {
                const __half2 s2 = __half2half2(s[x]);
                scaled(q[x].x, s2, o[x].h[0], o[x].h[1]);
                scaled(q[x].y, s2, o[x].h[2], o[x].h[3]);
            }
            *reinterpret_cast<uint4*>((x ? p.v_out : p.k_out) + out) = o[x].raw;
        }
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

// What is wrong with a scaling, or RC_SUCCESS.
int32_t check_scaling(int32_t rotary_dim, double base, int32_t scaling, double factor, double original_length, double keep_turns, double stretch_turns) {
    if (rotary_dim <= 0 || rotary_dim % 16 || rotary_dim > kMaxHeadDim)
        return fail(RC_INVALID_VALUE, "rotary_dim must be a multiple of 16 up to %d, got %d", kMaxHeadDim, rotary_dim);
    if (scaling < PPLB200_ROTARY_NONE || scaling > PPLB200_ROTARY_WAVELENGTH) return fail(RC_UNSUPPORTED, "unknown rotary scaling %d", scaling);
    if (!(base > 1.0) || !std::isfinite(base)) return fail(RC_INVALID_VALUE, "the base must be above 1");
    if (scaling != PPLB200_ROTARY_NONE && (!(factor >= 1.0) || !std::isfinite(factor))) return fail(RC_INVALID_VALUE, "the factor must be at least 1");
    const bool blend = scaling == PPLB200_ROTARY_YARN || scaling == PPLB200_ROTARY_WAVELENGTH;
    if (blend && (!(original_length > 0.0) || !std::isfinite(original_length) || !(stretch_turns > 0.0) || !(keep_turns > stretch_turns) || !std::isfinite(keep_turns)))
        return fail(RC_INVALID_VALUE, "a blend needs original_length > 0 and keep_turns > stretch_turns > 0");
    return RC_SUCCESS;
}

// The words of a scaling that has been checked: put(i, word) for each of rotary_dim / 2 planes; returns the factor on the values.
// The frequencies in 64-bit mantissas (long double): a word is off by a few of its units, and an angle by that times the position.
template <class Put>
float turn_words(int32_t rotary_dim, double base, int32_t scaling, double factor, double original_length, double keep_turns, double stretch_turns, Put put) {
    const bool blend = scaling == PPLB200_ROTARY_YARN || scaling == PPLB200_ROTARY_WAVELENGTH;
    const long double two_pi = 6.283185307179586476925286766559005768L, ld_base = base, ld_factor = factor;
    const double rd = rotary_dim, turn = (double)two_pi;
    const long double b = scaling == PPLB200_ROTARY_NTK ? ld_base * std::pow(ld_factor, (long double)rd / (rd - 2.0)) : ld_base;
    // planes between which YARN blends: those that turn keep_turns and stretch_turns times within the original length
    double first = 0.0, last = 0.0;
    if (scaling == PPLB200_ROTARY_YARN) {
        first = std::fmax(std::floor(rd * std::log(original_length / (keep_turns * turn)) / (2.0 * std::log(base))), 0.0);
        last = std::fmin(std::ceil(rd * std::log(original_length / (stretch_turns * turn)) / (2.0 * std::log(base))), rd - 1.0);
    }
    for (int32_t i = 0; i < rotary_dim / 2; ++i) {
        long double f = i ? std::pow(b, -2.0L * i / rd) : 1.0L;
        if (scaling == PPLB200_ROTARY_LINEAR) f /= ld_factor;
        if (blend) {
            const long double keep = scaling == PPLB200_ROTARY_YARN ? 1.0L - (i - first) / (long double)std::fmax(last - first, 0.001)
                                                                    : (original_length * f / two_pi - stretch_turns) / ((long double)keep_turns - stretch_turns);
            const long double part = std::fmin(std::fmax(keep, 0.0L), 1.0L);
            f = f * part + f / ld_factor * (1.0L - part);
        }
        put(i, (uint64_t)std::floor(f / two_pi * 0x1p64L + 0.5L)); // f <= 1: below 2^62
    }
    return scaling == PPLB200_ROTARY_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
}

// RC_SUCCESS, with the axes in p, or what is wrong with them.
int32_t take_axes(const pplb200_rotary_axes* axes, int64_t tokens, RotaryKvParams& p) {
    if (!axes) return fail(RC_INVALID_VALUE, "null axes");
    if (axes->axes < 1 || axes->axes > PPLB200_ROTARY_MAX_AXES) return fail(RC_UNSUPPORTED, "1 to %d axes, got %d", PPLB200_ROTARY_MAX_AXES, axes->axes);
    if (!axes->axis_of_plane || ((uintptr_t)axes->axis_of_plane & 3)) return fail(RC_INVALID_VALUE, "axis_of_plane must be a 4-byte aligned pointer");
    if (axes->axis_stride < 0 || (axes->axes > 1 && axes->axis_stride > 0 && axes->axis_stride < tokens)) // 0: all axes have the same, as text among images has
        return fail(RC_INVALID_VALUE, "the positions of the axes overlap in part");
    p.axis_of_plane = axes->axis_of_plane;
    p.axis_stride = axes->axis_stride;
    p.axes = axes->axes;
    return RC_SUCCESS;
}

int32_t rotary_call(pplb200_stream_t stream, const pplb200_rotary_args* a, const pplb200_rotary_axes* axes, bool several) {
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
    if (several && (rc = take_axes(axes, a->tokens, p)) != RC_SUCCESS) return rc;
    p.src[0] = (const half*)a->q; p.src[1] = (const half*)a->k;
    p.dst[0] = (half*)a->q_out; p.dst[1] = (half*)a->k_out;
    p.src_stride[0] = a->q_stride; p.src_stride[1] = a->k_stride;
    p.dst_stride[0] = a->q_out_stride; p.dst_stride[1] = a->k_out_stride;
    p.heads[Q] = a->q_heads; p.heads[K] = a->k_heads;
    p.tokens = a->tokens; p.positions = a->positions; p.turns = a->turns;
    p.head_dim = a->head_dim; p.rotary_dim = a->rotary_dim; p.interleaved = a->interleaved;
    p.magnitude = a->magnitude;
    return launch_rotary_kv((cudaStream_t)stream, p);
}

int32_t write_call(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_kv_write_args* a, const pplb200_rotary_axes* axes, bool several) {
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
    if (several && (rc = take_axes(axes, a->tokens, p)) != RC_SUCCESS) return rc;
    if (several && !a->rotary_dim) return fail(RC_INVALID_VALUE, "axes without rotary_dim");
    p.src[0] = (const half*)a->q; p.src[1] = (const half*)a->k; p.src[2] = (const half*)a->v;
    p.dst[0] = (half*)a->q_out;
    p.src_stride[0] = a->q_stride; p.src_stride[1] = a->k_stride; p.src_stride[2] = a->v_stride;
    p.dst_stride[0] = a->q_out_stride;
    p.heads[Q] = q_heads; p.heads[K] = p.heads[V] = cache->kv_heads;
    p.tokens = a->tokens; p.positions = a->positions; p.slots = a->slots; p.turns = a->turns;
    p.head_dim = cache->head_dim; p.rotary_dim = a->rotary_dim; p.interleaved = a->interleaved;
    p.magnitude = a->magnitude;
    p.store = 1;
    p.cache = *cache;
    return launch_rotary_kv((cudaStream_t)stream, p);
}

} // namespace
} // namespace pplb200

using namespace pplb200;

extern "C" {

int32_t pplb200_rotary_frequencies(int32_t rotary_dim, double base, int32_t scaling, double factor, double original_length,
                                   double keep_turns, double stretch_turns, uint64_t* turns_host, float* magnitude_host) {
    const int32_t rc = check_scaling(rotary_dim, base, scaling, factor, original_length, keep_turns, stretch_turns);
    if (rc != RC_SUCCESS) return rc;
    if (!turns_host || !magnitude_host) return fail(RC_INVALID_VALUE, "null pointer");
    *magnitude_host = turn_words(rotary_dim, base, scaling, factor, original_length, keep_turns, stretch_turns, [&](int32_t i, uint64_t word) { turns_host[i] = word; });
    return RC_SUCCESS;
}

int32_t pplb200_rotary_axes_frequencies(int32_t rotary_dim, double base, int32_t scaling, double factor, double original_length,
                                        double keep_turns, double stretch_turns, int32_t axes, const int32_t* planes_host, int32_t alternating,
                                        int32_t restart, uint64_t* turns_host, uint8_t* axis_of_plane_host, float* magnitude_host) {
    const int32_t rc = check_scaling(rotary_dim, base, scaling, factor, original_length, keep_turns, stretch_turns);
    if (rc != RC_SUCCESS) return rc;
    if (!planes_host || !turns_host || !axis_of_plane_host || !magnitude_host) return fail(RC_INVALID_VALUE, "null pointer");
    if (axes < 1 || axes > PPLB200_ROTARY_MAX_AXES) return fail(RC_UNSUPPORTED, "1 to %d axes, got %d", PPLB200_ROTARY_MAX_AXES, axes);
    const int32_t planes = rotary_dim / 2;
    int64_t together = 0;
    for (int32_t a = 0; a < axes; ++a) {
        if (planes_host[a] < 0) return fail(RC_INVALID_VALUE, "axis %d has %d planes", a, planes_host[a]);
        together += planes_host[a];
    }
    if (together != planes) return fail(RC_INVALID_VALUE, "the axes have %lld planes together, of %d", (long long)together, planes);
    int32_t left[PPLB200_ROTARY_MAX_AXES] = {}, at = 0;
    for (int32_t a = 0; a < axes; ++a) left[a] = planes_host[a];
    while (at < planes)
        for (int32_t a = 0; a < axes; ++a)
            for (int32_t n = alternating ? std::min(left[a], 1) : left[a]; n > 0; --n, --left[a]) axis_of_plane_host[at++] = (uint8_t)a;
    if (!restart) {
        *magnitude_host = turn_words(rotary_dim, base, scaling, factor, original_length, keep_turns, stretch_turns, [&](int32_t i, uint64_t word) { turns_host[i] = word; });
        return RC_SUCCESS;
    }
    for (int32_t a = 0; a < axes; ++a) {
        int32_t next = 0; // planes of the axis come in order
        *magnitude_host = turn_words(2 * planes_host[a], base, scaling, factor, original_length, keep_turns, stretch_turns, [&](int32_t, uint64_t word) {
            while (axis_of_plane_host[next] != a) ++next;
            turns_host[next++] = word;
        });
    }
    return RC_SUCCESS;
}

int32_t pplb200_rotary_fp16(pplb200_stream_t stream, const pplb200_rotary_args* args) { return rotary_call(stream, args, nullptr, false); }
int32_t pplb200_rotary_axes_fp16(pplb200_stream_t stream, const pplb200_rotary_args* args, const pplb200_rotary_axes* axes) {
    return rotary_call(stream, args, axes, true);
}
int32_t pplb200_kv_cache_write_fp16(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_kv_write_args* args) {
    return write_call(stream, cache, args, nullptr, false);
}
int32_t pplb200_kv_cache_write_axes_fp16(pplb200_stream_t stream, const pplb200_kv_cache* cache, const pplb200_kv_write_args* args, const pplb200_rotary_axes* axes) {
    return write_call(stream, cache, args, axes, true);
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
    KvReadParams p = {};
    p.cache = *cache;
    p.slots = slots; p.tokens = tokens;
    p.k_out = (half*)k_out; p.v_out = (half*)v_out;
    p.units = cache->kv_heads * (cache->head_dim / 8);
    // few tokens: fewer units a thread, so that there are blocks for all SMs
    const int64_t each = std::min<int64_t>(UNITS, std::max<int64_t>(1, tokens * p.units / (TPB * 1184LL)));
    p.tokens_here = (int32_t)std::min<int64_t>(TPB, std::max<int64_t>(1, TPB * each / p.units));
    const int64_t shares = std::min<int64_t>((p.units + TPB * each - 1) / (TPB * each), 65535);
    small_division(p.units, p.units_magic, p.units_shift);
    small_division(cache->head_dim / 8, p.head_magic, p.head_shift);
    const dim3 grid((unsigned)((tokens + p.tokens_here - 1) / p.tokens_here), (unsigned)shares);
    if (cache->quant_group) launch_ex(kv_read_kernel<true>, grid, dim3(TPB), (cudaStream_t)stream, true, p);
    else launch_ex(kv_read_kernel<false>, grid, dim3(TPB), (cudaStream_t)stream, true, p);
    return check_launch("cache read");
}

int64_t pplb200_kv_cache_offset(const pplb200_kv_cache* c, int64_t slot, int32_t head) {
    int64_t page;
    int32_t in_page;
    if (check_kv_cache(c) != RC_SUCCESS || head < 0 || head >= c->kv_heads || !kv_find(slot, c->num_pages, c->page_size, page, in_page)) return -1;
    return kv_row(page, in_page, head, c->page_stride, c->head_stride, c->token_stride);
}

} // extern "C"
