// Attention of one new token per sequence for a batch that shares a prefix: the prefix for the rows of all sequences at once, then each sequence's
// own tokens, whose sums are joined with the prefix's where the output is written.
#include "shared_prefix.cuh"

#include <cmath>
#include <cuda.h>

namespace pplb200 {
namespace {

using namespace prefix;

constexpr int64_t kMaxRows = 1 << 24;

constexpr int32_t block_tokens(int32_t head_dim) { return head_dim == 256 ? 64 : 128; }
constexpr int32_t most_tiles(int32_t head_dim, bool groups) { return head_dim < 256 && (!groups || head_dim == 64) ? 2 : 1; } // that tensor and shared memory have room for

// Parts that the prefix is cut into: at most so many that there is a CTA for every SM.
int32_t most_splits(int64_t items) { return (int32_t)std::max<int64_t>(1, kSms / items); }
// More are not worth their joining (splits_of).
int64_t worthwhile_splits(int64_t blocks) { return std::max<int64_t>(8, (int64_t)std::sqrt(8.0 * (double)blocks) + 1); }

// Tiles of rows that a CTA takes at once.  Two share what is loaded, and widened: a block of 128 tokens for both takes 2.04 us where it takes 1.09 for one in fp16 (heads of 64: 1.85 and 0.99),
// 3.7 and 2.13 over int8, and 2 to 5 of the latter more at the ends, for twice as many sums to be joined.  How many blocks a CTA goes through, and so which is less, depends on how either divides
// the SMs.  64 heads over 8, 32768 tokens, one tile and two, us: fp16 48 sequences (3 tiles) 62 and 73, 80 (5) 104 and 103, 112 (7) 147 and 144, 144 (9) 160 and 185; int8 rows 104 and 120, 193 and
// 174, 285 and 254, 287 and 332; 8 heads over one, fp16, 24, 40 and 56 tiles 58, 103, 148 and 61, 92, 122; over 4096 tokens 21, 31, 38 and 24, 31, 38.
int32_t tiles_at_once(int64_t rows, const pplb200_kv_cache& c, int64_t blocks) {
    const int64_t tiles = (rows + 127) / 128;
    if (most_tiles(c.head_dim, c.quant_group == 8) == 1 || tiles == 1) return 1;
    const auto through = [&](int64_t items) { // blocks of a CTA
        const int64_t splits = std::min<int64_t>({most_splits(c.kv_heads * items), blocks, worthwhile_splits(blocks)});
        return (double)((blocks + splits - 1) / splits);
    };
    const bool f16 = c.quant_group == 0;
    return (f16 ? 1.88 : 1.74) * through((tiles + 1) / 2) + (f16 && c.head_dim > 64 ? 5 : 2) < through(tiles) ? 2 : 1;
}
// Joining the parts costs about an eighth of a block each, which the square root balances (64 rows of one head, 32768 tokens: 22 us with 46 parts, 41 with 148).  The
// kernel for the own tokens fills `own_sms` SMs, and where these are left to it, it runs beside this one: up to four blocks a CTA more are worth it
// (16 rows of 8 heads, 4096 tokens: 13.2 us with 13 parts, 17.8 with 17; 4096 of int8 rows and 700 of their own each: 22.5, 33).
int32_t splits_of(int64_t items, int64_t own_sms, int64_t blocks, bool* beside = nullptr) {
    const int64_t all = std::min<int64_t>({most_splits(items), blocks, worthwhile_splits(blocks)});
    const int64_t spared = std::min(all, (kSms - own_sms) / items);
    const bool spare = spared > 0 && (blocks + spared - 1) / spared <= (blocks + all - 1) / all + 4;
    if (beside) *beside = spare;
    return (int32_t)(spare ? spared : all);
}

// Few rows of an int8 cache: the decode kernel, whose matrix instructions take 8 or 16 at once, widens with all of its warps, and is faster where a CTA would have several
// blocks (int8 rows, 8 rows of 8 heads over 1000, 4096 and 32768 tokens: 11.8, 15.7, 28 us, by tiles 12.5, 17.3, 48; 4 of 32 over 1000 13.3 and 17.1; 16 of 8 over 4096, 12345
// and 32768 19.6, 25, 36 and 17.7, 27, 47; groups of 8 19, 25, 38 and 17, 27, 55.  Other heads, rows of int8, 8 of 8 over 1000, 4096, 12345 and 32768: of 64 10.7, 12.9, 16.3, 20.4 and
// 9.6, 11.9, 20.0, 34.8; of 96 11.9, 15.6, 20, 29 and 11.6, 14.2, 24, 40; of 256 15.6, 19.0, 26, 40 and 13.2, 18.4, 35, 63.  In fp16 8 rows of 8 heads over 8000 and 32768
// 18.0, 32.4 and 16.2, 31.2).
constexpr int32_t kFewRows = 16;
bool by_decode(int64_t rows, const pplb200_kv_cache& c, int64_t blocks, int32_t splits) {
    return c.quant_group && rows <= kFewRows && blocks > splits * (rows <= 8 ? 1LL : 6LL);
}

// Workspace: what the decode kernel needs for the own tokens, which it begins to go through before the prefix's kernel ends; sums over the parts of the prefix, and what the decode
// kernel needs for few rows' prefix.
// Reference exponents and sums of weights, then sums of values.
int64_t part_bytes(int64_t sums, int32_t head_dim) { return round_up(sums * 8, 256) + round_up(sums * head_dim * 4, 256); }
// Sums for up to `rows` of a key head: fewer rows can need more, in more parts.
int64_t most_sums(int64_t rows, int32_t kv_heads) {
    int64_t most = 0;
    for (int64_t r = std::min<int64_t>(rows, 256); r > 0; r = std::min(rows, r + 256)) {
        most = std::max(most, kv_heads * r * most_splits(kv_heads * ((r + 255) / 256)));
        if (r == rows || r >= 256 * kSms) break; // (one part from there on)
    }
    return std::max(most, kv_heads * rows);
}

// A map of keys or values for boxes of box_rows tokens by 64 dimensions; false where there is none for such strides.
bool make_page_map(CUtensorMap* map, const pplb200_kv_cache& c, const void* base, int32_t box_rows) {
    static const decltype(&cuTensorMapEncodeTiled) encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess;
        return ok ? (decltype(&cuTensorMapEncodeTiled))f : nullptr;
    }();
    const int64_t strides_of[3] = {c.token_stride * 2, c.head_stride * 2, c.page_stride * 2};
    const int64_t extents[3] = {c.page_size, c.kv_heads, c.num_pages};
    cuuint64_t dims[4] = {(cuuint64_t)c.head_dim}, strides[3];
    for (int i = 0; i < 3; ++i) {
        if (extents[i] > 0x7fffffff || strides_of[i] >= 1LL << 40 || (strides_of[i] == 0 && extents[i] > 1)) return false;
        dims[1 + i] = (cuuint64_t)extents[i];
        strides[i] = (cuuint64_t)(strides_of[i] ? strides_of[i] : 16); // (of one: not used)
    }
    const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, steps[4] = {1, 1, 1, 1};
    return encode && encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int KIND>
int32_t launch_tiles(cudaStream_t stream, PrefixParams& p) {
    using T = Tile<D, KIND>;
    static_assert(T::SMEM + 18 * 1024 <= 232448);
    static_assert(T::NB == block_tokens(D) && T::TILES == most_tiles(D, KIND == CACHE_I8_GROUPS));
    p.box_rows = 0;
    if (KIND == CACHE_F16 && p.cache.page_size % 16 == 0 && p.cache.num_pages > 0) {
        const int32_t rows = std::min(p.cache.page_size & -p.cache.page_size, T::NB);
        if (make_page_map(&p.kmap, p.cache, p.cache.k, rows) && make_page_map(&p.vmap, p.cache, p.cache.v, rows)) p.box_rows = rows;
    }
    const cudaError_t e = cudaFuncSetAttribute(prefix_tile_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
    if (e != cudaSuccess) return fail(RC_DEVICE_RUNTIME_ERROR, "shared prefix: %s", cudaGetErrorString(e));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.items * p.splits));
    cfg.blockDim = dim3(T::THREADS);
    cfg.dynamicSmemBytes = T::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, prefix_tile_kernel<T>, p);
    return check_launch("shared prefix");
}
template <int D>
int32_t launch_kind(cudaStream_t stream, PrefixParams& p) {
    if (p.cache.quant_group == 0) return launch_tiles<D, CACHE_F16>(stream, p);
    if (p.cache.quant_group == 8) return launch_tiles<D, CACHE_I8_GROUPS>(stream, p);
    return launch_tiles<D, CACHE_I8_ROWS>(stream, p);
}
int32_t launch_prefix(cudaStream_t stream, PrefixParams& p) {
    if (p.cache.head_dim == 64) return launch_kind<64>(stream, p);
    if (p.cache.head_dim == 96) return launch_kind<96>(stream, p);
    if (p.cache.head_dim == 128) return launch_kind<128>(stream, p);
    return launch_kind<256>(stream, p);
}

} // namespace
} // namespace pplb200

using namespace pplb200;

extern "C" {

int64_t pplb200_shared_prefix_attention_workspace_bytes(int64_t batch, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
    if (batch < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || head_dim <= 0 || batch > kMaxRows / q_heads) return -1;
    const int32_t shared = q_heads / kv_heads;
    const int64_t rows = batch * shared, few = std::min<int64_t>(rows, kFewRows);
    return workspace_bytes(shared, head_dim) +
           std::max(part_bytes(most_sums(rows, kv_heads), head_dim), part_bytes(kv_heads * few, head_dim) + workspace_bytes(few, head_dim));
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
    const int64_t rows = a->batch * a->q_heads, tokens = prefix->num_pages * cache->page_size;
    char* const ws = (char*)a->ws;
    own.unit_tokens = cache->page_size;
    own.units_per_page = 1;
    own.num_units = own.num_pages;
    own.rows_per_head = shared;
    own.part_rows = rows;
    own.parts = 1;
    own.late_wait = true;
    own.ahead = (uint32_t*)(ws + kAhead);
    lay_out(own, ws, shared);
    const int64_t nb = block_tokens(cache->head_dim), blocks = std::max<int64_t>(1, (tokens + nb - 1) / nb);
    const int32_t tiles = tiles_at_once(a->batch * shared, *cache, blocks), items = (int32_t)(cache->kv_heads * ((a->batch * shared + 128 * tiles - 1) / (128 * tiles)));
    // Own tokens by a CTA for each sequence and key head, on SMs that are left to them, up to 1024 tokens (fp16, 32 sequences of 8 heads, 1000 tokens each behind 1000 31 us, 51 if
    // shared out; but 8 of one 18 and 15.4, and behind 12345 tokens, without SMs for them, 71 and 68); up to 512 in any case (64 of one head with 300 11.7, 20.4).
    bool beside;
    own.whole_tokens = a->batch * cache->kv_heads >= 32 ? 1024 : 512;
    int32_t splits = splits_of(items, sms_of_general(own), blocks, &beside);
    if (!beside && own.whole_tokens > 512) {
        own.whole_tokens = 512;
        splits = splits_of(items, sms_of_general(own), blocks);
    }
    const bool decode = by_decode(a->batch * shared, *cache, blocks, splits);
    if (decode) own.whole_tokens = 512;
    const int64_t sums = decode ? rows : rows * most_splits(cache->kv_heads * ((a->batch * shared + 255) / 256));
    own.part_tops = (float2*)(ws + workspace_bytes(shared, cache->head_dim));
    own.part_sums = (float*)((char*)own.part_tops + round_up(sums * 8, 256));
    if (decode) {
        // the prefix as one sequence, whose key heads are asked by the rows of all
        AttentionParams first = own;
        first.batch = 1;
        first.pages = prefix->pages;
        first.lengths = prefix->length;
        first.pages_stride = prefix->num_pages;
        first.tokens_in_table = tokens;
        first.parts = 0;
        first.late_wait = false;
        first.whole_tokens = 0;
        first.keep_parts = true;
        lay_out(first, (char*)own.part_tops + part_bytes(sums, cache->head_dim), a->batch * shared);
        first.arrived = (uint64_t*)(ws + kCounters);
        const int32_t done = launch_general((cudaStream_t)stream, first);
        if (done != RC_SUCCESS) return done;
    } else {
        PrefixParams p = {};
        p.q = own.q; p.q_stride = own.q_stride;
        p.pages = prefix->pages; p.length = prefix->length;
        p.tokens_in_table = tokens;
        p.num_pages = own.num_pages; p.rows = (int32_t)(a->batch * shared);
        p.rows_per_head = shared; p.q_heads = a->q_heads;
        small_division(shared, p.rows_magic, p.rows_shift);
        small_division(cache->page_size, p.page_magic, p.page_shift);
        p.scale_log2 = own.scale_log2;
        p.tiles = tiles; p.items = items; p.splits = splits;
        p.cache = *cache;
        p.part_rows = rows; p.part_tops = own.part_tops; p.part_sums = own.part_sums;
        p.ahead = own.ahead;
        const int32_t done = launch_prefix((cudaStream_t)stream, p);
        if (done != RC_SUCCESS) return done;
        own.parts = p.splits;
    }
    return launch_general((cudaStream_t)stream, own);
}

int32_t pplb200_shared_prefix_attention_status(int32_t reset) {
    void* word = nullptr;
    cudaStream_t mine; // no other stream of the device is waited for
    if (cudaGetSymbolAddress(&word, g_status) != cudaSuccess || cudaStreamCreateWithFlags(&mine, cudaStreamNonBlocking) != cudaSuccess) {
        cudaGetLastError();
        return -1;
    }
    unsigned int v = 0;
    bool ok = cudaMemcpyAsync(&v, word, sizeof(v), cudaMemcpyDeviceToHost, mine) == cudaSuccess && cudaStreamSynchronize(mine) == cudaSuccess;
    if (ok && reset && v) ok = cudaMemsetAsync(word, 0, sizeof(v), mine) == cudaSuccess && cudaStreamSynchronize(mine) == cudaSuccess;
    cudaStreamDestroy(mine);
    return ok ? (int32_t)v : -1;
}

} // extern "C"
