// The paged key-value cache: where a token's row lies, and the checks that the entry points share.
#pragma once

#include "common.cuh"
#include "../../include/pplb200_attention.h"

namespace pplb200 {

constexpr int kMaxHeadDim = 256;

// Offset of a row in units of the strides' elements.  64 bits throughout: a cache of a few layers passes 2^31 elements.
__host__ __device__ inline int64_t kv_row(int64_t page, int64_t in_page, int64_t head, int64_t page_stride, int64_t head_stride,
                                          int64_t token_stride) {
    return page * page_stride + head * head_stride + in_page * token_stride;
}

// Page of a slot, and the slot's place on it; false where the cache has no such slot.
__host__ __device__ inline bool kv_find(int64_t slot, int64_t num_pages, int32_t page_size, int64_t& page, int32_t& in_page) {
    if (slot < 0) return false;
    if ((uint64_t)slot >> 32) {
        page = slot / page_size;
        in_page = (int32_t)(slot - page * page_size);
    } else { // a 32-bit division is a quarter of the instructions
        page = (uint32_t)slot / (uint32_t)page_size;
        in_page = (int32_t)((uint32_t)slot - (uint32_t)page * (uint32_t)page_size);
    }
    return page < num_pages;
}

// n / d = n * magic >> shift for all n below 2^31: with 2^(s - 1) < d <= 2^s and magic = ceil(2^(31 + s) / d), magic * d exceeds 2^(31 + s)
// by less than d <= 2^s, which n < 2^31 keeps below 1 / d of the quotient.
inline void small_division(uint32_t d, uint32_t& magic, uint32_t& shift) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    shift = 31 + s;
    magic = (uint32_t)(((1ull << shift) + d - 1) / d);
}

// RC_SUCCESS, or the first thing wrong with the description (the text goes to pplb200_last_error()).
int32_t check_kv_cache(const pplb200_kv_cache* c);

} // namespace pplb200
