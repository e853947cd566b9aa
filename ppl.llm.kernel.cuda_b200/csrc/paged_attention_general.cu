// The GENERAL forms of decode attention: tables that differ from key head to key head, rows of several sequences, sums kept and joined.
#include "paged_attention.cuh"

namespace pplb200 {
namespace paged {

int32_t sms_of_general(AttentionParams& p) {
    int32_t sms = 0;
    launch_attention<true>(nullptr, p, &sms);
    return sms;
}

int32_t launch_general(cudaStream_t stream, AttentionParams& p) {
    small_division(p.unit_tokens, p.page_magic, p.page_shift);
    small_division(p.units_per_page, p.unit_magic, p.unit_shift);
    small_division(p.rows_per_head, p.rows_magic, p.rows_shift);
    return launch_attention<true>(stream, p);
}

} // namespace paged
} // namespace pplb200
