// Entry points of the attention of one new token over a paged key-value cache; the kernels are in fvs_kv_attend.cuh.
#include "fvs_kv_attend.cuh"

namespace fvs {
namespace kv {
extern template int launch_types<64>(fvs_stream_t, const AttendArgs&, int);
extern template int launch_types<96>(fvs_stream_t, const AttendArgs&, int);
extern template int launch_types<128>(fvs_stream_t, const AttendArgs&, int);
extern template int launch_types<192>(fvs_stream_t, const AttendArgs&, int);
extern template int launch_types<256>(fvs_stream_t, const AttendArgs&, int);
}  // namespace kv
}  // namespace fvs

using namespace fvs::kv;

// two partial results for each of the pieces: 3 for each CTA; CTAs of an SM times rows of a
// partial result are at most SM_ROWS
extern "C" int fvs_kv_attend_work(int dim) {
    if (dim < 1) return FVS_EINVAL;
    if (dim > 256) return FVS_ERANGE;
    return 2 * 3 * fvs_sm_count() * SM_ROWS * (dim + 2) * 4;
}

extern "C" int fvs_kv_attend(fvs_stream_t stream, const fvs_kv_cache* cache, int type, const void* q, int64_t q_seq,
                             int64_t q_head, int hq, const int32_t* table, int seqs, int wide, int64_t table_stride,
                             const int32_t* lens, float scale, void* out, float* lse, void* work,
                             int32_t* arrived) {
    if (int rc = check_cache(cache)) return rc;
    FVS_CHECK_ARG(type == FVS_F16 || type == FVS_BF16);
    FVS_CHECK_ARG(cache->type == FVS_I8 || cache->type == type);
    FVS_CHECK_ARG(seqs >= 0 && hq >= 1 && hq % cache->heads == 0);
    if (seqs == 0) return FVS_OK;
    if (int rc = check_table(table, seqs, wide, table_stride)) return rc;
    FVS_CHECK_ARG(q && ((uintptr_t)q & 15) == 0 && q_seq % 8 == 0 && q_head % 8 == 0 && q_seq >= 0 && q_head >= 0);
    FVS_CHECK_ARG(lens && out && ((uintptr_t)out & 15) == 0 && work && ((uintptr_t)work & 15) == 0 &&
                  arrived && ((uintptr_t)arrived & 7) == 0);
    if ((int64_t)seqs * hq > (1 << 28)) return FVS_ERANGE;
    AttendArgs a{*cache, {table, table_stride, seqs, wide}, q, q_seq, q_head, lens, out, lse, arrived,
                 (unsigned long long*)(arrived + 2), (float*)work, hq, hq / cache->heads, 1, scale * 1.4426950408889634f, 0, 0};
    // exact for numerators below 2^31: 2^shift <= page_mul * page < 2^shift + 2^(shift - 31)
    uint32_t bits = 0;
    while ((1ull << bits) < (uint64_t)cache->page) bits++;
    a.page_shift = 31 + bits;
    a.page_mul = (uint32_t)(((1ull << a.page_shift) + cache->page - 1) / cache->page);
    switch (cache->dim) {
        case 64: return launch_types<64>(stream, a, type);
        case 96: return launch_types<96>(stream, a, type);
        case 128: return launch_types<128>(stream, a, type);
        case 192: return launch_types<192>(stream, a, type);
        default: return launch_types<256>(stream, a, type);
    }
}
