// Appending with norms of the query and key heads: fvs_kv_append's kernel with the norm in the same pass (a unit of its
// own, so that the two sets of kernels compile side by side).
//
// x -> x / sqrt(mean x^2 + eps) * weight, then the rotation, all in fp32 and rounded once: the norm by itself would read and
// write every head once more.  Its cost beside the plain append is a sum over 16 elements a lane, two to four exchanges and
// the weights' loads, all behind the loads of the rows.
#include "fvs_kv_append.cuh"

using namespace fvs::kv;

extern "C" int fvs_kv_append_norm(fvs_stream_t stream, const fvs_kv_cache* cache, int type, const void* k, int64_t k_token,
                                  int64_t k_head, const void* v, int64_t v_token, int64_t v_head, const void* q,
                                  int64_t q_token, int64_t q_head, int hq, void* q_out, const int32_t* table, int seqs,
                                  int wide, int64_t table_stride, const int32_t* seq, const int32_t* idx,
                                  const int32_t* pos, int tokens, const float* cos, const float* sin, int positions,
                                  int rot, int pairs,
                                  const void* q_weight, const void* k_weight, int weight_type, float eps) {
    AppendArgs a;
    if (int rc = append_args(a, cache, type, k, k_token, k_head, v, v_token, v_head, q, q_token, q_head, hq, q_out, table,
                             seqs, wide, table_stride, seq, idx, pos, tokens, cos, sin, positions, rot, pairs))
        return rc;
    if (a.tokens == 0) return FVS_OK;
    FVS_CHECK_ARG(weight_type == FVS_F32 || weight_type == type);
    FVS_CHECK_ARG((((uintptr_t)q_weight | (uintptr_t)k_weight) & 15) == 0 && eps > 0.f && eps < 1e30f);
    a.q_weight = q_weight;
    a.k_weight = k_weight;
    a.weight_f32 = weight_type == FVS_F32;
    a.eps = eps;
    return append_launch<true>(stream, a, type, pairs == FVS_PAIRS_HALVES);
}
