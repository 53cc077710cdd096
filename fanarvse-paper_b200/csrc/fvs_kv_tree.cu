// Entry points of the attention of a tree of drafted tokens over a paged key-value cache; the kernels are in
// fvs_kv_tree.cuh.
#include <mutex>

#include "fvs_kv_tree.cuh"

namespace fvs {
namespace kv {
namespace tree {
extern template int launch_types<64>(fvs_stream_t, Args, int);
extern template int launch_types<96>(fvs_stream_t, Args, int);
extern template int launch_types<128>(fvs_stream_t, Args, int);
extern template int launch_types<192>(fvs_stream_t, Args, int);
extern template int launch_types<256>(fvs_stream_t, Args, int);
}
}  // namespace kv
}  // namespace fvs

using namespace fvs::kv;

// two partial results of each CTA, of as many rows as an item has, behind DESC words of each CTA: two CTAs of 128 rows an SM
// with heads up to 128, else one.  The same for every number of rows
extern "C" int fvs_kv_attend_tree_work(int dim, int rows) {
    if (dim < 1 || rows < 0) return FVS_EINVAL;
    if (dim > 256) return FVS_ERANGE;
    return fvs_sm_count() * (2 * tree::DESC * 4 + (dim <= 128 ? 2 : 1) * 2 * tree::ROWS * (dim + 2) * 4);
}

extern "C" int fvs_kv_attend_tree(fvs_stream_t stream, const fvs_kv_cache* cache, int type, const void* q, int64_t q_seq,
                                  int64_t q_node, int64_t q_head, int hq, const int32_t* table, int seqs, int wide,
                                  int64_t table_stride, const int32_t* lens, const int32_t* parents,
                                  int64_t parent_stride, const int32_t* counts, int nodes, float scale, void* out,
                                  float* lse, void* work) {
    if (int rc = check_cache(cache)) return rc;
    FVS_CHECK_ARG(type == FVS_F16 || type == FVS_BF16);
    FVS_CHECK_ARG(cache->type == FVS_I8 || cache->type == type);
    FVS_CHECK_ARG(seqs >= 0 && nodes >= 0 && hq >= 1 && hq % cache->heads == 0 && parent_stride >= 0);
    if (seqs == 0 || nodes == 0) return FVS_OK;
    if (int rc = check_table(table, seqs, wide, table_stride)) return rc;
    FVS_CHECK_ARG(q && ((uintptr_t)q & 15) == 0 && q_seq % 8 == 0 && q_node % 8 == 0 && q_head % 8 == 0);
    FVS_CHECK_ARG(q_seq >= 0 && q_node >= 0 && q_head >= 0);
    FVS_CHECK_ARG(lens && parents && out && ((uintptr_t)out & 15) == 0 && work && ((uintptr_t)work & 15) == 0);
    const int group = hq / cache->heads;
    if (nodes > FVS_TREE_NODES || (int64_t)nodes * group > (1 << 24) || (int64_t)wide * cache->page > 0x7fffff00ll - FVS_TREE_NODES)
        return FVS_ERANGE;
    tree::Args a{*cache, {table, table_stride, seqs, wide}, q, q_seq, q_node, q_head, lens, parents, counts, parent_stride,
                 nodes, hq, group, scale, out, lse, (float*)work, nullptr, 0, 0};
    // The second launch reads what the first leaves in the workspace.  Threads that launch on one stream share a workspace, so
    // no call's launches come between another's (ctypes gives up Python's lock meanwhile).
    static std::mutex both;
    const std::lock_guard<std::mutex> hold(both);
    switch (cache->dim) {
        case 64: return tree::launch_types<64>(stream, a, type);
        case 96: return tree::launch_types<96>(stream, a, type);
        case 128: return tree::launch_types<128>(stream, a, type);
        case 192: return tree::launch_types<192>(stream, a, type);
        default: return tree::launch_types<256>(stream, a, type);
    }
}
