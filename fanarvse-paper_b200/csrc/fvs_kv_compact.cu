// Moving rows inside a paged key-value cache: the rows of the drafted tokens that verification took, one behind the other.
//
// Row lens[b] + path[b, n] goes to place lens[b] + n.  A path rises, so n <= path[b, n] and no row's place is the source of
// a row before it: taken in order, with every row of a batch loaded before one of it is stored, nothing is overwritten
// before it was read.  A warp moves the rows of one sequence and key head, of k or of v, so that the order needs no more
// than a warp's barrier.  The call moves a few hundred KB and is bound by its latencies: the path, then the page table, then
// the rows, 16 bytes a lane and up to BATCH loads of a lane on the way at once.
#include "fvs_kv.cuh"

namespace fvs {
namespace kv {

constexpr int COMPACT_THREADS = 128, COMPACT_BATCH = 4;

struct CompactArgs {
    fvs_kv_cache c;
    Table tb;
    const int32_t *lens, *path;
    int nodes;
};

template <int D, int STORE>
__global__ void __launch_bounds__(COMPACT_THREADS) compact_kernel(CompactArgs a) {
    constexpr int EL = STORE == FVS_I8 ? 16 : 8, L = D / EL, AT_ONCE = 32 / L, ESZ = 16 / EL;
    const unsigned w = blockIdx.x * (COMPACT_THREADS / 32) + threadIdx.x / 32, per_seq = 2 * a.c.heads;
    const int b = (int)(w / per_seq);
    if (b >= a.tb.seqs) return;
    const int lane = threadIdx.x & 31, e = lane % L * EL, sub = lane / L;
    const int part = (int)(w % per_seq), head = part >> 1;
    uint8_t* rows = (uint8_t*)((part & 1) ? a.c.v : a.c.k) + ((int64_t)head * a.c.head_stride + e) * ESZ;
    float* scales = STORE != FVS_I8 ? nullptr : ((part & 1) ? a.c.v_scale : a.c.k_scale) + (int64_t)head * a.c.scale_head_stride;
    const int start = __ldg(a.lens + b);
    const int32_t* path = a.path + (int64_t)b * a.nodes;
    int before = -1;  // the path's last node of the chunk before
    for (int n0 = 0; n0 < a.nodes; n0 += 32) {
        // a lane looks up the source and the place of one row
        const int n = n0 + lane;
        const int node = n < a.nodes ? __ldg(path + n) : -1;
        int last = __shfl_up_sync(0xffffffffu, node, 1);
        if (lane == 0) last = before;
        const unsigned stop = __ballot_sync(0xffffffffu, node < 0), wrong = __ballot_sync(0xffffffffu, node >= 0 && (node <= last || node >= a.nodes));
        int count = stop ? __ffs(stop) - 1 : 32;
        const bool bad = start < 0 || (wrong && __ffs(wrong) - 1 < count);
        if (bad) {
            if (lane == 0) atomicOr(a.c.status, BAD_INDEX);
            count = start < 0 ? 0 : __ffs(wrong) - 1;  // no row from there on
        }
        int page = 0, slot = 0, to_page = 0, to_slot = 0;
        bool there = lane < count && node != n;  // else the row lies in its place already
        if (there) {
            // two lookups, each reporting what it finds (a sum past 31 bits is no place of any table)
            const bool from = place(a.c, a.tb, b, (int)min((int64_t)start + node, (int64_t)INT32_MAX), page, slot);
            const bool to = place(a.c, a.tb, b, (int)min((int64_t)start + n, (int64_t)INT32_MAX), to_page, to_slot);
            there = from && to;
        }
        const unsigned moves = __ballot_sync(0xffffffffu, there);
        for (int r0 = 0; r0 < count; r0 += AT_ONCE * COMPACT_BATCH) {
            uint4 raw[COMPACT_BATCH];
            float scale[COMPACT_BATCH];
#pragma unroll
            for (int u = 0; u < COMPACT_BATCH; u++) {
                const int r = r0 + u * AT_ONCE + sub;
                const int pg = __shfl_sync(0xffffffffu, page, r & 31), sl = __shfl_sync(0xffffffffu, slot, r & 31);
                if (sub < AT_ONCE && r < count && (moves >> r & 1)) {
                    raw[u] = *(const uint4*)(rows + ((int64_t)pg * a.c.page_stride + (int64_t)sl * a.c.slot_stride) * ESZ);
                    if (STORE == FVS_I8 && e == 0)
                        scale[u] = scales[(int64_t)pg * a.c.scale_page_stride + (int64_t)sl * a.c.scale_slot_stride];
                }
            }
            __syncwarp();
#pragma unroll
            for (int u = 0; u < COMPACT_BATCH; u++) {
                const int r = r0 + u * AT_ONCE + sub;
                const int pg = __shfl_sync(0xffffffffu, to_page, r & 31), sl = __shfl_sync(0xffffffffu, to_slot, r & 31);
                if (sub < AT_ONCE && r < count && (moves >> r & 1)) {
                    *(uint4*)(rows + ((int64_t)pg * a.c.page_stride + (int64_t)sl * a.c.slot_stride) * ESZ) = raw[u];
                    if (STORE == FVS_I8 && e == 0)
                        scales[(int64_t)pg * a.c.scale_page_stride + (int64_t)sl * a.c.scale_slot_stride] = scale[u];
                }
            }
            __syncwarp();
        }
        if (count < 32) return;
        before = __shfl_sync(0xffffffffu, node, 31);
    }
}

template <int STORE>
static void launch_compact(fvs_stream_t stream, const CompactArgs& a) {
    const int64_t warps = (int64_t)a.tb.seqs * 2 * a.c.heads;
    const unsigned grid = (unsigned)((warps + COMPACT_THREADS / 32 - 1) / (COMPACT_THREADS / 32));
    switch (a.c.dim) {
        case 64: compact_kernel<64, STORE><<<grid, COMPACT_THREADS, 0, stream>>>(a); break;
        case 96: compact_kernel<96, STORE><<<grid, COMPACT_THREADS, 0, stream>>>(a); break;
        case 128: compact_kernel<128, STORE><<<grid, COMPACT_THREADS, 0, stream>>>(a); break;
        case 192: compact_kernel<192, STORE><<<grid, COMPACT_THREADS, 0, stream>>>(a); break;
        default: compact_kernel<256, STORE><<<grid, COMPACT_THREADS, 0, stream>>>(a); break;
    }
}

}  // namespace kv
}  // namespace fvs

using namespace fvs::kv;

extern "C" int fvs_kv_compact(fvs_stream_t stream, const fvs_kv_cache* cache, const int32_t* table, int seqs, int wide,
                              int64_t table_stride, const int32_t* lens, const int32_t* path, int nodes) {
    if (int rc = check_cache(cache)) return rc;
    FVS_CHECK_ARG(seqs >= 0 && nodes >= 0);
    if (seqs == 0 || nodes == 0) return FVS_OK;
    if (int rc = check_table(table, seqs, wide, table_stride)) return rc;
    FVS_CHECK_ARG(lens && path);
    if ((int64_t)seqs * 2 * cache->heads > 0x7fffff00ll) return FVS_ERANGE;
    const CompactArgs a{*cache, {table, table_stride, seqs, wide}, lens, path, nodes};
    // 16-bit types move alike
    cache->type == FVS_I8 ? launch_compact<FVS_I8>(stream, a) : launch_compact<FVS_F16>(stream, a);
    return fvs_launch_status();
}
