// Verification of drafted tokens against a target model's probabilities, from given random numbers (new: what follows the
// attention of a tree of drafted tokens; the reference ends with the found rows' ids).
//
// Behind the last node taken (at first the sequence's end) the target's probabilities are p and the draft's q.  The node's
// children are tried in order: with r_0 = p and m_0 = 1, child c of token x is taken if u_c m_k q(x) < r_k(x), else
// r_{k+1} = max(r_k - m_k q, 0) and m_{k+1} = sum r_{k+1}, unless that is 0.  Where none is taken the next token is drawn from
// r_k: the first whose running sum passes u_last sum(r_k).  Taken this way the tokens are distributed as the target's own.
//
// All of it is in fp64: p and q are exact in it and so is a first difference of numbers less than 2^29 apart, so that a
// decision depends on the order of a sum only within 1e-16 of its border.
//
// Whether a node is taken without a refusal before it needs two numbers, gathered for all nodes at once; a whole row (and
// the draft's) is read only for a node's refused child and for the last draw, a pass over V (1 + draft) elements each: the
// floor is one pass, more of a row come from L2.  A cluster of CTAs shares a row, since one SM reads it at 1/148 of the
// memory's rate; the sums of its CTAs are exchanged through distributed shared memory and added in order of rank, so that
// every CTA comes to the same numbers and walks the same path by itself.
// What bounds it: a sequence's passes behind one another, each with a cluster's barrier at its end.  64 x 16 nodes over
// 131072 tokens take 45 us with up to four passes of a sequence (140 in all, 120 MB): 35 % of the issue slots, warps wait for
// loads and for the barrier.  Asking L2 for a warp's part ahead of the loads changed nothing.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "fvs_common.cuh"

namespace cg = cooperative_groups;

namespace fvs {
namespace drafts {

constexpr int THREADS = 256, WARPS = THREADS / 32, NODES = 256, CTAS = 8;
constexpr int AHEAD = 2;  // loads of 16 bytes of a row that a lane has on the way (64 x 16 nodes over
                          // 131072 tokens: 45 us, with three 50, with four 53: registers spill and code is fetched again)
constexpr int RUN = 8;    // elements of a thread in the draw

struct Rows {  // [seqs, nodes + 1, vocab], strides in elements; null: none
    const void* at;
    int64_t seq, row;
};

struct Args {
    Rows target, draft;
    const int32_t *parents, *tokens, *counts;
    const float* u;
    int64_t parent_stride;  // 0: one tree for all
    int seqs, nodes, vocab;
    int32_t *path, *kept, *token;
};

__device__ __forceinline__ float sane(float x) { return x > 0.f && x < __int_as_float(0x7f800000) ? x : 0.f; }  // else no probability
template <typename T>
__device__ __forceinline__ float value(const T* p) { return sane((float)*p); }

// 16 bytes of a row from element `at` on: one load where all of them are the row's (and its skew is the vectors'), else
// those elements that are, and zeros
template <typename T>
__device__ __forceinline__ uint4 load(const T* row, int at, int vocab, bool aligned) {
    constexpr int VEC = 16 / sizeof(T);
    if (aligned && at >= 0 && at + VEC <= vocab) return __ldg((const uint4*)(row + at));
    uint4 raw = make_uint4(0, 0, 0, 0);
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; i++)
        if (at + i >= 0 && at + i < vocab) e[i] = row[at + i];
    return raw;
}

struct Shared {
    double left[NODES];   // r_k of the node's token, while its parent is the last node taken
    double qx[NODES];
    float u[NODES + 1];
    int parent[NODES], tok[NODES];
    int refused[NODES];      // tokens refused in it (drafts without probabilities)
    double warp[WARPS], scan[WARPS];
    double total[2][CTAS];   // of each CTA, two passes in turn
    int found, positive;
};

// r_k of element v of the present row: as every m_j and q is at least 0, max(.. max(p - m_0 q, 0) .. - m_{k-1} q, 0) is max(p -
// M q, 0) with M their sum.  M is 1 for k = 1, and a difference of two fp32 numbers less than 2^29 apart is exact in fp64.
__device__ __forceinline__ double rest_of(float p, float q, double M) {
    const double r = fma(-M, (double)q, (double)p);
    // the sign over both words: a comparison of fp64 numbers and two selections took 49 us where this takes 45
    const int keep = ~(__double2hiint(r) >> 31);
    return __hiloint2double(__double2hiint(r) & keep, __double2loint(r) & keep);
}
template <bool DRAFT>
__device__ __forceinline__ double rest(float p, float q, int v, const Shared& s, int k, double M) {
    if (DRAFT) return rest_of(p, q, M);
    for (int j = 0; j < k; j++) p = v == s.refused[j] ? 0.f : p;
    return p;
}

// sum of r_n over N times 16 bytes, the first of them from element v on, 32 lanes' vectors apart
template <typename T, bool DRAFT, int N>
__device__ __forceinline__ double sum_of(const uint4 (&praw)[N], const uint4 (&qraw)[N], int v, const Shared& s, int n, double M) {
    constexpr int VEC = 16 / sizeof(T);
    float p[N * VEC], q[N * VEC];
    uint32_t most = 0;  // above every number's bits where something is negative or not finite
#pragma unroll
    for (int i = 0; i < N * VEC; i++) {
        p[i] = (float)reinterpret_cast<const T*>(&praw[i / VEC])[i % VEC];
        most = max(most, __float_as_uint(p[i]));
        if (DRAFT) {
            q[i] = (float)reinterpret_cast<const T*>(&qraw[i / VEC])[i % VEC];
            most = max(most, __float_as_uint(q[i]));
        }
    }
    if (__builtin_expect(most >= 0x7f800000u, 0)) {
#pragma unroll
        for (int i = 0; i < N * VEC; i++) {
            p[i] = sane(p[i]);
            if (DRAFT) q[i] = sane(q[i]);
        }
    }
    if (!DRAFT) {
#pragma unroll 1
        for (int j = 0; j < n; j++) {
            const int at = s.refused[j] - v;
#pragma unroll
            for (int i = 0; i < N * VEC; i++)
                if (at == i / VEC * 32 * VEC + i % VEC) p[i] = 0.f;
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < N * VEC; i += 2)
        sum += DRAFT ? rest_of(p[i], q[i], M) + rest_of(p[i + 1], q[i + 1], M) : (double)p[i] + (double)p[i + 1];
    return sum;
}

template <typename T, bool DRAFT>
__global__ void __launch_bounds__(THREADS, 4) verify_kernel(Args a) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ Shared s;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int b = blockIdx.x / ctas, tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const T* target = (const T*)a.target.at + b * a.target.seq;
    const T* draft = (const T*)a.draft.at + b * a.draft.seq;
    const int nodes = a.counts ? min(max(__ldg(a.counts + b), 0), a.nodes) : a.nodes;
    for (int i = tid; i < nodes; i += THREADS) {
        const int up = __ldg(a.parents + b * a.parent_stride + i), x = __ldg(a.tokens + (int64_t)b * a.nodes + i);
        const bool ok = up >= -1 && up < i && x >= 0 && x < a.vocab;
        s.parent[i] = ok ? up : -2;  // never taken
        s.tok[i] = x;
        s.u[i] = __ldg(a.u + (int64_t)b * (a.nodes + 1) + i);
        s.left[i] = ok ? (double)value(target + (up + 1) * a.target.row + x) : 0.0;
        s.qx[i] = !ok ? 0.0 : DRAFT ? (double)value(draft + (up + 1) * a.draft.row + x) : 1.0;
    }
    int last = -1, kept = 0, k = 0, turn = 0;
    double total = 0.0;
    bool summed = false;  // total and the warps' sums are those of r_k
    // The parts of a row that the cluster's warps sum lie side by side: vectors of 16 bytes, the first of them beginning
    // `skew` elements before the row where that is not aligned.
    auto skew_of = [&](const T* row) { return (int)((uintptr_t)row / sizeof(T) % VEC); };
    auto span_of = [&](int skew) { return ((a.vocab + skew + VEC - 1) / VEC + ctas * WARPS - 1) / (ctas * WARPS); };
    // sums of r_n over the row behind `last`; ends with all of the cluster's threads having them
    auto pass = [&](int n, double M) {
        const T *p = target + (last + 1) * a.target.row, *q = draft + (last + 1) * a.draft.row;
        const int skew = skew_of(p), span = span_of(skew), lo = (rank * WARPS + warp) * span;
        const int hi = min((a.vocab + skew + VEC - 1) / VEC, lo + span);
        const bool alike = DRAFT && skew_of(q) == skew, both = DRAFT && n > 0;
        double sum = 0.0;
        for (int j0 = lo + lane; j0 < hi; j0 += 32 * AHEAD) {
            uint4 pv[AHEAD], qv[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const int j = j0 + 32 * i;
                const int at = j < hi ? j * VEC - skew : a.vocab;  // none behind the part
                pv[i] = load(p, at, a.vocab, true);
                qv[i] = both ? load(q, at, a.vocab, alike) : make_uint4(0, 0, 0, 0);
            }
            sum += sum_of<T, DRAFT, AHEAD>(pv, qv, j0 * VEC - skew, s, n, M);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) s.warp[warp] = sum;
        __syncthreads();
        if (tid < ctas) {
            double all = 0.0;
#pragma unroll
            for (int w = 0; w < WARPS; w++) all += s.warp[w];
            *cluster.map_shared_rank(&s.total[turn][rank], tid) = all;
        }
        cluster.sync();
        double all = 0.0;
        for (int r = 0; r < ctas; r++) all += s.total[turn][r];
        return all;
    };
    cluster.sync();  // every CTA has begun and has its nodes
    double mass = 1.0, M = 0.0;  // m_k, m_0 + .. + m_{k-1}
    for (int i = 0; i < nodes; i++) {  // children come after their parents
        if (s.parent[i] != last) continue;
        if ((double)s.u[i] * mass * s.qx[i] < s.left[i]) {
            if (rank == 0 && tid == 0) a.path[(int64_t)b * a.nodes + kept] = i;
            last = i;
            kept++;
            k = 0;
            mass = 1.0;
            M = 0.0;
            summed = false;
            continue;
        }
        if (!DRAFT) {
            if (tid == 0) s.refused[k] = s.tok[i];
            __syncthreads();
        }
        const double m = pass(k + 1, M + mass);
        turn ^= 1;
        summed = m > 0.0;
        if (m > 0.0) {
            for (int c = tid; c < nodes; c += THREADS) {
                if (s.parent[c] != last) continue;
                if (DRAFT)
                    s.left[c] = fmax(__dsub_rn(s.left[c], __dmul_rn(mass, s.qx[c])), 0.0);
                else if (s.tok[c] == s.tok[i])
                    s.left[c] = 0.0;
            }
            __syncthreads();
            M += mass;
            mass = m;
            total = m;
            k++;
        }
    }
    if (!summed) {
        __syncthreads();
        total = pass(k, M);
    } else {
        turn ^= 1;  // the buffer of the last pass
    }
    // the draw: the first CTA, warp and element at which the running sum passes the limit
    const double limit = (double)__ldg(a.u + (int64_t)b * (a.nodes + 1) + a.nodes) * total;
    int owner = -1, some = -1;
    double before = 0.0;
    for (int r = 0; r < ctas; r++) {
        const double all = s.total[turn][r];
        if (all > 0.0) some = r;
        if (before + all > limit) {
            owner = r;
            break;
        }
        if (r < ctas - 1) before += all;
    }
    const bool none = owner < 0;  // a limit that no sum passes (u of 1, say): the last element with a probability
    if (none) owner = some;
    if (rank == 0 && tid == 0) {
        a.kept[b] = kept;
        if (owner < 0) a.token[b] = -1;
    }
    if (rank == 0)
        for (int n = kept + tid; n < a.nodes; n += THREADS) a.path[(int64_t)b * a.nodes + n] = -1;
    if (rank == owner) {
        int w = 0, positive = -1;
        bool over = false;
        for (; w < WARPS; w++) {
            if (s.warp[w] > 0.0) positive = w;
            if (!none && before + s.warp[w] > limit) {
                over = true;
                break;
            }
            if (w < WARPS - 1) before += s.warp[w];
        }
        if (!over) w = positive;  // the sums' rounding, or none
        const T *p = target + (last + 1) * a.target.row, *q = draft + (last + 1) * a.draft.row;
        const int skew = skew_of(p), span = span_of(skew);
        const int from = max(0, (rank * WARPS + w) * span * VEC - skew), to = min(a.vocab, (rank * WARPS + w + 1) * span * VEC - skew);
        if (tid == 0) s.found = INT_MAX, s.positive = -1;
        __syncthreads();
        for (int v0 = from; v0 < to; v0 += THREADS * RUN) {
            const int v = v0 + tid * RUN;
            double x[RUN], sum = 0.0;
#pragma unroll
            for (int j = 0; j < RUN; j++) {
                x[j] = v + j < to ? rest<DRAFT>(value(p + v + j), DRAFT && k > 0 ? value(q + v + j) : 0.f, v + j, s, k, M) : 0.0;
                sum += x[j];
            }
            double upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            if (lane == 31) s.scan[warp] = upto;
            __syncthreads();
            double add = before, all = before;
#pragma unroll
            for (int j = 0; j < WARPS; j++) {
                if (j < warp) add += s.scan[j];
                all += s.scan[j];
            }
            add += upto - sum;
#pragma unroll
            for (int j = 0; j < RUN; j++) {
                add += x[j];
                if (x[j] > 0.0) {
                    if (over && add > limit) atomicMin(&s.found, v + j);
                    atomicMax(&s.positive, v + j);
                }
            }
            before = all;
            __syncthreads();
            if (s.found != INT_MAX) break;
        }
        if (tid == 0) a.token[b] = s.found != INT_MAX ? s.found : s.positive;
    }
    cluster.sync();  // no CTA ends while another may still write its sums
}

template <typename T>
static int launch(fvs_stream_t stream, const Args& a) {
    // CTAs of a row: as many as run at once, four an SM, and at least 2048 elements each
    int ctas = 1;
    while (ctas < CTAS && ctas * 2 * a.seqs <= 4 * fvs_sm_count() && a.vocab >= ctas * 2 * 2048) ctas *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.seqs * ctas));
    cfg.blockDim = dim3(THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)ctas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = a.draft.at ? cudaLaunchKernelEx(&cfg, verify_kernel<T, true>, a) : cudaLaunchKernelEx(&cfg, verify_kernel<T, false>, a);
    return e == cudaSuccess ? fvs_launch_status() : (int)e;
}

}  // namespace drafts
}  // namespace fvs

using namespace fvs::drafts;

extern "C" int fvs_verify(fvs_stream_t stream, int type, const void* target, int64_t target_seq, int64_t target_row,
                          const void* draft, int64_t draft_seq, int64_t draft_row, const int32_t* parents,
                          int64_t parent_stride, const int32_t* tokens, const int32_t* counts, const float* u, int seqs,
                          int nodes, int vocab, int32_t* path, int32_t* kept, int32_t* token) {
    FVS_CHECK_ARG(type == FVS_F16 || type == FVS_BF16 || type == FVS_F32);
    FVS_CHECK_ARG(seqs >= 0 && nodes >= 0 && vocab >= 1);
    if (seqs == 0) return FVS_OK;
    const uintptr_t odd = type == FVS_F32 ? 3 : 1;
    FVS_CHECK_ARG(target && u && kept && token && (nodes == 0 || (parents && tokens && path)));
    FVS_CHECK_ARG(((uintptr_t)target & odd) == 0 && ((uintptr_t)draft & odd) == 0);
    FVS_CHECK_ARG(target_seq >= 0 && target_row >= 0 && draft_seq >= 0 && draft_row >= 0 && parent_stride >= 0);
    if (nodes > NODES || vocab > (1 << 30) || seqs > (1 << 27)) return FVS_ERANGE;
    const Args a{{target, target_seq, target_row}, {draft, draft_seq, draft_row}, parents, tokens, counts, u, parent_stride,
                 seqs, nodes, vocab, path, kept, token};
    return type == FVS_F32 ? launch<float>(stream, a) : type == FVS_F16 ? launch<__half>(stream, a) : launch<__nv_bfloat16>(stream, a);
}
