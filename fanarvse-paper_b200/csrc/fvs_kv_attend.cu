// Attention of one new token per sequence over a paged key-value cache (new; see include/fanar_b200.h).
//
// One pass over the keys with the running maximum m and sum l of the softmax: a tile of keys with scores s changes them to
// m' = max(m, max s), l' = l e^(m - m') + sum e^(s - m'), and the accumulated output by o' = o e^(m - m') + sum
// e^(s - m') v.  Scores are kept in units of log2 (scale * log2 e folded into q), all of it in fp32.
#include "fvs_kv.cuh"

namespace fvs {
namespace kv {

struct AttendArgs {
    fvs_kv_cache c;
    Table tb;
    const void* q;
    int64_t q_seq, q_head;
    const int32_t* lens;
    void* out;
    float* lse;
    int hq;
    float scale2;  // scale * log2 e
};

constexpr int THREADS = 128;

template <int TYPE>
__device__ __forceinline__ float element(const void* p, int64_t i) {
    if (TYPE == FVS_F16) return __half2float(((const __half*)p)[i]);
    if (TYPE == FVS_BF16) return __bfloat162float(((const __nv_bfloat16*)p)[i]);
    return (float)((const int8_t*)p)[i];
}

__device__ __forceinline__ float block_reduce(float x, bool is_max, float* scratch) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float y = __shfl_xor_sync(0xffffffffu, x, o);
        x = is_max ? fmaxf(x, y) : x + y;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    x = scratch[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; w++) x = is_max ? fmaxf(x, scratch[w]) : x + scratch[w];
    return x;
}

// One CTA per (query head, sequence): a thread scores one key of a tile of 128, then owns output elements.
template <int TYPE, int STORE>
__global__ void __launch_bounds__(THREADS) attend_kernel(AttendArgs a) {
    __shared__ float sq[256], sp[THREADS], scratch[THREADS / 32];
    __shared__ int64_t srow[THREADS];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, D = a.c.dim;
    const int kvh = h / (a.hq / a.c.heads);
    for (int i = tid; i < D; i += THREADS)
        sq[i] = element<TYPE>(a.q, b * a.q_seq + h * a.q_head + i) * a.scale2;
    int len = __ldg(a.lens + b);
    if (len > (int64_t)a.tb.wide * a.c.page) {
        len = a.tb.wide * a.c.page;
        atomicOr(a.c.status, BAD_INDEX);
    }
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    __syncthreads();
    for (int t0 = 0; t0 < len; t0 += THREADS) {
        const int t = t0 + tid;
        int page, slot;
        bool seen = t < len && place(a.c, a.tb, b, t, page, slot);
        if (seen && a.c.fill) seen = slot < __ldg(a.c.fill + page);
        float s = -INFINITY;
        srow[tid] = -1;
        float vs = 1.f;
        if (seen) {
            const int64_t row = page * a.c.page_stride + kvh * a.c.head_stride + slot * a.c.slot_stride;
            srow[tid] = row;
            float dot = 0.f;
            for (int i = 0; i < D; i++) dot = fmaf(sq[i], element<STORE>(a.c.k, row + i), dot);
            s = dot;
            if (STORE == FVS_I8) {
                const int64_t at = page * a.c.scale_page_stride + kvh * a.c.scale_head_stride + slot * a.c.scale_slot_stride;
                s *= __ldg(a.c.k_scale + at);
                vs = __ldg(a.c.v_scale + at);
            }
        }
        const float m1 = fmaxf(m, block_reduce(s, true, scratch));
        const float base = m1 == -INFINITY ? 0.f : m1;
        const float p = exp2f(s - base), corr = exp2f(m - base);
        l = l * corr + block_reduce(seen ? p : 0.f, false, scratch);
        sp[tid] = p * vs;
        m = m1;
        __syncthreads();
        o0 *= corr;
        o1 *= corr;
        for (int n = 0; n < min(THREADS, len - t0); n++) {
            const int64_t row = srow[n];
            if (row < 0) continue;
            if (tid < D) o0 = fmaf(sp[n], element<STORE>(a.c.v, row + tid), o0);
            if (tid + THREADS < D) o1 = fmaf(sp[n], element<STORE>(a.c.v, row + tid + THREADS), o1);
        }
        __syncthreads();
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t o = ((int64_t)b * a.hq + h) * D;
    for (int n = 0; n < 2; n++) {
        const int i = tid + n * THREADS;
        const float x = l == 0.f ? 0.f : (n ? o1 : o0) * inv;
        if (i >= D) break;
        if (TYPE == FVS_F16)
            ((__half*)a.out)[o + i] = __float2half_rn(x);
        else
            ((__nv_bfloat16*)a.out)[o + i] = __float2bfloat16_rn(x);
    }
    if (tid == 0 && a.lse) a.lse[(int64_t)b * a.hq + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace kv
}  // namespace fvs

using namespace fvs::kv;

extern "C" int fvs_kv_attend_work(int seqs, int hq, int dim) {
    if (seqs < 1 || hq < 1 || dim < 1) return FVS_EINVAL;
    if ((int64_t)seqs * hq > (1 << 28)) return FVS_ERANGE;
    return seqs * hq * 4;
}

extern "C" int fvs_kv_attend(fvs_stream_t stream, const fvs_kv_cache* cache, int type, const void* q, int64_t q_seq,
                             int64_t q_head, int hq, const int32_t* table, int seqs, int wide, int64_t table_stride,
                             const int32_t* lens, float scale, void* out, float* lse, void* work) {
    if (int rc = check_cache(cache)) return rc;
    FVS_CHECK_ARG(type == FVS_F16 || type == FVS_BF16);
    FVS_CHECK_ARG(cache->type == FVS_I8 || cache->type == type);
    FVS_CHECK_ARG(seqs >= 0 && hq >= 1 && hq % cache->heads == 0);
    if (seqs == 0) return FVS_OK;
    if (int rc = check_table(table, seqs, wide, table_stride)) return rc;
    FVS_CHECK_ARG(q && ((uintptr_t)q & 15) == 0 && q_seq % 8 == 0 && q_head % 8 == 0 && q_seq >= 0 && q_head >= 0);
    FVS_CHECK_ARG(lens && out && ((uintptr_t)out & 15) == 0 && work && ((uintptr_t)work & 15) == 0);
    if (seqs > 65535) return FVS_ERANGE;
    AttendArgs a{*cache, {table, table_stride, seqs, wide}, q, q_seq, q_head, lens, out, lse, hq,
                 scale * 1.4426950408889634f};
    const dim3 grid(hq, seqs);
    if (type == FVS_F16) {
        if (cache->type == FVS_I8)
            attend_kernel<FVS_F16, FVS_I8><<<grid, THREADS, 0, stream>>>(a);
        else
            attend_kernel<FVS_F16, FVS_F16><<<grid, THREADS, 0, stream>>>(a);
    } else {
        if (cache->type == FVS_I8)
            attend_kernel<FVS_BF16, FVS_I8><<<grid, THREADS, 0, stream>>>(a);
        else
            attend_kernel<FVS_BF16, FVS_BF16><<<grid, THREADS, 0, stream>>>(a);
    }
    return fvs_launch_status();
}
