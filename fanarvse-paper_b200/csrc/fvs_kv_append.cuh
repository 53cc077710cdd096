// Appending to a paged key-value cache: the kernel of fvs_kv_append and fvs_kv_append_norm.
//
// What counts is bytes on the way: a warp loads up to 16 heads of one token's q, k or v (under way while the token's place,
// its cosines and the norm's weights are looked up), then stores them and ends; nothing is done one after another.  A head
// of D elements is D / 16 lanes' (in a group of 4, 8 or 16; each lane holds two chunks of 8 elements, those that a rotation
// by halves pairs), so that the sum of a norm is one or two exchanges among its lanes' group.
#pragma once
#include "fvs_kv.cuh"

namespace fvs {
namespace kv {

constexpr int THREADS = 256;
// loads of a lane that are on the way together: 35 us with two at 9000 tokens of 48 heads of 64 (39 with one or four: a
// lane's work after them, or its registers, grow)
constexpr int BATCH = 2;

struct Heads {  // token and head strides in elements
    const void* at;
    int64_t token, head;
};

struct AppendArgs {
    fvs_kv_cache c;
    Table tb;
    Heads k, v, q;
    void* q_out;
    const int32_t *seq, *idx, *pos;
    const float *cos, *sin;
    int hq, tokens, positions, rot;
    int q_warps, k_warps;  // of a token for q and for k (as many for v)
    const void *q_weight, *k_weight;  // of the norms [dim], null: that head is not normed
    int weight_f32;                   // else of the new rows' type
    float eps;
};

// lanes of a head of D elements
template <int D>
struct Lanes {
    static constexpr int used = D / 16;
    static constexpr int group = used <= 4 ? 4 : used <= 8 ? 8 : 16;
};

// (a, b) -> (a cos - b sin, b cos + a sin): each product and sum rounded by itself, so that the stored codes are those of
// the same expression elsewhere
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
    const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    a = x;
}

// four values as rounded int8 (half to even; at most 127 in magnitude here, 0 for a not-a-number)
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    uint32_t r;
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(r) : "r"(__float2int_rn(d)), "r"(__float2int_rn(c)));
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(__float2int_rn(b)), "r"(__float2int_rn(a)), "r"(r));
    return r;
}

// the larger magnitude; not-a-numbers stay
__device__ __forceinline__ float max_abs(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}

// TYPE: of the new rows; STORE: of the cache (TYPE or int8); HALVES: pairs (i, i + rot/2), else neighbours (2i, 2i + 1);
// NORM: x -> x / sqrt(mean x^2 + eps) * weight before the rotation, for the heads that have weights
template <int D, int TYPE, int STORE, bool HALVES, bool NORM>
__global__ void __launch_bounds__(THREADS) append_kernel(AppendArgs a) {
    using T = typename Elem<TYPE>::T;
    constexpr int L = Lanes<D>::group, AT_ONCE = 32 / L;
    const unsigned w = blockIdx.x * (THREADS / 32) + threadIdx.x / 32, warps = a.q_warps + 2 * a.k_warps;
    const int token = (int)(w / warps);
    if (token >= a.tokens) return;
    const int lane = threadIdx.x & 31, j = lane % L, sub = lane / L;
    // this warp's heads of q, k or v
    int part = (int)(w % warps);
    const bool is_q = part < a.q_warps;
    if (!is_q) part -= a.q_warps;
    const bool is_k = !is_q && part < a.k_warps;
    if (!is_q && !is_k) part -= a.k_warps;
    const Heads src = is_q ? a.q : is_k ? a.k : a.v;
    const int heads = is_q ? a.hq : a.c.heads, share = is_q ? a.q_warps : a.k_warps;
    const int per = ((heads + share - 1) / share + AT_ONCE - 1) / AT_ONCE * AT_ONCE;
    const int head0 = part * per + sub, end = min(heads, part * per + per), count = end - part * per;
    // the lane's two chunks, of neighbouring lanes side by side in memory
    int e0, e1;
    bool turn0, turn1;
    const int turning = a.rot / 16;
    if (HALVES) {
        turn0 = turn1 = j < turning;
        e0 = turn0 ? 8 * j : a.rot + 8 * (j - turning);
        e1 = e0 + (turn0 ? a.rot / 2 : (D - a.rot) / 2);
    } else {
        e0 = 8 * j;
        e1 = e0 + D / 2;
        turn0 = e0 < a.rot;
        turn1 = e1 < a.rot;
    }
    const bool used = j < Lanes<D>::used;
    uint4 raw[BATCH][2];
    const T* from = (const T*)src.at + token * src.token + head0 * src.head;
#pragma unroll
    for (int u = 0; u < BATCH; u++) {
        raw[u][0] = raw[u][1] = make_uint4(0, 0, 0, 0);
        if (u * AT_ONCE < count && used && head0 + u * AT_ONCE < end) {
            raw[u][0] = *(const uint4*)(from + e0);
            raw[u][1] = *(const uint4*)(from + e1);
        }
        from += AT_ONCE * src.head;
    }
    const void* weight = !NORM ? nullptr : is_q ? a.q_weight : is_k ? a.k_weight : nullptr;  // the same for a whole warp
    float w0[8], w1[8];
    if (NORM && weight && used) {
        if (a.weight_f32) {
            const float *p0 = (const float*)weight + e0, *p1 = (const float*)weight + e1;
            *(float4*)w0 = __ldg((const float4*)p0), *(float4*)(w0 + 4) = __ldg((const float4*)p0 + 1);
            *(float4*)w1 = __ldg((const float4*)p1), *(float4*)(w1 + 4) = __ldg((const float4*)p1 + 1);
        } else {
            up8<TYPE>(__ldg((const uint4*)((const T*)weight + e0)), w0);
            up8<TYPE>(__ldg((const uint4*)((const T*)weight + e1)), w1);
        }
    }
    int page = 0, slot = 0;
    const int t = __ldg(a.idx + token), pos = a.pos ? __ldg(a.pos + token) : t;
    bool there = place(a.c, a.tb, a.seq ? __ldg(a.seq + token) : token, t, page, slot);
    if (there && a.rot && (unsigned)pos >= (unsigned)a.positions) {
        atomicOr(a.c.status, BAD_INDEX);
        there = false;
    }
    float c[8], s[8];
    const bool turns = (is_q || is_k) && there && used && (turn0 || turn1);
    if (turns) {
        const float *pc = a.cos + (int64_t)pos * (a.rot / 2), *ps = a.sin + (int64_t)pos * (a.rot / 2);
        const int o0 = HALVES ? e0 : e0 / 2, o1 = HALVES ? e0 + 4 : turn1 ? e1 / 2 : o0;
        *(float4*)c = __ldg((const float4*)(pc + o0));
        *(float4*)s = __ldg((const float4*)(ps + o0));
        *(float4*)(c + 4) = __ldg((const float4*)(pc + o1));
        *(float4*)(s + 4) = __ldg((const float4*)(ps + o1));
    }
    if (!there && !is_q) return;  // a whole warp
    const int64_t to_scale = page * a.c.scale_page_stride + slot * a.c.scale_slot_stride + head0 * a.c.scale_head_stride;
    const int64_t to = is_q ? ((int64_t)token * a.hq + head0) * D
                            : page * a.c.page_stride + slot * a.c.slot_stride + head0 * a.c.head_stride;
    const int64_t step = is_q ? AT_ONCE * D : AT_ONCE * a.c.head_stride;
    void* dst = is_q ? a.q_out : is_k ? a.c.k : a.c.v;
#pragma unroll
    for (int u = 0; u < BATCH; u++) {
        if (u * AT_ONCE >= count) break;  // a whole warp
        const bool live = used && head0 + u * AT_ONCE < end;
        const bool codes = STORE == FVS_I8 && !is_q;
        float x0[8], x1[8];
        const bool norms = NORM && weight && there;  // the same for a whole warp
        if (turns || codes || norms) {
            up8<TYPE>(raw[u][0], x0);
            up8<TYPE>(raw[u][1], x1);
        }
        if (norms) {  // lanes without a part of the head hold zeros
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < 8; n++) sum = fmaf(x0[n], x0[n], fmaf(x1[n], x1[n], sum));
#pragma unroll
            for (int o = L / 2; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float r = __frsqrt_rn(fmaf(sum, 1.f / D, a.eps));
            if (used) {
#pragma unroll
                for (int n = 0; n < 8; n++) x0[n] = x0[n] * r * w0[n], x1[n] = x1[n] * r * w1[n];
            }
        }
        if (turns) {
            if (HALVES) {
#pragma unroll
                for (int n = 0; n < 8; n++) turn(x0[n], x1[n], c[n], s[n]);
            } else {
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    turn(x0[2 * n], x0[2 * n + 1], c[n], s[n]);
                    if (turn1) turn(x1[2 * n], x1[2 * n + 1], c[4 + n], s[4 + n]);
                }
            }
        }
        if (codes) {
            float m = 0.f;
#pragma unroll
            for (int n = 0; n < 8; n++) m = max_abs(m, max_abs(x0[n], x1[n]));
#pragma unroll
            for (int o = L / 2; o; o >>= 1) m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (!live) continue;
            const float scale = m < 0x1p-126f ? 0.f : __fmul_rn(m, 1.f / 127.f);
            if (m < 0x1p-100f) {  // 127 / m could be infinite: the row 2^64 larger has the same codes.  Subnormal rows: zeros
                const float up = m < 0x1p-126f ? 0.f : 0x1p64f;
                m *= up;
#pragma unroll
                for (int n = 0; n < 8; n++) x0[n] *= up, x1[n] *= up;
            }
            const float inv = m > 0.f ? __fmul_rn(__frcp_rn(m), 127.f) : 0.f;
            uint32_t code[4];
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const float* x = (n < 2 ? x0 : x1) + (n & 1) * 4;
                code[n] = codes4(__fmul_rn(x[0], inv), __fmul_rn(x[1], inv), __fmul_rn(x[2], inv), __fmul_rn(x[3], inv));
            }
            int8_t* p = (int8_t*)dst + to + u * step;
            *(uint2*)(p + e0) = make_uint2(code[0], code[1]);
            *(uint2*)(p + e1) = make_uint2(code[2], code[3]);
            if (j == 0) (is_k ? a.c.k_scale : a.c.v_scale)[to_scale + u * AT_ONCE * a.c.scale_head_stride] = scale;
        } else if (live) {
            if (turns || norms) raw[u][0] = down8<TYPE>(x0), raw[u][1] = down8<TYPE>(x1);
            if (!there) raw[u][0] = raw[u][1] = make_uint4(0, 0, 0, 0);  // a query without a place
            T* p = (T*)dst + to + u * step;
            *(uint4*)(p + e0) = raw[u][0];
            *(uint4*)(p + e1) = raw[u][1];
        }
    }
}

static bool heads_ok(const void* p, int64_t token, int64_t head, int d) {
    return p && ((uintptr_t)p & 15) == 0 && token % 8 == 0 && head % 8 == 0 && token >= 0 && (head >= d || head == 0);
}

template <int D, bool NORM>
static void launch_append(fvs_stream_t stream, AppendArgs a, int type, bool halves) {
    constexpr int most = 32 / Lanes<D>::group * BATCH;  // heads of a warp
    a.q_warps = (a.hq + most - 1) / most;
    a.k_warps = (a.c.heads + most - 1) / most;
    const int64_t warps = (int64_t)a.tokens * (a.q_warps + 2 * a.k_warps);
    const unsigned grid = (unsigned)((warps + THREADS / 32 - 1) / (THREADS / 32));
    const bool i8 = a.c.type == FVS_I8;
    if (type == FVS_F16) {
        if (i8)
            halves ? append_kernel<D, FVS_F16, FVS_I8, true, NORM><<<grid, THREADS, 0, stream>>>(a)
                   : append_kernel<D, FVS_F16, FVS_I8, false, NORM><<<grid, THREADS, 0, stream>>>(a);
        else
            halves ? append_kernel<D, FVS_F16, FVS_F16, true, NORM><<<grid, THREADS, 0, stream>>>(a)
                   : append_kernel<D, FVS_F16, FVS_F16, false, NORM><<<grid, THREADS, 0, stream>>>(a);
    } else {
        if (i8)
            halves ? append_kernel<D, FVS_BF16, FVS_I8, true, NORM><<<grid, THREADS, 0, stream>>>(a)
                   : append_kernel<D, FVS_BF16, FVS_I8, false, NORM><<<grid, THREADS, 0, stream>>>(a);
        else
            halves ? append_kernel<D, FVS_BF16, FVS_BF16, true, NORM><<<grid, THREADS, 0, stream>>>(a)
                   : append_kernel<D, FVS_BF16, FVS_BF16, false, NORM><<<grid, THREADS, 0, stream>>>(a);
    }
}

// host: the checks that both entry points make; fills a (tokens 0: nothing to do)
static inline int append_args(AppendArgs& a, const fvs_kv_cache* cache, int type, const void* k, int64_t k_token,
                              int64_t k_head, const void* v, int64_t v_token, int64_t v_head, const void* q,
                              int64_t q_token, int64_t q_head, int hq, void* q_out, const int32_t* table, int seqs,
                              int wide, int64_t table_stride, const int32_t* seq, const int32_t* idx,
                              const int32_t* pos, int tokens, const float* cos, const float* sin, int positions,
                              int rot, int pairs) {
    if (int rc = check_cache(cache)) return rc;
    FVS_CHECK_ARG(type == FVS_F16 || type == FVS_BF16);
    FVS_CHECK_ARG(cache->type == FVS_I8 || cache->type == type);
    FVS_CHECK_ARG(tokens >= 0 && hq >= 0 && rot >= 0 && (pairs == FVS_PAIRS_HALVES || pairs == FVS_PAIRS_NEIGHBOURS));
    if (tokens == 0) {
        a.tokens = 0;
        return FVS_OK;
    }
    if (int rc = check_table(table, seqs, wide, table_stride)) return rc;
    FVS_CHECK_ARG(idx && (seq || tokens <= seqs));
    FVS_CHECK_ARG(heads_ok(k, k_token, k_head, cache->dim) && heads_ok(v, v_token, v_head, cache->dim));
    if (hq) FVS_CHECK_ARG(heads_ok(q, q_token, q_head, cache->dim) && q_out && ((uintptr_t)q_out & 15) == 0);
    if (rot)
        FVS_CHECK_ARG(rot % 16 == 0 && rot <= cache->dim && cos && sin && positions >= 1 &&
                      (((uintptr_t)cos | (uintptr_t)sin) & 15) == 0);
    if ((int64_t)tokens * (hq + 2 * (int64_t)cache->heads) > 0x7fffff00ll) return FVS_ERANGE;
    a = AppendArgs{*cache, {table, table_stride, seqs, wide}, {k, k_token, k_head}, {v, v_token, v_head},
                 {q, q_token, q_head}, q_out, seq, idx, pos, cos, sin, hq, tokens, positions, rot, 0, 0, nullptr, nullptr, 0, 0.f};
    return FVS_OK;
}

template <bool NORM>
static int append_launch(fvs_stream_t stream, const AppendArgs& a, int type, bool halves) {
    if (a.tokens == 0) return FVS_OK;
    switch (a.c.dim) {
        case 64: launch_append<64, NORM>(stream, a, type, halves); break;
        case 96: launch_append<96, NORM>(stream, a, type, halves); break;
        case 128: launch_append<128, NORM>(stream, a, type, halves); break;
        case 192: launch_append<192, NORM>(stream, a, type, halves); break;
        default: launch_append<256, NORM>(stream, a, type, halves); break;
    }
    return fvs_launch_status();
}

}  // namespace kv
}  // namespace fvs
