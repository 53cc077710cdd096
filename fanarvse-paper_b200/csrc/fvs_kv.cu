// Writing a paged key-value cache and reading it back (new: the reference ends with the found rows' ids; here the
// passages behind these ids have keys and values in pages).
//
// fvs_kv_append: rotates the query and key heads of new tokens by their positions and stores keys and values at their
// places.  fvs_kv_read: copies rows out as floating point.  Both move every byte once: a head of D elements is handled by
// D / 16 lanes (4 to 16 of them, in a group of 4, 8 or 16), each of which holds two chunks of 8 elements -- for a
// rotation by halves the chunks j and j + rot / 16, so that both elements of each pair are in the lane's registers.
#include "fvs_kv.cuh"

namespace fvs {
namespace kv {

constexpr int THREADS = 256;

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

// TYPE: of the new rows; STORE: of the cache (TYPE or int8); HALVES: pairs (i, i + rot/2), else neighbours (2i, 2i + 1)
template <int D, int TYPE, int STORE, bool HALVES>
__global__ void __launch_bounds__(THREADS) append_kernel(AppendArgs a) {
    using T = typename Elem<TYPE>::T;
    constexpr int L = Lanes<D>::group;
    const unsigned unit = blockIdx.x * (THREADS / L) + threadIdx.x / L;  // (token, row of its heads)
    const int j = threadIdx.x % L;
    const unsigned rows = a.hq + 2 * a.c.heads;
    const int token = (int)(unit / rows), row = (int)(unit % rows);
    const bool live = token < a.tokens && j < Lanes<D>::used;
    int page = 0, slot = 0, pos = 0;
    bool there = false;
    if (live) {
        const int t = __ldg(a.idx + token);
        pos = a.pos ? __ldg(a.pos + token) : t;
        there = place(a.c, a.tb, a.seq ? __ldg(a.seq + token) : token, t, page, slot);
        if (there && a.rot && (unsigned)pos >= (unsigned)a.positions) {
            atomicOr(a.c.status, BAD_INDEX);
            there = false;
        }
    }
    const bool is_q = row < a.hq, is_k = !is_q && row < a.hq + a.c.heads;
    const Heads& src = is_q ? a.q : is_k ? a.k : a.v;
    const int head = is_q ? row : is_k ? row - a.hq : row - a.hq - a.c.heads;
    // the lane's two chunks
    const int turning = a.rot / 16;  // lanes that rotate
    const bool turns = j < turning && (is_q || is_k);
    int e0, e1;
    if (HALVES && j < turning) {
        e0 = 8 * j;
        e1 = e0 + a.rot / 2;
    } else {
        e0 = 16 * j;
        e1 = e0 + 8;
    }
    float x0[8], x1[8];
    if (there) {
        const T* p = (const T*)src.at + token * src.token + head * src.head;
        up8<TYPE>(*(const uint4*)(p + e0), x0);
        up8<TYPE>(*(const uint4*)(p + e1), x1);
        if (turns) {
            // HALVES: pair i = e0 + n, n < 8; neighbours: pairs e0 / 2 + n
            const int64_t o = (int64_t)pos * (a.rot / 2) + 8 * j;
            const float4 c0 = __ldg((const float4*)(a.cos + o)), c1 = __ldg((const float4*)(a.cos + o + 4));
            const float4 s0 = __ldg((const float4*)(a.sin + o)), s1 = __ldg((const float4*)(a.sin + o + 4));
            const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
            const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
            if (HALVES) {
#pragma unroll
                for (int n = 0; n < 8; n++) turn(x0[n], x1[n], c[n], s[n]);
            } else {
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    turn(x0[2 * n], x0[2 * n + 1], c[n], s[n]);
                    turn(x1[2 * n], x1[2 * n + 1], c[4 + n], s[4 + n]);
                }
            }
        }
    } else {
#pragma unroll
        for (int n = 0; n < 8; n++) x0[n] = x1[n] = 0.f;
    }
    if (STORE == FVS_I8) {
        // the row's largest magnitude as ordered bits: a not-a-number is larger than infinity, so it is not lost
        uint32_t top = 0;
#pragma unroll
        for (int n = 0; n < 8; n++)
            top = max(top, max(__float_as_uint(x0[n]) & 0x7fffffffu, __float_as_uint(x1[n]) & 0x7fffffffu));
#pragma unroll
        for (int o = L / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (!is_q) {
            if (!there) return;
            const float m = __uint_as_float(top);
            const float inv = m > 0.f ? fminf(__fmul_rn(__frcp_rn(m), 127.f), 3.402823466e38f) : 0.f;
            uint32_t w[4];
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const float* x = n < 2 ? x0 : x1;
                w[n] = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int code = max(-127, min(127, __float2int_rn(__fmul_rn(x[(n & 1) * 4 + i], inv))));
                    w[n] |= (uint32_t)(code & 0xff) << (8 * i);
                }
            }
            int8_t* p = (int8_t*)(is_k ? a.c.k : a.c.v) + page * a.c.page_stride + head * a.c.head_stride +
                        slot * a.c.slot_stride;
            *(uint2*)(p + e0) = make_uint2(w[0], w[1]);
            *(uint2*)(p + e1) = make_uint2(w[2], w[3]);
            if (j == 0)
                (is_k ? a.c.k_scale : a.c.v_scale)[page * a.c.scale_page_stride + head * a.c.scale_head_stride +
                                                   slot * a.c.scale_slot_stride] = __fmul_rn(m, 1.f / 127.f);
            return;
        }
    }
    if (!live) return;
    T* p;
    if (is_q) {
        p = (T*)a.q_out + ((int64_t)token * a.hq + head) * D;  // zeros where the token has no place
    } else {
        if (!there) return;
        p = (T*)(is_k ? a.c.k : a.c.v) + page * a.c.page_stride + head * a.c.head_stride + slot * a.c.slot_stride;
    }
    *(uint4*)(p + e0) = down8<TYPE>(x0);
    *(uint4*)(p + e1) = down8<TYPE>(x1);
}

struct ReadArgs {
    fvs_kv_cache c;
    Table tb;
    void *k, *v;
    const int32_t *seq, *idx;
    int tokens;
};

// rows of the cache as TYPE, zeros where a token has no place: a lane moves 16 elements
template <int D, int STORE, int TYPE>
__global__ void __launch_bounds__(THREADS) read_kernel(ReadArgs a) {
    constexpr int L = D / 16;
    const unsigned unit = blockIdx.x * (THREADS / L) + threadIdx.x / L;
    const int j = threadIdx.x % L;
    const unsigned rows = 2 * a.c.heads;
    const int token = (int)(unit / rows), row = (int)(unit % rows);
    if (token >= a.tokens || threadIdx.x >= THREADS / L * L) return;
    const bool is_k = row < a.c.heads;
    const int head = is_k ? row : row - a.c.heads;
    int page, slot;
    const bool there =
        place(a.c, a.tb, a.seq ? __ldg(a.seq + token) : token, __ldg(a.idx + token), page, slot);
    float x[16];
#pragma unroll
    for (int n = 0; n < 16; n++) x[n] = 0.f;
    if (there) {
        const int64_t o = page * a.c.page_stride + head * a.c.head_stride + slot * a.c.slot_stride + 16 * j;
        if (STORE == FVS_I8) {
            const uint4 w4 = __ldg((const uint4*)((const int8_t*)(is_k ? a.c.k : a.c.v) + o));
            const float s = __ldg((is_k ? a.c.k_scale : a.c.v_scale) + page * a.c.scale_page_stride +
                                  head * a.c.scale_head_stride + slot * a.c.scale_slot_stride);
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int n = 0; n < 16; n++) x[n] = __fmul_rn((float)(int8_t)(w[n / 4] >> (8 * (n % 4))), s);
        } else {
            const uint16_t* p = (const uint16_t*)(is_k ? a.c.k : a.c.v) + o;
            float lo[8], hi[8];
            up8<STORE == FVS_I8 ? FVS_F16 : STORE>(__ldg((const uint4*)p), lo);
            up8<STORE == FVS_I8 ? FVS_F16 : STORE>(__ldg((const uint4*)(p + 8)), hi);
#pragma unroll
            for (int n = 0; n < 8; n++) x[n] = lo[n], x[8 + n] = hi[n];
        }
    }
    const int64_t o = ((int64_t)token * a.c.heads + head) * D + 16 * j;
    void* out = is_k ? a.k : a.v;
    if (TYPE == FVS_F32) {
#pragma unroll
        for (int n = 0; n < 4; n++)
            *(float4*)((float*)out + o + 4 * n) = make_float4(x[4 * n], x[4 * n + 1], x[4 * n + 2], x[4 * n + 3]);
    } else {
        float lo[8], hi[8];
#pragma unroll
        for (int n = 0; n < 8; n++) lo[n] = x[n], hi[n] = x[8 + n];
        uint4* p = (uint4*)((uint16_t*)out + o);
        p[0] = down8<TYPE == FVS_F32 ? FVS_F16 : TYPE>(lo);
        p[1] = down8<TYPE == FVS_F32 ? FVS_F16 : TYPE>(hi);
    }
}

static bool heads_ok(const void* p, int64_t token, int64_t head, int d) {
    return p && ((uintptr_t)p & 15) == 0 && token % 8 == 0 && head % 8 == 0 && token >= 0 && (head >= d || head == 0);
}

template <int D>
static void launch_append(fvs_stream_t stream, const AppendArgs& a, int type, bool halves) {
    constexpr unsigned per = THREADS / Lanes<D>::group;
    const unsigned grid = ((unsigned)a.tokens * (a.hq + 2 * a.c.heads) + per - 1) / per;
    const bool i8 = a.c.type == FVS_I8;
    if (type == FVS_F16) {
        if (i8)
            halves ? append_kernel<D, FVS_F16, FVS_I8, true><<<grid, THREADS, 0, stream>>>(a)
                   : append_kernel<D, FVS_F16, FVS_I8, false><<<grid, THREADS, 0, stream>>>(a);
        else
            halves ? append_kernel<D, FVS_F16, FVS_F16, true><<<grid, THREADS, 0, stream>>>(a)
                   : append_kernel<D, FVS_F16, FVS_F16, false><<<grid, THREADS, 0, stream>>>(a);
    } else {
        if (i8)
            halves ? append_kernel<D, FVS_BF16, FVS_I8, true><<<grid, THREADS, 0, stream>>>(a)
                   : append_kernel<D, FVS_BF16, FVS_I8, false><<<grid, THREADS, 0, stream>>>(a);
        else
            halves ? append_kernel<D, FVS_BF16, FVS_BF16, true><<<grid, THREADS, 0, stream>>>(a)
                   : append_kernel<D, FVS_BF16, FVS_BF16, false><<<grid, THREADS, 0, stream>>>(a);
    }
}

template <int D, int STORE>
static void launch_read(fvs_stream_t stream, const ReadArgs& a, int type) {
    constexpr unsigned per = THREADS / (D / 16);
    const unsigned grid = ((unsigned)a.tokens * 2 * a.c.heads + per - 1) / per;
    if (type == FVS_F16)
        read_kernel<D, STORE, FVS_F16><<<grid, THREADS, 0, stream>>>(a);
    else if (type == FVS_BF16)
        read_kernel<D, STORE, FVS_BF16><<<grid, THREADS, 0, stream>>>(a);
    else
        read_kernel<D, STORE, FVS_F32><<<grid, THREADS, 0, stream>>>(a);
}

}  // namespace kv
}  // namespace fvs

using namespace fvs::kv;

extern "C" int fvs_kv_append(fvs_stream_t stream, const fvs_kv_cache* cache, int type, const void* k, int64_t k_token,
                             int64_t k_head, const void* v, int64_t v_token, int64_t v_head, const void* q,
                             int64_t q_token, int64_t q_head, int hq, void* q_out, const int32_t* table, int seqs,
                             int wide, int64_t table_stride, const int32_t* seq, const int32_t* idx,
                             const int32_t* pos, int tokens, const float* cos, const float* sin, int positions,
                             int rot, int pairs) {
    if (int rc = check_cache(cache)) return rc;
    FVS_CHECK_ARG(type == FVS_F16 || type == FVS_BF16);
    FVS_CHECK_ARG(cache->type == FVS_I8 || cache->type == type);
    FVS_CHECK_ARG(tokens >= 0 && hq >= 0 && rot >= 0 && (pairs == FVS_PAIRS_HALVES || pairs == FVS_PAIRS_NEIGHBOURS));
    if (tokens == 0) return FVS_OK;
    if (int rc = check_table(table, seqs, wide, table_stride)) return rc;
    FVS_CHECK_ARG(idx && (seq || tokens <= seqs));
    FVS_CHECK_ARG(heads_ok(k, k_token, k_head, cache->dim) && heads_ok(v, v_token, v_head, cache->dim));
    if (hq) FVS_CHECK_ARG(heads_ok(q, q_token, q_head, cache->dim) && q_out && ((uintptr_t)q_out & 15) == 0);
    if (rot)
        FVS_CHECK_ARG(rot % 16 == 0 && rot <= cache->dim && cos && sin && positions >= 1 &&
                      (((uintptr_t)cos | (uintptr_t)sin) & 15) == 0);
    if ((int64_t)tokens * (hq + 2 * (int64_t)cache->heads) > 0x7fffff00ll) return FVS_ERANGE;
    AppendArgs a{*cache, {table, table_stride, seqs, wide}, {k, k_token, k_head}, {v, v_token, v_head},
                 {q, q_token, q_head}, q_out, seq, idx, pos, cos, sin, hq, tokens, positions, rot};
    const bool halves = pairs == FVS_PAIRS_HALVES;
    switch (cache->dim) {
        case 64: launch_append<64>(stream, a, type, halves); break;
        case 96: launch_append<96>(stream, a, type, halves); break;
        case 128: launch_append<128>(stream, a, type, halves); break;
        case 192: launch_append<192>(stream, a, type, halves); break;
        default: launch_append<256>(stream, a, type, halves); break;
    }
    return fvs_launch_status();
}

extern "C" int fvs_kv_read(fvs_stream_t stream, const fvs_kv_cache* cache, int type, void* k, void* v,
                           const int32_t* table, int seqs, int wide, int64_t table_stride, const int32_t* seq,
                           const int32_t* idx, int tokens) {
    if (int rc = check_cache(cache)) return rc;
    FVS_CHECK_ARG(type == FVS_F16 || type == FVS_BF16 || type == FVS_F32);
    FVS_CHECK_ARG(tokens >= 0);
    if (tokens == 0) return FVS_OK;
    if (int rc = check_table(table, seqs, wide, table_stride)) return rc;
    FVS_CHECK_ARG(idx && (seq || tokens <= seqs) && k && v && (((uintptr_t)k | (uintptr_t)v) & 15) == 0);
    if ((int64_t)tokens * 2 * cache->heads > 0x7fffff00ll) return FVS_ERANGE;
    ReadArgs a{*cache, {table, table_stride, seqs, wide}, k, v, seq, idx, tokens};
#define FVS_KV_READ(D)                                                                     \
    (cache->type == FVS_I8    ? launch_read<D, FVS_I8>(stream, a, type)                    \
     : cache->type == FVS_F16 ? launch_read<D, FVS_F16>(stream, a, type)                   \
                              : launch_read<D, FVS_BF16>(stream, a, type))
    switch (cache->dim) {
        case 64: FVS_KV_READ(64); break;
        case 96: FVS_KV_READ(96); break;
        case 128: FVS_KV_READ(128); break;
        case 192: FVS_KV_READ(192); break;
        default: FVS_KV_READ(256); break;
    }
#undef FVS_KV_READ
    return fvs_launch_status();
}
