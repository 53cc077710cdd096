// Writing a paged key-value cache and reading it back (new: the reference ends with the found rows' ids; here the
// passages behind these ids have keys and values in pages).
//
// fvs_kv_append: rotates the query and key heads of new tokens by their positions and stores keys and values at their
// places.  fvs_kv_read: copies rows out as floating point.  Both move every byte once and are bound by memory.  A warp
// works for one token: its place and its cosines are looked up once, then it takes the token's heads (of q, k and v in
// turn) a few at a time with the next heads' loads in flight.  A head of D elements is D / 16 lanes' (append: in a group of
// 4, 8 or 16; each lane holds two chunks of 8 elements, those that a rotation by halves pairs) or D / 8 lanes' (read).
// With few tokens a token's heads are spread over several warps.
#include "fvs_kv.cuh"

namespace fvs {
namespace kv {

constexpr int THREADS = 256;
constexpr int BATCH = 4;  // heads of a lane whose loads are in flight together

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
    int spread;  // warps of a token
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
    constexpr int L = Lanes<D>::group, AT_ONCE = 32 / L;
    const unsigned w = blockIdx.x * (THREADS / 32) + threadIdx.x / 32;
    const int token = (int)(w / (unsigned)a.spread);
    if (token >= a.tokens) return;
    const int lane = threadIdx.x & 31, j = lane % L, sub = lane / L;
    const int rows = a.hq + 2 * a.c.heads;
    // this warp's heads
    const int per = ((rows + a.spread - 1) / a.spread + AT_ONCE - 1) / AT_ONCE * AT_ONCE;
    const int begin = (int)(w % (unsigned)a.spread) * per, end = min(rows, begin + per);
    int page = 0, slot = 0;
    const int t = __ldg(a.idx + token), pos = a.pos ? __ldg(a.pos + token) : t;
    bool there = place(a.c, a.tb, a.seq ? __ldg(a.seq + token) : token, t, page, slot);
    if (there && a.rot && (unsigned)pos >= (unsigned)a.positions) {
        atomicOr(a.c.status, BAD_INDEX);
        there = false;
    }
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
    float c[8], s[8];
#pragma unroll
    for (int n = 0; n < 8; n++) c[n] = 1.f, s[n] = 0.f;
    if (there && used && (turn0 || turn1)) {
        const float *pc = a.cos + (int64_t)pos * (a.rot / 2), *ps = a.sin + (int64_t)pos * (a.rot / 2);
        const int o0 = HALVES ? e0 : e0 / 2, o1 = HALVES ? e0 + 4 : e1 / 2;
        *(float4*)c = __ldg((const float4*)(pc + o0));
        *(float4*)s = __ldg((const float4*)(ps + o0));
        if (HALVES || turn1) {
            *(float4*)(c + 4) = __ldg((const float4*)(pc + o1));
            *(float4*)(s + 4) = __ldg((const float4*)(ps + o1));
        }
    }
    const int64_t to = page * a.c.page_stride + slot * a.c.slot_stride;
    const int64_t to_scale = page * a.c.scale_page_stride + slot * a.c.scale_slot_stride;
    for (int row0 = begin; row0 < end; row0 += AT_ONCE * BATCH) {
        uint4 raw[BATCH][2];
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            const int row = row0 + u * AT_ONCE + sub;
            raw[u][0] = raw[u][1] = make_uint4(0, 0, 0, 0);
            if (there && used && row < end) {
                const bool is_q = row < a.hq, is_k = row < a.hq + a.c.heads;
                const Heads& src = is_q ? a.q : is_k ? a.k : a.v;
                const int head = is_q ? row : is_k ? row - a.hq : row - a.hq - a.c.heads;
                const T* p = (const T*)src.at + token * src.token + head * src.head;
                raw[u][0] = *(const uint4*)(p + e0);
                raw[u][1] = *(const uint4*)(p + e1);
            }
        }
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            const int row = row0 + u * AT_ONCE + sub;
            const bool is_q = row < a.hq, is_k = !is_q && row < a.hq + a.c.heads;
            const int head = is_q ? row : is_k ? row - a.hq : row - a.hq - a.c.heads;
            float x0[8], x1[8];
            up8<TYPE>(raw[u][0], x0);
            up8<TYPE>(raw[u][1], x1);
            if (is_q || is_k) {
                if (HALVES) {
                    if (turn0) {
#pragma unroll
                        for (int n = 0; n < 8; n++) turn(x0[n], x1[n], c[n], s[n]);
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        if (turn0) turn(x0[2 * n], x0[2 * n + 1], c[n], s[n]);
                        if (turn1) turn(x1[2 * n], x1[2 * n + 1], c[4 + n], s[4 + n]);
                    }
                }
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
                    if (!there || !used || row >= end) continue;
                    const float m = __uint_as_float(top);
                    const float inv = m > 0.f ? fminf(__fmul_rn(__frcp_rn(m), 127.f), 3.402823466e38f) : 0.f;
                    uint32_t code[4];
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        const float* x = n < 2 ? x0 : x1;
                        code[n] = 0;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int y = max(-127, min(127, __float2int_rn(__fmul_rn(x[(n & 1) * 4 + i], inv))));
                            code[n] |= (uint32_t)(y & 0xff) << (8 * i);
                        }
                    }
                    int8_t* p = (int8_t*)(is_k ? a.c.k : a.c.v) + to + head * a.c.head_stride;
                    *(uint2*)(p + e0) = make_uint2(code[0], code[1]);
                    *(uint2*)(p + e1) = make_uint2(code[2], code[3]);
                    if (j == 0)
                        (is_k ? a.c.k_scale : a.c.v_scale)[to_scale + head * a.c.scale_head_stride] = __fmul_rn(m, 1.f / 127.f);
                    continue;
                }
            }
            if (!used || row >= end || (!is_q && !there)) continue;
            T* p = is_q ? (T*)a.q_out + ((int64_t)token * a.hq + head) * D  // zeros where the token has no place
                        : (T*)(is_k ? a.c.k : a.c.v) + to + head * a.c.head_stride;
            *(uint4*)(p + e0) = down8<TYPE>(x0);
            *(uint4*)(p + e1) = down8<TYPE>(x1);
        }
    }
}

struct ReadArgs {
    fvs_kv_cache c;
    Table tb;
    void *k, *v;
    const int32_t *seq, *idx;
    int tokens, spread;
};

// rows of the cache as TYPE, zeros where a token has no place: a lane moves 8 elements of a row
template <int D, int STORE, int TYPE>
__global__ void __launch_bounds__(THREADS) read_kernel(ReadArgs a) {
    constexpr int L = D / 8, AT_ONCE = 32 / L, ESZ = STORE == FVS_I8 ? 1 : 2;
    const unsigned w = blockIdx.x * (THREADS / 32) + threadIdx.x / 32;
    const int token = (int)(w / (unsigned)a.spread);
    if (token >= a.tokens) return;
    const int lane = threadIdx.x & 31, e = lane % L * 8, sub = lane / L;
    const int rows = 2 * a.c.heads;
    const int per = ((rows + a.spread - 1) / a.spread + AT_ONCE - 1) / AT_ONCE * AT_ONCE;
    const int begin = (int)(w % (unsigned)a.spread) * per, end = min(rows, begin + per);
    int page = 0, slot = 0;
    const bool there = place(a.c, a.tb, a.seq ? __ldg(a.seq + token) : token, __ldg(a.idx + token), page, slot);
    const int64_t from = page * a.c.page_stride + slot * a.c.slot_stride + e;
    const int64_t from_scale = page * a.c.scale_page_stride + slot * a.c.scale_slot_stride;
    for (int row0 = begin; row0 < end; row0 += AT_ONCE * BATCH) {
        uint4 raw[BATCH];
        float scale[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            const int row = row0 + u * AT_ONCE + sub;
            const bool is_k = row < a.c.heads;
            const int head = is_k ? row : row - a.c.heads;
            raw[u] = make_uint4(0, 0, 0, 0);
            scale[u] = 0.f;
            if (there && sub < AT_ONCE && row < end) {
                const uint8_t* p = (const uint8_t*)(is_k ? a.c.k : a.c.v) + (from + head * a.c.head_stride) * ESZ;
                if (STORE == FVS_I8) {
                    *(uint2*)&raw[u] = __ldg((const uint2*)p);
                    scale[u] = __ldg((is_k ? a.c.k_scale : a.c.v_scale) + from_scale + head * a.c.scale_head_stride);
                } else {
                    raw[u] = __ldg((const uint4*)p);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            const int row = row0 + u * AT_ONCE + sub;
            if (sub >= AT_ONCE || row >= end) continue;
            const bool is_k = row < a.c.heads;
            const int head = is_k ? row : row - a.c.heads;
            const int64_t o = ((int64_t)token * a.c.heads + head) * D + e;
            void* out = is_k ? a.k : a.v;
            float x[8];
            if (STORE == FVS_I8) {
                const uint32_t word[2] = {raw[u].x, raw[u].y};
#pragma unroll
                for (int n = 0; n < 8; n++) x[n] = there ? __fmul_rn((float)(int8_t)(word[n / 4] >> (8 * (n % 4))), scale[u]) : 0.f;
            } else {
                up8<STORE == FVS_I8 ? FVS_F16 : STORE>(raw[u], x);
            }
            if (TYPE == FVS_F32) {
                *(float4*)((float*)out + o) = make_float4(x[0], x[1], x[2], x[3]);
                *(float4*)((float*)out + o + 4) = make_float4(x[4], x[5], x[6], x[7]);
            } else {
                *(uint4*)((uint16_t*)out + o) = TYPE == STORE ? raw[u] : down8<TYPE == FVS_F32 ? FVS_F16 : TYPE>(x);
            }
        }
    }
}

// warps of a token: one, more where that would leave SMs without work (`at_once`: heads that a warp takes at a time)
static int spread_of(int tokens, int rows, int at_once) {
    const int want = (32 * fvs_sm_count() + tokens - 1) / tokens, most = (rows + at_once - 1) / at_once;
    return want < 1 ? 1 : want < most ? want : most;
}
static unsigned grid_of(int tokens, int spread) { return (unsigned)(((int64_t)tokens * spread + THREADS / 32 - 1) / (THREADS / 32)); }

static bool heads_ok(const void* p, int64_t token, int64_t head, int d) {
    return p && ((uintptr_t)p & 15) == 0 && token % 8 == 0 && head % 8 == 0 && token >= 0 && (head >= d || head == 0);
}

template <int D>
static void launch_append(fvs_stream_t stream, AppendArgs a, int type, bool halves) {
    a.spread = spread_of(a.tokens, a.hq + 2 * a.c.heads, 32 / Lanes<D>::group);
    const unsigned grid = grid_of(a.tokens, a.spread);
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
static void launch_read(fvs_stream_t stream, ReadArgs a, int type) {
    a.spread = spread_of(a.tokens, 2 * a.c.heads, 32 / (D / 8));
    const unsigned grid = grid_of(a.tokens, a.spread);
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
                 {q, q_token, q_head}, q_out, seq, idx, pos, cos, sin, hq, tokens, positions, rot, 1};
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
    ReadArgs a{*cache, {table, table_stride, seqs, wide}, k, v, seq, idx, tokens, 1};
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
