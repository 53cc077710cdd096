// Writing a paged key-value cache and reading it back (new: the reference ends with the found rows' ids; here the
// passages behind these ids have keys and values in pages).
//
// fvs_kv_append: rotates the query and key heads of new tokens by their positions and stores keys and values at their
// places.  fvs_kv_read: copies rows out as floating point.  Both move every byte once and are bound by memory, so what
// counts is bytes on the way: a warp loads up to 16 heads of one token's q, k or v (append: under way while the token's
// place and its cosines are looked up) or the rows of several tokens (read: their places looked up side by side), then
// stores them and ends; nothing is done one after another.  A head of D elements is D / 16 lanes' (append: in a group of 4,
// 8 or 16; each lane holds two chunks of 8 elements, those that a rotation by halves pairs) or a lane's per 16 bytes (read).
#include "fvs_kv.cuh"

namespace fvs {
namespace kv {

constexpr int THREADS = 256;
// loads of a lane that are on the way together: append takes 35 us with two at 9000 tokens of 48 heads of 64 (39 with one
// or four: a lane's work after them, or its registers, grow), read 23 us with four at 31000 tokens of 8 int8 rows of 96 (25
// with two; each lane looking its places up by itself, without the exchange below, took 20.5 us there)
constexpr int BATCH = 2, READ_BATCH = 4;

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

// TYPE: of the new rows; STORE: of the cache (TYPE or int8); HALVES: pairs (i, i + rot/2), else neighbours (2i, 2i + 1)
template <int D, int TYPE, int STORE, bool HALVES>
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
        if (turns || codes) {
            up8<TYPE>(raw[u][0], x0);
            up8<TYPE>(raw[u][1], x1);
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
            if (turns) raw[u][0] = down8<TYPE>(x0), raw[u][1] = down8<TYPE>(x1);
            if (!there) raw[u][0] = raw[u][1] = make_uint4(0, 0, 0, 0);  // a query without a place
            T* p = (T*)dst + to + u * step;
            *(uint4*)(p + e0) = raw[u][0];
            *(uint4*)(p + e1) = raw[u][1];
        }
    }
}

struct ReadArgs {
    fvs_kv_cache c;
    Table tb;
    void *k, *v;
    const int32_t *seq, *idx;
    int tokens, per;  // tokens of a warp, at most 32
    int spread;       // warps that share a token's rows
    float inv_rows;
};

// rows of the cache as TYPE, zeros where a token has no place: a lane moves 16 bytes of a row.  A warp's lanes look up
// the places of its tokens side by side; then all their rows are on the way together.
template <int D, int STORE, int TYPE>
__global__ void __launch_bounds__(THREADS) read_kernel(ReadArgs a) {
    constexpr int EL = STORE == FVS_I8 ? 16 : 8, L = D / EL, AT_ONCE = 32 / L, ESZ = 16 / EL;
    const unsigned w = blockIdx.x * (THREADS / 32) + threadIdx.x / 32;
    const int first = (int)(w / (unsigned)a.spread * (unsigned)a.per);
    if (first >= a.tokens) return;
    const int n = min(a.per, a.tokens - first);
    const int lane = threadIdx.x & 31, e = lane % L * EL, sub = lane / L;
    const int rows = 2 * a.c.heads;
    int page = 0, slot = 0;
    bool there = false;
    if (lane < n) there = place(a.c, a.tb, a.seq ? __ldg(a.seq + first + lane) : first + lane, __ldg(a.idx + first + lane), page, slot);
    if (!there) page = -1;
    // i / rows; exact while a warp has several tokens, of fewer than 2 * 32 * READ_BATCH rows then
    auto token_of = [&](int i) { return n == 1 ? 0 : (int)(((float)i + 0.5f) * a.inv_rows); };
    for (int i0 = (int)(w % (unsigned)a.spread) * AT_ONCE * READ_BATCH; i0 < n * rows; i0 += a.spread * AT_ONCE * READ_BATCH) {
        uint4 raw[READ_BATCH];
        float scale[READ_BATCH];
#pragma unroll
        for (int u = 0; u < READ_BATCH; u++) {
            const int i = i0 + u * AT_ONCE + sub, t = min(token_of(i), n - 1), row = i - t * rows;
            const bool is_k = row < a.c.heads;
            const int head = is_k ? row : row - a.c.heads;
            const int pg = __shfl_sync(0xffffffffu, page, t), sl = __shfl_sync(0xffffffffu, slot, t);
            raw[u] = make_uint4(0, 0, 0, 0);
            scale[u] = 0.f;
            if (pg >= 0 && sub < AT_ONCE && i < n * rows) {
                const uint8_t* p = (const uint8_t*)(is_k ? a.c.k : a.c.v) +
                                   ((int64_t)pg * a.c.page_stride + (int64_t)head * a.c.head_stride + (int64_t)sl * a.c.slot_stride + e) * ESZ;
                raw[u] = __ldg((const uint4*)p);
                if (STORE == FVS_I8)
                    scale[u] = __ldg((is_k ? a.c.k_scale : a.c.v_scale) + (int64_t)pg * a.c.scale_page_stride +
                                     (int64_t)head * a.c.scale_head_stride + (int64_t)sl * a.c.scale_slot_stride);
            }
        }
#pragma unroll
        for (int u = 0; u < READ_BATCH; u++) {
            const int i = i0 + u * AT_ONCE + sub, t = token_of(i), row = i - t * rows;
            if (sub >= AT_ONCE || i >= n * rows) continue;
            const bool is_k = row < a.c.heads;
            const int64_t o = ((int64_t)(first + t) * a.c.heads + (is_k ? row : row - a.c.heads)) * D + e;
            void* out = is_k ? a.k : a.v;
            if (TYPE == STORE) {
                *(uint4*)((uint16_t*)out + o) = raw[u];
                continue;
            }
            const uint32_t word[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
            for (int m0 = 0; m0 < EL; m0 += 8) {
                float x[8];
#pragma unroll
                for (int m = 0; m < 8; m += 2) {
                    if (STORE == FVS_I8) {
                        // the byte code + 128 in the mantissa of 2^23
                        const uint32_t u4 = word[(m0 + m) / 4] ^ 0x80808080u;
                        x[m] = __fmul_rn(__uint_as_float(__byte_perm(u4, 0x4b000000u, 0x7440 + m % 4)) - 8388736.f, scale[u]);
                        x[m + 1] = __fmul_rn(__uint_as_float(__byte_perm(u4, 0x4b000000u, 0x7441 + m % 4)) - 8388736.f, scale[u]);
                    } else {
                        const float2 two = Elem<STORE == FVS_I8 ? FVS_F16 : STORE>::up(word[m / 2]);
                        x[m] = two.x, x[m + 1] = two.y;
                    }
                }
                if (TYPE == FVS_F32) {
                    *(float4*)((float*)out + o + m0) = make_float4(x[0], x[1], x[2], x[3]);
                    *(float4*)((float*)out + o + m0 + 4) = make_float4(x[4], x[5], x[6], x[7]);
                } else {
                    *(uint4*)((uint16_t*)out + o + m0) = down8<TYPE == FVS_F32 ? FVS_F16 : TYPE>(x);
                }
            }
        }
    }
}

static bool heads_ok(const void* p, int64_t token, int64_t head, int d) {
    return p && ((uintptr_t)p & 15) == 0 && token % 8 == 0 && head % 8 == 0 && token >= 0 && (head >= d || head == 0);
}

template <int D>
static void launch_append(fvs_stream_t stream, AppendArgs a, int type, bool halves) {
    constexpr int most = 32 / Lanes<D>::group * BATCH;  // heads of a warp
    a.q_warps = (a.hq + most - 1) / most;
    a.k_warps = (a.c.heads + most - 1) / most;
    const int64_t warps = (int64_t)a.tokens * (a.q_warps + 2 * a.k_warps);
    const unsigned grid = (unsigned)((warps + THREADS / 32 - 1) / (THREADS / 32));
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
    // as many tokens as a warp has on the way at once (more of them per warp, one after another, took half as long again)
    const int at_once = 32 / (D / (STORE == FVS_I8 ? 16 : 8)) * READ_BATCH, per = at_once / (2 * a.c.heads);
    a.per = per < 1 ? 1 : per < 32 ? per : 32;
    a.spread = per < 1 ? (2 * a.c.heads + at_once - 1) / at_once : 1;
    a.inv_rows = 1.f / (2 * a.c.heads);
    const int64_t warps = (int64_t)((a.tokens + a.per - 1) / a.per) * a.spread;
    const unsigned grid = (unsigned)((warps + THREADS / 32 - 1) / (THREADS / 32));
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
                 {q, q_token, q_head}, q_out, seq, idx, pos, cos, sin, hq, tokens, positions, rot, 0, 0};
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
    ReadArgs a{*cache, {table, table_stride, seqs, wide}, k, v, seq, idx, tokens, 1, 1, 0.f};
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
