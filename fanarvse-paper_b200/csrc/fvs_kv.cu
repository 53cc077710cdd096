// Writing a paged key-value cache and reading it back (new: the reference ends with the found rows' ids; here the
// passages behind these ids have keys and values in pages).
//
// fvs_kv_append: rotates the query and key heads of new tokens by their positions and stores keys and values at their
// places (the kernel: fvs_kv_append.cuh).  fvs_kv_read: copies rows out as floating point.  Both move every byte once and
// are bound by memory: a warp of read takes the rows of several tokens, looks their places up side by side, then loads and
// stores 16 bytes a lane and ends.
#include "fvs_kv_append.cuh"

namespace fvs {
namespace kv {

// loads of a lane that are on the way together: 23 us with four at 31000 tokens of 8 int8 rows of 96 (25 with two; each
// lane looking its places up by itself, without the exchange below, took 20.5 us there)
constexpr int READ_BATCH = 4;

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
    AppendArgs a;
    if (int rc = append_args(a, cache, type, k, k_token, k_head, v, v_token, v_head, q, q_token, q_head, hq, q_out, table,
                             seqs, wide, table_stride, seq, idx, pos, tokens, cos, sin, positions, rot, pairs))
        return rc;
    return append_launch<false>(stream, a, type, pairs == FVS_PAIRS_HALVES);
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
