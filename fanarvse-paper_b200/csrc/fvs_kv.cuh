// What the paged key-value cache's kernels share: the cache's layout, its element types, where a logical token lies.
#pragma once
#include <cuda_bf16.h>

#include "fvs_common.cuh"

namespace fvs {
namespace kv {

// Element types by the codes of include/fanar_b200.h.
template <int TYPE>
struct Elem;
template <>
struct Elem<FVS_F16> {
    using T = __half;
    static __device__ __forceinline__ float2 up(uint32_t x) { return __half22float2(*reinterpret_cast<__half2*>(&x)); }
    static __device__ __forceinline__ uint32_t down(float a, float b) {
        const __half2 r = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};
template <>
struct Elem<FVS_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float2 up(uint32_t x) {
        return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t down(float a, float b) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};
// 16 consecutive bytes of 16-bit elements as fp32 and back (one rounding per element)
template <int TYPE>
__device__ __forceinline__ void up8(const uint4& x, float (&f)[8]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 p = Elem<TYPE>::up(w[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}
template <int TYPE>
__device__ __forceinline__ uint4 down8(const float (&f)[8]) {
    return make_uint4(Elem<TYPE>::down(f[0], f[1]), Elem<TYPE>::down(f[2], f[3]), Elem<TYPE>::down(f[4], f[5]),
                      Elem<TYPE>::down(f[6], f[7]));
}

// The page table of a call: table[seq * stride + t / page] is the page of logical token t, -1 where there is none.
struct Table {
    const int32_t* at;
    int64_t stride;
    int32_t seqs, wide;
};

constexpr int BAD_INDEX = 1;  // status bit: an index outside its table (the access was skipped)

// Page and slot of token `t` of sequence `b`; false where it has no place (t < 0, a hole) or an index is out of range,
// which also sets the status word.
__device__ __forceinline__ bool place(const fvs_kv_cache& c, const Table& tb, int b, int t, int& page, int& slot) {
    if (t < 0) return false;
    const int p = (int)((unsigned)t / (unsigned)c.page);
    bool bad = (unsigned)b >= (unsigned)tb.seqs || p >= tb.wide;
    page = -1;
    slot = t - p * c.page;
    if (!bad) {
        page = __ldg(tb.at + (int64_t)b * tb.stride + p);
        bad = page >= c.pages;
    }
    if (bad) atomicOr(c.status, BAD_INDEX);
    return !bad && page >= 0;
}

// host: the checks that every entry point makes of a cache
static inline int check_cache(const fvs_kv_cache* c) {
    FVS_CHECK_ARG(c && c->k && c->v && c->status && c->pages >= 1 && c->heads >= 1 && c->page >= 1);
    FVS_CHECK_ARG(c->type == FVS_F16 || c->type == FVS_BF16 || c->type == FVS_I8);
    const int64_t per = c->type == FVS_I8 ? 16 : 8;  // elements in 16 bytes
    FVS_CHECK_ARG(c->page_stride % per == 0 && c->head_stride % per == 0 && c->slot_stride % per == 0);
    FVS_CHECK_ARG(c->page_stride >= 0 && c->head_stride >= 0 && c->slot_stride >= c->dim);
    FVS_CHECK_ARG(((((uintptr_t)c->k) | ((uintptr_t)c->v)) & 15) == 0);
    if (c->type == FVS_I8)
        FVS_CHECK_ARG(c->k_scale && c->v_scale && c->scale_page_stride >= 0 && c->scale_head_stride >= 0 &&
                      c->scale_slot_stride >= 1);
    const int d = c->dim;
    if (!(d == 64 || d == 96 || d == 128 || d == 192 || d == 256)) return FVS_ERANGE;
    return FVS_OK;
}
static inline int check_table(const int32_t* table, int seqs, int wide, int64_t stride) {
    FVS_CHECK_ARG(table && seqs >= 1 && wide >= 1 && stride >= 0);
    return FVS_OK;
}

}  // namespace kv
}  // namespace fvs
