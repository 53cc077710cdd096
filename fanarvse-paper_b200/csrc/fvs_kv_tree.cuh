// Attention of a tree of drafted tokens over a paged key-value cache (new: the reference ends with the found rows' ids).
//
// Node i of sequence b lies at logical place lens[b] + i and sees every token before lens[b], its ancestors and itself:
// out = sum_t softmax_t(scale <q, k_t>) v_t.  The nodes' query heads of one key head are the rows of one product: rows =
// nodes * (hq / heads), so that keys and values are read once for all of them.  With 4 rows * dim flops per 4 * dim bytes of a
// 16-bit key and value, memory bounds a call up to about 250 rows and the matrix instructions above that.
//
// A CTA per SM, a share of equal cost each of all items (sequence, key head, up to 128 * MT rows), cut anywhere between
// tiles of KEYS keys; what is cut goes through the workspace and join_kernel.  Inside a CTA, a stream of tiles:
//   producer warps (4): look up each key's page and copy its row of k and of v into a ring of slots, in the layout of a
//     128-byte swizzled tile whatever the page size; a key that is not there becomes zeros.  int8 codes are widened to 16 bits
//     on the way (exact), their scales go beside the tile.
//   one thread of a warp issues the products: S = Q K^T into one of two TMEM buffers, and, when the rows' weights lie there
//     in place of S, O += P V; the next tile's S is issued before this tile's O, so that the exponentials overlap both.
//   softmax warpgroups (W), a thread per row: maximum, weights, sum.  With 128 rows (MT = 1) two of them take turns at the
//     tiles, each with an O of its own, added at the end; with 256 rows (MT = 2) each has its rows; heads wider than 128
//     leave TMEM for one O only.
//
// Rounding: scores, maxima, sums and O are fp32.  A weight enters the second product as two parts of the 16-bit type (its
// rounded value and the rounded rest): 17 bits with bf16, 22 with fp16, where one part would double the error that the output's
// own rounding makes; a third has no room in TMEM.  int8 codes are multiplied as bf16 with their key's scale in the weight.
// The running maximum is moved only when it rises by more than 2^SLACK: O need not be rescaled at most tiles, and the
// quotient is the same.
#pragma once
#include <type_traits>

#include "fvs_kv.cuh"
#include "fvs_tcgen05.cuh"

namespace fvs {
namespace kv {
namespace tree {
using namespace fvs::tcg;

constexpr int ROWS = 128;     // rows of a matrix instruction
constexpr int INFO = 4;       // tiles whose keys' flags and scales are held
constexpr int SEGS = 4;       // segments that the scheduler is ahead
constexpr int ITEM_COST = 2;  // cost of an item in tiles: its queries' copy and its output
constexpr int GAVE_UP = 2;    // status bit: a bounded wait ran out

struct Args {
    fvs_kv_cache c;
    Table tb;
    const void* q;
    int64_t q_seq, q_node, q_head;
    const int32_t *lens, *parents, *counts;
    int64_t parent_stride;
    int nodes, hq, group;
    float scale;
    void* out;
    float* lse;
    float* work;     // two partial results of each CTA: [dim][rows] O, then [rows] maxima (log2), [rows] sums
    int32_t* desc;   // 8 words of each CTA: what join_kernel reads
    uint32_t wait_limit;
};


template <int D>
struct Shape {
    static constexpr int KEYS = D <= 128 ? 128 : 64;
    static constexpr int W = D <= 128 ? 2 : 1;
    static constexpr int BLOCKS = (D + 63) / 64;  // 128-byte columns of a tile
    static constexpr int SLOT = KEYS * 128 * BLOCKS;
    static constexpr int THREADS = 32 * (4 * W + 4 + 2);  // softmax, producers, matrix instructions and scheduler
    static constexpr int O0 = 2 * KEYS;  // TMEM columns: two S, then W of O
    static_assert(O0 + W * D <= 512, "tensor memory columns");
};
constexpr int BARS = 64 * 8, INFO_BYTES = 16 + 2 * 128 * 4, MERGE_BYTES = 2 * 2 * ROWS * 8;
constexpr int SEG_BYTES = 48, MASK_BYTES = 2 * 4 * ROWS * 4;  // masks: a row's 128 bits for each softmax thread
constexpr int MISC = BARS + INFO * INFO_BYTES + MERGE_BYTES + 64 + SEGS * SEG_BYTES + MASK_BYTES;
template <int D, int MT>
struct Plan {
    using S = Shape<D>;
    static constexpr int Q = MT * ROWS * 128 * S::BLOCKS;
    static constexpr int FIT = (232448 - 1024 - MISC - Q) / S::SLOT;
    static constexpr int SLOTS = FIT > 12 ? 12 : FIT;
    static constexpr int BYTES = 1024 + Q + SLOTS * S::SLOT + MISC;
    static_assert(SLOTS >= 4, "two tiles of keys and of values");
};

// A sequence's share of the work: its items are (key head, row tile), of `tiles` tiles each.
struct Seq {
    int n, count, keys, tiles, rts;
};
template <int KEYS, int RT>
__device__ __forceinline__ Seq sequence(const Args& a, int b) {
    Seq s;
    const int64_t room = (int64_t)a.tb.wide * a.c.page;
    s.n = (int)min((int64_t)max(__ldg(a.lens + b), 0), room);
    s.count = a.counts ? min(max(__ldg(a.counts + b), 0), a.nodes) : a.nodes;
    s.keys = (int)min((int64_t)s.n + s.count, room);
    s.tiles = (s.keys + KEYS - 1) / KEYS;
    s.rts = (s.count * a.group + RT - 1) / RT;
    return s;
}
__device__ __forceinline__ int64_t cost_of(const Args& a, const Seq& s) {
    return (int64_t)s.rts * a.c.heads * (ITEM_COST + s.tiles);
}

struct Seg {             // tiles [t0, t1) of one item; t0 == t1: no more
    int b, head, rt, rows, t0, t1, n, keys, tiles, item;
};

// Walks over the segments of a CTA (the scheduler's).
template <int KEYS, int RT>
struct Walk {
    int64_t base, start, end;  // cost before the item, and the CTA's share
    int item, b;               // item of the sequence
    Seq s;
    __device__ __forceinline__ void begin(const Args& a, int first, int64_t first_base, int64_t from, int64_t to) {
        start = from;
        end = to;
        b = first;
        base = first_base;
        item = -1;
        if (from < to) {
            s = sequence<KEYS, RT>(a, b);
            const int each = ITEM_COST + s.tiles;
            item = (int)((from - first_base) / each) - 1;
            base = first_base + (int64_t)item * each;
        }
    }
    __device__ __forceinline__ bool next(const Args& a, Seg& g) {
        if (start >= end) return false;
        while (true) {
            base += ITEM_COST + s.tiles;
            item++;
            while (item >= s.rts * a.c.heads) {
                item = 0;
                if (base >= end || ++b >= a.tb.seqs) return false;
                s = sequence<KEYS, RT>(a, b);
            }
            if (base >= end) return false;
            const int64_t first = start - base - ITEM_COST, last = end - base - ITEM_COST;
            g.t0 = first > 0 ? (int)first : 0;
            g.t1 = last < s.tiles ? (int)last : s.tiles;
            if (g.t0 >= g.t1) continue;
            g.b = b;
            g.item = item;
            g.head = item / s.rts;
            g.rt = item - g.head * s.rts;
            g.rows = min(RT, s.count * a.group - g.rt * RT);
            g.n = s.n;
            g.keys = s.keys;
            g.tiles = s.tiles;
            return true;
        }
    }
};

__device__ __forceinline__ uint32_t idesc(int N, bool bf16, bool transposed) {
    const uint32_t t = bf16 ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | ((transposed ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
}
// values as the second operand: keys are the rows of 128 bytes, so N runs along memory; column blocks `lbo` bytes apart,
// eight keys 1024 bytes apart
__device__ __forceinline__ uint64_t values_desc(uint32_t addr, uint32_t lbo) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// waits for the loads so far, those into r among them: what reads r comes behind
__device__ __forceinline__ void tmem_wait32(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// the barrier counts this thread when all of its copies so far have landed
__device__ __forceinline__ void copies_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float exp2_of(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// two fp32 operations in one instruction
struct Two {
    uint64_t x;
};
__device__ __forceinline__ Two two(float a, float b) {
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.x) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 one(Two a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.x));
    return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.x) : "l"(a.x), "l"(b.x), "l"(c.x));
    return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.x) : "l"(a.x), "l"(b.x));
    return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.x) : "l"(a.x), "l"(b.x));
    return r;
}
// four int8 codes as 16-bit values, exactly: fp16 by 1024 + 128 + code in the mantissa; bf16 by the low seven bits behind
// 128, less 128 or, for a negative code, 256
template <int TYPE>
__device__ __forceinline__ void widen4(uint32_t x, uint32_t& lo, uint32_t& hi) {
    if (TYPE == FVS_F16) {
        const __half2 off = __half2half2(__ushort_as_half(0x6480));
        x ^= 0x80808080u;
        const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
        const __half2 ra = __hsub2(*reinterpret_cast<const __half2*>(&a), off), rb = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
        lo = *reinterpret_cast<const uint32_t*>(&ra);
        hi = *reinterpret_cast<const uint32_t*>(&rb);
    } else {
        const uint32_t a = __byte_perm(x, 0x43434343u, 0x4140), b = __byte_perm(x, 0x43434343u, 0x4342);
        const uint32_t va = a & 0xff7fff7fu, sa = a & 0xff80ff80u, vb = b & 0xff7fff7fu, sb = b & 0xff80ff80u;
        const __nv_bfloat162 ra = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&va), *reinterpret_cast<const __nv_bfloat162*>(&sa));
        const __nv_bfloat162 rb = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&vb), *reinterpret_cast<const __nv_bfloat162*>(&sb));
        lo = *reinterpret_cast<const uint32_t*>(&ra);
        hi = *reinterpret_cast<const uint32_t*>(&rb);
    }
}

template <int D, int TYPE, int STORE, int MT>
__global__ void __launch_bounds__(Shape<D>::THREADS, 1) tree_kernel(Args a) {
    using S = Shape<D>;
    using P = Plan<D, MT>;
    constexpr bool I8 = STORE == FVS_I8;
    constexpr int KEYS = S::KEYS, W = S::W, RT = ROWS * MT, SLOTS = P::SLOTS, CHUNKS = KEYS / 32;
    constexpr int VTYPE = I8 ? FVS_BF16 : TYPE;  // of weights and values
    // weights: of fp16 values in the upper part of fp16's range, 2^(LIFT + SLACK) at most
    constexpr float SLACK = VTYPE == FVS_F16 ? 4.f : 8.f, LIFT = VTYPE == FVS_F16 ? 11.f : 0.f;
    static_assert(MT == 1 || W == 2, "256 rows need two softmax warpgroups");

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = saddr(smem);
    const uint32_t q_smem = sbase, ring = sbase + P::Q;
    uint8_t* misc = smem + P::Q + SLOTS * S::SLOT;
    const uint32_t bars = saddr(misc);
    auto full = [&](int s) { return bars + 8 * s; };
    auto empty = [&](int s) { return bars + 8 * (12 + s); };
    auto info_full = [&](int s) { return bars + 8 * (24 + s); };
    auto info_empty = [&](int s) { return bars + 8 * (24 + INFO + s); };
    auto s_full = [&](int s) { return bars + 8 * (32 + s); };
    auto p_full = [&](int s) { return bars + 8 * (34 + s); };
    auto pv_done = [&](int w) { return bars + 8 * (36 + w); };
    const uint32_t q_full = bars + 8 * 38, q_empty = bars + 8 * 39, o_free = bars + 8 * 40, merge_bar = bars + 8 * 41,
                   drain = bars + 8 * 42;
    auto seg_full = [&](int s) { return bars + 8 * (43 + s); };
    auto seg_empty = [&](int s) { return bars + 8 * (43 + SEGS + s); };
    volatile Seg* segs = reinterpret_cast<volatile Seg*>(misc + BARS + INFO * INFO_BYTES + MERGE_BYTES + 64);
    uint8_t* info = misc + BARS;
    float2* merge = reinterpret_cast<float2*>(misc + BARS + INFO * INFO_BYTES);  // [2][W][ROWS]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + BARS + INFO * INFO_BYTES + MERGE_BYTES);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int64_t* s_place = reinterpret_cast<int64_t*>(tmem_slot + 2);  // total, sequence, cost before it

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int W_PROD = 4 * W, W_MMA = 4 * W + 4;
    const uint32_t WL = a.wait_limit;

    if (tid == 0) {
        for (int s = 0; s < SLOTS; s++) {
            mbar_init(full(s), 128);
            mbar_init(empty(s), 1);
        }
        for (int s = 0; s < INFO; s++) {
            mbar_init(info_full(s), 4);
            mbar_init(info_empty(s), 4 * MT);
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(s_full(s), 1);
            mbar_init(p_full(s), 128);
            mbar_init(pv_done(s), 1);
        }
        mbar_init(q_full, 128);
        mbar_init(q_empty, 1);
        mbar_init(o_free, 128 * W);
        mbar_init(merge_bar, 128 * W);
        mbar_init(drain, 1);
        for (int s = 0; s < SEGS; s++) {
            mbar_init(seg_full(s), 1);
            mbar_init(seg_empty(s), 4 * W + 4 + 1);
        }
        *abort = 0;
        s_place[0] = s_place[1] = s_place[2] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        proxy_fence();
    }
    if (warp == W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // ---------------------------------------------------------------- this CTA's share
    {
        // a thread adds up a run of sequences; where the share begins, its thread finds the sequence
        const int per = (a.tb.seqs + S::THREADS - 1) / S::THREADS;
        const int b0 = min(a.tb.seqs, tid * per), b1 = min(a.tb.seqs, b0 + per);
        int64_t mine = 0;
        for (int b = b0; b < b1; b++) {
            const Seq s = sequence<KEYS, RT>(a, b);
            mine += cost_of(a, s);
            if (blockIdx.x == 0 && s.count > 0 && (int64_t)__ldg(a.lens + b) + s.count > (int64_t)a.tb.wide * a.c.page)
                atomicOr(a.c.status, BAD_INDEX);
        }
        int64_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        int64_t* sums = reinterpret_cast<int64_t*>(smem);  // the ring is not in use yet
        if (lane == 31) sums[warp] = upto;
        __syncthreads();
        int64_t before = upto - mine, total = 0;
        for (int w = 0; w < S::THREADS / 32; w++) {
            if (w < warp) before += sums[w];
            total += sums[w];
        }
        const int64_t from = total * (int64_t)blockIdx.x / gridDim.x;
        if (from >= before && from < before + mine) {
            int b = b0;
            for (;; b++) {
                const int64_t cost = cost_of(a, sequence<KEYS, RT>(a, b));
                if (from < before + cost) break;
                before += cost;
            }
            s_place[1] = b;
            s_place[2] = before;
        }
        if (tid == 0) {
            s_place[0] = total;
            int32_t* d = a.desc + 8 * blockIdx.x;  // no share of a cut item yet; whether there is any share
            d[0] = d[5] = -1;
            d[7] = from < total * ((int64_t)blockIdx.x + 1) / gridDim.x;
        }
        // rows of nodes that a sequence does not have
        if (a.counts)
            for (int b = blockIdx.x; b < a.tb.seqs; b += gridDim.x) {
                const int count = min(max(__ldg(a.counts + b), 0), a.nodes);
                const int64_t r0 = ((int64_t)b * a.nodes + count) * a.hq, r1 = ((int64_t)b + 1) * a.nodes * a.hq;
                uint4* out = reinterpret_cast<uint4*>(a.out);
                for (int64_t i = r0 * (D / 8) + tid; i < r1 * (D / 8); i += S::THREADS) out[i] = make_uint4(0, 0, 0, 0);
                if (a.lse)
                    for (int64_t i = r0 + tid; i < r1; i += S::THREADS) a.lse[i] = __int_as_float(0xff800000);
            }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const float scale2 = a.scale * 1.4426950408889634f;  // of scores in powers of two

    if (warp >= W_PROD && warp < W_MMA) {
        // ------------------------------------------------------------ producers
        constexpr int PER = KEYS / 4;              // keys of a warp
        constexpr int CH = (I8 ? D / 16 : D / 8);  // 16-byte chunks of a stored row
        constexpr int TURNS = PER * CH / 32;
        static_assert(PER * CH % 32 == 0, "whole turns");
        constexpr uint32_t NONE = 0xffffffffu;
        const int pw = warp - W_PROD, key = pw * PER + (lane % PER);
        const uint8_t *kbase = (const uint8_t*)a.c.k, *vbase = (const uint8_t*)a.c.v;
        int slot = 0, phase = 1, tile = 0;  // the first pass over the ring finds it free
        int b = 0, head = 0, keys = 0;      // of the segment
        bool ok = true;
        // where key `key` of tile t lies, in 16 bytes from the tensor's first, and its scales
        uint32_t at, next_at;
        float ks = 0.f, vs = 0.f;
        auto lookup = [&](int t) {
            const int x = t * KEYS + key;
            next_at = NONE;
            if (I8) ks = vs = 0.f;
            if (x < keys) {
                int page, s;
                if (place(a.c, a.tb, b, x, page, s) && (!a.c.fill || s < __ldg(a.c.fill + page))) {
                    const int64_t e = (int64_t)page * a.c.page_stride + (int64_t)s * a.c.slot_stride + (int64_t)head * a.c.head_stride;
                    next_at = (uint32_t)(e / (I8 ? 16 : 8));
                    if (I8) {
                        const int64_t se = (int64_t)page * a.c.scale_page_stride + (int64_t)s * a.c.scale_slot_stride + (int64_t)head * a.c.scale_head_stride;
                        ks = __ldg(a.c.k_scale + se);
                        vs = __ldg(a.c.v_scale + se);
                    }
                }
            }
        };
        auto advance = [&]() {
            if (++slot == SLOTS) slot = 0, phase ^= 1;
        };
        // chunk c of key k in a slot
        auto chunk = [&](int k, int c) { return (uint32_t)((c >> 3) * (KEYS * 128) + k * 128 + (((c & 7) ^ (k & 7)) << 4)); };
        // the rows that this lane copies chunks of, a turn each: the same for keys and values
        uint32_t rows[TURNS];
        auto exchange = [&](uint32_t x) {
#pragma unroll
            for (int i = 0; i < TURNS; i++) rows[i] = __shfl_sync(0xffffffffu, x, (i * 32 + lane) / CH);
        };
        auto copy = [&](const uint8_t* base, bool all) {
            const uint32_t dst = ring + slot * S::SLOT;
            if (all) {
#pragma unroll
                for (int i = 0; i < TURNS; i++) {
                    const int id = i * 32 + lane, r = id / CH, c = id - r * CH;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + chunk(pw * PER + r, c)), "l"(base + c * 16 + (uint64_t)rows[i] * 16) : "memory");
                }
            } else {
#pragma unroll
                for (int i = 0; i < TURNS; i++) {
                    const int id = i * 32 + lane, r = id / CH, c = id - r * CH;
                    const bool there = rows[i] != NONE;
                    cp_async16(dst + chunk(pw * PER + r, c), base + (there ? c * 16 + (uint64_t)rows[i] * 16 : 0), there);
                }
            }
            copies_arrive(full(slot));
        };
        // int8 codes: keys and values of the next tile are on their way in registers
        uint4 rk[I8 ? TURNS : 1], rv[I8 ? TURNS : 1];
        auto fetch = [&](uint4* raw, const uint8_t* base) {
#pragma unroll
            for (int i = 0; i < (I8 ? TURNS : 0); i++) {
                const int id = i * 32 + lane, r = id / CH, c = id - r * CH;
                raw[i] = make_uint4(0, 0, 0, 0);
                if (rows[i] != NONE) raw[i] = __ldg((const uint4*)(base + c * 16 + (uint64_t)rows[i] * 16));
            }
        };
        auto widen = [&](uint4* raw, auto type) {
            constexpr int T = decltype(type)::value;
            const uint32_t dst = ring + slot * S::SLOT;
#pragma unroll
            for (int i = 0; i < (I8 ? TURNS : 0); i++) {
                const int id = i * 32 + lane, r = id / CH, c = 2 * (id - r * CH), k = pw * PER + r;
                uint32_t w[8];
                widen4<T>(raw[i].x, w[0], w[1]);
                widen4<T>(raw[i].y, w[2], w[3]);
                widen4<T>(raw[i].z, w[4], w[5]);
                widen4<T>(raw[i].w, w[6], w[7]);
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + chunk(k, c)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + chunk(k, c + 1)), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
            }
            proxy_fence();
            mbar_arrive(full(slot));
        };
        for (int seg = 0; ok; seg++) {
            if (!warp_wait(seg_full(seg % SEGS), (seg / SEGS) & 1, abort, WL)) break;
            const volatile Seg& g = segs[seg % SEGS];
            const int t0 = g.t0, t1 = g.t1;
            b = g.b, head = g.head, keys = g.keys;
            if (t0 >= t1) break;
            lookup(t0);
            at = next_at;
            if (I8) {
                exchange(at);
                fetch(rk, kbase);
                fetch(rv, vbase);
            }
            for (int t = t0; t < t1 && ok; t++, tile++) {
                // flags and scales
                const int is = tile % INFO;
                if (!warp_wait(info_empty(is), ((tile / INFO) & 1) ^ 1, abort, WL)) { ok = false; break; }
                const unsigned there = __ballot_sync(0xffffffffu, at != NONE);
                uint8_t* mine = info + is * INFO_BYTES;
                if (lane == 0) {
                    if (PER == 32)
                        reinterpret_cast<uint32_t*>(mine)[pw] = there;
                    else
                        reinterpret_cast<uint16_t*>(mine)[pw] = (uint16_t)there;
                }
                if (I8 && lane < PER) {
                    float* sc = reinterpret_cast<float*>(mine + 16);
                    sc[key] = ks * scale2;  // scores in powers of two
                    sc[128 + key] = vs;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(info_full(is));
                if (!I8) exchange(at);
                if (t + 1 < t1) {
                    lookup(t + 1);
                    at = next_at;
                }
                if (!warp_wait(empty(slot), phase, abort, WL)) { ok = false; break; }
                if (I8) {
                    widen(rk, std::integral_constant<int, TYPE>());
                    if (t + 1 < t1) {
                        exchange(at);
                        fetch(rk, kbase);
                    }
                } else {
                    copy(kbase, there == 0xffffffffu);
                }
                advance();
                if (!warp_wait(empty(slot), phase, abort, WL)) { ok = false; break; }
                if (I8) {
                    widen(rv, std::integral_constant<int, FVS_BF16>());
                    if (t + 1 < t1) fetch(rv, vbase);
                } else {
                    copy(vbase, there == 0xffffffffu);
                }
                advance();
                if (t == t0) {
                    // the rows' queries, behind the first tile: their buffer is free when the segment before has its scores
                    if (!warp_wait(q_empty, (seg & 1) ^ 1, abort, WL)) { ok = false; break; }
                    constexpr int QCH = D / 8;
                    const int rt = g.rt, live_rows = g.rows;
                    for (int id = pw * 32 + lane; id < RT * QCH; id += 128) {
                        const int r = id / QCH, c = id - r * QCH, mt = r / ROWS, k = r - mt * ROWS, row = rt * RT + r;
                        const bool live = r < live_rows;
                        const int node = live ? row / a.group : 0, h = live ? row - node * a.group : 0;
                        const uint16_t* src = (const uint16_t*)a.q + (int64_t)b * a.q_seq + (int64_t)node * a.q_node + (int64_t)(head * a.group + h) * a.q_head + c * 8;
                        cp_async16(q_smem + mt * (ROWS * 128 * S::BLOCKS) + (c >> 3) * (ROWS * 128) + k * 128 + (((c & 7) ^ (k & 7)) << 4), src, live);
                    }
                    copies_arrive(q_full);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(seg_empty(seg % SEGS));
        }
        cp_async_wait_all();
    } else if (warp >= W_MMA) {
        // ------------------------------------------------------------ the matrix instructions' thread
        if (warp == W_MMA && lane == 0) {
            const uint32_t id_s = idesc(KEYS, TYPE == FVS_BF16, false), id_o = idesc(D, VTYPE == FVS_BF16, true);
            int kslot = 0, kphase = 0, vslot = 1, vphase = 0;  // keys in even places of the stream, values in odd ones
            int unit = 0;
            bool ok = true;
            auto scores = [&](int u, int mt) {
                const uint32_t d = tmem + (u & 1) * KEYS, ab = q_smem + mt * (ROWS * 128 * S::BLOCKS), bb = ring + kslot * S::SLOT;
#pragma unroll
                for (int k = 0; k < D / 16; k++)
                    mma_ss(d, sw128_desc(ab + (k >> 2) * (ROWS * 128) + (k & 3) * 32), sw128_desc(bb + (k >> 2) * (KEYS * 128) + (k & 3) * 32), id_s, k > 0);
                mma_commit(s_full(u & 1));
            };
            auto step = [&](int& s, int& ph) {
                s += 2;
                if (s >= SLOTS) s -= SLOTS, ph ^= 1;
            };
            // O += P V of unit u (the tile k of its segment)
            auto outputs = [&](int u, int k, int mt) {
                if (mt == 0 && !mbar_wait(full(vslot), vphase, abort, WL)) return false;
                if (!mbar_wait(p_full(u & 1), (u >> 1) & 1, abort, WL)) return false;
                proxy_fence();
                tc_fence_after();
                const int w = W == 2 ? u & 1 : 0;
                const uint32_t d = tmem + S::O0 + w * D, p = tmem + (u & 1) * KEYS, vb = ring + vslot * S::SLOT;
                const bool first = k < (W == 2 && MT == 1 ? 2 : 1);
#pragma unroll
                for (int i = 0; i < KEYS / 16; i++) {
                    const uint64_t v = values_desc(vb + i * 2048, KEYS * 128);
                    mma_ts(d, p + 32 * (i >> 1) + 8 * (i & 1), v, id_o, !(first && i == 0));
                    mma_ts(d, p + 32 * (i >> 1) + 8 * (i & 1) + 16, v, id_o, true);
                }
                mma_commit(pv_done(w));
                if (mt == MT - 1) {
                    mma_commit(empty(vslot));
                    step(vslot, vphase);
                }
                return true;
            };
            for (int seg = 0;; seg++) {
                if (!mbar_wait(seg_full(seg % SEGS), (seg / SEGS) & 1, abort, WL)) break;
                const int tiles = segs[seg % SEGS].t1 - segs[seg % SEGS].t0, units = tiles * MT;
                mbar_arrive(seg_empty(seg % SEGS));
                if (tiles == 0 || !mbar_wait(q_full, seg & 1, abort, WL)) break;
                for (int x = 0; x < units && ok; x++, unit++) {
                    const int mt = MT == 2 ? x & 1 : 0;
                    if (mt == 0 && !mbar_wait(full(kslot), kphase, abort, WL)) { ok = false; break; }
                    proxy_fence();
                    tc_fence_after();
                    scores(unit, mt);
                    if (mt == MT - 1) {
                        mma_commit(empty(kslot));
                        step(kslot, kphase);
                    }
                    if (x == units - 1) mma_commit(q_empty);
                    if (x == 0) {
                        // O's first products of this segment come behind the reads of the one before
                        if (seg > 0 && !mbar_wait(o_free, (seg - 1) & 1, abort, WL)) ok = false;
                    } else if (!outputs(unit - 1, MT == 2 ? (x - 1) >> 1 : x - 1, MT == 2 ? (x - 1) & 1 : 0)) {
                        ok = false;
                    }
                }
                if (!ok || !outputs(unit - 1, tiles - 1, MT - 1)) break;
            }
            mma_commit(drain);  // what was issued has to end before the CTA does
            mbar_drain(drain, 0);
        } else if (warp == W_MMA + 1 && lane == 0) {
            // -------------------------------------------------------- the scheduler
            Walk<KEYS, RT> walk;
            const int64_t total = s_place[0];
            walk.begin(a, (int)s_place[1], s_place[2], total * (int64_t)blockIdx.x / gridDim.x, total * ((int64_t)blockIdx.x + 1) / gridDim.x);
            bool more = true;
            for (int seg = 0; more; seg++) {
                Seg g;
                more = walk.next(a, g);
                if (!more) g.t0 = g.t1 = 0;
                if (!mbar_wait(seg_empty(seg % SEGS), ((seg / SEGS) & 1) ^ 1, abort, WL)) break;
                volatile Seg& to = segs[seg % SEGS];
                to.t0 = g.t0, to.t1 = g.t1;
                if (more) to.b = g.b, to.head = g.head, to.rt = g.rt, to.rows = g.rows, to.n = g.n, to.keys = g.keys, to.tiles = g.tiles, to.item = g.item;
                mbar_arrive(seg_full(seg % SEGS));
            }
        }
        __syncwarp();
    } else if (warp < W_PROD) {
        // ------------------------------------------------------------ softmax, a thread per row
        const int w = warp >> 2, r = (warp & 3) * 32 + lane;  // warpgroup, TMEM lane
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        uint32_t* mask = reinterpret_cast<uint32_t*>(misc + BARS + INFO * INFO_BYTES + MERGE_BYTES + 64 + SEGS * SEG_BYTES) + w * 4 * ROWS + r;
        const float lift = scale2 == 0.f ? 1.f : fabsf(scale2);  // the sign, and a scale of 0, are in the scores
        int tile = 0;
        bool ok = true;
        for (int seg = 0;; seg++) {
            if (!warp_wait(seg_full(seg % SEGS), (seg / SEGS) & 1, abort, WL)) { ok = false; break; }
            const volatile Seg& g = segs[seg % SEGS];
            const int t0 = g.t0, t1 = g.t1;
            if (t0 >= t1) break;
            const int mine = MT == 2 ? w * ROWS + r : r;            // row of the item's row tile
            const bool warp_live = mine - lane < g.rows;
            const int row = g.rt * RT + mine;
            const int node = mine < g.rows ? row / a.group : 0;
            float m = __int_as_float(0xff800000), l = 0.f;
            bool any = false;                                       // units of this warpgroup in this segment
            int last = -1;                                          // the last of them
            for (int t = t0; t < t1; t++, tile++) {
                int u = MT == 2 ? 2 * tile + w : tile;
                if (MT == 1 && W == 2 && (u & 1) != w) continue;
                const int n_th = W == 2 ? u >> 1 : u;               // of this warpgroup
                const int is = tile % INFO;
                if (!warp_wait(info_full(is), (tile / INFO) & 1, abort, WL) || !warp_wait(s_full(u & 1), (u >> 1) & 1, abort, WL)) { ok = false; break; }
                tc_fence_after();
                const uint32_t s_tmem = lanes + (u & 1) * KEYS;
                const uint8_t* inf = info + is * INFO_BYTES;
                if (warp_live) {
                    uint32_t see[CHUNKS];
                    bool all = true;
#pragma unroll
                    for (int k = 0; k < CHUNKS; k++) see[k] = reinterpret_cast<const uint32_t*>(inf)[k];
                    const int x0 = t * KEYS - g.n;                // of the tile's first key behind the sequence
                    if (x0 + KEYS > 0) {
                        uint32_t tree[CHUNKS];
#pragma unroll
                        for (int k = 0; k < CHUNKS; k++) {
                            const int before = min(max(-x0 - 32 * k, 0), 32);  // keys of the sequence itself
                            tree[k] = before == 32 ? 0xffffffffu : (1u << before) - 1u;
                        }
                        const int32_t* up = a.parents + (int64_t)g.b * a.parent_stride;
                        for (int i = node; i >= 0 && i >= x0;) {
                            const int at = i - x0;
#pragma unroll
                            for (int k = 0; k < CHUNKS; k++)
                                if (at >> 5 == k) tree[k] |= 1u << (at & 31);
                            const int p = __ldg(up + i);
                            i = p < i ? p : -1;
                        }
#pragma unroll
                        for (int k = 0; k < CHUNKS; k++) see[k] &= tree[k];
                    }
#pragma unroll
                    for (int k = 0; k < CHUNKS; k++) all &= see[k] == 0xffffffffu;
                    const bool odd = __any_sync(0xffffffffu, !all) || (!I8 && scale2 <= 0.f);
                    if (odd) {
#pragma unroll
                        for (int k = 0; k < CHUNKS; k++) mask[k * ROWS] = see[k];
                    }
                    const float* ks = reinterpret_cast<const float*>(inf + 16);
                    // Two passes over the row's scores in TMEM, 32 at a time: the largest, then the weights.  (All of a
                    // tile's at once leave no registers, and unrolled code no place in the instruction cache: both took up
                    // to half as long again.)
                    uint32_t s[32];
                    // what the scores are before `lift`: with the key's scale and in powers of two (int8), with their sign;
                    // masked where the tile is not plain
                    auto fetch = [&](int k) {
                        tmem_ld32(s_tmem + 32 * k, s);
                        tmem_wait32(s);
                        if (I8) {
#pragma unroll
                            for (int j = 0; j < 32; j += 4) {
                                const float4 f = *reinterpret_cast<const float4*>(ks + 32 * k + j);
                                const float2 y = one(mul2(two(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), two(f.x, f.y)));
                                const float2 z = one(mul2(two(__uint_as_float(s[j + 2]), __uint_as_float(s[j + 3])), two(f.z, f.w)));
                                s[j] = __float_as_uint(y.x), s[j + 1] = __float_as_uint(y.y);
                                s[j + 2] = __float_as_uint(z.x), s[j + 3] = __float_as_uint(z.y);
                            }
                        }
                        if (odd) {
                            const uint32_t word = reinterpret_cast<const volatile uint32_t*>(mask)[k * ROWS];
                            const float sign = I8 ? 1.f : scale2 < 0.f ? -1.f : scale2 == 0.f ? 0.f : 1.f;
#pragma unroll
                            for (int j = 0; j < 32; j++) s[j] = word >> j & 1 ? __float_as_uint(__uint_as_float(s[j]) * sign) : 0xff800000u;
                        }
                    };
                    float tops[4];
#pragma unroll
                    for (int y = 0; y < 4; y++) tops[y] = __int_as_float(0xff800000);
#pragma unroll 1
                    for (int k = 0; k < CHUNKS; k++) {
                        fetch(k);
#pragma unroll
                        for (int j = 0; j < 32; j += 8) {
#pragma unroll
                            for (int y = 0; y < 4; y++)
                                tops[y] = fmaxf(tops[y], fmaxf(__uint_as_float(s[j + y]), __uint_as_float(s[j + y + 4])));
                        }
                    }
                    float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                    if (!I8) top *= lift;
                    const bool rises = any ? top > m + SLACK : true;
                    if (__any_sync(0xffffffffu, rises)) {
                        const float to = fmaxf(m, top);
                        if (any) {
                            const float by = m == to ? 1.f : exp2_of(m - to);
                            l *= by;
                            if (!warp_wait(pv_done(w), (n_th - 1) & 1, abort, WL)) { ok = false; break; }
                            tc_fence_after();
#pragma unroll 1
                            for (int k = 0; k < D; k += 16) {
                                uint32_t o[16];
                                tmem_ld16(lanes + S::O0 + w * D + k, o);
                                tmem_wait16(o);
#pragma unroll
                                for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * by);
                                tmem_st16(lanes + S::O0 + w * D + k, o);
                            }
                        }
                        m = to;
                    }
                    const float off = m == __int_as_float(0xff800000) ? 0.f : m;
                    const Two minus = two(-off, -off), factor = two(lift, lift);
                    Two sums[2] = {two(0.f, 0.f), two(0.f, 0.f)};
#pragma unroll 1
                    for (int k = 0; k < CHUNKS; k++) {
                        fetch(k);
#pragma unroll
                        for (int h = 0; h < 32; h += 16) {
                            uint32_t hi[8], lo[8];
#pragma unroll
                            for (int j = 0; j < 16; j += 2) {
                                const Two raw = two(__uint_as_float(s[h + j]), __uint_as_float(s[h + j + 1]));
                                const float2 x = one(I8 ? add2(raw, minus) : fma2(raw, factor, minus));
                                Two p = two(exp2_of(x.x), exp2_of(x.y));
                                sums[(j / 2) & 1] = add2(sums[(j / 2) & 1], p);
                                if (I8) {
                                    const float2 f = *reinterpret_cast<const float2*>(ks + 128 + 32 * k + h + j);
                                    p = mul2(p, two(f.x, f.y));
                                }
                                if (LIFT != 0.f) p = mul2(p, two(2048.f, 2048.f));
                                const float2 w2 = one(p);
                                hi[j / 2] = Elem<VTYPE>::down(w2.x, w2.y);
                                const float2 got = Elem<VTYPE>::up(hi[j / 2]);
                                const float2 rest = one(add2(p, two(-got.x, -got.y)));
                                lo[j / 2] = Elem<VTYPE>::down(rest.x, rest.y);
                            }
                            tmem_st8(s_tmem + 32 * k + h / 2, hi);
                            tmem_st8(s_tmem + 32 * k + 16 + h / 2, lo);
                        }
                    }
                    const float2 sum = one(add2(sums[0], sums[1]));
                    l += sum.x + sum.y;
                    tmem_st_wait();
                }
                any = true;
                last = n_th;
                // With one warpgroup its O may still be behind by two products here, which a parity cannot tell from none;
                // with two, S(u) came behind the warpgroup's last product.
                if (W == 1 && n_th > 0 && !warp_wait(pv_done(w), (n_th - 1) & 1, abort, WL)) { ok = false; break; }
                tc_fence_before();
                __syncwarp();
                mbar_arrive(p_full(u & 1));
                if (lane == 0) mbar_arrive(info_empty(is));
            }
            if (!ok) break;
            // ---------------------------------------------------------------- the segment's result
            const bool whole = t0 == 0 && t1 == g.tiles;
            float* part = a.work + (int64_t)(2 * blockIdx.x + (t0 == 0 ? 1 : 0)) * RT * (D + 2);
            if (any && !warp_wait(pv_done(w), last & 1, abort, WL)) { ok = false; break; }
            float scale0, scale1 = 0.f;  // of this thread's O and, with two for a row, of the other
            int c0 = 0, c1 = D;
            bool has0 = any, has1 = false;
            if (MT == 1 && W == 2) {
                // both warpgroups have a share of each row: each adds up half of the columns
                merge[((seg & 1) * 2 + w) * ROWS + r] = make_float2(m, l);
                mbar_arrive(merge_bar);
                if (!warp_wait(merge_bar, seg & 1, abort, WL)) { ok = false; break; }
                has1 = t1 - t0 > 1 || !any;
                if (has1) {
                    // the other's last unit: the segment's last tile, or the one before it
                    const int end_tile = tile - 1, other = (end_tile & 1) == w ? end_tile - 1 : end_tile;
                    if (!warp_wait(pv_done(w ^ 1), (other >> 1) & 1, abort, WL)) { ok = false; break; }
                }
                const float2 o = merge[((seg & 1) * 2 + (w ^ 1)) * ROWS + r];
                const float to = fmaxf(m, o.x);
                scale0 = m == to ? 1.f : exp2_of(m - to);
                scale1 = o.x == to ? 1.f : exp2_of(o.x - to);
                l = l * scale0 + o.y * scale1;
                m = to;
                c0 = w == 0 ? 0 : D / 2;
                c1 = c0 + D / 2;
            } else {
                scale0 = 1.f;
            }
            tc_fence_after();
            const bool live = mine < g.rows;
            if (warp_live) {
                const int h = live ? row - node * a.group : 0;
                const int64_t o_row = ((int64_t)g.b * a.nodes + node) * a.hq + g.head * a.group + h;
                const float down = LIFT != 0.f ? 1.f / 2048.f : 1.f;
                const float by = whole ? (l == 0.f ? 0.f : down / l) : down;
                const float f0 = scale0 * by, f1 = scale1 * by;
#pragma unroll 1
                for (int k = c0; k < c1; k += 16) {
                    uint32_t x[16], y[16];
                    if (has0) tmem_ld16(lanes + S::O0 + w * D + k, x);
                    if (has1) tmem_ld16(lanes + S::O0 + (w ^ 1) * D + k, y);
                    if (has0) tmem_wait16(x);
                    if (has1) tmem_wait16(y);
                    float o[16];
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        o[j] = has0 ? __uint_as_float(x[j]) * f0 : 0.f;
                        if (has1) o[j] = fmaf(__uint_as_float(y[j]), f1, o[j]);
                    }
                    if (whole && live) {
                        uint16_t* out = (uint16_t*)a.out + o_row * D + k;
#pragma unroll
                        for (int j = 0; j < 16; j += 8) {
                            float e[8];
#pragma unroll
                            for (int z = 0; z < 8; z++) e[z] = l == 0.f ? 0.f : o[j + z];
                            *reinterpret_cast<uint4*>(out + j) = down8<TYPE>(e);
                        }
                    } else if (live) {
#pragma unroll
                        for (int j = 0; j < 16; j++) part[(k + j) * RT + mine] = o[j];
                    }
                }
                if (live && (MT == 2 || W == 1 || w == 0)) {
                    if (whole) {
                        if (a.lse) a.lse[o_row] = l == 0.f ? __int_as_float(0xff800000) : (m + log2f(l)) * 0.6931471805599453f;
                    } else {
                        part[D * RT + mine] = m;
                        part[(D + 1) * RT + mine] = l;
                    }
                }
            }
            tc_fence_before();
            mbar_arrive(o_free);
            // what join_kernel reads: the item that begins here and goes on, and the one that came from the CTA before
            if (tid == 0 && !whole) {
                int32_t* d = a.desc + 8 * blockIdx.x;
                const int item = g.item;
                if (t0 == 0) {
                    d[0] = g.b, d[1] = item, d[2] = g.head, d[3] = g.rt, d[4] = g.rows;
                } else {
                    d[5] = g.b, d[6] = item;
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(seg_empty(seg % SEGS));
        }
        if (!ok && lane == 0) atomicOr(a.c.status, GAVE_UP);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == W_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    if (*abort && tid == 0) atomicOr(a.c.status, GAVE_UP);
}

// Adds the shares of the items that were cut.  Block (c, rows of 32): the item that begins in CTA c and goes on in the CTAs
// behind it, each of which left one share.
template <int D, int TYPE, int RT>
__global__ void __launch_bounds__(256) join_kernel(Args a, int ctas) {
    extern __shared__ float weight[];  // [shares][32]
    __shared__ float s_m[8][32], s_l[8][32];
    const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int32_t* d = a.desc + 8 * c;
    const int b = d[0], item = d[1], head = d[2], rt = d[3], rows = d[4];
    const int row = blockIdx.y * 32 + lane;
    if (b < 0 || (int)blockIdx.y * 32 >= rows) return;
    // the CTAs behind that have a share of it: none between them has another item
    int upto = c + 1;
    while (upto < ctas && ((a.desc[8 * upto + 5] == b && a.desc[8 * upto + 6] == item) || a.desc[8 * upto + 7] == 0)) upto++;
    auto part = [&](int i) { return a.work + (int64_t)(2 * (c + i) + (i == 0 ? 1 : 0)) * RT * (D + 2); };
    auto has = [&](int i) { return i == 0 || (a.desc[8 * (c + i) + 5] == b && a.desc[8 * (c + i) + 6] == item); };
    const int shares = upto - c;
    float m = __int_as_float(0xff800000);
    for (int i = warp; i < shares; i += 8) {
        const float x = has(i) && row < rows ? part(i)[D * RT + row] : __int_as_float(0xff800000);
        weight[i * 32 + lane] = x;
        m = fmaxf(m, x);
    }
    s_m[warp][lane] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) m = fmaxf(m, s_m[w][lane]);
    float l = 0.f;
    for (int i = warp; i < shares; i += 8) {
        const float x = weight[i * 32 + lane], by = x == m ? 1.f : exp2_of(x - m);
        const bool there = has(i) && row < rows;
        weight[i * 32 + lane] = there ? by : 0.f;
        if (there) l = fmaf(part(i)[(D + 1) * RT + row], by, l);
    }
    s_l[warp][lane] = l;
    __syncthreads();
    l = 0.f;
#pragma unroll
    for (int w = 0; w < 8; w++) l += s_l[w][lane];
    if (row >= rows) return;
    const int at = rt * RT + row, node = at / a.group, h = at - node * a.group;
    const int64_t o_row = ((int64_t)b * a.nodes + node) * a.hq + head * a.group + h;
    constexpr int COLS = D / 8;
    float o[COLS];
#pragma unroll
    for (int j = 0; j < COLS; j++) o[j] = 0.f;
    for (int i = 0; i < shares; i++) {
        if (!has(i)) continue;
        const float by = weight[i * 32 + lane];
        const float* p = part(i) + (int64_t)warp * COLS * RT + row;
#pragma unroll
        for (int j = 0; j < COLS; j++) o[j] = fmaf(p[j * RT], by, o[j]);
    }
    const float by = l == 0.f ? 0.f : 1.f / l;
    uint16_t* out = (uint16_t*)a.out + o_row * D + warp * COLS;
#pragma unroll
    for (int j = 0; j < COLS; j += 4) {
        float e[4];
#pragma unroll
        for (int z = 0; z < 4; z++) e[z] = l == 0.f ? 0.f : o[j + z] * by;
        *reinterpret_cast<uint2*>(out + j) = make_uint2(Elem<TYPE>::down(e[0], e[1]), Elem<TYPE>::down(e[2], e[3]));
    }
    if (warp == 0 && a.lse) a.lse[o_row] = l == 0.f ? __int_as_float(0xff800000) : (m + log2f(l)) * 0.6931471805599453f;
}

template <int D, int TYPE, int STORE, int MT>
static int launch(fvs_stream_t stream, Args a) {
    using P = Plan<D, MT>;
    constexpr int RT = ROWS * MT;
    const int ctas = fvs_sm_count();
    const void* f = (const void*)tree_kernel<D, TYPE, STORE, MT>;
    cudaError_t e = fvs_ensure_smem(f, P::BYTES);
    if (e != cudaSuccess) return (int)e;
    a.wait_limit = pipeline_wait_limit();
    a.desc = (int32_t*)a.work;
    a.work = a.work + 8 * ctas;
    tree_kernel<D, TYPE, STORE, MT><<<ctas, Shape<D>::THREADS, P::BYTES, stream>>>(a);
    if (int rc = fvs_launch_status()) return rc;
    const int rows = a.nodes * a.group;
    join_kernel<D, TYPE, RT><<<dim3(ctas, ((rows < RT ? rows : RT) + 31) / 32), 256, ctas * 32 * 4, stream>>>(a, ctas);
    return fvs_launch_status();
}

// kernels over heads of D elements; MT: 256 rows of an item where there are more than 128
template <int D>
int launch_types(fvs_stream_t stream, const Args& a, int type) {
    const bool i8 = a.c.type == FVS_I8, two = Shape<D>::W == 2 && a.nodes * a.group > ROWS;
#define FVS_TREE(T, ST) (two ? launch<D, T, ST, Shape<D>::W>(stream, a) : launch<D, T, ST, 1>(stream, a))
    if (type == FVS_F16) return i8 ? FVS_TREE(FVS_F16, FVS_I8) : FVS_TREE(FVS_F16, FVS_F16);
    return i8 ? FVS_TREE(FVS_BF16, FVS_I8) : FVS_TREE(FVS_BF16, FVS_BF16);
#undef FVS_TREE
}

}  // namespace tree
}  // namespace kv
}  // namespace fvs
