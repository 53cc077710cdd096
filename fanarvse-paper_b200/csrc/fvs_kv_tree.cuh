// Attention of a tree of drafted tokens over a paged key-value cache (new: the reference ends with the found rows' ids).
//
// Node i of sequence b lies at logical place lens[b] + i and sees every token before lens[b], its ancestors and itself:
// out = sum_t softmax_t(scale <q, k_t>) v_t.  The nodes' query heads of one key head are the rows of one product: rows =
// nodes * (hq / heads), so that keys and values are read once for all of them.  With 6 rows * dim flops (both parts of a weight
// count) per 4 * dim bytes of a 16-bit key and value, memory bounds a call up to about 170 rows and the matrix instructions above.
//
// One or two CTAs an SM (Shape), each with a share of equal cost of all items (sequence, key head, up to 256 rows), cut anywhere
// between tiles of KEYS keys; what is cut goes through the workspace and join_kernel.  Inside a CTA, a stream of tiles:
//   producers: keys and values into a ring of slots in the layout of a 128-byte swizzled tile.  16-bit rows come by tensor
//     copies, a box for each piece of a page; pages of other than a multiple of 8 slots by 16-byte copies; int8 codes are
//     widened to 16 bits on the way (exact), their scales go beside the tile.  Flags of the keys that are there go beside it.
//   scheduler and relay (a warp): writes the CTA's segments ahead, and passes filled slots on behind a proxy fence.
//   matrix instructions (a thread for each softmax warpgroup): S = Q K^T into TMEM, and, when the rows' weights lie there in
//     place of S, O += P V; where TMEM has room a tile's S is issued before the O of the tile before.
//   softmax warpgroups, a thread per row: weights and their sum; at a segment's end the output or the share of one.
// What bounds it: up to 128 rows no unit (64 ragged requests of 64 rows: 83 us where the bytes take 48, a rate of 3.8 TB/s, tensor
// pipe 44 %, issue slots 31 %): a CTA's tiles wait for one another (copy, scores, weights, outputs; one O, so that a segment's
// products wait for the one before to be read out), and 8 us are the join.  With 256 rows the softmax warps, whose 11
// instructions and 2 exponentials for each pair of scores take 660 cycles for 32 columns of two warps of a quarter SM when they
// run alone (131000 tokens under 64 nodes: 218 us at best where memory takes 84 and the matrix instructions with two parts of each
// weight 126).
//
// Rounding: scores, maxima, sums and O are fp32.  A weight enters the second product as two parts of the 16-bit type, its
// rounded value and the rounded rest: 22 bits over fp16 values and over int8 codes (as fp16, their scale in the weight), 17 over
// bf16 values.  One part would double the error that the output's own rounding makes.  Outputs that are not the nearest
// number, 64 sequences of 1 to 7700 keys, one node, heads of 128: bf16 1 in 676 (attend, which has 24 bits, 1 in 4096, products
// in fp32 1 in 5958), fp16 1 in 333 (attend 512, fp32 705), over int8 codes 1 in 2427 bf16 ones (attend 4096, fp32 3121; 546 with
// two bf16 parts) and 1 in 349 fp16 ones (attend 809, fp32 705; 84 with two bf16 parts).  64 nodes over 131000 bf16 keys:
// 1 in 381, fp32 1 in 260.  A third bf16 part would be a third more of the matrix instructions, and half as much more of the TMEM
// that a tile's scores leave, which heads of 128 do not have.
// A row's weights are relative to a reference that rises only when they become large (LIMIT): O need not be rescaled at most
// tiles, and the quotient is the same.
#pragma once
#include <type_traits>

#include "fvs_kv.cuh"
#include "fvs_tcgen05.cuh"

namespace fvs {
namespace kv {
namespace tree {
using namespace fvs::tcg;

constexpr int ROWS = 128;     // rows of a matrix instruction
constexpr int INFO = 8;       // tiles whose keys' flags and scales are held
constexpr int SEGS = 4;       // segments that the scheduler is ahead
constexpr int ITEM_KEYS = 256;  // cost of an item, its queries' copy and its output, in keys (384: 64 ragged requests take 2 % longer)
constexpr int LEAST_COST = 4;  // of a CTA's share, in tiles
constexpr int GAVE_UP = 2;     // status bit: a bounded wait ran out
constexpr int SEG_BYTES = 48;
constexpr int DESC = 16;
// Words of a CTA's descriptor: the item that begins in it and goes on in others (sequence or -1, item, key head, row tile, rows),
// the item that it continues (sequence or -1, item), HAS_SHARE and NOT_FINITE, then where its share begins (sequence; cost
// before that and of all, 64 bits each).
constexpr int HAS_SHARE = 1, NOT_FINITE = 2;  // NOT_FINITE: an O of an item that it computed whole is not finite

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
    int32_t* desc;   // DESC words of each CTA: what join_kernel reads
    uint32_t wait_limit;
    int box;         // keys of a tensor copy, a power of two that divides the page
};
struct Maps {  // of keys and values: element, slot, head, page
    CUtensorMap k, v;
};

// How a kernel uses an SM, by head size and 128 * MT rows of an item.
template <int D, int STORE, int MT, int QR>
struct Shape {
    static_assert(MT == 1 || D <= 128, "tensor memory holds one O of a wide head");
    static_assert(QR == ROWS || (MT == 1 && D <= 128), "fewer rows of queries");
    // CTAs of an SM: with 128 rows of heads up to 128 two, whose beginnings and ends overlap (one CTA whose two softmax
    // warpgroups took turns at the tiles took 115 us where this took 107, at 64 ragged requests of 64 rows)
    static constexpr int CTAS = MT == 1 && D <= 128 ? 2 : 1;
    static constexpr int W = MT;  // softmax warpgroups
    // keys of a tile: 128 where the codes' widening is the slower part (388 us where 64 took 436, at 24 long int8 contexts under
    // 32 nodes), else 64, whose scores are computed a tile ahead (229 where 128 took 254, at 131000 tokens under 64 nodes)
    static constexpr int KEYS = MT == 2 && STORE == FVS_I8 ? 128 : 64;
    // keys whose weights enter O together, while the softmax warps are at the next ones: half a tile (131000 tokens under 64
    // nodes: 217 us, 220 with whole tiles), whole tiles with two CTAs an SM (64 ragged requests: 83 us, 89 with halves)
    static constexpr int PART = CTAS == 2 ? KEYS : KEYS / 2;
    static constexpr int COLUMNS = 512 / CTAS;                                       // of tensor memory
    static constexpr int BUFFERS = MT == 2 ? 256 / KEYS : CTAS == 2 ? 2 : 4;         // of scores in it
    static constexpr int LEAD = BUFFERS == W ? 0 : 1;  // units whose scores are issued before a unit's outputs wait
    static constexpr int PRODUCERS = CTAS == 2 ? 2 : 4;  // warps
    static constexpr int BLOCKS = (D + 63) / 64;         // 128-byte columns of a tile
    static constexpr int SLOT = KEYS * 128 * BLOCKS;
    static constexpr int THREADS = 32 * (4 * W + PRODUCERS + W + 1);  // softmax, producers, matrix instructions, scheduler
    static constexpr int O0 = BUFFERS * KEYS;                         // columns of the scores, then W of O
    static_assert(O0 + W * D <= COLUMNS, "tensor memory columns");
    // shared memory: queries, the ring, then barriers, the tiles' flags and scales, segments and masks
    static constexpr int Q = MT * QR * 128 * BLOCKS;
    static constexpr int BARS = 96 * 8, INFO_BYTES = 16 + 2 * KEYS * 4, MASK_BYTES = W * ROWS * (KEYS / 32) * 4;
    static constexpr int MISC = BARS + INFO * INFO_BYTES + 64 + SEGS * SEG_BYTES + MASK_BYTES;
    static constexpr int FIT = ((CTAS == 2 ? 115712 : 232448) - 1024 - MISC - Q) / SLOT;
    static constexpr int SLOTS = FIT > 12 ? 12 : FIT;
    static constexpr int BYTES = 1024 + Q + SLOTS * SLOT + MISC;
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
template <int KEYS>
__device__ __forceinline__ int64_t cost_of(const Args& a, const Seq& s) {
    return (int64_t)s.rts * a.c.heads * (ITEM_KEYS / KEYS + s.tiles);
}

// Where the share of CTA c begins: of equal cost, of as many CTAs as have LEAST_COST or more (what a cut costs)
__device__ __forceinline__ int64_t shares(int64_t total, int ctas) { return min((int64_t)ctas, max((int64_t)1, total / LEAST_COST)); }
__device__ __forceinline__ int64_t share(int64_t total, int64_t ctas, unsigned c) { return c >= ctas ? total : total * (int64_t)c / ctas; }

struct Seg {             // tiles [t0, t1) of one item; t0 == t1: no more
    int b, head, rt, rows, t0, t1, n, keys, tiles, item;
};

// Walks over the segments of a CTA (the scheduler's).
template <int KEYS, int RT>
struct Walk {
    static constexpr int ITEM_COST = ITEM_KEYS / KEYS;
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
// The scale of a row of int8 keys.  It multiplies the score, where the formula multiplies the codes: with an infinite one their
// products with q's elements are infinities of both signs, a not-a-number together.
__device__ __forceinline__ float key_scale(const float* at) {
    const float x = __ldg(at);
    return __fadd_rn(__fsub_rn(x, x), x);
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
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait8(uint32_t (&r)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])::"memory");
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
// whether the phase with the given parity is complete, without waiting
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done;
}
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

__device__ __forceinline__ float log2_of(float x) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
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

// QR: rows of queries that shared memory holds, 64 where an item has no more: the matrix instructions read 128, the others of
// whatever lies behind (their scores and outputs go to rows that nobody reads), and the ring has a slot more (64 ragged requests
// are 3 % faster)
// BOXES: 16-bit rows come by tensor copies (pages of a multiple of 8 slots); else by the producers' lanes, 16 bytes each, whose
// traffic delays every wait on a barrier (104 us instead of 88 at 64 ragged requests)
template <int D, int TYPE, int STORE, int MT, int QR, bool BOXES>
__global__ void __launch_bounds__(Shape<D, STORE, MT, QR>::THREADS, Shape<D, STORE, MT, QR>::CTAS)
    tree_kernel(Args a, const __grid_constant__ Maps maps) {
    using S = Shape<D, STORE, MT, QR>;
    constexpr bool I8 = STORE == FVS_I8;
    constexpr int KEYS = S::KEYS, BUFFERS = S::BUFFERS, PART = S::PART, PARTS = KEYS / PART, W = S::W, RT = ROWS * MT, SLOTS = S::SLOTS, LEAD = S::LEAD;
    constexpr int INFO_BYTES = S::INFO_BYTES, PRODUCERS = S::PRODUCERS;
    constexpr int VTYPE = I8 ? FVS_F16 : TYPE;  // of weights and values
    // The most that 32 weights may add up to before their reference rises; over fp16 values they lie in the upper part of
    // fp16's range, LIMIT * LIFT at most.  Over int8 codes it is the weights times the values' scales that enter the product:
    // the reference follows these, 2^UP below the largest, and the weights alone only have to stay in fp32's range, their sum over
    // 2^31 keys too (scales outside 2^-FAR to 2^FAR count as its ends; a weight is 2^(UP + FAR) at most where the reference rises).
    constexpr float UP = 9.f, FAR = 80.f, MOST = 0x1p95f;
    constexpr float LIMIT = I8 ? 127.f * 512.f : VTYPE == FVS_F16 ? 127.f : 4096.f, LIFT = !I8 && VTYPE == FVS_F16 ? 512.f : 1.f;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = saddr(smem);
    const uint32_t q_smem = sbase, ring = sbase + S::Q;
    uint8_t* misc = smem + S::Q + SLOTS * S::SLOT;
    const uint32_t bars = saddr(misc);
    auto full = [&](int s) { return bars + 8 * s; };
    auto empty = [&](int s) { return bars + 8 * (12 + s); };
    auto info_full = [&](int s) { return bars + 8 * (24 + s); };
    auto info_empty = [&](int s) { return bars + 8 * (32 + s); };
    auto s_full = [&](int u) { return bars + 8 * (80 + u % BUFFERS); };
    auto p_full = [&](int u, int part) { return bars + 8 * (88 + u % BUFFERS * PARTS + part); };  // PART keys
    auto pv_half = [&](int u) { return bars + 8 * (84 + u % BUFFERS); };
    auto pv_done = [&](int u) { return bars + 8 * (48 + u % BUFFERS); };
    auto round_of = [&](int u) { return (uint32_t)(u / BUFFERS) & 1u; };  // parity of unit u's phase of these
    auto seg_full = [&](int s) { return bars + 8 * (52 + s); };
    auto seg_empty = [&](int s) { return bars + 8 * (52 + SEGS + s); };
    const uint32_t q_full = bars + 8 * 60, q_empty = bars + 8 * 61, o_free = bars + 8 * 62,
                   drain = bars + 8 * 64, q_landed = bars + 8 * 65;
    auto landed = [&](int s) { return bars + 8 * (66 + s); };
    volatile Seg* segs = reinterpret_cast<volatile Seg*>(misc + S::BARS + INFO * INFO_BYTES + 64);
    uint8_t* info = misc + S::BARS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + S::BARS + INFO * INFO_BYTES);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int64_t* s_place = reinterpret_cast<int64_t*>(tmem_slot + 2);  // total, sequence, cost before it

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int W_PROD = 4 * W, W_MMA = 4 * W + PRODUCERS;
    const uint32_t WL = a.wait_limit;

    if (tid == 0) {
        for (int s = 0; s < SLOTS; s++) {
            mbar_init(landed(s), BOXES ? 1 : 32 * PRODUCERS);
            mbar_init(full(s), 1);
            mbar_init(empty(s), MT);
        }
        for (int s = 0; s < INFO; s++) {
            mbar_init(info_full(s), BOXES ? 1 : PRODUCERS);
            mbar_init(info_empty(s), 4 * MT);
        }
        for (int u = 0; u < BUFFERS; u++) {
            mbar_init(s_full(u), 1);
            for (int part = 0; part < PARTS; part++) mbar_init(p_full(u, part), 4);
            if (PARTS == 2) mbar_init(pv_half(u), 1);
            mbar_init(pv_done(u), 1);
        }
        mbar_init(q_landed, 32 * (BOXES ? PRODUCERS - 1 : PRODUCERS));
        mbar_init(q_full, 1);
        mbar_init(q_empty, W);
        mbar_init(o_free, 128 * W);
        mbar_init(drain, W);
        for (int s = 0; s < SEGS; s++) {
            mbar_init(seg_full(s), 1);
            mbar_init(seg_empty(s), 4 * W + PRODUCERS + W);
        }
        *abort = 0;
        s_place[0] = s_place[1] = s_place[2] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        proxy_fence();
    }
    if (warp == W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(tmem_slot)), "r"((uint32_t)S::COLUMNS) : "memory");
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
            mine += cost_of<KEYS>(a, s);
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
        const int64_t ctas = shares(total, gridDim.x), from = share(total, ctas, blockIdx.x);
        if (from >= before && from < before + mine) {
            int b = b0;
            for (;; b++) {
                const int64_t cost = cost_of<KEYS>(a, sequence<KEYS, RT>(a, b));
                if (from < before + cost) break;
                before += cost;
            }
            s_place[1] = b;
            s_place[2] = before;
        }
        if (tid == 0) {
            s_place[0] = total;
            int32_t* d = a.desc + DESC * blockIdx.x;  // no share of a cut item yet
            d[0] = d[5] = -1;
            d[7] = from < share(total, ctas, blockIdx.x + 1) ? HAS_SHARE : 0;
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
    if (tid == 0) {
        int32_t* d = a.desc + DESC * blockIdx.x;
        d[8] = (int32_t)s_place[1];
        *reinterpret_cast<int64_t*>(d + 10) = s_place[2];
        *reinterpret_cast<int64_t*>(d + 12) = s_place[0];
    }
    const uint32_t tmem = *tmem_slot;
    const float scale2 = a.scale * 1.4426950408889634f;  // of scores in powers of two

    // chunk c of 16 bytes of row k of a 128-byte swizzled tile of `rows` rows
    auto swizzled = [](int rows, int k, int c) { return (uint32_t)((c >> 3) * (rows * 128) + k * 128 + (((c & 7) ^ (k & 7)) << 4)); };
    // a segment's queries into their buffer by warp qw of qn: 32 rows at a time, addresses by a lane each
    auto queries = [&](const volatile Seg& g, int qw, int qn) {
        constexpr int QCH = D / 8;
        constexpr uint32_t NONE = 0xffffffffu;
        const int b = g.b, head = g.head, rt = g.rt, live_rows = g.rows;
#pragma unroll 1
        for (int r0 = qw * 32; r0 < MT * QR; r0 += 32 * qn) {
            const int row = rt * RT + r0 + lane;
            uint32_t from = NONE;
            if (r0 + lane < live_rows) {
                const int node = row / a.group, h = head * a.group + row - node * a.group;
                from = (uint32_t)(((int64_t)b * a.q_seq + (int64_t)node * a.q_node + (int64_t)h * a.q_head) / 8);
            }
            const int mt = r0 / ROWS, k0 = r0 - mt * ROWS;
            const uint32_t dst = q_smem + mt * (ROWS * 128 * S::BLOCKS);
#pragma unroll 4
            for (int i = 0; i < QCH; i++) {
                const int id = i * 32 + lane, r = id / QCH, c = id - r * QCH;
                const uint32_t at = __shfl_sync(0xffffffffu, from, r);
                cp_async16(dst + swizzled(QR, k0 + r, c), (const uint8_t*)a.q + (at == NONE ? 0 : c * 16 + (uint64_t)at * 16), at != NONE);
            }
        }
        copies_arrive(q_landed);
    };
    if (BOXES && warp >= W_PROD && warp < W_MMA) {
        // ------------------------------------------------------------ producers by tensor copies
        if (warp == W_PROD) {
            // A lane looks up a box: those of as many tiles at once as the lanes go to (a lookup is two or three loads behind one
            // another).  A box comes whole if it has any keys; the scores of what it holds beside them are masked, and the
            // relay puts zeros in place of those values.
            const int box = a.box, boxes = KEYS / box, ahead = 32 / boxes;
            int slot = 0, phase = 1, tile = 0, issued = 0;
            bool ok = true;
            int page, at, have, next_page = 0, next_at = 0, next_have = 0;
            int b_page = 0, b_at = 0, b_have = 0;  // of the lane's box of the tiles that were looked up
            for (int seg = 0; ok; seg++) {
                if (!warp_wait(seg_full(seg % SEGS), (seg / SEGS) & 1, abort, WL)) break;
                const volatile Seg& g = segs[seg % SEGS];
                const int t0 = g.t0, t1 = g.t1, b = g.b, head = g.head, keys = g.keys;
                if (t0 >= t1) break;
                auto lookup = [&](int t) {
                    const int x = t * KEYS + lane * box;
                    next_have = 0;
                    if ((unsigned)x < (unsigned)keys && place(a.c, a.tb, b, x, next_page, next_at)) {
                        next_have = min(box, keys - x);
                        if (a.c.fill) next_have = max(0, min(next_have, __ldg(a.c.fill + next_page) - next_at));
                    }
                };
                // the boxes of `mine` lanes into the next slot
                auto copy = [&](const CUtensorMap* map, bool mine) {
                    const int n = __popc(__ballot_sync(0xffffffffu, mine));
                    if (lane == 0) mbar_expect_tx(landed(slot), n * box * 128 * S::BLOCKS);
                    __syncwarp();
                    if (mine) {
#pragma unroll
                        for (int c = 0; c < S::BLOCKS; c++)
                            asm volatile(
                                "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                                    ring + slot * S::SLOT + c * (KEYS * 128) + lane * box * 128),
                                "l"(map), "r"(c * 64), "r"(at), "r"(head), "r"(page), "r"(landed(slot))
                                : "memory");
                    }
                    if (++slot == SLOTS) slot = 0, phase ^= 1;
                    issued++;
                };
                lookup(t0);
                for (int t = t0, i = ahead; t < t1; t++, tile++) {
                    if (i == ahead) b_page = next_page, b_at = next_at, b_have = next_have, i = 0;
                    const int from = (i * boxes + lane) & 31;
                    page = __shfl_sync(0xffffffffu, b_page, from);
                    at = __shfl_sync(0xffffffffu, b_at, from);
                    have = __shfl_sync(0xffffffffu, b_have, from);
                    if (lane >= boxes) have = 0;
                    i++;
                    const int is = tile % INFO, first = lane * box;
                    uint32_t lo = 0, hi = 0;  // flags of the tile's keys
                    if (have > 0) {
                        const uint64_t mine = (have == 64 ? ~0ull : (1ull << have) - 1) << first;
                        lo = (uint32_t)mine, hi = (uint32_t)(mine >> 32);
                    }
                    lo = __reduce_or_sync(0xffffffffu, lo);
                    hi = __reduce_or_sync(0xffffffffu, hi);
                    if (!warp_wait(info_empty(is), ((tile / INFO) & 1) ^ 1, abort, WL)) { ok = false; break; }
                    if (lane == 0) {
                        *reinterpret_cast<uint2*>(info + is * INFO_BYTES) = make_uint2(lo, hi);
                        mbar_arrive(info_full(is));
                    }
                    if (!warp_wait(empty(slot), phase, abort, WL)) { ok = false; break; }
                    copy(&maps.k, have > 0);
                    if (!warp_wait(empty(slot), phase, abort, WL)) { ok = false; break; }
                    copy(&maps.v, have > 0);
                    if (i == 1 && t + ahead < t1) lookup(t + ahead);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(seg_empty(seg % SEGS));
            }
            // no copy is under way when the CTA ends, whatever became of its waits
            for (int i = max(0, issued - SLOTS); i < issued; i++) mbar_drain(landed(i % SLOTS), (i / SLOTS) & 1);
        } else {
            for (int seg = 0;; seg++) {
                if (!warp_wait(seg_full(seg % SEGS), (seg / SEGS) & 1, abort, WL)) break;
                const volatile Seg& g = segs[seg % SEGS];
                if (g.t0 >= g.t1 || !warp_wait(q_empty, (seg & 1) ^ 1, abort, WL)) break;
                queries(g, warp - W_PROD - 1, PRODUCERS - 1);
                __syncwarp();
                if (lane == 0) mbar_arrive(seg_empty(seg % SEGS));
            }
            cp_async_wait_all();
        }
    } else if (!BOXES && warp >= W_PROD && warp < W_MMA) {
        // ------------------------------------------------------------ producers by their lanes
        constexpr int PER = KEYS / PRODUCERS;      // keys of a warp
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
                        ks = key_scale(a.c.k_scale + se);
                        vs = __ldg(a.c.v_scale + se);
                    }
                }
            }
        };
        auto advance = [&]() {
            if (++slot == SLOTS) slot = 0, phase ^= 1;
        };
        // chunk c of key k in a slot
        auto chunk = [&](int k, int c) { return swizzled(KEYS, k, c); };
        // the rows that this lane copies chunks of, a turn each: the same for keys and values
        uint32_t rows[TURNS];
        auto exchange = [&](uint32_t x) {
#pragma unroll
            for (int i = 0; i < TURNS; i++) rows[i] = __shfl_sync(0xffffffffu, x, (i * 32 + lane) / CH);
        };
        auto copy = [&](const uint8_t* base) {
            const uint32_t dst = ring + slot * S::SLOT;
#pragma unroll
            for (int i = 0; i < TURNS; i++) {
                const int id = i * 32 + lane, r = id / CH, c = id - r * CH;
                const bool there = rows[i] != NONE;
                cp_async16(dst + chunk(pw * PER + r, c), base + (there ? c * 16 + (uint64_t)rows[i] * 16 : 0), there);
            }
            copies_arrive(landed(slot));
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
            mbar_arrive(landed(slot));
        };
        for (int seg = 0; ok; seg++) {
            if (!warp_wait(seg_full(seg % SEGS), (seg / SEGS) & 1, abort, WL)) break;
            const volatile Seg& g = segs[seg % SEGS];
            const int t0 = g.t0, t1 = g.t1;
            b = g.b, head = g.head, keys = g.keys;
            if (t0 >= t1) break;
            // before the first tile if the segment before has all its scores, else behind it
            const bool asked = __all_sync(0xffffffffu, mbar_test(q_empty, (seg & 1) ^ 1));
            if (asked) queries(g, pw, PRODUCERS);
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
                    sc[KEYS + key] = vs;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(info_full(is));
                if (!I8) exchange(at);
                if (t + 1 < t1) {
                    lookup(t + 1);
                    at = next_at;
                }
#pragma unroll 1
                for (int op = 0; op < 2; op++) {  // keys, then values
                    if (!warp_wait(empty(slot), phase, abort, WL)) { ok = false; break; }
                    if (!I8) {
                        copy(op ? vbase : kbase);
                    } else if (op == 0) {
                        widen(rk, std::integral_constant<int, TYPE>());
                        if (t + 1 < t1) {
                            exchange(at);
                            fetch(rk, kbase);
                        }
                    } else {
                        widen(rv, std::integral_constant<int, FVS_F16>());
                        if (t + 1 < t1) fetch(rv, vbase);
                    }
                    advance();
                }
                if (!ok) break;
                if (t == t0 && !asked && !(ok = warp_wait(q_empty, (seg & 1) ^ 1, abort, WL))) break;
                if (t == t0 && !asked) queries(g, pw, PRODUCERS);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(seg_empty(seg % SEGS));
        }
        cp_async_wait_all();
    } else if (warp >= W_MMA) {
        // A thread for each softmax warpgroup issues its matrix instructions: a unit's outputs (O += P V) PART keys at a time as
        // its weights come, and right behind the last ones the next unit's scores (S = Q K^T), which take the weights'
        // place; instructions of one thread run in order.  An instruction is issued when the one before it has begun and a
        // single thread is slow, so what it need not wait for between instructions it does before or behind them.
        if (warp < W_MMA + W && lane == 0) {
            const int w = warp - W_MMA;
            const uint32_t id_s = idesc(KEYS, TYPE == FVS_BF16, false), id_o = idesc(D, VTYPE == FVS_BF16, true);
            int kslot = 0, kphase = 0, vslot = 1, vphase = 0;
            int tile = 0;  // tiles of this CTA before the segment
            bool ok = true;
            const uint64_t q_desc = sw128_desc(q_smem + (MT == 2 ? w * (ROWS * 128 * S::BLOCKS) : 0)), k_desc = sw128_desc(ring),
                           v_desc = values_desc(ring, KEYS * 128);
            auto step = [&](int& slot, int& phase) {
                slot += 2;
                if (slot >= SLOTS) slot -= SLOTS, phase ^= 1;
            };
            // S of unit u: keys in the next slot, which is full
            auto scores = [&](int u) {
                const uint32_t d = tmem + (u % BUFFERS) * KEYS;
                const uint64_t bd = k_desc + (uint32_t)(kslot * (S::SLOT / 16));
#pragma unroll
                for (int k = 0; k < D / 16; k++)
                    mma_ss(d, q_desc + ((k >> 2) * (QR * 128 / 16) + (k & 3) * 2), bd + ((k >> 2) * (KEYS * 128 / 16) + (k & 3) * 2), id_s, k > 0);
                mma_commit(s_full(u));
                mma_commit(empty(kslot));
                step(kslot, kphase);
            };
            for (int seg = 0; ok; seg++) {
                if (!mbar_wait(seg_full(seg % SEGS), (seg / SEGS) & 1, abort, WL)) break;
                const int tiles = segs[seg % SEGS].t1 - segs[seg % SEGS].t0;
                mbar_arrive(seg_empty(seg % SEGS));
                if (tiles == 0 || !mbar_wait(q_full, seg & 1, abort, WL)) break;
                const int units = tiles;
                auto unit = [&](int x) { return W * (tile + x) + w; };
                int asked = 0;
                // the next unit's scores, if its keys are there
                auto ask = [&](int most) {
                    if (asked < min(units, most) && mbar_test(full(kslot), kphase)) {
                        tc_fence_after();
                        scores(unit(asked));
                        if (++asked == units) mma_commit(q_empty);
                    }
                };
                // waits for a barrier and asks meanwhile (what is waited for may need the scores)
                auto wait = [&](uint32_t bar, uint32_t parity, int most) {
                    for (uint32_t it = 0; it < WL; it++) {
                        ask(most);
                        if (mbar_test(bar, parity)) return true;
                        if ((it & 255u) == 255u && *abort) return false;
                    }
                    *abort = 1;
                    return false;
                };
                // O's first products of this segment come behind the reads of the one before
                if (seg > 0) ok = wait(o_free, (seg - 1) & 1, 1 + LEAD);
#pragma unroll 1
                for (int x = 0; x < units && ok; x++) {
                    const int u = unit(x);
                    const uint32_t d = tmem + S::O0 + w * D, p = tmem + (u % BUFFERS) * KEYS;
                    const uint64_t v = v_desc + (uint32_t)(vslot * (S::SLOT / 16));
#pragma unroll
                    for (int part = 0; part < PARTS; part++) {
                        if (!(ok = wait(p_full(u, part), round_of(u), x + 1 + LEAD))) break;
                        if (part == 0 && !(ok = mbar_wait(full(vslot), vphase, abort, WL))) break;
                        tc_fence_after();
#pragma unroll
                        for (int i = PART / 16 * part; i < PART / 16 * (part + 1); i++) {
                            mma_ts(d, p + 32 * (i >> 1) + 8 * (i & 1), v + i * 128, id_o, x + i > 0);
                            mma_ts(d, p + 32 * (i >> 1) + 8 * (i & 1) + 16, v + i * 128, id_o, true);
                        }
                        if (part < PARTS - 1) mma_commit(pv_half(u));
                    }
                    if (!ok) break;
                    if (LEAD == 0) ask(x + 2);  // right behind, in place of the weights
                    mma_commit(pv_done(u));
                    mma_commit(empty(vslot));
                    step(vslot, vphase);
                }
                tile += tiles;
            }
            mma_commit(drain);  // what was issued has to end before the CTA does
            mbar_drain(drain, 0);
        } else if (warp == W_MMA + W) {
            // -------------------------------------------------------- the scheduler, which is also the relay
            // What the producers wrote becomes visible to the matrix instructions by a fence between the two.  The
            // instructions' own thread would wait at it until those it has issued are done (100 cycles for each
            // instruction instead of 67).
            Walk<KEYS, RT> walk;
            const int64_t total = s_place[0];
            const int64_t ctas = shares(total, gridDim.x);
            walk.begin(a, (int)s_place[1], s_place[2], share(total, ctas, blockIdx.x), share(total, ctas, blockIdx.x + 1));
            int slot = 0, phase = 0, told = 0, tile = 0;
            bool more = true, ok = true;
            auto pass = [&](bool values) {
                if (!warp_wait(landed(slot), phase, abort, WL)) return false;
                if (BOXES && values) {  // zeros for keys that are not there: a weight of 0 times anything is not 0
                    const int is = tile % INFO;
                    if (!warp_wait(info_full(is), (tile / INFO) & 1, abort, WL)) return false;
                    const uint2 there = *reinterpret_cast<const uint2*>(info + is * INFO_BYTES);
                    if ((there.x & there.y) != 0xffffffffu) {
                        constexpr int CH = D / 8;
                        for (int id = lane; id < KEYS * CH; id += 32) {
                            const int k = id / CH, c = id - k * CH;
                            if (!((k < 32 ? there.x >> k : there.y >> (k - 32)) & 1))
                                asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(ring + slot * S::SLOT + swizzled(KEYS, k, c)), "r"(0) : "memory");
                        }
                    }
                }
                proxy_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(full(slot));
                if (++slot == SLOTS) slot = 0, phase ^= 1;
                return true;
            };
            for (int seg = 0; ok; seg++) {
                for (; more && told <= seg + 1; told++) {  // a segment ahead
                    Seg g;
                    more = walk.next(a, g);
                    if (!more) g.t0 = g.t1 = 0;
                    if (!warp_wait(seg_empty(told % SEGS), ((told / SEGS) & 1) ^ 1, abort, WL)) { ok = false; break; }
                    if (lane == 0) {
                        volatile Seg& to = segs[told % SEGS];
                        to.t0 = g.t0, to.t1 = g.t1;
                        if (more) to.b = g.b, to.head = g.head, to.rt = g.rt, to.rows = g.rows, to.n = g.n, to.keys = g.keys, to.tiles = g.tiles, to.item = g.item;
                        mbar_arrive(seg_full(told % SEGS));
                    }
                    __syncwarp();
                }
                if (!ok) break;
                const int tiles = segs[seg % SEGS].t1 - segs[seg % SEGS].t0;
                if (tiles == 0) break;
                for (int t = 0; t < tiles; t++, tile++) {
                    if (!(ok = pass(false)) || !(ok = pass(true))) break;
                    if (t == 0) {
                        if (!(ok = warp_wait(q_landed, seg & 1, abort, WL))) break;
                        proxy_fence();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(q_full);
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp < W_PROD) {
        // ------------------------------------------------------------ softmax, a thread per row
        const int w = warp >> 2, r = (warp & 3) * 32 + lane;  // warpgroup, TMEM lane
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        uint32_t* mask = reinterpret_cast<uint32_t*>(misc + S::BARS + INFO * INFO_BYTES + 64 + SEGS * SEG_BYTES) + w * (KEYS / 32) * ROWS + r;
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
            const int n = g.n;
            float m = __int_as_float(0xff800000), l = 0.f;
            bool any = false;                                       // units of this warpgroup in this segment
            int last = -1;                                          // the last of them
            for (int t = t0; t < t1; t++, tile++) {
                const int u = W * tile + w;
                const int is = tile % INFO;
                if (!warp_wait(info_full(is), (tile / INFO) & 1, abort, WL) || !warp_wait(s_full(u), round_of(u), abort, WL)) { ok = false; break; }
                tc_fence_after();
                const uint32_t s_tmem = lanes + (u % BUFFERS) * KEYS;
                const uint8_t* inf = info + is * INFO_BYTES;
                if (warp_live) {
                    constexpr int WORDS = KEYS / 32;
                    uint32_t see[WORDS];
                    uint32_t all = 0xffffffffu;
#pragma unroll
                    for (int k = 0; k < WORDS; k++) see[k] = reinterpret_cast<const uint32_t*>(inf)[k], all &= see[k];
                    const int x0 = t * KEYS - n;  // of the tile's first key behind the sequence
                    bool odd = all != 0xffffffffu || (!I8 && scale2 <= 0.f);
                    if (x0 + KEYS > 0) {
                        uint32_t tree[WORDS];
                        all = 0xffffffffu;
#pragma unroll
                        for (int k = 0; k < WORDS; k++) {
                            const int before = min(max(-x0 - 32 * k, 0), 32);  // keys of the sequence itself
                            tree[k] = before == 32 ? 0xffffffffu : (1u << before) - 1u;
                        }
                        const int32_t* up = a.parents + (int64_t)g.b * a.parent_stride;
                        for (int i = node; i >= 0 && i >= x0;) {
                            const int at = i - x0;
#pragma unroll
                            for (int k = 0; k < WORDS; k++)
                                if (at >> 5 == k) tree[k] |= 1u << (at & 31);
                            const int p = __ldg(up + i);
                            i = p < i ? p : -1;
                        }
#pragma unroll
                        for (int k = 0; k < WORDS; k++) see[k] &= tree[k], all &= see[k];
                        odd = odd || __any_sync(0xffffffffu, all != 0xffffffffu);
                    }
                    if (odd) {
#pragma unroll
                        for (int k = 0; k < WORDS; k++) mask[k * ROWS] = see[k];
                    }
                    const float* ks = reinterpret_cast<const float*>(inf + 16);
                    // The row's scores 32 at a time: weights above the reference `m`, unless their sum says that one of them is
                    // far above it, which is rare: then m rises and the 32 are taken again.  (A largest score
                    // for every 32 took 90 of 730 cycles, all of a tile's scores at once left no registers, and unrolled
                    // code no place in the instruction cache.)
                    const Two factor = two(lift, lift);
                    // 32 scores: with the key's scale, in powers of two (int8), masked, and with the scale's sign
                    auto scores = [&](uint32_t (&s)[32], int k) {
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
                        if (__builtin_expect(odd, 0)) {
                            const uint32_t word = mask[k * ROWS];
                            const float sign = I8 ? 1.f : scale2 < 0.f ? -1.f : scale2 == 0.f ? 0.f : 1.f;
#pragma unroll
                            for (int j = 0; j < 32; j++) s[j] = word >> j & 1 ? __float_as_uint(__uint_as_float(s[j]) * sign) : 0xff800000u;
                        }
                    };
                    bool raise = !any, need = raise;  // no reference yet; of the warp, of this row
#pragma unroll 1
                    for (int k = 0; k < KEYS / 32;) {
                        uint32_t s[32];
                        scores(s, k);
                        if (__builtin_expect(raise, 0)) {
                            float top = __int_as_float(0xff800000);
#pragma unroll
                            for (int j = 0; j < 32; j++) {
                                const float x = __uint_as_float(s[j]);
                                top = fmaxf(top, I8 ? x + fminf(fmaxf(log2_of(fabsf(ks[KEYS + 32 * k + j])), -FAR), FAR) - UP : x);
                            }
                            if (!I8) top *= lift;
                            const float to = need ? fmaxf(m, top) : m, by = m == to ? 1.f : exp2_of(m - to);
                            m = to;
                            l *= by;
                            const bool half = PARTS == 2 && k >= PART / 32;  // the tile's first weights may be in O
                            tmem_st_wait();  // weights, or an O that rose before, that are read again below
                            if (any || half) {
                                ok = ok && warp_wait(half ? pv_half(u) : pv_done(last), round_of(half ? u : last), abort, WL);
                                tc_fence_after();
#pragma unroll 1
                                for (int x = 0; x < D; x += 16) {
                                    uint32_t o[16];
                                    tmem_ld16(lanes + S::O0 + w * D + x, o);
                                    tmem_wait16(o);
#pragma unroll
                                    for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * by);
                                    tmem_st16(lanes + S::O0 + w * D + x, o);
                                }
                            }
                            if (PART == 64 && (k & 1)) {  // the 32 weights before are not in O yet
#pragma unroll 1
                                for (int x = 0; x < 16; x += 8) {
                                    uint32_t hi[8], lo[8];
                                    tmem_ld8(s_tmem + 32 * (k - 1) + x, hi);
                                    tmem_ld8(s_tmem + 32 * (k - 1) + 16 + x, lo);
                                    tmem_wait8(hi);
                                    tmem_wait8(lo);
#pragma unroll
                                    for (int j = 0; j < 8; j++) {
                                        const float2 y = Elem<VTYPE>::up(hi[j]), z = Elem<VTYPE>::up(lo[j]);
                                        const float p = (y.x + z.x) * by, q = (y.y + z.y) * by;
                                        hi[j] = Elem<VTYPE>::down(p, q);
                                        const float2 got = Elem<VTYPE>::up(hi[j]);
                                        lo[j] = Elem<VTYPE>::down(p - got.x, q - got.y);
                                    }
                                    tmem_st8(s_tmem + 32 * (k - 1) + x, hi);
                                    tmem_st8(s_tmem + 32 * (k - 1) + 16 + x, lo);
                                }
                            }
                        }
                        const float off = m == __int_as_float(0xff800000) ? 0.f : m;
                        const Two minus = two(-off, -off);
                        Two sums[2] = {two(0.f, 0.f), two(0.f, 0.f)};
                        Two scaled[2] = {two(0.f, 0.f), two(0.f, 0.f)};  // int8: sums with the values' scales
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            float4 f;
                            if (I8) f = *reinterpret_cast<const float4*>(ks + KEYS + 32 * k + j);
#pragma unroll
                            for (int y = 0; y < 2; y++) {
                                const int i = j + 2 * y;
                                const Two raw = two(__uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                                const float2 x = one(I8 ? add2(raw, minus) : fma2(raw, factor, minus));
                                Two p = two(exp2_of(x.x), exp2_of(x.y));
                                sums[y] = add2(sums[y], p);
                                if (I8) {
                                    p = mul2(p, y ? two(f.z, f.w) : two(f.x, f.y));
                                    scaled[y] = add2(scaled[y], p);
                                }
                                const float2 w2 = one(p);
                                s[i] = __float_as_uint(w2.x), s[i + 1] = __float_as_uint(w2.y);
                            }
                        }
                        const float2 pair = one(add2(sums[0], sums[1]));
                        const float sum = pair.x + pair.y;
                        // (not-a-numbers and rows that have seen nothing yet are taken again once)
                        if (I8) {
                            const float2 both = one(add2(scaled[0], scaled[1]));
                            need = !(both.x + both.y <= LIMIT && sum <= MOST) || m == __int_as_float(0xff800000);
                        } else {
                            need = !(sum <= LIMIT) || m == __int_as_float(0xff800000);
                        }
                        if (__any_sync(0xffffffffu, need) && !raise) {
                            raise = true;
                            continue;
                        }
                        raise = false;
                        l += sum;
#pragma unroll
                        for (int h = 0; h < 32; h += 16) {
                            uint32_t hi[8], lo[8];
#pragma unroll
                            for (int j = 0; j < 16; j += 4) {
#pragma unroll
                                for (int y = 0; y < 2; y++) {
                                    Two p = two(__uint_as_float(s[h + j + 2 * y]), __uint_as_float(s[h + j + 2 * y + 1]));
                                    if (LIFT != 1.f) p = mul2(p, two(LIFT, LIFT));
                                    const float2 w2 = one(p);
                                    hi[j / 2 + y] = Elem<VTYPE>::down(w2.x, w2.y);
                                    const float2 got = Elem<VTYPE>::up(hi[j / 2 + y]);
                                    const float2 rest = one(fma2(two(got.x, got.y), two(-1.f, -1.f), p));
                                    lo[j / 2 + y] = Elem<VTYPE>::down(rest.x, rest.y);
                                }
                            }
                            tmem_st8(s_tmem + 32 * k + h / 2, hi);
                            tmem_st8(s_tmem + 32 * k + 16 + h / 2, lo);
                        }
                        if ((k + 1) % (PART / 32) == 0) {
                            tmem_st_wait();
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(p_full(u, k / (PART / 32)));
                        }
                        k++;
                    }
                    if (!ok) break;
                } else {
#pragma unroll
                    for (int part = 0; part < PARTS; part++)
                        if (lane == 0) mbar_arrive(p_full(u, part));
                }
                any = true;
                last = u;
                __syncwarp();
                if (lane == 0) mbar_arrive(info_empty(is));
            }
            if (!ok) break;
            // ---------------------------------------------------------------- the segment's result
            const bool whole = t0 == 0 && t1 == g.tiles;
            float* part = a.work + (int64_t)(2 * blockIdx.x + (t0 == 0 ? 1 : 0)) * RT * (D + 2);
            if (!warp_wait(pv_done(last), round_of(last), abort, WL)) { ok = false; break; }
            tc_fence_after();
            const bool live = mine < g.rows;
            if (warp_live) {
                const int h = live ? row - node * a.group : 0;
                const int64_t o_row = ((int64_t)g.b * a.nodes + node) * a.hq + g.head * a.group + h;
                const float down = 1.f / LIFT;
                const float by = whole ? (l == 0.f ? 0.f : down / l) : down;
                Two finite = two(0.f, 0.f);  // not-a-number if an element of O is not finite
#pragma unroll 1
                for (int k = 0; k < D; k += 16) {
                    uint32_t x[16];
                    tmem_ld16(lanes + S::O0 + w * D + k, x);
                    tmem_wait16(x);
                    float o[16];
#pragma unroll
                    for (int j = 0; j < 16; j += 2) finite = fma2(two(__uint_as_float(x[j]), __uint_as_float(x[j + 1])), two(0.f, 0.f), finite);
#pragma unroll
                    for (int j = 0; j < 16; j++) o[j] = __uint_as_float(x[j]) * by;
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
                if (live) {
                    if (whole) {
                        const float2 sure = one(finite);
                        // (a sum of weights that is not finite either is not-a-number in the formula too)
                        if (!(sure.x + sure.y == 0.f) && l > 0.f && l < -__int_as_float(0xff800000)) a.desc[DESC * blockIdx.x + 7] = HAS_SHARE | NOT_FINITE;
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
                int32_t* d = a.desc + DESC * blockIdx.x;
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
    if (warp == W_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)S::COLUMNS));
    if (*abort && tid == 0) atomicOr(a.c.status, GAVE_UP);
}

// ---------------------------------------------------------------- outputs that are not finite
// The products multiply every value of a tile by every row's weights, those of keys that a row does not see by zeros, and a
// weight's second part may be negative: a value that is not finite makes not-a-numbers of outputs that the formula gives as an
// infinity, or that it has no part in.  Large weights of large finite values may add up to an infinity.  Such outputs (an O that
// is not finite where the sum of weights is) are computed again from the formula, behind everything else, by the block that
// holds them: a column is what its values that are not finite make of it (weights are above zero), or, where a row sees none,
// the mean of its values by weights of at most one.  Finite inputs pay for a look at O and for the blocks of this code: 24 long
// int8 contexts under 32 nodes 386 us (381 without), 32 x 10 passages 63.3 (61.7), 131000 tokens under 64 nodes nothing.  Others
// pay for what is computed again: of those 131000 tokens 2 ms for an infinite value in one key head, 92 for a not-a-number
// in a node, whose siblings' scores are taken again; one short passage 60 and 120 us.
constexpr int JOIN_COLS = 32, JOIN_THREADS = 256, JOIN_LEAST = 96;  // JOIN_LEAST: CTAs whose maxima leave room for a Redo
constexpr int AGAIN = 4;                                            // rows at once

// a key's row, and its scales
struct Stored {
    const uint8_t *k, *v;
    float ks, vs;
};
template <int STORE>
__device__ __forceinline__ bool stored(const Args& a, int b, int head, int x, Stored& r) {
    int page, slot;
    if (!place(a.c, a.tb, b, x, page, slot) || (a.c.fill && slot >= __ldg(a.c.fill + page))) return false;
    const int64_t e = (int64_t)page * a.c.page_stride + (int64_t)slot * a.c.slot_stride + (int64_t)head * a.c.head_stride;
    constexpr int ESZ = STORE == FVS_I8 ? 1 : 2;
    r.k = (const uint8_t*)a.c.k + e * ESZ;
    r.v = (const uint8_t*)a.c.v + e * ESZ;
    r.ks = r.vs = 1.f;
    if (STORE == FVS_I8) {
        const int64_t se = (int64_t)page * a.c.scale_page_stride + (int64_t)slot * a.c.scale_slot_stride + (int64_t)head * a.c.scale_head_stride;
        r.ks = key_scale(a.c.k_scale + se);
        r.vs = __ldg(a.c.v_scale + se);
    }
    return true;
}
// 8 elements of a stored row
template <int STORE>
__device__ __forceinline__ void elements(const uint8_t* at, int first, float (&f)[8]) {
    if (STORE == FVS_I8) {
        const uint2 x = __ldg((const uint2*)(at + first));
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = (float)(int8_t)((i < 4 ? x.x : x.y) >> (8 * (i & 3)));
    } else {
        up8<STORE == FVS_I8 ? FVS_F16 : STORE>(__ldg((const uint4*)(at + 2 * first)), f);
    }
}
__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < __int_as_float(0x7f800000); }

struct Kinds {  // a bit for each of 32 columns
    uint32_t nan, up, down;
    __device__ __forceinline__ void add(const Kinds& x) {
        if (x.nan) atomicOr(&nan, x.nan);
        if (x.up) atomicOr(&up, x.up);
        if (x.down) atomicOr(&down, x.down);
    }
};
// what redo() keeps in shared memory
struct Redo {
    float q[AGAIN][256];
    float m[JOIN_THREADS / 32][AGAIN], l[JOIN_THREADS / 32][AGAIN];
    float o[JOIN_THREADS / 32][AGAIN][JOIN_COLS];
    uint32_t sees[AGAIN][FVS_TREE_NODES / 32];
    Kinds all, tree[AGAIN];
};

// Rows [row0, row0 + 32) of an item's row tile, those of `which`, columns [col, col + 32): outputs that are not finite, by the
// whole block, four lanes a key.  refs: a number near each row's largest score (log2), or null: a.lse has it, or, without one,
// the scores are looked at first (a row whose sum of weights is not finite is not-a-number in the formula too, and is left).
template <int D, int TYPE, int STORE, int RT>
__device__ __noinline__ void redo(const Args& a, Redo& s, int b, int head, int rt, int rows, int n, int keys, int row0, int col, uint32_t which,
                                  const float* refs) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane & 3;
    constexpr int STEP = JOIN_THREADS / 4;  // keys at once
    const float scale2 = a.scale * 1.4426950408889634f;
    const int before = min(n, keys);  // keys of the sequence, which all rows see
    bool known = false;               // what the values of the sequence's keys are, in s.all
    // (out and lse are read past the cache that other kernels' results may not be in)
    for (int r0 = 0; r0 < min(32, rows - row0); r0 += AGAIN) {
        uint32_t wrong[AGAIN], any = 0;
        int64_t at[AGAIN];
        float ref[AGAIN];
#pragma unroll
        for (int r = 0; r < AGAIN; r++) {
            wrong[r] = 0;
            if (row0 + r0 + r >= rows || !(which >> (r0 + r) & 1)) continue;
            const int row = rt * RT + row0 + r0 + r, node = row / a.group, h = head * a.group + row - node * a.group;
            at[r] = ((int64_t)b * a.nodes + node) * a.hq + h;
            const float was = Elem<TYPE>::up((uint32_t)__ldcg((const uint16_t*)a.out + at[r] * D + col + lane)).x;
            ref[r] = refs ? refs[r0 + r] : a.lse ? __ldcg(a.lse + at[r]) * 1.4426950408889634f : 0.f;
            if (is_finite(ref[r])) wrong[r] = __ballot_sync(0xffffffffu, !is_finite(was));  // the same in every warp
            any |= wrong[r];
        }
        __syncthreads();  // every warp has looked
        if (any == 0) continue;
        if (!known) {
            if (tid == 0) s.all = Kinds{0, 0, 0};
            __syncthreads();
        }
        // what is not finite in this lane's columns
        auto kinds = [&](const Stored& k) {
            Kinds x = {0, 0, 0};
            float f[8];
            elements<STORE>(k.v, col + 8 * sub, f);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float y = f[j] * k.vs;
                if (!is_finite(y)) (y > 0.f ? x.up : y < 0.f ? x.down : x.nan) |= 1u << (8 * sub + j);
            }
            return x;
        };
        if (!known) {
            known = true;
            for (int x = tid >> 2; x < before; x += STEP) {
                Stored k;
                if (stored<STORE>(a, b, head, x, k)) s.all.add(kinds(k));
            }
        }
        if (tid < AGAIN) {
            s.tree[tid] = Kinds{0, 0, 0};
            for (int i = 0; i < FVS_TREE_NODES / 32; i++) s.sees[tid][i] = 0;
            const int32_t* up = a.parents + (int64_t)b * a.parent_stride;
            const int row = row0 + r0 + tid;
            for (int i = row < rows ? (rt * RT + row) / a.group : -1; i >= 0;) {
                s.sees[tid][i >> 5] |= 1u << (i & 31);
                const int p = __ldg(up + i);
                i = p < i ? p : -1;
            }
        }
        for (int i = tid; i < AGAIN * D; i += JOIN_THREADS) {
            const int r = i / D, e = i - r * D, row = rt * RT + row0 + r0 + r, node = row / a.group, h = head * a.group + row - node * a.group;
            s.q[r][e] = row0 + r0 + r >= rows ? 0.f
                            : Elem<TYPE>::up((uint32_t)((const uint16_t*)a.q)[(int64_t)b * a.q_seq + (int64_t)node * a.q_node + (int64_t)h * a.q_head + e]).x;
        }
        __syncthreads();
        auto seen = [&](int r, int x) { return x < n || (s.sees[r][(x - n) >> 5] >> ((x - n) & 31) & 1); };
        for (int x = before + (tid >> 2); x < keys; x += STEP) {
            Stored k;
            if (!stored<STORE>(a, b, head, x, k)) continue;
            const Kinds of_node = kinds(k);
            for (int r = 0; r < AGAIN; r++)
                if (seen(r, x)) s.tree[r].add(of_node);
        }
        __syncthreads();
        bool scores = !refs && !a.lse;
#pragma unroll
        for (int r = 0; r < AGAIN; r++)
            scores = scores || (wrong[r] & ~(s.all.nan | s.all.up | s.all.down | s.tree[r].nan | s.tree[r].up | s.tree[r].down));
        float l[AGAIN] = {}, o[AGAIN][8] = {};
        if (scores) {
            // the rows' scores of a key, by its four lanes together
            auto score = [&](const Stored& k, bool there, float (&y)[AGAIN]) {
#pragma unroll
                for (int r = 0; r < AGAIN; r++) y[r] = 0.f;
                if (there) {
#pragma unroll 1
                    for (int e = 8 * sub; e < D; e += 32) {
                        float f[8];
                        elements<STORE>(k.k, e, f);
#pragma unroll
                        for (int r = 0; r < AGAIN; r++) {
#pragma unroll
                            for (int j = 0; j < 8; j++) y[r] = fmaf(s.q[r][e + j], f[j], y[r]);
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < AGAIN; r++) {
                    y[r] += __shfl_xor_sync(0xffffffffu, y[r], 1);
                    y[r] += __shfl_xor_sync(0xffffffffu, y[r], 2);
                    y[r] *= k.ks * scale2;
                }
            };
            if (!refs && !a.lse) {
                float m[AGAIN];
#pragma unroll
                for (int r = 0; r < AGAIN; r++) m[r] = __int_as_float(0xff800000);
                auto join = [&](int r, float om, float ol) {
                    const float top = fmaxf(m[r], om);
                    l[r] = l[r] * (m[r] == top ? 1.f : exp2_of(m[r] - top)) + ol * (om == top ? 1.f : exp2_of(om - top));
                    m[r] = top;
                };
                for (int x0 = 0; x0 < keys; x0 += STEP) {
                    const int x = x0 + (tid >> 2);
                    Stored k = {nullptr, nullptr, 0.f, 0.f};
                    const bool there = x < keys && stored<STORE>(a, b, head, x, k);
                    float y[AGAIN];
                    score(k, there, y);
#pragma unroll
                    for (int r = 0; r < AGAIN; r++)
                        if (there && seen(r, x)) join(r, y[r], 1.f);
                }
#pragma unroll
                for (int r = 0; r < AGAIN; r++) {
#pragma unroll
                    for (int i = 16; i >= 4; i >>= 1) {
                        const float om = __shfl_xor_sync(0xffffffffu, m[r], i), ol = __shfl_xor_sync(0xffffffffu, l[r], i);
                        join(r, om, ol);
                    }
                    if (lane == 0) s.m[warp][r] = m[r], s.l[warp][r] = l[r];
                }
                __syncthreads();
#pragma unroll
                for (int r = 0; r < AGAIN; r++) {
                    m[r] = __int_as_float(0xff800000), l[r] = 0.f;
                    for (int w = 0; w < JOIN_THREADS / 32; w++) join(r, s.m[w][r], s.l[w][r]);
                    ref[r] = m[r];
                    if (!is_finite(l[r])) wrong[r] = 0;
                    l[r] = 0.f;
                }
                __syncthreads();
            }
            for (int x0 = 0; x0 < keys; x0 += STEP) {
                const int x = x0 + (tid >> 2);
                Stored k = {nullptr, nullptr, 0.f, 0.f};
                const bool there = x < keys && stored<STORE>(a, b, head, x, k);
                float y[AGAIN], f[8];
                score(k, there, y);
                if (!there) continue;
                elements<STORE>(k.v, col + 8 * sub, f);
#pragma unroll
                for (int j = 0; j < 8; j++) f[j] = is_finite(f[j] * k.vs) ? f[j] * k.vs : 0.f;
#pragma unroll
                for (int r = 0; r < AGAIN; r++) {
                    if (!seen(r, x)) continue;
                    const float p = exp2_of(y[r] - ref[r]);
                    l[r] += p;
#pragma unroll
                    for (int j = 0; j < 8; j++) o[r][j] = fmaf(p, f[j], o[r][j]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < AGAIN; r++) {
#pragma unroll
            for (int i = 16; i >= 4; i >>= 1) {
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], i);
#pragma unroll
                for (int j = 0; j < 8; j++) o[r][j] += __shfl_xor_sync(0xffffffffu, o[r][j], i);
            }
            if (lane < 4) {
                if (lane == 0) s.l[warp][r] = l[r];
#pragma unroll
                for (int j = 0; j < 8; j++) s.o[warp][r][8 * sub + j] = o[r][j];
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < AGAIN; r++)
            if (warp == r && (wrong[r] >> lane & 1)) {
                float x = 0.f, sum = 0.f;
                for (int w = 0; w < JOIN_THREADS / 32; w++) x += s.o[w][r][lane], sum += s.l[w][r];
                const bool nan = (s.all.nan | s.tree[r].nan) >> lane & 1, up = (s.all.up | s.tree[r].up) >> lane & 1, down = (s.all.down | s.tree[r].down) >> lane & 1;
                x = nan || (up && down) ? __int_as_float(0x7fc00000) : up ? __int_as_float(0x7f800000) : down ? __int_as_float(0xff800000) : x / sum;
                ((uint16_t*)a.out)[at[r] * D + col + lane] = (uint16_t)Elem<TYPE>::down(x, 0.f);
            }
        __syncthreads();
    }
}

// what join_kernel's block has of such rows: those of the cut item in `which`, and items that its CTA computed whole
template <int D, int TYPE, int STORE, int RT, int KEYS>
__device__ __noinline__ void redo_block(const Args& a, Redo& s, int ctas, uint32_t which, const float* refs) {
    const int c = blockIdx.x, row0 = blockIdx.y * 32, col = blockIdx.z * JOIN_COLS;
    const int32_t* desc = a.desc + DESC * c;
    __syncthreads();
    if (which) {
        const Seq q = sequence<KEYS, RT>(a, desc[0]);
        redo<D, TYPE, STORE, RT>(a, s, desc[0], desc[2], desc[3], desc[4], q.n, q.keys, row0, col, which, refs);
    }
    if (!(desc[7] & NOT_FINITE)) return;
    Walk<KEYS, RT> walk;
    const int64_t total = *reinterpret_cast<const int64_t*>(desc + 12), have = shares(total, ctas);
    walk.begin(a, desc[8], *reinterpret_cast<const int64_t*>(desc + 10), share(total, have, c), share(total, have, c + 1));
    Seg g;
    while (walk.next(a, g))
        if (g.t0 == 0 && g.t1 == g.tiles && row0 < g.rows)
            redo<D, TYPE, STORE, RT>(a, s, g.b, g.head, g.rt, g.rows, g.n, g.keys, row0, col, 0xffffffffu, nullptr);
}

// Adds the shares of the items that were cut.  Block (c, 32 rows, 32 columns): the item that begins in CTA c and goes on in
// the CTAs behind it, each of which left one share.  The shares are read once, from L2 mostly, and what bounds it is the
// latency of its loads behind one another (descriptors, maxima and sums, O).  Then, where there are any, the outputs that are
// not finite, of this item and of those that CTA c computed whole.  Blocks of an SM, which redo_block's registers would cut to
// two: as many as the maxima leave room for with 296 CTAs, five; over int8 codes of 256 rows eight (24 long int8 contexts under
// 32 nodes: 386 us, 389 with five), over 16-bit ones five as well (131000 tokens under 64 nodes: 246 us, 250 with eight).
template <int D, int TYPE, int STORE, int RT, int KEYS>
__global__ void __launch_bounds__(JOIN_THREADS, RT == 256 && STORE == FVS_I8 ? 8 : 5) join_kernel(const __grid_constant__ Args a, int ctas) {
    constexpr int COLS = JOIN_COLS / 8;  // of a thread
    extern __shared__ float tops[];      // maxima [shares][32], no share's -infinity
    __shared__ float s_m[8][32], s_l[8][32];
    __shared__ int s_upto;
    __shared__ uint8_t s_has[512];
    __shared__ uint32_t s_wrong;         // rows with an O that is not finite
    __shared__ float s_ref[32];          // their sums' logarithms
    static_assert(sizeof(Redo) <= JOIN_LEAST * 32 * 4, "redo's memory takes that of the maxima");
    const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) s_upto = ctas, s_wrong = 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // all of the shares are there
    const int32_t* desc = a.desc + DESC * c;
    const int4 d = *reinterpret_cast<const int4*>(desc);
    const int b = d.x, item = d.y, head = d.z, rt = d.w, rows = desc[4], flags = desc[7];
    const int row = blockIdx.y * 32 + lane, col0 = blockIdx.z * JOIN_COLS;
    __syncthreads();
    if (b >= 0 && (int)blockIdx.y * 32 < rows) {
        // the CTAs behind that have a share of it: none between them has another item, some may have nothing at all
        for (int x = c + (int)threadIdx.x; x < ctas; x += JOIN_THREADS) {
            const int4 e = *reinterpret_cast<const int4*>(a.desc + DESC * x + 4);
            const bool has = x == c || (e.y == b && e.z == item);
            s_has[x - c] = has;
            if (!has && e.w != 0) atomicMin(&s_upto, x);
        }
        __syncthreads();
        const int shares = s_upto - c;
        auto part = [&](int i) { return a.work + (int64_t)(2 * (c + i) + (i == 0 ? 1 : 0)) * RT * (D + 2); };
        constexpr float NONE = -__builtin_huge_valf();
        float m = NONE, l = 0.f;
#pragma unroll 2
        for (int i = warp; i < shares; i += 8) {
            const bool there = s_has[i] && row < rows;
            const float x = there ? part(i)[D * RT + row] : NONE, y = there ? part(i)[(D + 1) * RT + row] : 0.f;
            tops[i * 32 + lane] = x;
            const float top = fmaxf(m, x);
            l = l * (m == top ? 1.f : exp2_of(m - top)) + y * (x == top ? 1.f : exp2_of(x - top));
            m = top;
        }
        s_m[warp][lane] = m;
        s_l[warp][lane] = l;
        __syncthreads();
        m = NONE;
#pragma unroll
        for (int w = 0; w < 8; w++) m = fmaxf(m, s_m[w][lane]);
        l = 0.f;
#pragma unroll
        for (int w = 0; w < 8; w++) l = fmaf(s_l[w][lane], s_m[w][lane] == m ? 1.f : exp2_of(s_m[w][lane] - m), l);
        if (row < rows) {
            const int at = rt * RT + row, node = at / a.group, h = at - node * a.group;
            const int64_t o_row = ((int64_t)b * a.nodes + node) * a.hq + head * a.group + h;
            const int col = col0 + warp * COLS;
            float o[COLS] = {};
#pragma unroll 4
            for (int i = 0; i < shares; i++) {
                const float top = tops[i * 32 + lane], by = top == m ? 1.f : exp2_of(top - m);
                const float* p = part(i) + col * RT + row;
                float x[COLS];
#pragma unroll
                for (int j = 0; j < COLS; j++) x[j] = p[j * RT];  // of a CTA without a share: anything, and not added
#pragma unroll
                for (int j = 0; j < COLS; j++)
                    if (top != NONE) o[j] = fmaf(x[j], by, o[j]);
            }
            const float by = l == 0.f ? 0.f : 1.f / l;
            uint32_t packed[COLS / 2];
            float finite = 0.f;  // not-a-number if an element of O is not finite
#pragma unroll
            for (int j = 0; j < COLS; j += 2) {
                packed[j / 2] = l == 0.f ? 0u : Elem<TYPE>::down(o[j] * by, o[j + 1] * by);
                finite = fmaf(o[j], 0.f, fmaf(o[j + 1], 0.f, finite));
            }
            uint16_t* out = (uint16_t*)a.out + o_row * D + col;
#pragma unroll
            for (int j = 0; j < COLS / 2; j++) reinterpret_cast<uint32_t*>(out)[j] = packed[j];
            if (blockIdx.z == 0 && warp == 0 && a.lse) a.lse[o_row] = l == 0.f ? NONE : (m + log2f(l)) * 0.6931471805599453f;
            if (finite != 0.f && l > 0.f && is_finite(l)) atomicOr(&s_wrong, 1u << lane), s_ref[lane] = m + log2f(l);
        }
        __syncthreads();
    }
    if (s_wrong || (flags & NOT_FINITE)) redo_block<D, TYPE, STORE, RT, KEYS>(a, *reinterpret_cast<Redo*>(tops), ctas, s_wrong, s_ref);
}

// the tensor maps of a 16-bit cache; false where tensor copies cannot take it
static bool make_maps(const fvs_kv_cache& c, Maps& maps, int& box) {
    box = 64;
    while (c.page % box) box /= 2;
    const EncodeTiledFn encode = encode_fn();
    if (box < 8 || !encode || c.slot_stride < 1 || c.head_stride < 1 || c.page_stride < 1) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)c.dim, (cuuint64_t)c.page, (cuuint64_t)c.heads, (cuuint64_t)c.pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c.slot_stride * 2, (cuuint64_t)c.head_stride * 2, (cuuint64_t)c.page_stride * 2};
    const cuuint32_t tile[4] = {64, (cuuint32_t)box, 1, 1}, ones[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = c.type == FVS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    for (int i = 0; i < 2; i++)
        if (encode(i ? &maps.v : &maps.k, type, 4, i ? c.v : c.k, dims, strides, tile, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
    return true;
}

template <int D, int TYPE, int STORE, int MT, int QR, bool BOXES>
static int launch(fvs_stream_t stream, Args a, const Maps& maps) {
    using S = Shape<D, STORE, MT, QR>;
    constexpr int RT = ROWS * MT;
    const int ctas = fvs_sm_count() * S::CTAS;
    const void* f = (const void*)tree_kernel<D, TYPE, STORE, MT, QR, BOXES>;
    cudaError_t e = fvs_ensure_smem(f, S::BYTES);
    if (e != cudaSuccess) return (int)e;
    a.wait_limit = pipeline_wait_limit();
    a.desc = (int32_t*)a.work;
    a.work = a.work + DESC * ctas;
    tree_kernel<D, TYPE, STORE, MT, QR, BOXES><<<ctas, S::THREADS, S::BYTES, stream>>>(a, maps);
    if (int rc = fvs_launch_status()) return rc;
    const int rows = a.nodes * a.group;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, ((rows < RT ? rows : RT) + 31) / 32, D / JOIN_COLS);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = (ctas > JOIN_LEAST ? ctas : JOIN_LEAST) * 32 * 4;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, join_kernel<D, TYPE, STORE, RT, S::KEYS>, a, ctas);
    if (e != cudaSuccess) return (int)e;
    return fvs_launch_status();
}

// kernels over heads of D elements, by the rows of an item: 256 at a time where there are more than 128, queries of 64 where
// there are no more (heads wider than 128: always 128)
template <int D, int TYPE, int STORE, bool BOXES>
static int launch_rows(fvs_stream_t stream, const Args& a, const Maps& maps) {
    constexpr bool narrow = D <= 128;
    const int rows = a.nodes * a.group;
    if (narrow && rows > ROWS) return launch<D, TYPE, STORE, narrow ? 2 : 1, ROWS, BOXES>(stream, a, maps);
    if (narrow && rows <= 64) return launch<D, TYPE, STORE, 1, narrow ? 64 : ROWS, BOXES>(stream, a, maps);
    return launch<D, TYPE, STORE, 1, ROWS, BOXES>(stream, a, maps);
}
template <int D>
int launch_types(fvs_stream_t stream, Args a, int type) {
    Maps maps = {};
    // what the other copies and the queries hold of an address: 32 bits of 16 bytes
    const int64_t last = (a.c.pages - 1) * a.c.page_stride + (a.c.heads - 1) * a.c.head_stride + (a.c.page - 1) * a.c.slot_stride;
    const int64_t last_q = (a.tb.seqs - 1) * a.q_seq + (a.nodes - 1) * a.q_node + (a.hq - 1) * a.q_head, most = 0xfffffff0ll;
    const bool small = last / (a.c.type == FVS_I8 ? 16 : 8) < most;
    if (last_q / 8 >= most || (a.c.type == FVS_I8 && !small)) return FVS_ERANGE;
    if (a.c.type == FVS_I8) return type == FVS_F16 ? launch_rows<D, FVS_F16, FVS_I8, false>(stream, a, maps) : launch_rows<D, FVS_BF16, FVS_I8, false>(stream, a, maps);
    if (make_maps(a.c, maps, a.box)) return type == FVS_F16 ? launch_rows<D, FVS_F16, FVS_F16, true>(stream, a, maps) : launch_rows<D, FVS_BF16, FVS_BF16, true>(stream, a, maps);
    if (!small) return FVS_ERANGE;
    return type == FVS_F16 ? launch_rows<D, FVS_F16, FVS_F16, false>(stream, a, maps) : launch_rows<D, FVS_BF16, FVS_BF16, false>(stream, a, maps);
}

}  // namespace tree
}  // namespace kv
}  // namespace fvs
