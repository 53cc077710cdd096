// Attention of one new token per sequence over a paged key-value cache (new; see include/fanar_b200.h).
//
// One pass over the keys with the running maximum m and sum l of the softmax: a tile of keys with scores s changes them to
// m' = max(m, max s), l' = l 2^(m - m') + sum 2^(s - m'), and the accumulated output by o' = o 2^(m - m') + sum
// 2^(s - m') v.  Scores are in units of log2 (scale * log2 e); m, l, o and all sums are fp32.
//
// Work.  A unit is 16 keys of one (sequence, key head, group of up to 8 NT query heads) item.  The items in order, each
// of ITEM_COST + its units, are cut into ranges of equal cost, one for each CTA of four warps, so that any mix of
// lengths keeps every SM busy and a long sequence is split without the host knowing any length.  The warps of a CTA take
// an item's units in turn and add up their results in shared memory; an item of few units is one warp's.  A range that
// holds a whole item writes its output; parts of an item go to the workspace, and the CTA that finishes an item's last
// part (counted by an atomic, joined in range order, so that results do not depend on the order of arrival) joins them.
//
// A warp copies its units' key and value rows with cp.async into a ring of its own (no block barrier between units; page
// numbers are looked up two units ahead of the copy) and multiplies with mma.sync m16n8k16.  Both products run
// transposed, S^T = K Q^T and O^T = V^T P^T: the 16 keys (then 16 output elements) fill the M side whatever the number of
// query heads that share a key head, and 8 heads fill N, where heads on M would leave half of a tile empty for 8 or
// fewer.  The probabilities pass from one layout to the other with movmatrix.  mma.sync and not tcgen05: each key feeds at
// most 16 query rows, so the bound is the cache's bytes (2 G / element size flops per byte), and tcgen05's 128-row
// tiles would be padded eightfold and more.
//
// The maximum moves only when a score passes it by more than 8 (a factor of 2^8 keeps fp32 sums and 16-bit probabilities
// in range), so most units need one vote instead of shuffles and a rescale.
//
// Rounding: probabilities enter the second product in 16 bits (the type of v; fp16 for int8 codes), like the output
// itself; l sums them in fp32 before that.  int8 codes are exact in fp16; their key scale multiplies the fp32 score, their
// value scale the probability, divided by the largest power of two met so far so that it stays in fp16's range; queries
// over int8 codes are brought to fp16 by a power of two for each head.
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
    int32_t* arrived;  // [items], zero between calls
    float* parts;
    int hq, group;     // query heads, query heads of a key head
    float scale2;      // scale * log2 e
};

constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int UNIT = 16;       // keys
constexpr int ITEM_COST = 3;   // of an item beside its units (loading q, adding up and writing), in units
constexpr float SLACK = 8.f;   // how far (log2) a score may pass the running maximum before it moves

template <int D, int STORE, int NT_>
struct Shape {
    static constexpr bool I8 = STORE == FVS_I8;
    static constexpr int NT = NT_;
    static constexpr int ROWS = 8 * NT;              // query heads of an item
    static constexpr int RB = D * (I8 ? 1 : 2);      // bytes of a row
    // row strides in shared memory that keep every access below free of bank conflicts: 16-bit rows are read by ldmatrix
    // (an odd number of 16-byte chunks); int8 keys 8 bytes a lane from 4 rows at a time (stride
    // = 32 or 96 mod 128), int8 values 4 bytes a lane from every second row (twice the stride = 32 or 96 mod 128)
    static constexpr int KS = I8 ? (D == 96 ? 160 : D + 32) : RB + 16;
    static constexpr int VS = RB + 16;
    static constexpr int SCALES = UNIT * (KS + VS);  // byte offset of the scales [2][16]
    static constexpr int MASK = SCALES + (I8 ? 128 : 0);
    static constexpr int STAGE = MASK + 16;
    static constexpr int OS = D + 4;                 // row stride (floats) of a staged output tile
    static constexpr int OBYTES = ROWS * OS * 4;
    static constexpr bool O_IN_RING = OBYTES <= STAGE;
    static constexpr int CTAS = RB <= 128 && NT == 1 ? 3 : RB <= 256 ? 2 : 1;  // per SM
    static constexpr int BUDGET = (227 * 1024) / CTAS - 1024 - 1024 - (O_IN_RING ? 0 : WARPS * OBYTES);
    static constexpr int FIT = BUDGET / (WARPS * STAGE);
    static constexpr int S = FIT > 6 ? 6 : FIT;      // ring stages
    static_assert(S >= 2, "ring");
    static constexpr int RING = S * STAGE;           // bytes per warp
    static constexpr int SMEM = WARPS * (RING + (O_IN_RING ? 0 : OBYTES));
    static constexpr int PART = ROWS * (D + 2);      // floats of a partial result
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at));
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <int TYPE>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (TYPE == FVS_F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// weight of a part with maximum and sum `ml` in a join whose maximum is mx (a part of not-a-numbers alone keeps them)
__device__ __forceinline__ float weight(float2 ml, float mx) {
    return ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2_fast(ml.x - mx);
}
// two codes (bytes chosen by `sel` from w ^ 0x80808080) as fp16: 0x6400 | u is 1024 + u, less 1152 is the signed code
__device__ __forceinline__ uint32_t codes2(uint32_t w, uint32_t sel) {
    const uint32_t x = __byte_perm(w, 0x64646464u, sel);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&y);
}

__device__ __forceinline__ int seq_len(const AttendArgs& a, int b) {
    const int len = __ldg(a.lens + b);
    const int64_t room = (int64_t)a.tb.wide * a.c.page;
    return len > room ? (int)room : max(len, 0);
}
__device__ __forceinline__ int units_of(int len) { return (int)(((unsigned)len + UNIT - 1) / UNIT); }

// A place in the order of all items: unit u of item hh (of per_seq) of sequence b.
struct Place {
    int b, hh, u;
};

// An item, with the units [u, end) of it that lie in a CTA's range.
struct Item {
    int b, hh, len, n, u, end;
};
__device__ __forceinline__ void clip(Item& it, const Place& stop) {
    it.end = it.b == stop.b && it.hh == stop.hh ? stop.u : it.n;
}
// the next item of the range; false at its end
__device__ __forceinline__ bool next_item(const AttendArgs& a, Item& it, const Place& stop, int per_seq) {
    if (++it.hh == per_seq) {
        it.hh = 0;
        do {
            if (++it.b > stop.b || it.b >= a.tb.seqs) return false;
            it.len = seq_len(a, it.b);
            it.n = units_of(it.len);
        } while (it.n == 0);
    }
    it.u = 0;
    clip(it, stop);
    return it.b < stop.b || (it.b == stop.b && it.hh <= stop.hh && it.end > 0);
}

// One key of a unit on its way from the page table to the copy.
struct Lookup {
    int entry, slot, head, fill;
    bool live;  // there is such a unit
};

template <int D, int TYPE, int STORE, int NT>
__global__ void __launch_bounds__(THREADS, Shape<D, STORE, NT>::CTAS) attend_kernel(AttendArgs a) {
    using Sh = Shape<D, STORE, NT>;
    constexpr bool I8 = Sh::I8;
    constexpr int MT = I8 ? FVS_F16 : TYPE;  // type of the matrix instructions' operands
    constexpr int S = Sh::S;
    extern __shared__ __align__(16) uint8_t ring_all[];
    __shared__ int64_t s_sum[WARPS];
    __shared__ int s_none[WARPS];
    __shared__ int64_t s_before[THREADS];  // cost (for one item of each sequence) before each thread's sequences
    __shared__ Place s_place[2];           // where this CTA's range begins and ends
    __shared__ int64_t s_base;             // cost before the first sequence of the range
    __shared__ float s_ml[WARPS][Sh::ROWS][2];
    __shared__ int s_tile[WARPS], s_last;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = lane >> 2, c4 = lane & 3;
    const int split = (a.group + Sh::ROWS - 1) / Sh::ROWS;  // items of a key head
    const int per_seq = a.c.heads * split;
    const int B = a.tb.seqs;

    // ---- cost of all sequences (each thread a run of them)
    const int chunk = (B + THREADS - 1) / THREADS;
    const int b_hi = min(B, (tid + 1) * chunk);
    int64_t mine = 0;
    int none = 0;
    for (int b0 = tid * chunk; b0 < b_hi; b0 += 8) {
        unsigned sum = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (b0 + j < b_hi) {
                const int n = units_of(seq_len(a, b0 + j));
                sum += n ? n + ITEM_COST : 0;
                none += n == 0;
            }
        }
        mine += sum;
    }
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    none = __reduce_add_sync(0xffffffffu, none);
    if (lane == 31) s_sum[warp] = incl;
    if (lane == 0) s_none[warp] = none;
    __syncthreads();
    int64_t before = incl - mine, total = 0;
    none = 0;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
        if (w < warp) before += s_sum[w];
        total += s_sum[w];
        none += s_none[w];
    }
    s_before[tid] = before;
    total *= per_seq;
    if (blockIdx.x == 0)
        for (int b = tid; b < B; b += THREADS)
            if (__ldg(a.lens + b) > (int64_t)a.tb.wide * a.c.page) atomicOr(a.c.status, BAD_INDEX);
    if (none) {  // sequences without a token: this CTA's share of all
        for (int b0 = 0; b0 < B; b0 += gridDim.x * 32) {
            const int b = b0 + lane * gridDim.x + blockIdx.x;
            for (uint32_t z = __ballot_sync(0xffffffffu, b < B && __ldg(a.lens + (b < B ? b : 0)) <= 0); z; z &= z - 1) {
                const int64_t bz = b0 + (int64_t)(__ffs(z) - 1) * gridDim.x + blockIdx.x;
                uint4* o = (uint4*)((uint16_t*)a.out + bz * a.hq * D);
                for (int i = tid; i < a.hq * D / 8; i += THREADS) o[i] = make_uint4(0, 0, 0, 0);
                if (a.lse)
                    for (int i = tid; i < a.hq; i += THREADS) a.lse[bz * a.hq + i] = -INFINITY;
            }
        }
    }
    // ---- this CTA's range of the cost.  Unit u of an item that begins at cost x lies at x + ITEM_COST + u.  A cut nearer
    // than `near` units to an item's begin or end moves there: joining two parts costs more than that
    int64_t per = (total + gridDim.x - 1) / gridDim.x;
    if (per < 16) per = 16;
    if (blockIdx.x * per >= total) return;
    const int near = per > 64 ? (int)(per / 8) : 8;
    const int alone = per > 128 ? 16 : (int)(per / 8);  // items of up to so many units are one warp's
    __syncthreads();
    if (warp < 2) {
        const int64_t g = (blockIdx.x + warp) * per;
        if (g >= total) {
            if (lane == 0) s_place[warp] = Place{B, 0, 0};
        } else {
            int at = 0;  // the last run of sequences that begins at or before g
#pragma unroll
            for (int j = 0; j < THREADS / 32; j++) at += s_before[j * 32 + lane] * per_seq <= g;
            at = (int)__reduce_add_sync(0xffffffffu, (unsigned)at) - 1;
            int64_t base = s_before[at];
            for (int b0 = at * chunk; b0 < B; b0 += 32) {
                const int n = b0 + lane < B ? units_of(seq_len(a, b0 + lane)) : 0;
                const int64_t cost = n ? n + ITEM_COST : 0;
                int64_t upto = cost;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += x;
                }
                const uint32_t past = __ballot_sync(0xffffffffu, (base + upto) * per_seq > g);
                if (past) {
                    if (lane == __ffs(past) - 1) {
                        const int64_t in = g - (base + upto - cost) * per_seq;
                        const int hh = (int)(in / cost), u = (int)(in - hh * cost) - ITEM_COST;
                        s_place[warp] = u < near ? Place{b0 + lane, hh, 0} : n - u < near ? Place{b0 + lane, hh + 1, 0} : Place{b0 + lane, hh, u};
                        if (warp == 0) s_base = base + upto - cost;
                    }
                    break;
                }
                base += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
    }
    __syncthreads();
    const Place stop = s_place[1];
    Item now;  // the item under computation
    now.b = s_place[0].b;
    now.hh = s_place[0].hh;
    now.len = seq_len(a, now.b);
    now.n = units_of(now.len);
    now.u = s_place[0].u;
    clip(now, stop);
    int64_t base = s_base;
    bool more = true;
    if (now.hh == per_seq) {  // moved past the sequence's last item
        const int b = now.b;
        now.hh--;
        more = next_item(a, now, stop, per_seq);
        if (now.b != b) base += units_of(seq_len(a, b)) + ITEM_COST;
    } else {
        more = now.b < stop.b || (now.b == stop.b && (now.hh < stop.hh || (now.hh == stop.hh && now.u < stop.u)));
    }
    if (!more) return;
    // the units that this warp copies: every fourth of an item, all of one that it has alone
    Item ahead = now;
    bool any = true;
    auto owner = [&](const Item& it) { return (it.b * per_seq + it.hh) % WARPS; };
    auto settle = [&]() {
        while (any && ahead.u >= ahead.end) {
            any = next_item(a, ahead, stop, per_seq);
            if (any) ahead.u = ahead.n > alone ? warp : owner(ahead) == warp ? 0 : ahead.end;
        }
    };
    ahead.u = ahead.n > alone ? ahead.u + warp : owner(ahead) == warp ? 0 : ahead.end;
    settle();

    uint8_t* ring = ring_all + warp * Sh::RING;
    const uint32_t ring_at = smem_addr(ring);

    // ---- copies, two lookups ahead
    auto look = [&]() {
        Lookup k;
        k.entry = -1;
        k.slot = 0;
        k.head = 0;
        k.live = any;
        if (any) {
            const int t = ahead.u * UNIT + (lane & 15);
            if (t < ahead.len) {
                const int p = (int)((unsigned)t / (unsigned)a.c.page);
                k.slot = t - p * a.c.page;
                k.entry = __ldg(a.tb.at + (int64_t)ahead.b * a.tb.stride + p);
            }
            k.head = ahead.hh / split;
            ahead.u += ahead.n > alone ? WARPS : 1;
            settle();
        }
        return k;
    };
    auto look_fill = [&](Lookup& k) {
        if (k.entry >= a.c.pages) {
            atomicOr(a.c.status, BAD_INDEX);
            k.entry = -1;
        }
        k.fill = a.c.fill && k.entry >= 0 ? __ldg(a.c.fill + k.entry) : 0x7fffffff;
    };
    auto issue = [&](const Lookup& k, int slot) {
        const bool live = k.entry >= 0 && k.slot < k.fill;
        const uint32_t mask = __ballot_sync(0xffffffffu, live);
        const int64_t row = live ? (int64_t)k.entry * a.c.page_stride + (int64_t)k.head * a.c.head_stride +
                                       (int64_t)k.slot * a.c.slot_stride
                                 : 0;
        const uint32_t st = ring_at + slot * Sh::STAGE;
        constexpr int PER = Sh::RB / 16;  // chunks of a row
        constexpr int ESZ = I8 ? 1 : 2;
#pragma unroll
        for (int i = 0; i < UNIT * PER / 32; i++) {
            const int at = i * 32 + lane, key = at / PER, ch = at % PER;
            const int64_t off = __shfl_sync(0xffffffffu, row, key) * ESZ + ch * 16;
            const bool on = (mask >> key) & 1;
            copy16(st + key * Sh::KS + ch * 16, (const uint8_t*)a.c.k + off, on);
            copy16(st + UNIT * Sh::KS + key * Sh::VS + ch * 16, (const uint8_t*)a.c.v + off, on);
        }
        if (I8) {
            const int64_t at = live ? (int64_t)k.entry * a.c.scale_page_stride + (int64_t)k.head * a.c.scale_head_stride +
                                          (int64_t)k.slot * a.c.scale_slot_stride
                                    : 0;
            copy4(st + Sh::SCALES + lane * 4, (lane < 16 ? a.c.k_scale : a.c.v_scale) + at, live);
        }
        if (lane == 0) *(uint32_t*)(ring + slot * Sh::STAGE + Sh::MASK) = mask & 0xffffu;
    };
    Lookup la = look();
    look_fill(la);
    Lookup lb = look();
    int ready = 0;                                         // next slot to fill
    auto feed = [&]() {
        if (la.live) issue(la, ready);
        copies_commit();
        ready = ready + 1 == S ? 0 : ready + 1;
        la = lb;
        look_fill(la);
        lb = look();
    };
#pragma unroll 1
    for (int i = 0; i < S - 1; i++) feed();

    // ---- the range's items
    int slot = 0;
#pragma unroll 1
    for (; more;) {
        const bool solo = now.n <= alone;
        const int kvh = now.hh / split, h0 = kvh * a.group + (now.hh % split) * Sh::ROWS;
        const int rows = min(Sh::ROWS, a.group - (now.hh % split) * Sh::ROWS);
        const Item it = now;
        const int64_t it_begin = base * per_seq + (int64_t)now.hh * (now.n + ITEM_COST);
        more = next_item(a, now, stop, per_seq);
        if (now.b != it.b) base += it.n + ITEM_COST;
        if (solo && owner(it) != warp) continue;
        auto team_sync = [&]() {
            if (solo)
                __syncwarp();
            else
                __syncthreads();
        };

        // q as the B operand: head r of each 8, elements of the order in which the keys' rows come
        uint32_t qf[NT][D / 16][2];
        float mul[NT][2];  // what a raw product is multiplied with, for heads 2 c4 and 2 c4 + 1
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int h = t * 8 + r;
            const uint16_t* qp = (const uint16_t*)a.q + it.b * a.q_seq + (int64_t)(h0 + h) * a.q_head;
            if (I8) {
                uint2 raw[D / 16];
                float top = 0.f;
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    raw[k] = h < rows ? __ldg((const uint2*)(qp + (k / 2) * 32 + c4 * 8 + (k & 1) * 4)) : make_uint2(0, 0);
                    const float2 x = Elem<TYPE>::up(raw[k].x), y = Elem<TYPE>::up(raw[k].y);
                    top = fmaxf(top, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))));
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e = max(1, min(252, (int)(__float_as_uint(top) >> 23)));  // 2^(e - 127) <= top
                const float down = __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    const float2 x = Elem<TYPE>::up(raw[k].x), y = Elem<TYPE>::up(raw[k].y);
                    qf[t][k][0] = Elem<FVS_F16>::down(x.x * down, x.y * down);
                    qf[t][k][1] = Elem<FVS_F16>::down(y.x * down, y.y * down);
                }
                const float up = a.scale2 * __uint_as_float((uint32_t)e << 23);
                mul[t][0] = __shfl_sync(0xffffffffu, up, c4 * 8);
                mul[t][1] = __shfl_sync(0xffffffffu, up, c4 * 8 + 4);
            } else {
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    qf[t][k][0] = h < rows ? __ldg((const uint32_t*)(qp + k * 16 + c4 * 2)) : 0u;
                    qf[t][k][1] = h < rows ? __ldg((const uint32_t*)(qp + k * 16 + c4 * 2 + 8)) : 0u;
                }
                mul[t][0] = mul[t][1] = a.scale2;
            }
        }
        float m[NT][2], l[NT][2], o[D / 16][NT][4];
        int vexp = 1;  // int8: value scales are divided by 2^(vexp - 126)
#pragma unroll
        for (int t = 0; t < NT; t++) m[t][0] = m[t][1] = -INFINITY, l[t][0] = l[t][1] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; i++)
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int x = 0; x < 4; x++) o[i][t][x] = 0.f;

#pragma unroll 1
        for (int u = solo ? it.u : it.u + warp; u < it.end; u += solo ? 1 : WARPS) {
            copies_wait<S - 2>();
            __syncwarp();
            feed();
            const uint32_t st = ring_at + slot * Sh::STAGE;
            const uint8_t* stp = ring + slot * Sh::STAGE;
            slot = slot + 1 == S ? 0 : slot + 1;
            const uint32_t mask = *(const uint32_t*)(stp + Sh::MASK);
            if (mask == 0) continue;
            // S^T = K Q^T, in two chains
            float s[NT][4], s2[NT][4];
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int x = 0; x < 4; x++) s[t][x] = s2[t][x] = 0.f;
            if (I8) {
#pragma unroll
                for (int k = 0; k < D / 32; k++) {
                    uint2 lo = *(const uint2*)(stp + r * Sh::KS + k * 32 + c4 * 8);
                    uint2 hi = *(const uint2*)(stp + (r + 8) * Sh::KS + k * 32 + c4 * 8);
                    lo.x ^= 0x80808080u, lo.y ^= 0x80808080u, hi.x ^= 0x80808080u, hi.y ^= 0x80808080u;
                    const uint32_t f0[4] = {codes2(lo.x, 0x4140), codes2(hi.x, 0x4140), codes2(lo.x, 0x4342), codes2(hi.x, 0x4342)};
                    const uint32_t f1[4] = {codes2(lo.y, 0x4140), codes2(hi.y, 0x4140), codes2(lo.y, 0x4342), codes2(hi.y, 0x4342)};
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        mma<MT>(s[t], f0, qf[t][2 * k][0], qf[t][2 * k][1]);
                        mma<MT>(s2[t], f1, qf[t][2 * k + 1][0], qf[t][2 * k + 1][1]);
                    }
                }
            } else {
                const uint32_t at = st + (lane & 15) * Sh::KS + (lane >> 4) * 16;
#pragma unroll
                for (int k = 0; k < D / 16; k += 2) {
                    uint32_t f0[4], f1[4];
                    ldm4(f0, at + k * 32);
                    ldm4(f1, at + k * 32 + 32);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        mma<MT>(s[t], f0, qf[t][k][0], qf[t][k][1]);
                        mma<MT>(s2[t], f1, qf[t][k + 1][0], qf[t][k + 1][1]);
                    }
                }
            }
            const bool on0 = (mask >> r) & 1, on1 = (mask >> (r + 8)) & 1;
            float ks0 = 1.f, ks1 = 1.f, vs0 = 1.f, vs1 = 1.f;
            if (I8) {
                const float* sc = (const float*)(stp + Sh::SCALES);
                ks0 = sc[r], ks1 = sc[r + 8], vs0 = sc[16 + r], vs1 = sc[24 + r];
            }
            bool moved = false;
#pragma unroll
            for (int t = 0; t < NT; t++) {
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const float raw = s[t][x] + s2[t][x];
                    const float y = I8 ? raw * (x < 2 ? ks0 : ks1) * mul[t][x & 1] : raw * mul[t][x & 1];
                    s[t][x] = (x < 2 ? on0 : on1) ? y : -INFINITY;
                }
                moved |= fmaxf(s[t][0], s[t][2]) > m[t][0] + SLACK || fmaxf(s[t][1], s[t][3]) > m[t][1] + SLACK;
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int t = 0; t < NT; t++) {
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        float y = fmaxf(s[t][x], s[t][x + 2]);
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, d));
                        y = fmaxf(y, m[t][x]);
                        const float f = y == -INFINITY ? 1.f : exp2_fast(m[t][x] - y);
                        m[t][x] = y;
                        l[t][x] *= f;
#pragma unroll
                        for (int i = 0; i < D / 16; i++) o[i][t][x] *= f, o[i][t][x + 2] *= f;
                    }
                }
            }
            if (I8) {
                const uint32_t big = max(__float_as_uint(vs0) & 0x7fffffffu, __float_as_uint(vs1) & 0x7fffffffu);
                const int e = min(252, (int)(__reduce_max_sync(0xffffffffu, big) >> 23));
                if (e > vexp) {
                    const float f = e - vexp >= 126 ? 0.f : __uint_as_float((uint32_t)(127 - (e - vexp)) << 23);
                    vexp = e;
#pragma unroll
                    for (int i = 0; i < D / 16; i++)
#pragma unroll
                        for (int t = 0; t < NT; t++)
#pragma unroll
                            for (int x = 0; x < 4; x++) o[i][t][x] *= f;
                }
                const float down = __uint_as_float((uint32_t)(253 - vexp) << 23);
                vs0 *= down, vs1 *= down;
            }
            // p, and p as the B operand of the second product
            uint32_t pf[NT][2];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const float z0 = m[t][0] == -INFINITY ? 0.f : m[t][0], z1 = m[t][1] == -INFINITY ? 0.f : m[t][1];
                float p0 = exp2_fast(s[t][0] - z0), p1 = exp2_fast(s[t][1] - z1);
                float p2 = exp2_fast(s[t][2] - z0), p3 = exp2_fast(s[t][3] - z1);
                l[t][0] += p0 + p2;
                l[t][1] += p1 + p3;
                if (I8) p0 *= vs0, p1 *= vs0, p2 *= vs1, p3 *= vs1;
                pf[t][0] = transpose8x8(Elem<MT>::down(p0, p1));
                pf[t][1] = transpose8x8(Elem<MT>::down(p2, p3));
            }
            // O^T += V^T P^T
            if (I8) {
                const uint8_t* v = stp + UNIT * Sh::KS + r * 4;
#pragma unroll
                for (int j = 0; j < D / 32; j++) {
                    const uint32_t v0 = *(const uint32_t*)(v + (2 * c4) * Sh::VS + j * 32) ^ 0x80808080u;
                    const uint32_t v1 = *(const uint32_t*)(v + (2 * c4 + 1) * Sh::VS + j * 32) ^ 0x80808080u;
                    const uint32_t v2 = *(const uint32_t*)(v + (2 * c4 + 8) * Sh::VS + j * 32) ^ 0x80808080u;
                    const uint32_t v3 = *(const uint32_t*)(v + (2 * c4 + 9) * Sh::VS + j * 32) ^ 0x80808080u;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t x = __byte_perm(v0, v1, h ? 0x7362 : 0x5140), y = __byte_perm(v2, v3, h ? 0x7362 : 0x5140);
                        const uint32_t f[4] = {codes2(x, 0x4140), codes2(x, 0x4342), codes2(y, 0x4140), codes2(y, 0x4342)};
#pragma unroll
                        for (int t = 0; t < NT; t++) mma<MT>(o[2 * j + h][t], f, pf[t][0], pf[t][1]);
                    }
                }
            } else {
                const uint32_t at = st + UNIT * Sh::KS + ((lane >> 4) * 8 + (lane & 7)) * Sh::VS + ((lane >> 3) & 1) * 16;
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    uint32_t f[4];
                    ldm4t(f, at + i * 32);
#pragma unroll
                    for (int t = 0; t < NT; t++) mma<MT>(o[i][t], f, pf[t][0], pf[t][1]);
                }
            }
        }

        // ---- the item's result: the warps' tiles through shared memory (each warp's ring slot that its next copy fills)
        __syncwarp();
        float* tile = Sh::O_IN_RING ? (float*)(ring + ready * Sh::STAGE)
                                    : (float*)(ring_all + WARPS * Sh::RING + warp * Sh::OBYTES);
        const float vup = I8 ? __uint_as_float((uint32_t)(vexp + 1) << 23) : 1.f;
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                float y = l[t][x];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) y += __shfl_xor_sync(0xffffffffu, y, d);
                const int row = t * 8 + 2 * c4 + x;
                if (r == 0) s_ml[warp][row][0] = m[t][x], s_ml[warp][row][1] = y;
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    float* p = tile + row * Sh::OS + (I8 ? (i / 2) * 32 + 4 * r + 2 * (i & 1) : i * 16 + r);
                    p[0] = o[i][t][x] * vup;
                    p[I8 ? 1 : 8] = o[i][t][x + 2] * vup;
                }
            }
        }
        if (lane == 0) s_tile[warp] = (int)((uint8_t*)tile - ring_all);
        team_sync();
        const bool whole = it.u == 0 && it.end == it.n;
        const int tt = solo ? lane : tid, nthr = solo ? 32 : THREADS;
        const int w_lo = solo ? warp : 0, w_hi = solo ? warp + 1 : WARPS;
        // an item's first part is its CTA's second one: that CTA may hold the last part of another
        float* part = a.parts + (int64_t)(2 * blockIdx.x + (it.u == 0)) * Sh::PART;
        constexpr int Q4 = D / 4;
        auto finish = [&](int row, int d, float mx, float sum, const float4& acc) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int64_t h = (int64_t)it.b * a.hq + h0 + row;
            *(uint2*)((uint16_t*)a.out + h * D + d) =
                sum == 0.f ? make_uint2(0, 0)
                           : make_uint2(Elem<TYPE>::down(acc.x * inv, acc.y * inv), Elem<TYPE>::down(acc.z * inv, acc.w * inv));
            if (d == 0 && a.lse) a.lse[h] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * 0.6931471805599453f;
        };
        for (int i = tt; i < rows * Q4; i += nthr) {
            const int row = i / Q4, d = (i - row * Q4) * 4;
            float mx = -INFINITY;
            for (int w = w_lo; w < w_hi; w++) mx = fmaxf(mx, s_ml[w][row][0]);
            float sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int w = w_lo; w < w_hi; w++) {
                const float f = weight(make_float2(s_ml[w][row][0], s_ml[w][row][1]), mx);
                const float4 x = *(const float4*)((const float*)(ring_all + s_tile[w]) + row * Sh::OS + d);
                if (f != 0.f) {
                    sum += s_ml[w][row][1] * f;
                    acc.x += x.x * f, acc.y += x.y * f, acc.z += x.z * f, acc.w += x.w * f;
                }
            }
            if (whole) {
                finish(row, d, mx, sum, acc);
            } else {
                *(float4*)(part + row * D + d) = acc;
                if (d == 0) *(float2*)(part + Sh::ROWS * D + 2 * row) = make_float2(mx, sum);
            }
        }
        if (!whole) {  // never alone: an item of so few units is not cut
            __threadfence();
            __syncthreads();
            // the cuts inside the item lie at multiples of per; parts - 1 of them, the first at t_lo * per
            const int t_lo = (int)((it_begin + ITEM_COST + near + per - 1) / per);
            const int parts = (int)((it_begin + ITEM_COST + it.n - near) / per) - t_lo + 2;
            if (tid == 0) {
                const int64_t item = (int64_t)it.b * per_seq + it.hh;
                s_last = atomicAdd(a.arrived + item, 1) == parts - 1;
                if (s_last) a.arrived[item] = 0;
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                for (int i = tid; i < rows * Q4; i += THREADS) {
                    const int row = i / Q4, d = (i - row * Q4) * 4;
                    const float* from = a.parts + (int64_t)2 * (t_lo - 1) * Sh::PART;
                    float mx = -INFINITY;
                    for (int t = 0; t < parts; t++)
                        mx = fmaxf(mx, __ldcg(from + (int64_t)(2 * t + (t == 0)) * Sh::PART + Sh::ROWS * D + 2 * row));
                    float sum = 0.f;
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int t = 0; t < parts; t++) {
                        const float* p = from + (int64_t)(2 * t + (t == 0)) * Sh::PART;
                        const float2 ml = __ldcg((const float2*)(p + Sh::ROWS * D + 2 * row));
                        const float4 x = __ldcg((const float4*)(p + row * D + d));
                        const float f = weight(ml, mx);
                        if (f != 0.f) {
                            sum += ml.y * f;
                            acc.x += x.x * f, acc.y += x.y * f, acc.z += x.z * f, acc.w += x.w * f;
                        }
                    }
                    finish(row, d, mx, sum, acc);
                }
            }
        }
        team_sync();  // the tiles' slots may be filled again
    }
    copies_wait<0>();
}

// query heads of an item, in eights: 16 rows' accumulators and queries fit the registers up to D = 128
template <int D>
static int eights(int group) {
    return group <= 8 || D > 128 ? 1 : 2;
}
static int rows_of(int dim, int group) { return 8 * (group <= 8 || dim > 128 ? 1 : 2); }

template <int D, int TYPE, int STORE, int NT>
static int launch_nt(fvs_stream_t stream, const AttendArgs& a) {
    using Sh = Shape<D, STORE, NT>;
    auto kernel = attend_kernel<D, TYPE, STORE, NT>;
    if (cudaError_t e = fvs_ensure_smem((const void*)kernel, Sh::SMEM)) return (int)e;
    // no more CTAs than the page tables' room can fill
    const int64_t room = (int64_t)a.tb.wide * a.c.page;
    const int64_t units = ((room < 0x7fffffff ? room : 0x7fffffff) + UNIT - 1) / UNIT * a.tb.seqs * a.c.heads *
                          ((a.group + Sh::ROWS - 1) / Sh::ROWS);
    int64_t grid = (units + WARPS - 1) / WARPS;
    const int64_t full = (int64_t)fvs_sm_count() * Sh::CTAS;
    if (grid > full) grid = full;
    kernel<<<(unsigned)grid, THREADS, Sh::SMEM, stream>>>(a);
    return fvs_launch_status();
}
template <int D, int TYPE, int STORE>
static int launch(fvs_stream_t stream, const AttendArgs& a) {
    if (eights<D>(a.group) == 1) return launch_nt<D, TYPE, STORE, 1>(stream, a);
    return launch_nt<D, TYPE, STORE, D <= 128 ? 2 : 1>(stream, a);
}
template <int D>
static int launch_types(fvs_stream_t stream, const AttendArgs& a, int type) {
    if (type == FVS_F16)
        return a.c.type == FVS_I8 ? launch<D, FVS_F16, FVS_I8>(stream, a) : launch<D, FVS_F16, FVS_F16>(stream, a);
    return a.c.type == FVS_I8 ? launch<D, FVS_BF16, FVS_I8>(stream, a) : launch<D, FVS_BF16, FVS_BF16>(stream, a);
}

}  // namespace kv
}  // namespace fvs

using namespace fvs::kv;

// two partial results for each of up to 3 CTAs on every SM
extern "C" int fvs_kv_attend_work(int dim) {
    if (dim < 1) return FVS_EINVAL;
    if (dim > 256) return FVS_ERANGE;
    return 2 * 3 * fvs_sm_count() * 16 * (dim + 2) * 4;
}

extern "C" int fvs_kv_attend(fvs_stream_t stream, const fvs_kv_cache* cache, int type, const void* q, int64_t q_seq,
                             int64_t q_head, int hq, const int32_t* table, int seqs, int wide, int64_t table_stride,
                             const int32_t* lens, float scale, void* out, float* lse, void* work,
                             int32_t* arrived) {
    if (int rc = check_cache(cache)) return rc;
    FVS_CHECK_ARG(type == FVS_F16 || type == FVS_BF16);
    FVS_CHECK_ARG(cache->type == FVS_I8 || cache->type == type);
    FVS_CHECK_ARG(seqs >= 0 && hq >= 1 && hq % cache->heads == 0);
    if (seqs == 0) return FVS_OK;
    if (int rc = check_table(table, seqs, wide, table_stride)) return rc;
    FVS_CHECK_ARG(q && ((uintptr_t)q & 15) == 0 && q_seq % 8 == 0 && q_head % 8 == 0 && q_seq >= 0 && q_head >= 0);
    FVS_CHECK_ARG(lens && out && ((uintptr_t)out & 15) == 0 && work && ((uintptr_t)work & 15) == 0 &&
                  arrived);
    if ((int64_t)seqs * hq > (1 << 28)) return FVS_ERANGE;
    AttendArgs a{*cache, {table, table_stride, seqs, wide}, q, q_seq, q_head, lens, out, lse, arrived,
                 (float*)work, hq, hq / cache->heads, scale * 1.4426950408889634f};
    switch (cache->dim) {
        case 64: return launch_types<64>(stream, a, type);
        case 96: return launch_types<96>(stream, a, type);
        case 128: return launch_types<128>(stream, a, type);
        case 192: return launch_types<192>(stream, a, type);
        default: return launch_types<256>(stream, a, type);
    }
}
