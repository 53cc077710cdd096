// Attention of one new token per sequence over a paged key-value cache (new; see include/fanar_b200.h).
//
// One pass over the keys with the running maximum m and sum l of the softmax: a tile of keys with scores s changes them to
// m' = max(m, max s), l' = l 2^(m - m') + sum 2^(s - m'), and the accumulated output by o' = o 2^(m - m') + sum
// 2^(s - m') v.  Scores are in units of log2 (scale * log2 e); m, l, o and all sums are fp32.
//
// Work.  A unit is 16 keys (32 of at most 128 bytes) of one (sequence, key head, group of up to 8 NT query heads) item.
// The items in order, each of ITEM_COST + its units, are cut into pieces of equal cost, one for each CTA of four warps, so
// that any mix of lengths keeps every SM busy and a long sequence is split without the host knowing any length.  The warps
// of a CTA take an item's units in turn and add up their results in shared memory; an item of few units is one warp's,
// taken when it is through with the one before.  A piece that holds a whole item writes its output; parts of an item go to
// the workspace, and the CTA that finishes an item's last part (counted by an atomic, joined in the order of the keys, so
// that results do not depend on the order of arrival) joins them.
//
// A warp copies its units' key and value rows with cp.async into a ring of its own (no block barrier between units; page
// numbers are looked up two units ahead of the copy) and multiplies with mma.sync m16n8k16.  Both products run
// transposed, S^T = K Q^T and O^T = V^T P^T: the 16 keys (then 16 output elements) fill the M side whatever the number of
// query heads that share a key head, and 8 heads fill N, where heads on M would leave half of a tile empty for 8 or
// fewer.  The probabilities pass from one layout to the other with movmatrix.  mma.sync and not tcgen05: each key feeds at
// most 16 query rows, so the bound is the cache's bytes (2 G / element size flops per byte), and tcgen05's 128-row
// tiles would be padded eightfold and more.
//
// The maximum moves only when a score passes it by more than SLACK, so most units need one vote instead of shuffles and a
// rescale.  Weights that become fp16 are taken 2^BELOW larger than the softmax's, near fp16's upper end: without that a key at
// 2^-25 of the largest weight vanished from the second product and not from l.
//
// Rounding: l sums the probabilities in fp32.  They enter the second product as the sum of 16-bit numbers, two fp16 ones with
// 21 bits together (fp16 caches, int8 codes) or three bf16 ones with 24, so that outputs are as near as fp32's sums bring
// them.  One fp16 number each made the error against 64 bits 1.4 times that (fp16 outputs); with two bf16 ones (16 bits) an
// output in 300 was on the neighbouring bf16 number, with three one in 3000 (64 sequences of 1 to 8192 keys).  Two fp16 parts
// take 2 to 4 % longer than one, 5 to 9 % over long int8 sequences, the third bf16 part 0.5 % (heads of 128) to 4 % (of 64).
// int8 codes are exact in fp16 (see codes2).  Their key scale multiplies the fp32 score, their value scale the probability, and
// a power of two for each head brings that product to fp16's range, by the largest product met so far (by the largest scale,
// one large row of no weight would take the others' bits).  Queries over int8 codes are brought to fp16 by a power of two for
// each head, their largest element to the upper end of its range.
//
// Measured on one B200 (6550 GB/s measured copy rate), calls back to back: 131071 bf16 keys of 8 heads of 128, 32 query
// heads, 102 to 105 us (5.2 TB/s), four such sequences 347 us (6.2 TB/s); 64 sequences of 1 to 8192 keys 65 us (4.8 TB/s);
// int8 codes, 48 sequences of 2048 to 16384 keys, 64 query heads, 141 us with two inputs in turn and 155 with more (4.2 to
// 4.6 TB/s, bound by 510 warp instructions for 16 keys of a head, copies, setup and joins included), 192 such sequences
// 530 to 570 us (4.6 to 5.0 TB/s); 2000 sequences of 1 to 200 int8 keys 38 us (per item, not per byte); one sequence of 100
// keys 10 us (waits for memory in a row).
#pragma once
#include <limits.h>

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
    int32_t* counts;   // the next piece of work, the CTAs that are done; zero between calls
    unsigned long long* arrived;  // [items] parts that are there, 16 bits for each of a CTA's warps; zero between calls
    float* parts;
    int hq, group;     // query heads, query heads of a key head
    int split;         // items of a key head
    float scale2;      // scale * log2 e
    uint32_t page_mul, page_shift;  // t / page = t * page_mul >> page_shift for t < 2^31
};

constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int ITEM_COST = 3;   // of an item beside its units (loading q, adding up, writing), in units; 3 to 10 make 2 % of difference
constexpr int SM_ROWS = 32;    // rows of partial results that an SM's CTAs may hold at a time
// How far (log2) a score may pass the running maximum before it moves, and how far below it the reference m lies.
// fp16 weights use its range: 2^(SLACK + BELOW) = 2^TOP at most, and 2^-25 / 2^BELOW = 2^-36 of the largest is the least.
// bf16 ones have fp32's range.  Weights over int8 codes are multiplied by the value scale first, and that product has a
// reference of its own with the same two distances.
template <int STORE> constexpr float SLACK = STORE == FVS_BF16 ? 8.f : 4.f;
template <int STORE> constexpr float BELOW = STORE == FVS_F16 ? 11.f : 0.f;
constexpr float TOP = 15.f;

template <int D, int STORE, int NT_>
struct Shape {
    static constexpr bool I8 = STORE == FVS_I8;
    static constexpr int NT = NT_;
    static constexpr int ROWS = 8 * NT;              // query heads of an item
    static constexpr int RB = D * (I8 ? 1 : 2);      // bytes of a row
    static constexpr int TILES = RB <= 128 ? 2 : 1;  // of 16 keys in a unit: one lookup, vote and loop turn for 4 KB of keys
    static constexpr int UNIT = 16 * TILES;
    // Rows in shared memory, so that no access below has bank conflicts.  Rows of 128 bytes: their 16-byte chunks permuted
    // by the row; others: padded, 16-bit rows (read by ldmatrix) to an odd number of chunks, int8 keys (8 bytes a lane from
    // 4 rows at a time) to 32 or 96 mod 128 bytes, int8 values (4 bytes a lane from every second row) to half of that.
    static constexpr bool SWZ = RB == 128;
    static constexpr int KS = SWZ ? RB : I8 ? (D == 96 ? 160 : D + 32) : RB + 16;
    static constexpr int VS = SWZ ? RB : RB + 16;
    static __device__ __forceinline__ int k_chunk(int row, int ch) { return !SWZ ? ch : I8 ? ch ^ (2 * (row & 3)) : ch ^ (row & 7); }
    static __device__ __forceinline__ int v_chunk(int row, int ch) { return !SWZ ? ch : I8 ? ch ^ (row & 6) : ch ^ (row & 7); }
    static constexpr int VALUES = UNIT * KS;                  // byte offset of the value rows
    static constexpr int SCALES = VALUES + UNIT * VS;         // of the scales [2][UNIT]
    static constexpr int MASK = SCALES + (I8 ? 8 * UNIT : 0);  // of the word of visible keys
    static constexpr int STAGE = MASK + 16;
    static constexpr int OS = D + 4;                 // row stride (floats) of a staged output tile
    static_assert(ROWS * OS * 4 <= STAGE, "an output tile fits a ring slot");
    static constexpr bool Q_SMEM = D > 128 && NT > 1;         // q's fragments would not fit the registers
    static_assert(!(I8 && Q_SMEM), "not built: see launch");
    static constexpr int QBYTES = Q_SMEM ? ROWS * D * 2 : 0;
    // CTAs per SM: three (12 warps hide each other's latencies; 168 registers a thread) where two stages fit: 64 ragged bf16
    // sequences of 8 heads of 128 take 66 us against 73 with two CTAs of three stages, 48 long int8 ones 141 against 155.  Heads
    // of 64 spill at 168 registers: two CTAs take 43 us there against 46 (131071 keys 62 and 63; 2000 short int8 sequences 31
    // and 35, 48 long ones 115 and 116).  16-bit heads of 96 spill as well, and gain on some calls (ragged 62 us against 66 with
    // two CTAs) what they lose on others (131071 keys 90 and 87).
    static constexpr int CTAS = NT == 1 && (D == 128 || (D == 96 && !I8)) ? 3 : RB <= 256 && !Q_SMEM ? 2 : 1;
    static constexpr int BUDGET = (227 * 1024) / CTAS - 1024 - 2560 - QBYTES;
    static constexpr int FIT = BUDGET / (WARPS * STAGE);
    static constexpr int S = FIT > 4 ? 4 : FIT;      // ring stages
    static_assert(S >= 2 && CTAS * ROWS <= SM_ROWS, "ring, workspace");
    static constexpr int TAKEN = 8;  // more items than a warp has on the way: units in the ring, lookups, one in reserve
    static_assert(S + 4 <= TAKEN, "taken");
    static constexpr int RING = S * STAGE;           // bytes per warp
    static constexpr int SMEM = WARPS * RING + QBYTES;
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
__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^x of a whole number, exactly; 0 below fp32's normal range
__device__ __forceinline__ float power2(float x) { return __uint_as_float((uint32_t)(127 + max(-127, min(127, (int)x))) << 23); }
// weight of a part with maximum and sum `ml` in a join whose maximum is mx (a part of not-a-numbers alone keeps them)
__device__ __forceinline__ float weight(float2 ml, float mx) {
    return ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2_fast(ml.x - mx);
}
// A weight as the sum of 16-bit numbers, two fp16 or three bf16 ones: its upper bits, those below them (`last` if these are the
// end, which is rounded), and so on.  Beside values that may be infinite (POS) each part stays above zero, so that an infinite
// value times it is no not-a-number.
template <int TYPE>
constexpr int PARTS = TYPE == FVS_F16 ? 2 : 3;
template <int TYPE, bool POS, bool LAST>
__device__ __forceinline__ uint32_t part2(float& a, float& b) {
    constexpr float LEAST = TYPE == FVS_F16 ? 0x1p-24f : 1.2e-38f;  // the smallest number, the smallest normal one
    constexpr uint32_t UPPER = TYPE == FVS_F16 ? 0xffffe000u : 0xffff0000u;
    if (LAST) return Elem<TYPE>::down(POS ? fmaxf(a, LEAST) : a, POS ? fmaxf(b, LEAST) : b);
    const float ua = __uint_as_float(__float_as_uint(a) & UPPER), ub = __uint_as_float(__float_as_uint(b) & UPPER);
    const uint32_t r = TYPE == FVS_F16 ? Elem<TYPE>::down(ua, ub) : __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    a -= ua, b -= ub;
    if (POS) a = fmaxf(a, LEAST), b = fmaxf(b, LEAST);
    return r;
}
// Two codes as fp16: the byte u = code + 128 under 0x64 is 1024 + u, and 1152 less is the code, exactly.  (Leaving the 128 in
// the products and taking it out of their sums spares the subtraction, but the sums then round at 128 sum |q|: a row with
// one large element, or one stored with an infinity, is not what the codes say.)
__device__ __forceinline__ uint32_t codes2(uint32_t u, uint32_t sel) {
    const uint32_t x = __byte_perm(u, 0x64646464u, sel), off = 0x64806480u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&off));
    return *reinterpret_cast<const uint32_t*>(&r);
}
constexpr uint32_t LOW = 0x4140, HIGH = 0x4342;  // the lower and the upper two codes of a word

__device__ __forceinline__ int seq_len(const AttendArgs& a, int b) {
    const int len = __ldg(a.lens + b);
    const int64_t room = (int64_t)a.tb.wide * a.c.page;
    return len > room ? (int)room : max(len, 0);
}
template <int UNIT>
__device__ __forceinline__ int units_of(int len) {
    return (int)(((unsigned)len + UNIT - 1) / UNIT);
}

// A place in the order of all items: unit u of part `sub` (of `split`) of the query heads of key head `head` of sequence b.
struct Place {
    int b, head, sub, u;
    __device__ __forceinline__ bool same_item(int ob, int oh, int os) const { return b == ob && head == oh && sub == os; }
};

// An item, with the units [u, end) of it that lie in a piece.
struct Item {
    int b, head, sub, len, n, u, end;
};
// the next item of the piece that ends at `stop`; false if there is none
template <int UNIT>
__device__ __forceinline__ bool next_item(const AttendArgs& a, Item& it, const Place& stop) {
    if (it.end < it.n || stop.same_item(it.b, it.head, it.sub)) return false;  // the piece ends in this one
    if (++it.sub == a.split) {
        it.sub = 0;
        if (++it.head == a.c.heads) {
            it.head = 0;
            do {
                if (++it.b > stop.b || it.b >= a.tb.seqs) return false;
                it.len = seq_len(a, it.b);
                it.n = units_of<UNIT>(it.len);
            } while (it.n == 0);
        }
    }
    it.u = 0;
    it.end = stop.same_item(it.b, it.head, it.sub) ? stop.u : it.n;
    return it.end > 0;
}

// One key of a unit on its way from the page table to the copy.
struct Lookup {
    int entry;  // page, < 0: none, NO_UNIT: the piece has no such unit
    int slot, head, fill;
};
constexpr int NO_UNIT = INT_MIN;

// Cuts of the cost of all items: equal shares, one for each CTA, each share cut into `runs` pieces, the first of them
// long.  A CTA begins with its share's long piece; the short ones are taken as CTAs finish, since SMs differ in how fast
// memory serves them and the warps of an SM in how often they issue (148 SMs, int8, 192 requests of 2048 to 16384 keys: 594
// -> 570 us; 4 of 131071 bf16 keys 357 -> 342).  Below 512 units a share one piece each has the same time (48 such int8
// requests: 141 us both ways) and less to join.
struct Cuts {
    int64_t share, lead;  // of the cost: a share, its first piece
    int runs, small;      // pieces of a share, the cost of each but the first (the last one may be shorter)
    // pieces are numbered in the order of the cost
    __device__ __forceinline__ int64_t at(int64_t piece) const {
        const int64_t s = piece / runs;
        const int k = (int)(piece - s * runs);
        return s * share + (k ? min(share, lead + (int64_t)(k - 1) * small) : 0);
    }
    // number of the last cut at or before g
    __device__ __forceinline__ int upto(int64_t g) const {
        const int64_t s = g / share, in = g - s * share;
        return (int)(s * runs + (in < lead ? 0 : min((int64_t)runs - 1, 1 + (in - lead) / small)));
    }
    // number of the first cut at or after g
    __device__ __forceinline__ int from(int64_t g) const { return upto(g - 1) + 1; }
    // the n-th of the pieces that are taken as CTAs finish
    __device__ __forceinline__ int64_t taken(int n) const { return (int64_t)(n / (runs - 1)) * runs + 1 + n % (runs - 1); }
};

__device__ __forceinline__ float log_sum(float mx, float sum) {
    return sum == 0.f ? -INFINITY : (mx + log2f(sum)) * 0.6931471805599453f;
}
// An item of which a piece holds a part.
struct CutItem {
    int b, head, sub, t_lo, parts;
};
// Joins an item's parts: rows warp, warp + 4, ... (R of them at most) of `rows`.  Lane t holds the weights of parts t and t +
// 32, then four elements of the sums.  Loads that wait for the memory of a busy GPU cost 2000 cycles and more each time, so
// all weights are one wait and WAYS rows of parts another.
template <int D, int TYPE, int ROWS, int R, int WAYS>
__device__ __forceinline__ void join_parts(const float* from, int parts, int warp, int rows, uint16_t* out, float* lse) {
    const int lane = threadIdx.x & 31;
    constexpr int Q4 = D / 4, PART = ROWS * (D + 2), Q = (Q4 + 31) / 32, WK = 2, BATCH = WAYS / Q / R > 0 ? WAYS / Q / R : 1;
    auto part_at = [&](int t) { return from + (2 * t + (t == 0)) * PART; };
    float mx[R], sum[R];
    float4 acc[R][Q];
#pragma unroll
    for (int w = 0; w < R; w++) {
        mx[w] = -INFINITY, sum[w] = 0.f;
#pragma unroll
        for (int i = 0; i < Q; i++) acc[w][i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    auto row_of = [&](int w) { return min(warp + w * WARPS, rows - 1); };
    for (int t0 = 0; t0 < parts; t0 += 32 * WK) {
        float2 ml[R][WK];
#pragma unroll
        for (int w = 0; w < R; w++)
#pragma unroll
            for (int k = 0; k < WK; k++) {
                const int t = t0 + 32 * k + lane;
                ml[w][k] = t < parts ? __ldcg((const float2*)(part_at(t) + ROWS * D + 2 * row_of(w))) : make_float2(-INFINITY, 0.f);
            }
#pragma unroll
        for (int w = 0; w < R; w++) {
            float top = mx[w];
#pragma unroll
            for (int k = 0; k < WK; k++) top = fmaxf(top, ml[w][k].x);
#pragma unroll
            for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float f = weight(make_float2(mx[w], sum[w]), top);  // of what the parts before added up to
            mx[w] = top;
            if (f != 1.f) {
                sum[w] *= f;
#pragma unroll
                for (int i = 0; i < Q; i++) acc[w][i].x *= f, acc[w][i].y *= f, acc[w][i].z *= f, acc[w][i].w *= f;
            }
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < WK; k++) {
                const float f1 = weight(ml[w][k], top);
                s += ml[w][k].y * f1;
                ml[w][k].x = f1;
            }
#pragma unroll
            for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            sum[w] += s;
        }
#pragma unroll
        for (int k = 0; k < WK; k++) {
            const int n = min(32, parts - t0 - 32 * k);
            for (int j0 = 0; j0 < n; j0 += BATCH) {
                float4 x[BATCH][R][Q];
#pragma unroll
                for (int j = 0; j < BATCH; j++) {
                    const float* p = part_at(t0 + 32 * k + min(j0 + j, n - 1));
#pragma unroll
                    for (int w = 0; w < R; w++)
#pragma unroll
                        for (int i = 0; i < Q; i++)
                            if (i * 32 + lane < Q4) x[j][w][i] = __ldcg((const float4*)(p + row_of(w) * D) + i * 32 + lane);
                }
#pragma unroll
                for (int j = 0; j < BATCH; j++)
#pragma unroll
                    for (int w = 0; w < R; w++) {
                        const float f = __shfl_sync(0xffffffffu, ml[w][k].x, min(j0 + j, 31));
                        if (j0 + j < n && f != 0.f)
#pragma unroll
                            for (int i = 0; i < Q; i++) {
                                acc[w][i].x += x[j][w][i].x * f, acc[w][i].y += x[j][w][i].y * f;
                                acc[w][i].z += x[j][w][i].z * f, acc[w][i].w += x[j][w][i].w * f;
                            }
                    }
            }
        }
    }
#pragma unroll
    for (int w = 0; w < R; w++) {
        const int row = warp + w * WARPS;
        if (row >= rows) break;
        const float inv = sum[w] == 0.f ? 0.f : 1.f / sum[w];
#pragma unroll
        for (int i = 0; i < Q; i++)
            if (i * 32 + lane < Q4)
                *((uint2*)(out + row * D) + i * 32 + lane) = make_uint2(Elem<TYPE>::down(acc[w][i].x * inv, acc[w][i].y * inv),
                                                                        Elem<TYPE>::down(acc[w][i].z * inv, acc[w][i].w * inv));
        if (lse && lane == 0) lse[row] = log_sum(mx[w], sum[w]);
    }
}

template <int D, int TYPE, int STORE, int NT>
__global__ void __launch_bounds__(THREADS, Shape<D, STORE, NT>::CTAS) attend_kernel(AttendArgs a) {
    using Sh = Shape<D, STORE, NT>;
    constexpr bool I8 = Sh::I8;
    constexpr int MT = I8 ? FVS_F16 : TYPE;  // type of the matrix instructions' operands
    constexpr int S = Sh::S, UNIT = Sh::UNIT, TILES = Sh::TILES, TAKEN = Sh::TAKEN;
    extern __shared__ __align__(128) uint8_t ring_all[];
    __shared__ int64_t s_sum[WARPS];
    __shared__ int s_none[WARPS];
    __shared__ int64_t s_before[THREADS];  // cost (for one item of each sequence) before each thread's sequences
    __shared__ Place s_place[2];           // where a piece begins and ends
    __shared__ int64_t s_base;             // cost before the first sequence of the piece
    __shared__ float s_ml[WARPS][Sh::ROWS][2];
    __shared__ int s_tile[WARPS], s_next;
    __shared__ int s_short, s_taken[WARPS][TAKEN];
    __shared__ CutItem s_cut[2];
    __shared__ Cuts s_cuts;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = lane >> 2, c4 = lane & 3;
    const int split = a.split;
    const int per_seq = a.c.heads * split;
    const int B = a.tb.seqs;

    // ---- cost of all sequences (each thread a run of them)
    const int chunk = (B + THREADS - 1) / THREADS;
    const int b_hi = min(B, (tid + 1) * chunk);
    int64_t mine = 0;
    int none = 0;
    for (int b0 = tid * chunk; b0 < b_hi; b0 += 16) {
        unsigned sum = 0;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            if (b0 + j < b_hi) {
                const int n = units_of<UNIT>(seq_len(a, b0 + j));
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
    // ---- the pieces.  Unit u of an item that begins at cost x lies at x + ITEM_COST + u.  A cut nearer than `near` units
    // to an item's begin or end moves there: joining two parts costs more than that
    Cuts cuts;
    // a share holds 16 units or, if these are smaller, an item
    const int64_t items = (int64_t)(B - none) * per_seq;
    cuts.share = max(max((int64_t)1, min((int64_t)16, items ? total / items : 1)), (total + gridDim.x - 1) / gridDim.x);
    const bool shared = cuts.share >= 512;  // setting up another piece and joining its part costs more than it evens out below
    if (shared) {
        cuts.small = (int)((cuts.share + 7) / 8);
        cuts.lead = cuts.share - 2 * cuts.small;
        cuts.runs = 3;
    } else {
        cuts.small = (int)cuts.share;
        cuts.lead = cuts.share;
        cuts.runs = 1;
    }
    if (tid == 0) s_cuts = cuts;
    const int near = max(8, cuts.small / 8);
    // items of up to so many units are one warp's; fewer than 2 near, so that none of them is cut
    const int alone = Sh::Q_SMEM ? 0 : (int)min((int64_t)15, cuts.share / 4);
    uint8_t* ring = ring_all + warp * Sh::RING;
    const uint32_t ring_at = smem_addr(ring);
    const bool aligned = a.c.page % 16 == 0;  // a tile's keys lie in one page
    auto page_of = [&](int t) { return (int)(((uint64_t)(unsigned)t * a.page_mul) >> a.page_shift); };

    int64_t piece = (int64_t)blockIdx.x * cuts.runs;
#pragma unroll 1
    for (;; piece = s_cuts.taken(s_next)) {
    __syncthreads();
    if (s_cuts.at(piece) >= total) break;
    if (tid == THREADS - 1 && shared) s_next = atomicAdd(a.counts, 1);
    if (tid == 0) s_short = 0;
    if (warp < 2) {
        const int64_t g = s_cuts.at(piece + warp);
        if (g >= total) {
            if (lane == 0) s_place[warp] = Place{B, 0, 0, 0};
        } else {
            int at = 0;  // the last run of sequences that begins at or before g
#pragma unroll
            for (int j = 0; j < THREADS / 32; j++) at += s_before[j * 32 + lane] * per_seq <= g;
            at = (int)__reduce_add_sync(0xffffffffu, (unsigned)at) - 1;
            int64_t base = s_before[at];
            for (int b0 = at * chunk; b0 < B; b0 += 32) {
                const int n = b0 + lane < B ? units_of<UNIT>(seq_len(a, b0 + lane)) : 0;
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
                        int hh = (int)(in / cost), u = (int)(in - hh * cost) - ITEM_COST;
                        if (u < near)
                            u = 0;
                        else if (n - u < near)
                            hh++, u = 0;  // heads: past the sequence's last item
                        s_place[warp] = Place{b0 + lane, hh / split, hh % split, u};
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
    now.head = s_place[0].head;
    now.sub = s_place[0].sub;
    now.u = s_place[0].u;
    now.len = seq_len(a, now.b);
    now.n = units_of<UNIT>(now.len);
    int64_t base = s_base;
    bool more;
    if (now.head == a.c.heads) {  // moved past the sequence's last item
        const int cost = now.n + ITEM_COST;
        now.head--;
        now.sub = split - 1;
        now.end = now.n;
        more = next_item<UNIT>(a, now, stop);
        base += cost;
    } else {
        now.end = stop.same_item(now.b, now.head, now.sub) ? stop.u : now.n;
        more = now.u < now.end;
    }
    // the units that this warp copies: every fourth of an item, all of one that it has alone
    Item ahead = now;
    bool any = more;
    // The piece's short items are numbered as they come.  A warp takes the next number when it is through with the one it
    // had, so that the warps come out even, and remembers it for the computation that follows.
    int next = 0, number_ahead = 0, taken = 0;
    bool own = false;
    auto settle = [&]() {
        while (any && ahead.u >= ahead.end) {
            any = next_item<UNIT>(a, ahead, stop);
            if (own) {
                own = false;
                if (lane == 0) s_taken[warp][taken % TAKEN] = number_ahead = atomicAdd(&s_short, 1);
                number_ahead = __shfl_sync(0xffffffffu, number_ahead, 0);
                taken++;
            }
            if (any && ahead.n <= alone) {
                own = next++ == number_ahead;
                ahead.u = own ? 0 : ahead.end;
            } else {
                ahead.u += warp;
            }
        }
    };
    if (lane == 0) s_taken[warp][0] = number_ahead = atomicAdd(&s_short, 1);
    number_ahead = __shfl_sync(0xffffffffu, number_ahead, 0);
    taken = 1;
    own = any && ahead.n <= alone && next++ == number_ahead;
    if (any && ahead.n <= alone)
        ahead.u = own ? 0 : ahead.end;
    else
        ahead.u += warp;
    settle();

    // ---- copies, two lookups ahead
    auto look = [&]() {
        Lookup k;
        k.entry = NO_UNIT;
        k.slot = k.head = 0;
        if (any) {
            const int t = ahead.u * UNIT + (lane & (UNIT - 1));
            const int from = aligned ? t & ~15 : t;
            k.entry = -1;
            k.slot = INT_MAX;  // not one of the sequence's keys
            if (from < ahead.len) {
                const int p = page_of(from);
                if (t < ahead.len) k.slot = t - p * a.c.page;
                k.entry = max(-1, __ldg(a.tb.at + (int64_t)ahead.b * a.tb.stride + p));
            }
            k.head = ahead.head;
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
        k.fill = a.c.fill && k.entry >= 0 ? __ldg(a.c.fill + k.entry) : INT_MAX;
    };
    auto issue = [&](const Lookup& k, int slot) {
        const bool live = k.entry >= 0 && k.slot < k.fill;
        const uint32_t mask = __ballot_sync(0xffffffffu, live) & (UNIT == 32 ? 0xffffffffu : 0xffffu);
        const uint32_t st = ring_at + slot * Sh::STAGE;
        constexpr int PER = Sh::RB / 16;  // chunks of a row
        constexpr int ESZ = I8 ? 1 : 2;
        if (aligned) {
            // a tile's rows are one slot apart: each lane copies its chunk of every RPI-th row
            constexpr int RPI = PER > 16 ? 1 : PER > 8 ? 2 : PER > 4 ? 4 : 8;
            const int row = lane / PER, ch = lane % PER;
#pragma unroll
            for (int j = 0; j < TILES; j++) {
                const uint32_t m = (mask >> (16 * j)) & 0xffffu;
                const int slot0 = __shfl_sync(0xffffffffu, k.slot, 16 * j), entry = __shfl_sync(0xffffffffu, k.entry, 16 * j);
                if (m && row < RPI) {
                    const int64_t off = ((int64_t)entry * a.c.page_stride + (int64_t)k.head * a.c.head_stride +
                                         (int64_t)(slot0 + row) * a.c.slot_stride) * ESZ + ch * 16;
                    const uint8_t *pk = (const uint8_t*)a.c.k + off, *pv = (const uint8_t*)a.c.v + off;
                    const int64_t step = a.c.slot_stride * (RPI * ESZ);
                    // full tiles of dense rows have fixed distances: no address arithmetic.  The rest is a loop, for the
                    // instruction cache's sake (unrolled, large int8 calls take 140 and 577 us, as a loop 141 and 570)
                    if (a.c.slot_stride == D && m == 0xffffu) {
#pragma unroll
                        for (int i = 0; i < 16 / RPI; i++) {
                            const int key = 16 * j + i * RPI + row;
                            copy16(st + key * Sh::KS + Sh::k_chunk(key, ch) * 16, pk + i * RPI * Sh::RB, true);
                            copy16(st + Sh::VALUES + key * Sh::VS + Sh::v_chunk(key, ch) * 16, pv + i * RPI * Sh::RB, true);
                        }
                    } else {
#pragma unroll 1
                        for (int i = 0; i < 16 / RPI; i++) {
                            const int key = 16 * j + i * RPI + row;
                            const bool on = (m >> (i * RPI + row)) & 1;
                            copy16(st + key * Sh::KS + Sh::k_chunk(key, ch) * 16, on ? pk + i * step : (const uint8_t*)a.c.k, on);
                            copy16(st + Sh::VALUES + key * Sh::VS + Sh::v_chunk(key, ch) * 16, on ? pv + i * step : (const uint8_t*)a.c.v, on);
                        }
                    }
                }
            }
        } else {
            const int64_t at0 = live ? (int64_t)k.entry * a.c.page_stride + (int64_t)k.head * a.c.head_stride +
                                           (int64_t)k.slot * a.c.slot_stride
                                     : 0;
#pragma unroll (D > 128 ? 2 : UNIT * PER / 32)
            for (int i = 0; i < UNIT * PER / 32; i++) {
                const int at = i * 32 + lane, key = at / PER, ch = at % PER;
                const int64_t off = __shfl_sync(0xffffffffu, at0, key) * ESZ + ch * 16;
                const bool on = (mask >> key) & 1;
                copy16(st + key * Sh::KS + Sh::k_chunk(key, ch) * 16, (const uint8_t*)a.c.k + off, on);
                copy16(st + Sh::VALUES + key * Sh::VS + Sh::v_chunk(key, ch) * 16, (const uint8_t*)a.c.v + off, on);
            }
        }
        if (I8) {
            const int64_t at = live ? (int64_t)k.entry * a.c.scale_page_stride + (int64_t)k.head * a.c.scale_head_stride +
                                          (int64_t)k.slot * a.c.scale_slot_stride
                                    : 0;
            if (UNIT == 32) {
                copy4(st + Sh::SCALES + lane * 4, a.c.k_scale + at, live);
                copy4(st + Sh::SCALES + 128 + lane * 4, a.c.v_scale + at, live);
            } else {
                copy4(st + Sh::SCALES + lane * 4, (lane < 16 ? a.c.k_scale : a.c.v_scale) + at, live);
            }
        }
        if (lane == 0) *(uint32_t*)(ring + slot * Sh::STAGE + Sh::MASK) = mask;
    };
    Lookup la, lb;
    int ready = S - 1;  // the slot to be filled next
    {
        // the first lookups side by side, so that their latencies overlap
        Lookup l0[S + 1];
#pragma unroll
        for (int i = 0; i <= S; i++) l0[i] = look();
#pragma unroll
        for (int i = 0; i < S; i++) look_fill(l0[i]);
#pragma unroll
        for (int i = 0; i < S - 1; i++) {
            if (l0[i].entry != NO_UNIT) issue(l0[i], i);
            copies_commit();
        }
        la = l0[S - 1];
        lb = l0[S];
    }
    auto feed = [&]() {
        if (la.entry != NO_UNIT) issue(la, ready);
        copies_commit();
        ready = ready + 1 == S ? 0 : ready + 1;
        la = lb;
        look_fill(la);
        lb = look();
    };

    // ---- the piece's items
    int slot = 0, cut = 0, number = 0, done = 0;
    __syncwarp();
#pragma unroll 1
    for (; more;) {
        const bool solo = now.n <= alone;
        const int h0 = now.head * a.group + now.sub * Sh::ROWS;
        const int rows = min(Sh::ROWS, a.group - now.sub * Sh::ROWS);
        const Item it = now;
        const int64_t it_begin = base * per_seq + (int64_t)(now.head * split + now.sub) * (now.n + ITEM_COST);
        more = next_item<UNIT>(a, now, stop);
        if (now.b != it.b) base += it.n + ITEM_COST;
        if (solo) {
            if (number++ != s_taken[warp][done % TAKEN]) continue;
            done++;
        }

        // q as the B operand: head r of each 8, elements of the order in which the keys' rows come
        uint32_t qf[Sh::Q_SMEM ? 1 : NT][Sh::Q_SMEM ? 1 : D / 16][2];
        uint2* q_all = (uint2*)(ring_all + Sh::SMEM - Sh::QBYTES);
        float mul[NT][2];   // what a raw product is multiplied with, for heads 2 c4 and 2 c4 + 1
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int h = t * 8 + r;
            const uint16_t* qp = (const uint16_t*)a.q + it.b * a.q_seq + (int64_t)(h0 + h) * a.q_head;
            if constexpr (I8) {
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
                // the largest element (2^(e - 127) at least) to 2^14: one 2^-39 of it still has a bit in fp16
                const int e = max(15, min(254, (int)(__float_as_uint(top) >> 23)));
                const float down = __uint_as_float((uint32_t)(268 - e) << 23);
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    const float2 x = Elem<TYPE>::up(raw[k].x), y = Elem<TYPE>::up(raw[k].y);
                    const uint32_t f0 = Elem<FVS_F16>::down(x.x * down, x.y * down), f1 = Elem<FVS_F16>::down(y.x * down, y.y * down);
                    qf[t][k][0] = f0;
                    qf[t][k][1] = f1;
                }
                const float up = a.scale2 * __uint_as_float((uint32_t)(e - 14) << 23);
#pragma unroll
                for (int x = 0; x < 2; x++) mul[t][x] = __shfl_sync(0xffffffffu, up, c4 * 8 + 4 * x);
            } else {
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    if (Sh::Q_SMEM && k % WARPS != warp) continue;
                    const uint32_t f0 = h < rows ? __ldg((const uint32_t*)(qp + k * 16 + c4 * 2)) : 0u;
                    const uint32_t f1 = h < rows ? __ldg((const uint32_t*)(qp + k * 16 + c4 * 2 + 8)) : 0u;
                    if (Sh::Q_SMEM) {
                        q_all[(t * (D / 16) + k) * 32 + lane] = make_uint2(f0, f1);
                    } else {
                        qf[Sh::Q_SMEM ? 0 : t][Sh::Q_SMEM ? 0 : k][0] = f0;
                        qf[Sh::Q_SMEM ? 0 : t][Sh::Q_SMEM ? 0 : k][1] = f1;
                    }
                }
                mul[t][0] = mul[t][1] = a.scale2;
            }
        }
        if (Sh::Q_SMEM) __syncthreads();
        auto q_frag = [&](int t, int k) {
            if (Sh::Q_SMEM) return q_all[(t * (D / 16) + k) * 32 + lane];
            return make_uint2(qf[Sh::Q_SMEM ? 0 : t][Sh::Q_SMEM ? 0 : k][0], qf[Sh::Q_SMEM ? 0 : t][Sh::Q_SMEM ? 0 : k][1]);
        };
        float m[NT][2], l[NT][2], o[D / 16][NT][4];
        // int8: m is a whole number, the product of a weight and its value scale is at most 2^lim (in log2 units like m, a
        // whole number too) and enters the matrix instructions times down = 2^(m + TOP - lim)
        float lim[NT][2], down[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            m[t][0] = m[t][1] = lim[t][0] = lim[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.f;
            down[t][0] = down[t][1] = 1.f;
        }
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
            // S^T = K Q^T, each tile in two chains
            float s[TILES][NT][4];
#pragma unroll
            for (int j = 0; j < TILES; j++) {
                float s2[NT][4];
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int x = 0; x < 4; x++) s[j][t][x] = s2[t][x] = 0.f;
                if (I8) {
#pragma unroll
                    for (int k = 0; k < D / 32; k++) {
                        const int at = (16 * j + r) * Sh::KS + Sh::k_chunk(r, 2 * k) * 16 + c4 * 8;
                        uint2 lo = *(const uint2*)(stp + at), hi = *(const uint2*)(stp + at + 8 * Sh::KS);
                        lo.x ^= 0x80808080u, lo.y ^= 0x80808080u, hi.x ^= 0x80808080u, hi.y ^= 0x80808080u;
                        const uint32_t f0[4] = {codes2(lo.x, LOW), codes2(hi.x, LOW), codes2(lo.x, HIGH), codes2(hi.x, HIGH)};
                        const uint32_t f1[4] = {codes2(lo.y, LOW), codes2(hi.y, LOW), codes2(lo.y, HIGH), codes2(hi.y, HIGH)};
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            const uint2 q0 = q_frag(t, 2 * k), q1 = q_frag(t, 2 * k + 1);
                            mma<MT>(s[j][t], f0, q0.x, q0.y);
                            mma<MT>(s2[t], f1, q1.x, q1.y);
                        }
                    }
                } else {
                    const uint32_t at = st + (16 * j + (lane & 15)) * Sh::KS;
#pragma unroll
                    for (int k = 0; k < D / 16; k += 2) {
                        uint32_t f0[4], f1[4];
                        ldm4(f0, at + Sh::k_chunk(lane, 2 * k + (lane >> 4)) * 16);
                        ldm4(f1, at + Sh::k_chunk(lane, 2 * k + 2 + (lane >> 4)) * 16);
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            const uint2 q0 = q_frag(t, k), q1 = q_frag(t, k + 1);
                            mma<MT>(s[j][t], f0, q0.x, q0.y);
                            mma<MT>(s2[t], f1, q1.x, q1.y);
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int x = 0; x < 4; x++) s[j][t][x] = (s[j][t][x] + s2[t][x]) * mul[t][x & 1];
            }
            float vs[TILES][2], lv[TILES][2];  // int8: value scales, their log2
            bool moved = false;
#pragma unroll
            for (int j = 0; j < TILES; j++) {
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const int key = 16 * j + 8 * x + r;
                    const float* sc = (const float*)(stp + Sh::SCALES);
                    const float ks = I8 ? sc[key] : 1.f;
                    vs[j][x] = I8 ? sc[UNIT + key] : 1.f;
                    lv[j][x] = I8 ? log2_fast(fabsf(vs[j][x])) : 0.f;
                    const bool on = (mask >> key) & 1;
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            float& y = s[j][t][2 * x + h];
                            y = on ? (I8 ? y * ks : y) : -INFINITY;
                            moved |= y > m[t][h] + (SLACK<STORE> + BELOW<STORE>);
                            if (I8) moved |= y + lv[j][x] > lim[t][h];
                        }
                }
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int t = 0; t < NT; t++) {
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        float y = m[t][x];
#pragma unroll
                        for (int j = 0; j < TILES; j++) y = fmaxf(y, fmaxf(s[j][t][x], s[j][t][x + 2]) - BELOW<STORE>);
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, d));
                        float f;
                        if (I8) {
                            float g = -INFINITY;
#pragma unroll
                            for (int j = 0; j < TILES; j++) g = fmaxf(g, fmaxf(s[j][t][x] + lv[j][0], s[j][t][x + 2] + lv[j][1]));
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, d));
                            y = ceilf(y);
                            g = fmaxf(fmaxf(lim[t][x], ceilf(g) + SLACK<STORE>), y + (TOP - 126.f));  // down <= 2^126
                            l[t][x] *= power2(m[t][x] - y);
                            f = power2(lim[t][x] - g);
                            lim[t][x] = g;
                            down[t][x] = power2(y + TOP - g);
                        } else {
                            f = y == -INFINITY ? 1.f : exp2_fast(m[t][x] - y);
                            l[t][x] *= f;
                        }
                        m[t][x] = y;
#pragma unroll
                        for (int i = 0; i < D / 16; i++) o[i][t][x] *= f, o[i][t][x + 2] *= f;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < TILES; j++) {
                if (TILES > 1 && ((mask >> (16 * j)) & 0xffffu) == 0) continue;  // its rows were not copied
                // p, and p's parts as the B operands of the second product
                uint32_t pf[PARTS<MT>][NT][2];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const float z0 = m[t][0] == -INFINITY ? 0.f : m[t][0], z1 = m[t][1] == -INFINITY ? 0.f : m[t][1];
                    float p0 = exp2_fast(s[j][t][0] - z0), p1 = exp2_fast(s[j][t][1] - z1);
                    float p2 = exp2_fast(s[j][t][2] - z0), p3 = exp2_fast(s[j][t][3] - z1);
                    l[t][0] += p0 + p2;
                    l[t][1] += p1 + p3;
                    if (I8) {  // in this order: the scale times down could be infinite
                        p0 = p0 * vs[j][0] * down[t][0], p1 = p1 * vs[j][0] * down[t][1];
                        p2 = p2 * vs[j][1] * down[t][0], p3 = p3 * vs[j][1] * down[t][1];
                    }
#pragma unroll
                    for (int n = 0; n + 1 < PARTS<MT>; n++) {
                        pf[n][t][0] = transpose8x8(part2<MT, !I8, false>(p0, p1));
                        pf[n][t][1] = transpose8x8(part2<MT, !I8, false>(p2, p3));
                    }
                    pf[PARTS<MT> - 1][t][0] = transpose8x8(part2<MT, false, true>(p0, p1));
                    pf[PARTS<MT> - 1][t][1] = transpose8x8(part2<MT, false, true>(p2, p3));
                }
                // O^T += V^T P^T
                if (I8) {
#pragma unroll
                    for (int k = 0; k < D / 32; k++) {
                        // rows 2 c4, 2 c4 + 1 and 8 further: their chunks are permuted alike
                        const uint8_t* v = stp + Sh::VALUES + (16 * j + 2 * c4) * Sh::VS + Sh::v_chunk(2 * c4, 2 * k) * 16 + r * 4;
                        const uint32_t v0 = *(const uint32_t*)v ^ 0x80808080u, v1 = *(const uint32_t*)(v + Sh::VS) ^ 0x80808080u;
                        const uint32_t v2 = *(const uint32_t*)(v + 8 * Sh::VS) ^ 0x80808080u, v3 = *(const uint32_t*)(v + 9 * Sh::VS) ^ 0x80808080u;
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const uint32_t x = __byte_perm(v0, v1, h ? 0x7362 : 0x5140), y = __byte_perm(v2, v3, h ? 0x7362 : 0x5140);
                            const uint32_t f[4] = {codes2(x, LOW), codes2(x, HIGH), codes2(y, LOW), codes2(y, HIGH)};
#pragma unroll
                            for (int t = 0; t < NT; t++)
#pragma unroll
                                for (int n = 0; n < PARTS<MT>; n++) mma<MT>(o[2 * k + h][t], f, pf[n][t][0], pf[n][t][1]);
                        }
                    }
                } else {
                    const int row = (lane >> 4) * 8 + (lane & 7);
                    const uint32_t at = st + Sh::VALUES + (16 * j + row) * Sh::VS;
#pragma unroll
                    for (int i = 0; i < D / 16; i++) {
                        uint32_t f[4];
                        ldm4t(f, at + Sh::v_chunk(lane, 2 * i + ((lane >> 3) & 1)) * 16);
#pragma unroll
                        for (int t = 0; t < NT; t++)
#pragma unroll
                            for (int n = 0; n < PARTS<MT>; n++) mma<MT>(o[i][t], f, pf[n][t][0], pf[n][t][1]);
                    }
                }
            }
        }

        // ---- the item's result.  Each lane brings its heads' outputs to the maximum over the warps, and to their end where
        // the item is whole; the warps' tiles are then added up in shared memory (in each warp's ring slot that its next
        // copy fills)
        const bool whole = it.u == 0 && it.end == it.n;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[t][x] += __shfl_xor_sync(0xffffffffu, l[t][x], d);
                if (r == 0) *(float2*)s_ml[warp][t * 8 + 2 * c4 + x] = make_float2(m[t][x], l[t][x]);
            }
        __syncwarp();
        float* tile = (float*)(ring + ready * Sh::STAGE);
        if (lane == 0) s_tile[warp] = (int)((uint8_t*)tile - ring_all);
        if (!solo) __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int row = t * 8 + 2 * c4 + x;
                float mx = m[t][x], sum = l[t][x], f = 1.f;
                if (!solo) {
                    const float2 own = make_float2(mx, sum);
#pragma unroll
                    for (int w = 0; w < WARPS; w++) mx = fmaxf(mx, s_ml[w][row][0]);
                    sum = 0.f;
#pragma unroll
                    for (int w = 0; w < WARPS; w++) {
                        const float2 ml = *(const float2*)s_ml[w][row];
                        sum += ml.y * weight(ml, mx);
                    }
                    f = weight(own, mx);
                }
                if (whole) {
                    f = sum == 0.f ? 0.f : f / sum;
                    if (a.lse && r == 0 && (solo || warp == 0) && row < rows)
                        a.lse[(int64_t)it.b * a.hq + h0 + row] = log_sum(mx, sum);
                } else if (r == 0 && warp == 0) {
                    *(float2*)(a.parts + (2 * piece + (it.u == 0)) * Sh::PART + Sh::ROWS * D + 2 * row) = make_float2(mx, sum);
                }
                const bool none = f == 0.f;
                const float up = I8 ? power2(lim[t][x] - m[t][x] - TOP) : 1.f;
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    float* p = tile + row * Sh::OS + (I8 ? (i / 2) * 32 + 4 * r + 2 * (i & 1) : i * 16 + r);
                    p[0] = none ? 0.f : o[i][t][x] * f * up;
                    p[I8 ? 1 : 8] = none ? 0.f : o[i][t][x + 2] * f * up;
                }
            }
        }
        constexpr int Q4 = D / 4;
        uint16_t* out = (uint16_t*)a.out + ((int64_t)it.b * a.hq + h0) * D;
        if (solo) {  // never cut: an item of so few units
            __syncwarp();
            for (int i = lane; i < rows * Q4; i += 32) {
                const int row = i / Q4, d = (i - row * Q4) * 4;
                const float4 x = *(const float4*)(tile + row * Sh::OS + d);
                *(uint2*)(out + row * D + d) = make_uint2(Elem<TYPE>::down(x.x, x.y), Elem<TYPE>::down(x.z, x.w));
            }
            __syncwarp();
            continue;
        }
        __syncthreads();
        // an item's first part is its piece's second one: the piece may begin with the last part of another item
        float* part = a.parts + (2 * piece + (it.u == 0)) * Sh::PART;
        for (int i = tid; i < rows * Q4; i += THREADS) {
            const int row = i / Q4, d = (i - row * Q4) * 4;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float4 x = *(const float4*)((const float*)(ring_all + s_tile[w]) + row * Sh::OS + d);
                acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
            }
            if (whole)
                *(uint2*)(out + row * D + d) = make_uint2(Elem<TYPE>::down(acc.x, acc.y), Elem<TYPE>::down(acc.z, acc.w));
            else
                *(float4*)(part + row * D + d) = acc;
        }
        __syncthreads();  // the part is written, and the tiles' slots may be filled again
        if (whole) continue;
        // its place among the parts: the cuts inside the item are parts - 1, the first at cut t_lo
        if (tid == 0) {
            const int t_lo = s_cuts.from(it_begin + ITEM_COST + near);
            s_cut[cut] = CutItem{it.b, it.head, it.sub, t_lo, s_cuts.upto(it_begin + ITEM_COST + it.n - near) - t_lo + 2};
        }
        cut++;
    }
    copies_wait<0>();
    __syncthreads();
    // ---- parts of cut items (the piece's first and last): each warp counts for the rows that it would join, and whoever is
    // last joins them.  At the piece's end, where the registers are free and both waits for the counts are one
    constexpr int WAYS = Sh::CTAS > 2 || D < 128 ? 8 : 16;  // what the registers hold
    unsigned joins = 0;
    if (lane < cut) {
        const CutItem& it = s_cut[lane];
        unsigned long long* count = a.arrived + ((int64_t)it.b * per_seq + it.head * split + it.sub);
        __threadfence();
        if ((int)((atomicAdd(count, 1ull << (16 * warp)) >> (16 * warp)) & 0xffff) == it.parts - 1) {
            atomicAdd(count, 0ull - ((unsigned long long)it.parts << (16 * warp)));
            joins = 1;
        }
    }
    joins = __ballot_sync(0xffffffffu, joins);
    if (joins) __threadfence();
#pragma unroll 1
    for (; joins; joins &= joins - 1) {
        const CutItem it = s_cut[__ffs(joins) - 1];
        const int rows = min(Sh::ROWS, a.group - it.sub * Sh::ROWS);
        const int64_t row0 = (int64_t)it.b * a.hq + it.head * a.group + it.sub * Sh::ROWS;
        const float* from = a.parts + (int64_t)2 * (it.t_lo - 1) * Sh::PART;
        uint16_t* out = (uint16_t*)a.out + row0 * D;
        float* lse = a.lse ? a.lse + row0 : nullptr;
        if (warp >= rows) continue;
        if (rows <= WARPS)
            join_parts<D, TYPE, Sh::ROWS, 1, WAYS>(from, it.parts, warp, rows, out, lse);
        else
            join_parts<D, TYPE, Sh::ROWS, Sh::ROWS / WARPS, WAYS>(from, it.parts, warp, rows, out, lse);
    }
    if (!shared) break;
    }
    if (shared && tid == 0) {
        if (atomicAdd(a.counts + 1, 1) == (int)gridDim.x - 1) a.counts[0] = a.counts[1] = 0;
    }
}

template <int D, int TYPE, int STORE, int NT>
static int launch_nt(fvs_stream_t stream, AttendArgs a) {
    using Sh = Shape<D, STORE, NT>;
    auto kernel = attend_kernel<D, TYPE, STORE, NT>;
    if (cudaError_t e = fvs_ensure_smem((const void*)kernel, Sh::SMEM)) return (int)e;
    a.split = (a.group + Sh::ROWS - 1) / Sh::ROWS;
    // no more CTAs than the page tables' room can fill
    const int64_t room = (int64_t)a.tb.wide * a.c.page;
    const int64_t units = ((room < INT_MAX ? room : INT_MAX) + Sh::UNIT - 1) / Sh::UNIT * a.tb.seqs * a.c.heads * a.split;
    int64_t grid = (units + WARPS - 1) / WARPS;
    const int64_t full = (int64_t)fvs_sm_count() * Sh::CTAS;
    if (grid > full) grid = full;
    kernel<<<(unsigned)grid, THREADS, Sh::SMEM, stream>>>(a);
    return fvs_launch_status();
}
template <int D, int TYPE, int STORE>
static int launch(fvs_stream_t stream, const AttendArgs& a) {
    // wide int8 heads: two items of 8 rows take 68 us where one of 16 takes 87 (64 requests of 500 to 16000 keys, D = 256);
    // wide 16-bit heads: 128 and 95 us (all with weights in one part; with two 76 us, and 87 us for 16-bit heads)
    if (a.group <= 8 || (STORE == FVS_I8 && D > 128)) return launch_nt<D, TYPE, STORE, 1>(stream, a);
    return launch_nt<D, TYPE, STORE, (STORE == FVS_I8 && D > 128 ? 1 : 2)>(stream, a);
}
// one translation unit for each D (fvs_kv_attend_*.cu): together they took 80 s to compile, side by side 25
template <int D>
int launch_types(fvs_stream_t stream, const AttendArgs& a, int type) {
    if (type == FVS_F16)
        return a.c.type == FVS_I8 ? launch<D, FVS_F16, FVS_I8>(stream, a) : launch<D, FVS_F16, FVS_F16>(stream, a);
    return a.c.type == FVS_I8 ? launch<D, FVS_BF16, FVS_I8>(stream, a) : launch<D, FVS_BF16, FVS_BF16>(stream, a);
}

}  // namespace kv
}  // namespace fvs
