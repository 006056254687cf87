// Attention of a few query rows per KV head over the paged 8-bit cache: a step of decoding, or of a few drafted tokens.
//
// What bounds it: HBM, each code of the cache read once (a byte per value, against one multiply-add per query row).  So the work is laid out for
// the memory system, and the products go to mma.sync on registers: a tcgen05 tile has 128 rows, of which a step would fill 4 or 8.
//
// Shares.  The keys of all (sequence, KV head, row tile) problems lie behind one another in units of 4 x 32 keys, and the CTAs - as many as are resident
// at once - take equal parts of that line, whatever the lengths of the sequences; the host does not know them.  A CTA's piece of a problem is a segment.  A warp
// asks for the keys of its next segment while it still works on the one before, so the stream of loads does not stop between them; a segment's four shares are joined
// warp to warp, and a warp that has handed its own on goes on.
// A problem that several CTAs share leaves partial results (sums, maximum, weights' sum) in the workspace; the CTA that comes last adds them up in their
// order along the keys, so the result does not depend on which one that is.
//
// A warp's step: 4 KB of keys and of values, copied by its own lanes with cp.async: no warp waits for another.
// Both contractions are products of 8-bit integers (mma.sync m16n8k32, exact 32-bit sums), so the codes are operands as they lie there.  (As f16, four
// instructions went into each pair of codes: 530 per step of 4 KB, and the SMs, not HBM, were the bound: 5.0 TB/s.)
//   scores  S[16 rows x 8 keys] = Q K^T.  Queries are fixed-point numbers of 22 bits and sign under a power of two per row - half a step is 2^-23 of the row's largest value -
//           as three signed digits of 8 bits, a row of the MMA each.  Where digits would lose too much, scores are formed in fp32 from the queries themselves.
//           f16: values above 2^-11 of the largest are held as they are.  What the others lose is summed up for each row; where it could move a score's exponent by more than
//           2^-13 in some key of the step, all codes of which were +-128, the step goes to fp32.  (With two digits, 15 bits, keys that have no part in a query's few outliers
//           of 16 to 33 times the rest came out up to 1.2 % off.)
//           fp32: every value loses something, next to nothing beside its score as a rule.  A step goes to fp32 where that, 1 / sqrt(12) of a step each and a root of their sum of
//           squares, times codes of 128, could move an exponent by more than 2^-16: scores of some tens for ordinary rows.  (A rule on a row's values alone, whether a few are far larger than the rest,
//           let rows pass half of whose values were 300 times the others; with keys that had no part in those the result was 12 % off.)
//   values  O^T[16 dims x 8 rows] = V^T P^T.  Weights exp2(s - m), m the row's largest score in the step, are fixed-point numbers of 16 bits (f16 results) or 23
//           (fp32): half a step is 2^-17 or 2^-24 of the largest weight of the step.  Unsigned digits, an MMA each; the accumulator fragment of S holds just the
//           weights that the operand fragment wants, four tokens' bytes to a register, and a 4 x 4 transpose of bytes puts four tokens' codes side by side.
// A step's sums, joined from the digits, times exp2(m - running maximum) and the page's scale are added to fp32 sums.  The order of a contraction is free, so 16
// consecutive bytes of a key are a lane's operands of two MMAs.
//
// Measured: 3 requests over 50001 to 33334 keys, f16, 8 KV heads of 128: 53.5 us, 4.8 TB/s of the call and more between its ends; the rest is the start (which sequence, which page,
// first data: 5 us) and the joining of the parts (4 us).  64 requests over 1000 to 508 keys, fp32, 8 heads of 64: 23.3 us; with the whole CTA waiting at the end of each segment it
// took 2 us more.  24 requests of 4 tokens over 2000 to 1042 keys, f16, 6 heads to each of 4: 29.9 us; 24 query rows are three tiles of 8, each of which takes the keys once more,
// from L2.  64 requests over 8000 keys, f16, 8 heads of 128: 174 us; where all steps form their scores in fp32, 1235.
#pragma once

#include "paged.cuh"
#include "split_pair.cuh"

namespace rmlk {
namespace paged {

struct Attend {
    const void* q;
    void* out;
    int64_t qs, os;  // row strides
    int q_heads, group;
    float scale;
    int* status;
};

constexpr int COUNTERS = 4096;  // arrival counters at the head of a workspace; one for each CTA that begins a shared problem

template <typename T, int D, int NR_>
struct Few {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int NR = NR_;               // groups of 8 query rows in a tile
    static constexpr int ROWS = 8 * NR;
    static constexpr int KS = 4096 / D, NC = KS / 16;  // keys of a warp's step; groups of 16 of them: one page each
    static constexpr int UNIT = 4 * KS;
    static constexpr int STAGES = 2;
    static constexpr int K_BYTES = KS * D, STEP = 2 * K_BYTES;
    static constexpr int QT = NR + 1;             // row tiles of the scores' MMAs: (first, second digit) of each group, and the third digits of both
    static constexpr int DIGITS = F32 ? 3 : 2;    // of the weights
    static constexpr int RING = 4 * STAGES * STEP;
    static constexpr int FRAGS = D / 16 * NR;    // groups of four sums per lane
    static constexpr int HAND = 32 * (FRAGS * 16 + NR * 8);  // a warp's share on its way to another: sums, maxima, weights' sums
    static constexpr int SCALES = RING + 2 * HAND, SCAN = SCALES + 4 * STAGES * NC * 8, SEGMENTS = SCAN + 64, SMEM = SEGMENTS + 4 * 2 * 64;
    static constexpr int PER_SM = NR == 2 ? 2 : 3;
};
constexpr int MOST_PARTS = 32;  // CTAs for a problem, on average: each costs the last one a fraction of a microsecond
inline size_t few_workspace(int64_t d) { return COUNTERS * 4 + static_cast<size_t>(sm_count()) * 4 * 2 * (32 * (d / 16 * 2 * 16 + 2 * 8)); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// signed x signed (queries and keys), signed x unsigned (values and weights)
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_u8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
// Where 16-byte unit u of key r (of 16) lies in shared memory.  A warp copies 512 consecutive bytes at a time - half-filled lines in flight cost a quarter of the
// bandwidth - and reads units of keys r .. r + 7 (keys), or the same units of every other key (values): the units of a 128-byte line are exchanged so that
// neither meets bank conflicts.
template <int D>
__device__ __forceinline__ int unit_at(int r, int u) {
    if constexpr (D == 64) return (r >> 1) * 128 + ((((r & 1) * 4 + u) ^ (r & 6)) << 4);
    return r * 128 + ((u ^ (r & 6) ^ (r & 1) * 4) << 4);
}
// byte B of four words, in order
template <int B>
__device__ __forceinline__ uint32_t bytes_of(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
    return __byte_perm(__byte_perm(w0, w1, B | (B + 4) << 4), __byte_perm(w2, w3, B | (B + 4) << 4), 0x5410);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    return x + __shfl_xor_sync(0xffffffffu, x, 2);
}
// a / b for 0 <= a, 0 < b: nearly always in 32 bits.  A 64-bit division is 2 KB of instructions: inlined wherever one may be needed, they made kernels of 100 KB, which do not
// stay in the instruction cache.
__device__ __noinline__ int64_t divide_64(int64_t a, int64_t b) { return a / b; }
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
    return ((a | b) >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : divide_64(a, b);
}

// named barriers between two warps: one hands over and goes on, the other waits
template <int ID>
__device__ __forceinline__ void pair_arrive() { asm volatile("bar.arrive %0, 64;" ::"n"(ID) : "memory"); }
template <int ID>
__device__ __forceinline__ void pair_wait() { asm volatile("bar.sync %0, 64;" ::"n"(ID) : "memory"); }
enum { HAND_0 = 1, HAND_1, HAND_UP, FREE_0, FREE_1 };

// What a lane knows of a tile's rows: sums over keys of w v (dims (D / 8) g + 2 i, and + 1 in the upper two, of rows 2 c4, 2 c4 + 1), the largest score and the sum of
// the weights of rows g (and g + 8).
template <int D, int NR>
struct Share {
    float acc[D / 16][NR][4], top[NR], sum[NR];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int r = 0; r < NR; r++) {
            top[r] = -INFINITY;
            sum[r] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 16; i++) acc[i][r][0] = acc[i][r][1] = acc[i][r][2] = acc[i][r][3] = 0.f;
        }
    }
    // rows 2 c4 and 2 c4 + 1 of something that lanes hold for row g
    static __device__ __forceinline__ float2 of_sums(float f, int c4) { return make_float2(__shfl_sync(0xffffffffu, f, 8 * c4), __shfl_sync(0xffffffffu, f, 8 * c4 + 4)); }
    __device__ __forceinline__ void scale(int r, float f, int c4) {
        const float2 k = of_sums(f, c4);
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            acc[i][r][0] *= k.x;
            acc[i][r][1] *= k.y;
            acc[i][r][2] *= k.x;
            acc[i][r][3] *= k.y;
        }
    }
    // to and from memory that holds it lane by lane
    __device__ __forceinline__ void put(float* at, int lane) const {
#pragma unroll
        for (int r = 0; r < NR; r++) {
            *reinterpret_cast<float2*>(at + 128 * (D / 16) * NR + 64 * r + 2 * lane) = make_float2(top[r], sum[r]);
#pragma unroll
            for (int i = 0; i < D / 16; i++)
                *reinterpret_cast<float4*>(at + 128 * (i * NR + r) + 4 * lane) = make_float4(acc[i][r][0], acc[i][r][1], acc[i][r][2], acc[i][r][3]);
        }
    }
    __device__ __forceinline__ void get(const float* at, int lane) {
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const float2 t = __ldcg(reinterpret_cast<const float2*>(at + 128 * (D / 16) * NR + 64 * r + 2 * lane));
            top[r] = t.x;
            sum[r] = t.y;
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                const float4 x = __ldcg(reinterpret_cast<const float4*>(at + 128 * (i * NR + r) + 4 * lane));
                acc[i][r][0] = x.x;
                acc[i][r][1] = x.y;
                acc[i][r][2] = x.z;
                acc[i][r][3] = x.w;
            }
        }
    }
    // A share without keys has the maximum -inf and sums of zero (or NaN, which has to stay).
    __device__ __forceinline__ void join(int r, float other_top, float other_sum, int c4, float2& own, float2& other) {
        const float most = fmaxf(top[r], other_top);
        const float f = top[r] == -INFINITY ? 1.f : ex2(top[r] - most), o = other_top == -INFINITY ? 1.f : ex2(other_top - most);
        top[r] = most;
        sum[r] = fmaf(other_sum, o, sum[r] * f);
        own = of_sums(f, c4);
        other = of_sums(o, c4);
    }
    __device__ __forceinline__ void join(const Share& x, int c4) {
#pragma unroll
        for (int r = 0; r < NR; r++) {
            float2 f, o;
            join(r, x.top[r], x.sum[r], c4, f, o);
#pragma unroll
            for (int i = 0; i < D / 16; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][r][e] = fmaf(x.acc[i][r][e], e & 1 ? o.y : o.x, acc[i][r][e] * (e & 1 ? f.y : f.x));
        }
    }
    __device__ __forceinline__ void join_shared(const float* at, int lane, int c4) {
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const float2 t = *reinterpret_cast<const float2*>(at + 128 * (D / 16) * NR + 64 * r + 2 * lane);
            float2 f, o;
            join(r, t.x, t.y, c4, f, o);
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                const float4 x = *reinterpret_cast<const float4*>(at + 128 * (i * NR + r) + 4 * lane);
                acc[i][r][0] = fmaf(x.x, o.x, acc[i][r][0] * f.x);
                acc[i][r][1] = fmaf(x.y, o.y, acc[i][r][1] * f.y);
                acc[i][r][2] = fmaf(x.z, o.x, acc[i][r][2] * f.x);
                acc[i][r][3] = fmaf(x.w, o.y, acc[i][r][3] * f.y);
            }
        }
    }
};

// A step's products of queries and codes in fp32, as lanes hold them: rows g (and g + 8) of the tile from row0 on, keys 8 j + 2 c4 and the next.
template <int D, int NR>
struct Scores {
    float x[NR][4096 / D / 8][2];
};
template <typename T, int D, int NR>
__device__ __noinline__ Scores<D, NR> scores_in_fp32(const T* q, int64_t stride, int group, int64_t first, int h, int row0, int rows, const uint8_t* keys) {
    constexpr int J = 4096 / D / 8;
    const int g = (threadIdx.x & 31) >> 2, c4 = threadIdx.x & 3;
    Scores<D, NR> y;
#pragma unroll
    for (int r = 0; r < NR; r++) {
        const int row = row0 + g + 8 * r, token = row / group;
        const T* src = q + (first + token) * stride + (static_cast<int64_t>(h) * group + row - token * group) * D;
#pragma unroll
        for (int j = 0; j < J; j++) y.x[r][j][0] = y.x[r][j][1] = 0.f;
#pragma unroll 1
        for (int u = 0; u < D / 4; u++) {  // four dims at a time
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = row < rows ? static_cast<float>(src[4 * u + i]) : 0.f;
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(keys + j / 2 * (16 * D) + unit_at<D>(8 * (j & 1) + 2 * c4 + e, u >> 2) + 4 * (u & 3));
#pragma unroll
                    for (int i = 0; i < 4; i++) y.x[r][j][e] = fmaf(v[i], static_cast<float>(static_cast<int8_t>(w >> (8 * i))), y.x[r][j][e]);
                }
        }
    }
    return y;
}

template <typename T, int D, int NR>
__global__ void __launch_bounds__(128, Few<T, D, NR>::PER_SM) few_kernel(const Cache c, const Batch q, const Attend a, const int tiles, unsigned* counters, float* partials) {
    using L = Few<T, D, NR>;
    constexpr int ROWS = L::ROWS, KS = L::KS, NC = L::NC, PIECES = D / 64, SLOT = L::HAND / 4;
    dep_sync();
    extern __shared__ __align__(16) uint8_t smem[];
    float* s_hand = reinterpret_cast<float*>(smem + L::RING);
    int64_t* s_at = reinterpret_cast<int64_t*>(smem + L::SCAN);  // scan, where the share begins, at the end whether this CTA was the last one
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c4 = lane & 3;
    const int64_t table_keys = q.width << c.page_log;
    // keys behind the table have no page: one of them stands for all
    auto keys_of = [&](int b) { return min(static_cast<int64_t>(q.lens[b]), table_keys + 1); };
    auto units_of = [&](int b) { return max((keys_of(b) + L::UNIT - 1) / L::UNIT, int64_t(1)); };  // (a sequence without keys has rows to write all the same)
    const int64_t items = static_cast<int64_t>(c.kv_heads) * tiles;  // problems of a sequence

    // ---- this CTA's share of the line ----
    int64_t total, per, lo, hi, share_seq;  // share_seq: where the sequence that the share begins in begins on the line
    int share_b;
    unsigned workers, longer;  // the first `longer` workers have per + 1 units, the others per
    auto begin_of = [&](unsigned w) { return per * w + min(w, longer); };
    auto worker_of = [&](int64_t unit) {
        const int64_t head = (per + 1) * longer;
        return static_cast<unsigned>(unit < head ? divide(unit, per + 1) : longer + divide(unit - head, per));
    };
    {
        const int each = (q.batch + 127) / 128, b0 = min(tid * each, q.batch), b1 = min(b0 + each, q.batch);
        int64_t own = 0;
        for (int i = b0; i < b1; i++) own += units_of(i);
        own *= items;
        int64_t upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        if (lane == 31) s_at[warp] = upto;
        __syncthreads();
        total = s_at[0] + s_at[1] + s_at[2] + s_at[3];
        for (int w = 0; w < warp; w++) upto += s_at[w];
        workers = static_cast<unsigned>(min(min(static_cast<int64_t>(gridDim.x), total), MOST_PARTS * items * q.batch));
        if (blockIdx.x >= workers) return;
        per = divide(total, workers);
        longer = static_cast<unsigned>(total - per * workers);
        lo = begin_of(blockIdx.x);
        hi = begin_of(blockIdx.x + 1);
        __syncthreads();
        int64_t first = upto - own;
        if (first <= lo && lo < upto) {
            for (int i = b0; i < b1; i++) {
                const int64_t n = units_of(i) * items;
                if (lo < first + n) {
                    s_at[0] = i;
                    s_at[1] = first;
                    break;
                }
                first += n;
            }
        }
        __syncthreads();
        share_b = static_cast<int>(s_at[0]);
        share_seq = s_at[1];
    }
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * (L::STAGES * L::STEP);
    const uint8_t* ring_ptr = smem + warp * (L::STAGES * L::STEP);
    float2* scales = reinterpret_cast<float2*>(smem + L::SCALES) + warp * (L::STAGES * NC);  // of K and V, [stage][NC]
    const int rows = q.each * a.group;

    // A segment, as a warp sees it: its steps are the keys first_key + i UNIT.
    struct Segment {
        int b, h, tile, steps, left;  // left: keys from the warp's first to the segment's end
        int64_t seq, unit, units, taken, first_key;  // where the sequence and the segment begin on the line; units of a problem, of them in the segment
    };
    auto look = [&](Segment& s) {
        const int64_t keys = keys_of(s.b);
        s.units = units_of(s.b);
        const int64_t item = divide(s.unit - s.seq, s.units), unit0 = (s.unit - s.seq) - item * s.units;
        s.taken = min(s.units - unit0, hi - s.unit);
        s.h = static_cast<int>(item) / tiles;
        s.tile = static_cast<int>(item) - s.h * tiles;
        s.first_key = unit0 * L::UNIT + warp * KS;
        const int64_t left = min(keys, (unit0 + s.taken) * L::UNIT) - s.first_key;
        s.left = static_cast<int>(max(left, int64_t(0)));
        s.steps = (s.left + L::UNIT - 1) / L::UNIT;
    };
    auto move_on = [&](Segment& s) {
        s.unit += s.taken;
        if (s.unit - s.seq == s.units * items) {
            s.seq = s.unit;
            s.b++;
        }
        if (s.unit < hi) look(s);
    };

    // ---- the stream of loads ----
    // The segments that are asked for and worked on wait in shared memory: in registers they would push out what the steps need.  (Every lane writes the same and reads what it wrote.)
    struct Place {
        Segment s;
        __device__ __forceinline__ void put(const Segment& x) volatile {
            s.b = x.b, s.h = x.h, s.tile = x.tile, s.steps = x.steps, s.left = x.left;
            s.seq = x.seq, s.unit = x.unit, s.units = x.units, s.taken = x.taken, s.first_key = x.first_key;
        }
        __device__ __forceinline__ Segment get() volatile {
            Segment x;
            x.b = s.b, x.h = s.h, x.tile = s.tile, x.steps = s.steps, x.left = s.left;
            x.seq = s.seq, x.unit = s.unit, x.units = s.units, x.taken = s.taken, x.first_key = s.first_key;
            return x;
        }
    };
    static_assert(sizeof(Place) <= 64, "");
    volatile Place* const asked = reinterpret_cast<volatile Place*>(smem + L::SEGMENTS + 128 * warp);
    volatile Place* const at_work = reinterpret_cast<volatile Place*>(smem + L::SEGMENTS + 128 * warp + 64);
    int ask_steps;
    {
        Segment first;
        first.b = share_b;
        first.seq = share_seq;
        first.unit = lo;
        look(first);
        asked->put(first);
        at_work->put(first);
        ask_steps = first.steps;
    }
    int block = -1;  // page and head as one index; -1: no key there, -2: a key without a page
    constexpr int PAGED_STEPS = 32 / NC;  // pages of so many steps are looked up at a time, one per lane
    const int block_bytes = c.page * D;
    int fill = 0, fill_stage = 0;  // next step to be asked for, its place in the ring
    auto issue = [&]() {
        if (fill == ask_steps) {
            Segment ask = asked->get();
            while (fill == ask.steps && ask.unit < hi) {
                move_on(ask);
                fill = 0;
                if (ask.unit >= hi) ask.steps = 0;
            }
            asked->put(ask);
            ask_steps = ask.steps;
        }
        if (fill < ask_steps) {
            const int h = asked->s.h;
            const int64_t first_key = asked->s.first_key;
            const int in_batch = fill % PAGED_STEPS;
            if (in_batch == 0) {
                const int off = (fill + lane / NC) * L::UNIT + (lane % NC) * 16;
                block = -1;
                if (off < asked->s.left) {
                    const int64_t at = (first_key + off) >> c.page_log;
                    const int p = at < q.width ? q.table[static_cast<int64_t>(asked->s.b) * q.width + at] : -1;
                    block = p >= 0 && p < c.pages ? p * c.kv_heads + h : -2;
                    if (block == -2 && a.status) *a.status = RMLK_ERR_INVALID_ARG;
                }
            }
            const uint32_t dst = ring + fill_stage * L::STEP;
#pragma unroll
            for (int n = 0; n < NC; n++) {
                const int at = __shfl_sync(0xffffffffu, block, in_batch * NC + n), from = at < 0 ? h : at;  // (page 0 is read where there is none)
                if (lane < 2) {  // the scales of K and V: 0 where there is no key, NaN where a key has no page
                    float* to = reinterpret_cast<float*>(scales + fill_stage * NC + n) + lane;
                    if (at >= 0) copy_async<4>(static_cast<uint32_t>(__cvta_generic_to_shared(to)), (lane ? c.vs : c.ks) + at);
                    else *to = at == -1 ? 0.f : __int_as_float(0x7fc00000);
                }
                const int64_t off = static_cast<int64_t>(from) * block_bytes + ((static_cast<int>(first_key & 127) + fill * L::UNIT + 16 * n) & (c.page - 1)) * D;
#pragma unroll
                for (int j = 0; j < D / 32; j++) {
                    const uint32_t to = dst + n * (16 * D) + unit_at<D>((512 / D) * j + lane / (D / 16), lane % (D / 16));
                    copy_async<16>(to, c.k + off + j * 512 + lane * 16);
                    copy_async<16>(to + L::K_BYTES, c.v + off + j * 512 + lane * 16);
                }
            }
            fill++;
            if (++fill_stage == L::STAGES) fill_stage = 0;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // a finished tile; a row that sees nothing is 0
    auto store = [&](const Share<D, NR>& x, int b, int h, int tile) {
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const float2 l = Share<D, NR>::of_sums(x.sum[r], c4);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int row = tile * ROWS + 8 * r + 2 * c4 + e, token = row / a.group;
                if (row >= rows) continue;
                const float sum = e ? l.y : l.x, inv = sum == 0.f ? 0.f : 1.f / sum;
                T* dst = static_cast<T*>(a.out) + (static_cast<int64_t>(b) * q.each + token) * a.os + (static_cast<int64_t>(h) * a.group + row - token * a.group) * D + g * (D / 8);
#pragma unroll
                for (int i = 0; i < D / 16; i += 2) {
                    const float4 o = make_float4(x.acc[i][r][e] * inv, x.acc[i][r][2 + e] * inv, x.acc[i + 1][r][e] * inv, x.acc[i + 1][r][2 + e] * inv);
                    if constexpr (L::F32) *reinterpret_cast<float4*>(dst + 2 * i) = o;
                    else *reinterpret_cast<uint2*>(dst + 2 * i) = make_uint2(pack_f16(o.x, o.y), pack_f16(o.z, o.w));
                }
            }
        }
    };
    // the CTAs that share a segment's problem, from `first` on; whether the first one's is its second piece of the line
    struct Parts {
        unsigned first, count;
        int second;
    };
    auto parts_of = [&](const Segment& s) {
        const int64_t begin = s.seq + divide(s.unit - s.seq, s.units) * s.units;
        Parts p;
        p.first = worker_of(begin);
        p.count = worker_of(begin + s.units - 1) - p.first + 1;
        p.second = begin_of(p.first) != begin;
        return p;
    };
    bool last_first = false, last_second = false;  // (warp 0) this CTA was the last one to finish the problem of its first, its last segment
    int stage = 0;
    bool first = true, handed = false;  // first segment of the CTA; the hand-over places have been used

    while (true) {
        const int b = at_work->s.b, h = at_work->s.h, tile = at_work->s.tile, steps = at_work->s.steps;
        const int64_t keys = keys_of(b), first_key = at_work->s.first_key;
        const int64_t before = static_cast<int64_t>(q.lens[b]) - q.each;  // keys before the first new token

        // ---- queries: fragments of the scores' MMAs, and what each lane's rows see.  (Asked for first, looked at when the first keys are on their way.) ----
        auto relative = [&](int64_t key) { return static_cast<int>(max(min(key - first_key, int64_t(0x7fffff00)), int64_t(0))); };
        using Four = typename std::conditional<L::F32, float4, uint2>::type;  // four values
        Four qx[NR][4 * PIECES];
        float factor[NR];
        int sees[NR];  // keys from the warp's first on that the lane's rows see
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const int row = tile * ROWS + g + 8 * r, token = row / a.group;
            const bool in = row < rows;
            sees[r] = in ? relative(min(before + token + 1, keys)) : 0;
            const T* src = static_cast<const T*>(a.q) + (static_cast<int64_t>(b) * q.each + token) * a.qs + (static_cast<int64_t>(h) * a.group + row - token * a.group) * D + 16 * c4;
#pragma unroll
            for (int s = 0; s < 4 * PIECES; s++) {
                Four x = {};
                if (in) x = *reinterpret_cast<const Four*>(src + (s >> 2) * 64 + (s & 3) * 4);
                qx[r][s] = x;
            }
        }
        if (first) {
#pragma unroll
            for (int s = 0; s < L::STAGES - 1; s++) issue();
        }
        // what digits of the tile's queries may lose in an exponent, for keys under the scale 1: three digits, the first two of them (f16)
        float lost = 0.f, lost_by_two = 0.f;
        // digits: [32 dims][row tile]: rows g and g + 8 of the lane's first four dims, then of the next four
        uint32_t qf[2 * PIECES][L::QT][4];
        if constexpr (NR == 1) {
#pragma unroll
            for (int s = 0; s < 2 * PIECES; s++) qf[s][NR][1] = qf[s][NR][3] = 0;  // no second group
        }
#pragma unroll
        for (int r = 0; r < NR; r++) {
            auto four = [&](int s) {
                if constexpr (L::F32) {
                    return qx[r][s];
                } else {
                    const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&qx[r][s].x)), hi = __half22float2(*reinterpret_cast<const __half2*>(&qx[r][s].y));
                    return make_float4(lo.x, lo.y, hi.x, hi.y);
                }
            };
            uint32_t most = 0;
#pragma unroll
            for (int s = 0; s < 4 * PIECES; s++) {
                const float4 x = four(s);
                most = max(max(most, max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu)), max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu));
            }
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            // 2^e: the largest in [2^14, 2^15), times 2^8 for the third digit, but not above what signed digits hold, 127 127 127
            int e = scale_exponent(most < 0x7f800000u ? most : 0u);
            if (__uint_as_float(most) * exp2_int(e) > 32639.49f) e--;
            const float up = exp2_int(e), more = 256.f;
            // an infinity or a NaN makes NaN of the row
            factor[r] = most < 0x7f800000u ? a.scale * 1.44269504f / more * exp2_int(-e) : __int_as_float(0x7fc00000);
            float rest = 0.f;  // (f16) what three digits leave of the lane's values, in steps; squares of the third digits
            int thirds = 0;
#pragma unroll
            for (int s = 0; s < 4 * PIECES; s++) {
                const float4 x = four(s);
                const int v[4] = {__float2int_rn(x.x * up * more), __float2int_rn(x.y * up * more), __float2int_rn(x.z * up * more), __float2int_rn(x.w * up * more)};
                if constexpr (!L::F32)
                    rest += (fabsf(x.x * up * more - static_cast<float>(v[0])) + fabsf(x.y * up * more - static_cast<float>(v[1]))) +
                            (fabsf(x.z * up * more - static_cast<float>(v[2])) + fabsf(x.w * up * more - static_cast<float>(v[3])));
                // signed digits: the byte of v + 0x80 (+ 0x8000) carries what the digits below borrow
                const uint32_t d0 = bytes_of<0>(v[0], v[1], v[2], v[3]), d1 = bytes_of<1>(v[0] + 0x80, v[1] + 0x80, v[2] + 0x80, v[3] + 0x80);
                uint32_t(&f)[L::QT][4] = qf[s >> 1];
                const int at = 2 * (s & 1);
                f[r][at] = bytes_of<2>(v[0] + 0x8080, v[1] + 0x8080, v[2] + 0x8080, v[3] + 0x8080);
                f[r][at + 1] = d1;
                f[NR][at + r] = d0;
                if constexpr (!L::F32) thirds = __dp4a(static_cast<int>(d0), static_cast<int>(d0), thirds);
            }
            // (a row that is NaN has no part in these)
            if constexpr (L::F32) {
                // a step / sqrt(12) for each value; the limit is 2^-16 for it
                if (most > 0) lost = fmaxf(lost, fabsf(factor[r]) * ((D == 64 ? 2.3094011f : 3.2659863f) * 128.f * 8.f));
            } else {
                lost = fmaxf(lost, quad_sum(rest) * fabsf(factor[r]) * 128.f);
                lost_by_two = fmaxf(lost_by_two, sqrtf(quad_sum(static_cast<float>(thirds))) * fabsf(factor[r]) * 128.f);
            }
        }
        lost = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(lost)));
        if constexpr (!L::F32) lost_by_two = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(lost_by_two)));
        const int all_see = relative(min(before + 1 + (tile * ROWS) / a.group, keys));  // that every row of the tile sees

        Share<D, NR> own;
        own.clear();
        float(&acc)[D / 16][NR][4] = own.acc;
        float(&top)[NR] = own.top;
        float(&sum)[NR] = own.sum;
        for (int step = 0; step < steps; step++, stage = stage + 1 == L::STAGES ? 0 : stage + 1) {
            __syncwarp();  // the slot that is filled next has been read, its scales too
            issue();
            asm volatile("cp.async.wait_group %0;" ::"n"(L::STAGES - 1) : "memory");
            __syncwarp();  // (of all lanes)
            const uint8_t* at = ring_ptr + stage * L::STEP;
            // scales of V: the largest magnitude, and whether the others are of its size and sign; what is not finite; the largest scale of K
            float k_top = 0.f, v_most = 0.f, v_least = 0.f, v_low = INFINITY;
            bool broken = false;
#pragma unroll
            for (int n = 0; n < NC; n++) {
                const float2 kv = scales[stage * NC + n];
                const float size = fabsf(kv.y);
                broken = broken || !(fabsf(kv.x) < INFINITY) || !(size < INFINITY);
                k_top = fmaxf(k_top, fabsf(kv.x));
                v_most = fmaxf(v_most, kv.y);
                v_least = fminf(v_least, kv.y);
                if (size > 0.f) v_low = fminf(v_low, size);
            }
            const float v_top = fmaxf(v_most, -v_least);
            // ---- scores ----
            float x[NR][KS / 8][2];
#pragma unroll
            for (int j = 0; j < KS / 8; j++) {
                int s[L::QT][4] = {};
#pragma unroll
                for (int i = 0; i < PIECES; i++) {
                    const uint4 w = *reinterpret_cast<const uint4*>(at + j / 2 * (16 * D) + unit_at<D>(8 * (j & 1) + g, 4 * i + c4));
#pragma unroll
                    for (int t = 0; t < (L::F32 ? L::QT : NR); t++) {
                        mma_s8(s[t], qf[2 * i][t][0], qf[2 * i][t][1], qf[2 * i][t][2], qf[2 * i][t][3], w.x, w.y);
                        mma_s8(s[t], qf[2 * i + 1][t][0], qf[2 * i + 1][t][1], qf[2 * i + 1][t][2], qf[2 * i + 1][t][3], w.z, w.w);
                    }
                }
                const float ks = scales[stage * NC + j / 2].x;
#pragma unroll
                for (int r = 0; r < NR; r++) {
                    const float t = factor[r] * ks;
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float high = static_cast<float>(s[r][e] * 256 + s[r][2 + e]);
                        x[r][j][e] = (L::F32 ? fmaf(high, 256.f, static_cast<float>(s[NR][2 * r + e])) : high * 256.f) * t;
                    }
                }
            }
            if (!L::F32 && lost_by_two * k_top > 2.44140625e-4f) {  // 2^-12: the third digits too
#pragma unroll
                for (int j = 0; j < KS / 8; j++) {
                    int s[4] = {};
#pragma unroll
                    for (int i = 0; i < PIECES; i++) {
                        const uint4 w = *reinterpret_cast<const uint4*>(at + j / 2 * (16 * D) + unit_at<D>(8 * (j & 1) + g, 4 * i + c4));
                        mma_s8(s, qf[2 * i][NR][0], qf[2 * i][NR][1], qf[2 * i][NR][2], qf[2 * i][NR][3], w.x, w.y);
                        mma_s8(s, qf[2 * i + 1][NR][0], qf[2 * i + 1][NR][1], qf[2 * i + 1][NR][2], qf[2 * i + 1][NR][3], w.z, w.w);
                    }
                    const float ks = scales[stage * NC + j / 2].x;
#pragma unroll
                    for (int r = 0; r < NR; r++)
#pragma unroll
                        for (int e = 0; e < 2; e++) x[r][j][e] = fmaf(static_cast<float>(s[2 * r + e]), factor[r] * ks, x[r][j][e]);
                }
            }
            const bool wide = lost * k_top > 1.220703125e-4f;  // 2^-13
            if (wide) {
                float direct[NR];
#pragma unroll
                for (int r = 0; r < NR; r++) direct[r] = factor[r] == factor[r] ? a.scale * 1.44269504f : factor[r];
                const Scores<D, NR> y = scores_in_fp32<T, D, NR>(static_cast<const T*>(a.q), a.qs, a.group, static_cast<int64_t>(b) * q.each, h, tile * ROWS, rows, at);
#pragma unroll
                for (int j = 0; j < KS / 8; j++) {
                    const float ks = scales[stage * NC + j / 2].x;
#pragma unroll
                    for (int r = 0; r < NR; r++) {
                        x[r][j][0] = y.x[r][j][0] * (direct[r] * ks);
                        x[r][j][1] = y.x[r][j][1] * (direct[r] * ks);
                    }
                }
            }
            if (KS + step * L::UNIT > all_see) {
#pragma unroll
                for (int r = 0; r < NR; r++) {
                    const int see = sees[r] - step * L::UNIT;
#pragma unroll
                    for (int j = 0; j < KS / 8; j++) {
                        if (8 * j + 2 * c4 >= see) x[r][j][0] = -INFINITY;
                        if (8 * j + 2 * c4 + 1 >= see) x[r][j][1] = -INFINITY;
                    }
                }
            }
            if (broken) {  // rows that see such a page become NaN
#pragma unroll
                for (int r = 0; r < NR; r++)
#pragma unroll
                    for (int n = 0; n < NC; n++) {
                        const float2 kv = scales[stage * NC + n];
                        if (!(fabsf(kv.x) < INFINITY && fabsf(kv.y) < INFINITY) && 16 * n < sees[r] - step * L::UNIT) sum[r] = __int_as_float(0x7fc00000);
                    }
            }
            float weight[NR];  // of the step's sums: exp2(largest score of the step - running maximum)
            bool more = false;
            float most[NR];
#pragma unroll
            for (int r = 0; r < NR; r++) {
                float m = -INFINITY;
#pragma unroll
                for (int j = 0; j < KS / 8; j++) m = fmaxf(m, fmaxf(x[r][j][0], x[r][j][1]));
                most[r] = quad_max(m);
                more = more || most[r] > top[r];
            }
            if (__any_sync(0xffffffffu, more)) {
#pragma unroll
                for (int r = 0; r < NR; r++) {
                    const float m = fmaxf(top[r], most[r]), corr = top[r] == -INFINITY ? 0.f : ex2(top[r] - m);
                    top[r] = m;
                    sum[r] *= corr;
                    own.scale(r, corr, c4);
                }
            }
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const float shift = most[r] == -INFINITY ? 0.f : most[r];
                weight[r] = most[r] == -INFINITY ? 0.f : ex2(most[r] - top[r]);
                float part = 0.f;
#pragma unroll
                for (int j = 0; j < KS / 8; j++) {
                    x[r][j][0] = ex2(x[r][j][0] - shift);
                    x[r][j][1] = ex2(x[r][j][1] - shift);
                    part += x[r][j][0] + x[r][j][1];
                }
                sum[r] = fmaf(part, weight[r], sum[r]);
            }
            // ---- values ----
            // Scales of V go into the weights, relative to the step's largest.  Where they differ by more than 2^3, or in sign, a page at a time is taken, under its own.
            const bool even = v_low * 8.f >= v_top && !(v_most > 0.f && v_least < 0.f);
            constexpr float MOST = L::F32 ? 8388607.f : 65535.f;
            const int passes = NC == 1 || even ? 1 : NC;
#pragma unroll 1
            for (int pass = 0; pass < passes; pass++) {
                const float ref = passes == 1 ? (v_most > 0.f ? v_top : -v_top) : scales[stage * NC + pass].y, size = fabsf(ref);
                if (!(size > 0.f && size < INFINITY)) continue;  // nothing but zeros (or NaN, seen to above)
                // v / size for 0 <= v <= size: the reciprocal of a number near the lower end of fp32 would be infinite, of 2^64 times it is not
                const float up = size < 1.f ? 18446744073709551616.f : 1.f, per = 1.f / (size * up);
                uint32_t p[NR][NC][L::DIGITS];
#pragma unroll
                for (int n = 0; n < NC; n++) {
                    // (a page whose scale is not finite: its weights are 0, or the row is NaN already)
                    const float v = fabsf(scales[stage * NC + n].y), k = passes > 1 ? (n == pass ? MOST : 0.f) : v == size ? MOST : v < INFINITY ? v * up * per * MOST : 0.f;
#pragma unroll
                    for (int r = 0; r < NR; r++) {
                        // the lower bits of 2^23 + a number below 2^23 are that number
                        const uint32_t w0 = __float_as_uint(fmaf(x[r][2 * n][0], k, 8388608.f)), w1 = __float_as_uint(fmaf(x[r][2 * n][1], k, 8388608.f));
                        const uint32_t w2 = __float_as_uint(fmaf(x[r][2 * n + 1][0], k, 8388608.f)), w3 = __float_as_uint(fmaf(x[r][2 * n + 1][1], k, 8388608.f));
                        const uint32_t t01 = __byte_perm(w0, w1, 0x5140), t23 = __byte_perm(w2, w3, 0x5140);
                        p[r][n][0] = __byte_perm(t01, t23, 0x5410);
                        p[r][n][1] = __byte_perm(t01, t23, 0x7632);
                        if constexpr (L::F32) p[r][n][2] = bytes_of<2>(w0, w1, w2, w3);
                    }
                }
                float2 f[NR];
#pragma unroll
                for (int r = 0; r < NR; r++) f[r] = Share<D, NR>::of_sums(weight[r] * (L::F32 ? ref : ref * (1.f / MOST)), c4);
                uint32_t v[NC][4][D / 32];
#pragma unroll
                for (int n = 0; n < NC; n++)
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const int token = 2 * c4 + (t & 1) + (t >> 1) * 8;
                        const uint8_t* src = at + L::K_BYTES + n * (16 * D) + unit_at<D>(token, D == 64 ? g / 2 : g) + (D == 64 ? (g & 1) * 8 : 0);
                        if constexpr (D == 64) {
                            const uint2 w = *reinterpret_cast<const uint2*>(src);
                            v[n][t][0] = w.x;
                            v[n][t][1] = w.y;
                        } else {
                            const uint4 w = *reinterpret_cast<const uint4*>(src);
                            v[n][t][0] = w.x;
                            v[n][t][1] = w.y;
                            v[n][t][2] = w.z;
                            v[n][t][3] = w.w;
                        }
                    }
#pragma unroll
                for (int w = 0; w < D / 32; w++) {
                    uint32_t tr[NC][4];  // four tokens of each of the word's four dims
#pragma unroll
                    for (int n = 0; n < NC; n++) {
                        const uint32_t a01 = __byte_perm(v[n][0][w], v[n][1][w], 0x5140), a23 = __byte_perm(v[n][2][w], v[n][3][w], 0x5140);
                        const uint32_t b01 = __byte_perm(v[n][0][w], v[n][1][w], 0x7362), b23 = __byte_perm(v[n][2][w], v[n][3][w], 0x7362);
                        tr[n][0] = __byte_perm(a01, a23, 0x5410);
                        tr[n][1] = __byte_perm(a01, a23, 0x7632);
                        tr[n][2] = __byte_perm(b01, b23, 0x5410);
                        tr[n][3] = __byte_perm(b01, b23, 0x7632);
                    }
#pragma unroll
                    for (int k = 0; k < 2; k++) {
#pragma unroll
                        for (int r = 0; r < NR; r++) {
                            int o[L::DIGITS][4] = {};
#pragma unroll
                            for (int n = 0; n < NC; n += 2)
#pragma unroll
                                for (int t = 0; t < L::DIGITS; t++) mma_u8(o[t], tr[n][2 * k], tr[n][2 * k + 1], tr[n + 1][2 * k], tr[n + 1][2 * k + 1], p[r][n][t], p[r][n + 1][t]);
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                // (fp32: 1 / MOST goes to the digits; the scale of V, down to 2^-126, would keep next to no bits under it.  f16 has no such values.)
                                const float value = L::F32 ? fmaf(static_cast<float>(o[L::DIGITS - 1][e] * 256 + o[1][e]), 256.f / MOST, static_cast<float>(o[0][e]) * (1.f / MOST))
                                                           : static_cast<float>(o[1][e] * 256 + o[0][e]);
                                acc[2 * w + k][r][e] = fmaf(value, e & 1 ? f[r].y : f[r].x, acc[2 * w + k][r][e]);
                            }
                        }
                    }
                }
            }
        }

        Segment now = at_work->get();
        // ---- the four warps' shares: 2 to 0, 3 to 1, 1 to 0 ----
#pragma unroll
        for (int r = 0; r < NR; r++) sum[r] = quad_sum(sum[r]);
        if (warp >= 2) {
            if (handed) {
                if (warp == 2) pair_wait<FREE_0>();
                else pair_wait<FREE_1>();
            }
            own.put(s_hand + (warp - 2) * SLOT, lane);
            if (warp == 2) pair_arrive<HAND_0>();
            else pair_arrive<HAND_1>();
        } else if (warp == 1) {
            pair_wait<HAND_1>();
            own.join_shared(s_hand + SLOT, lane, c4);
            own.put(s_hand + SLOT, lane);  // (each lane where it has just read)
            pair_arrive<HAND_UP>();
        } else {
            pair_wait<HAND_0>();
            own.join_shared(s_hand, lane, c4);
            pair_arrive<FREE_0>();
            pair_wait<HAND_UP>();
            own.join_shared(s_hand + SLOT, lane, c4);
            pair_arrive<FREE_1>();
            if (now.taken == now.units) {
                store(own, now.b, now.h, now.tile);
            } else {
                own.put(partials + (static_cast<int64_t>(blockIdx.x) * 2 + (first ? 0 : 1)) * SLOT, lane);
                __threadfence();
                __syncwarp();
                if (lane == 0) {
                    const Parts p = parts_of(now);
                    const bool last = atomicInc(&counters[p.first], p.count - 1) == p.count - 1;  // back to zero with the last one
                    if (first) last_first = last;
                    else last_second = last;
                }
            }
        }
        handed = true;
        first = false;
        if (now.unit + now.taken == hi) break;
        move_on(now);
        at_work->put(now);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (warp == 2) pair_wait<FREE_0>();  // (no arrival is left open)
    if (warp == 3) pair_wait<FREE_1>();

    // ---- problems that are shared with other CTAs: at most the share's first and last ----
    if (warp == 0 && lane == 0) {
        s_at[0] = last_first;
        s_at[1] = last_second;
    }
    __syncthreads();
    auto finish = [&](const Segment& s) {
        // each warp joins a run of the parts, then the warps as above
        const Parts p = parts_of(s);
        const unsigned p0 = p.count * warp / 4, p1 = p.count * (warp + 1) / 4;
        auto part = [&](unsigned i) { return partials + (static_cast<int64_t>(p.first + i) * 2 + (i == 0 ? p.second : 0)) * SLOT; };
        constexpr int AHEAD = D / 16 * NR <= 8 ? 3 : 1;  // parts on their way at a time
        Share<D, NR> own;
        own.clear();
        for (unsigned i = p0; i < p1; i += AHEAD) {
            Share<D, NR> x[AHEAD];
#pragma unroll
            for (int e = 0; e < AHEAD; e++)
                if (i + e < p1) x[e].get(part(i + e), lane);
#pragma unroll
            for (int e = 0; e < AHEAD; e++)
                if (i + e < p1) own.join(x[e], c4);
        }
        // runs are joined from the front on: 1 to 0, 3 to 2, 2 to 0
        if (warp & 1) own.put(s_hand + (warp >> 1) * SLOT, lane);
        __syncthreads();
        if (!(warp & 1)) own.join_shared(s_hand + (warp >> 1) * SLOT, lane, c4);
        if (warp == 2) own.put(s_hand + SLOT, lane);
        __syncthreads();
        if (warp == 0) {
            own.join_shared(s_hand + SLOT, lane, c4);
            store(own, s.b, s.h, s.tile);
        }
    };
    if (s_at[0] | s_at[1]) {
        __threadfence();
        if (s_at[0]) {
            Segment head;
            head.b = share_b;
            head.seq = share_seq;
            head.unit = lo;
            look(head);
            finish(head);
        }
        __syncthreads();
        if (s_at[1]) finish(at_work->get());
    }
}

}  // namespace paged
}  // namespace rmlk
