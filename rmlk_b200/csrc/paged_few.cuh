// Attention of a few query rows per KV head over the paged 8-bit cache: a step of decoding, or of a few drafted tokens.
//
// What bounds it: HBM, each code of the cache read once (a byte per value, against one multiply-add per query row).  So the work is laid out for
// the memory system, and the products go to mma.sync on registers: a tcgen05 tile has 128 rows, of which a step would fill 4 or 8, and wants its operands in
// shared memory as f16, which costs more than the products themselves.
//
// Shares.  The keys of all (sequence, KV head, row tile) problems lie behind one another in units of 4 x 32 keys, and the CTAs - as many as are resident
// at once - take equal parts of that line, whatever the lengths of the sequences; the host does not know them.  A CTA's piece of a problem is a segment.  A warp
// asks for the keys of its next segment while it still works on the one before, so the stream of loads does not stop between them; a segment's four shares are joined
// warp to warp, and a warp that has handed its own on goes on.  (With the whole CTA waiting at each end, 64 requests over 1000 keys took 24 us.)
// A problem that several CTAs share leaves partial results (sums, maximum, weights' sum) in the workspace; the CTA that comes last adds them up in their
// order along the keys, so the result does not depend on which one that is.
//
// A warp's step: 32 keys.  Each lane copies by cp.async just the bytes that it will read itself; no lane waits for another.  The order of a contraction is
// free, so a lane's 16 consecutive bytes of a key are its operands of four MMAs (four dims to each), and bytes become f16 in registers:
// 0x6400 | (b ^ 0x80) is 1152 + b.
//   scores  S[16 rows x 8 keys]     = Q K^T: fp32 queries as pairs of f16, the high parts in rows 0-7, the low parts (2^11 times their size) in rows 8-15; f16
//                                     queries: 8 or 16 rows
//   values  O^T[16 dims x 8 rows] += V^T P^T over 16 keys: the accumulator fragment of S is the operand fragment of P^T as it is; two tokens' bytes side by side are V^T's
// Codes are exact in f16.  For fp32 results a step's O is formed from zero and added to fp32 sums, which keeps the MMA's truncating accumulator short; for f16 the
// accumulators stay in the MMAs.  Weights are 2^14 exp2(s - max): as pairs for fp32, as f16 for f16 results (2^-11 of a weight, as much as the result's own rounding).
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
    static constexpr bool PAIRS = sizeof(T) == 4;
    static constexpr int NR = NR_;               // groups of 8 query rows in a tile
    static constexpr int ROWS = 8 * NR;
    static constexpr int KS = 32, NC = KS / 16;  // keys of a warp's step; groups of 16 of them: one page each
    static constexpr int UNIT = 4 * KS;
    static constexpr int STAGES = D == 64 ? 3 : 2;
    static constexpr int K_BYTES = KS * D, STEP = 2 * K_BYTES;
    static constexpr int RING = 4 * STAGES * STEP;
    static constexpr int FRAGS = D / 16 * NR;    // groups of four sums per lane
    static constexpr int HAND = 32 * (FRAGS * 16 + NR * 8);  // a warp's share on its way to another: sums, maxima, weights' sums
    static constexpr int SCALES = RING + 2 * HAND, SCAN = SCALES + 4 * STAGES * NC * 8, SMEM = SCAN + 64;
    static constexpr int PER_SM = NR == 2 && D == 128 ? 2 : 3;
    static_assert(!PAIRS || NR == 1, "the low parts take rows 8-15");
};
constexpr int MOST_PARTS = 32;  // CTAs for a problem, on average: each costs the last one a fraction of a microsecond
inline size_t few_workspace(int64_t d) { return COUNTERS * 4 + static_cast<size_t>(sm_count()) * 4 * 2 * (32 * (d / 16 * 2 * 16 + 2 * 8)); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
// two bytes (of four that have 0x80 flipped) as f16: 1024 + u - 1152
__device__ __forceinline__ uint32_t two_f16(uint32_t flipped, uint32_t selector) {
    const uint32_t biased = __byte_perm(flipped, 0x64646464u, selector);
    const uint32_t offset = 0x64806480u;
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&biased), *reinterpret_cast<const __half2*>(&offset));
    return *reinterpret_cast<const uint32_t*>(&v);
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
// a / b for 0 <= a, 0 < b: nearly always in 32 bits, where a division is a fifth of the instructions
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
    return ((a | b) >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
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
        s.left = static_cast<int>(min(max(left, int64_t(0)), int64_t(0x7fffff00)));  // (2^31 keys are none of a cache's)
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
    Segment ask;
    ask.b = share_b;
    ask.seq = share_seq;
    ask.unit = lo;
    look(ask);
    Segment now = ask;
    int block = -1;  // page and head as one index; -1: no key there, -2: a key without a page
    constexpr int PAGED_STEPS = 32 / NC;  // pages of so many steps are looked up at a time, one per lane
    const int8_t* k_lane = c.k + g * D + c4 * 16;
    const int8_t* v_lane = c.v + 2 * c4 * D + g * (D / 8);
    const int block_bytes = c.page * D;
    int fill = 0, fill_stage = 0;  // next step to be asked for, its place in the ring
    auto issue = [&]() {
        while (fill == ask.steps && ask.unit < hi) {
            move_on(ask);
            fill = 0;
            if (ask.unit >= hi) ask.steps = 0;
        }
        if (fill < ask.steps) {
            const int in_batch = fill % PAGED_STEPS;
            if (in_batch == 0) {
                const int off = (fill + lane / NC) * L::UNIT + (lane % NC) * 16;
                block = -1;
                if (off < ask.left) {
                    const int64_t at = (ask.first_key + off) >> c.page_log;
                    const int p = at < q.width ? q.table[static_cast<int64_t>(ask.b) * q.width + at] : -1;
                    block = p >= 0 && p < c.pages ? p * c.kv_heads + ask.h : -2;
                    if (block == -2 && a.status) *a.status = RMLK_ERR_INVALID_ARG;
                }
            }
            const uint32_t dst = ring + fill_stage * L::STEP;
#pragma unroll
            for (int n = 0; n < NC; n++) {
                const int at = __shfl_sync(0xffffffffu, block, in_batch * NC + n), from = at < 0 ? ask.h : at;  // (page 0 is read where there is none)
                if (lane < 2) {  // the scales of K and V: 0 where there is no key, NaN where a key has no page
                    float* to = reinterpret_cast<float*>(scales + fill_stage * NC + n) + lane;
                    if (at >= 0) copy_async<4>(static_cast<uint32_t>(__cvta_generic_to_shared(to)), (lane ? c.vs : c.ks) + at);
                    else *to = at == -1 ? 0.f : __int_as_float(0x7fc00000);
                }
                const int64_t off = static_cast<int64_t>(from) * block_bytes + ((static_cast<int>(ask.first_key & 127) + fill * L::UNIT + 16 * n) & (c.page - 1)) * D;
                const int8_t* ks = k_lane + off;
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int i = 0; i < PIECES; i++) copy_async<16>(dst + ((2 * n + j) * PIECES + i) * 512 + lane * 16, ks + j * 8 * D + i * 64);
                const int8_t* vs = v_lane + off;
#pragma unroll
                for (int t = 0; t < 4; t++) copy_async<D / 8>(dst + L::K_BYTES + (4 * n + t) * (4 * D) + lane * (D / 8), vs + ((t & 1) + (t >> 1) * 8) * D);
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
                    if constexpr (L::PAIRS) *reinterpret_cast<float4*>(dst + 2 * i) = o;
                    else *reinterpret_cast<uint2*>(dst + 2 * i) = make_uint2(pack_f16(o.x, o.y), pack_f16(o.z, o.w));
                }
            }
        }
    };
    int stage = 0;
    bool first = true, handed = false;  // first segment of the CTA; the hand-over places have been used

    while (now.unit < hi) {
        const int b = now.b, h = now.h, tile = now.tile;
        const int64_t keys = keys_of(b), first_key = now.first_key;
        const int64_t before = static_cast<int64_t>(q.lens[b]) - q.each;  // keys before the first new token

        // ---- queries: fragments of the scores' MMAs, and what each lane's rows see.  (Asked for first, looked at when the first keys are on their way.) ----
        auto relative = [&](int64_t key) { return static_cast<int>(max(min(key - first_key, int64_t(0x7fffff00)), int64_t(0))); };
        constexpr int QF = L::PAIRS ? 4 : 2 * NR;  // registers of a fragment: rows g (high, low), or g and g + 8
        uint32_t qf[4 * PIECES][QF];
        float4 qx[L::PAIRS ? 4 * PIECES : 1];
        float factor[NR];
        int sees[NR];  // keys from the warp's first on that the lane's rows see
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const int row = tile * ROWS + g + 8 * r, token = row / a.group;
            const bool in = row < rows;
            sees[r] = in ? relative(min(before + token + 1, keys)) : 0;
            factor[r] = a.scale * 1.44269504f;
            const T* src = static_cast<const T*>(a.q) + (static_cast<int64_t>(b) * q.each + token) * a.qs + (static_cast<int64_t>(h) * a.group + row - token * a.group) * D + 16 * c4;
#pragma unroll
            for (int s = 0; s < 4 * PIECES; s++) {
                const T* at = src + (s >> 2) * 64 + (s & 3) * 4;
                if constexpr (L::PAIRS) {
                    qx[s] = in ? *reinterpret_cast<const float4*>(at) : make_float4(0.f, 0.f, 0.f, 0.f);
                } else {
                    const uint2 x = in ? *reinterpret_cast<const uint2*>(at) : make_uint2(0u, 0u);
                    qf[s][r] = x.x;
                    qf[s][NR + r] = x.y;
                }
            }
        }
        if (first) {
#pragma unroll
            for (int s = 0; s < L::STAGES - 1; s++) issue();
        }
        if constexpr (L::PAIRS) {
            uint32_t most = 0;
#pragma unroll
            for (int s = 0; s < 4 * PIECES; s++)
                most = max(max(most, max(finite_abs_bits(qx[s].x), finite_abs_bits(qx[s].y))), max(finite_abs_bits(qx[s].z), finite_abs_bits(qx[s].w)));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const int e = scale_exponent(most);
            const float up = exp2_int(e);
            factor[0] *= exp2_int(-e);
#pragma unroll
            for (int s = 0; s < 4 * PIECES; s++) {
                split2(qx[s].x * up, qx[s].y * up, qf[s][0], qf[s][1]);
                split2(qx[s].z * up, qx[s].w * up, qf[s][2], qf[s][3]);
            }
        }
        const int all_see = relative(min(before + 1 + (tile * ROWS) / a.group, keys));  // that every row of the tile sees

        Share<D, NR> own;
        own.clear();
        float(&acc)[D / 16][NR][4] = own.acc;
        float(&top)[NR] = own.top;
        float(&sum)[NR] = own.sum;
        float v_ref = 0.f, v_inv = 0.f, v_top = 0.f;  // the scale of V that the weights are relative to, its reciprocal, the largest so far
        for (int step = 0; step < now.steps; step++, stage = stage + 1 == L::STAGES ? 0 : stage + 1) {
            __syncwarp();  // the slot that is filled next has been read, its scales too
            issue();
            asm volatile("cp.async.wait_group %0;" ::"n"(L::STAGES - 1) : "memory");
            __syncwarp();  // (scales come from other lanes)
            const uint8_t* at = ring_ptr + stage * L::STEP;
            // ---- scores ----
            float s[KS / 8][4];
#pragma unroll
            for (int j = 0; j < KS / 8; j++) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
            for (int i = 0; i < PIECES; i++) {
#pragma unroll
                for (int j = 0; j < KS / 8; j++) {
                    const uint4 w = *reinterpret_cast<const uint4*>(at + (j * PIECES + i) * 512 + lane * 16);
                    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t f = word[k] ^ 0x80808080u;
                        const uint32_t(&qa)[QF] = qf[4 * i + k];
                        mma_16816(s[j], qa[0], QF == 4 ? qa[1] : 0u, QF == 4 ? qa[2] : qa[1], QF == 4 ? qa[3] : 0u, two_f16(f, 0x4140), two_f16(f, 0x4342));
                    }
                }
            }
            float x[NR][KS / 8][2];
            float most[NR];
#pragma unroll
            for (int r = 0; r < NR; r++) most[r] = top[r];
#pragma unroll
            for (int j = 0; j < KS / 8; j++) {
                const float ks = scales[stage * NC + j / 2].x;
                if constexpr (L::PAIRS) {
                    const float t = factor[0] * ks;
                    x[0][j][0] = fmaf(s[j][2], 1.f / SPLIT_LO, s[j][0]) * t;
                    x[0][j][1] = fmaf(s[j][3], 1.f / SPLIT_LO, s[j][1]) * t;
                } else {
#pragma unroll
                    for (int r = 0; r < NR; r++) {
                        const float t = factor[r] * ks;
                        x[r][j][0] = s[j][2 * r] * t;
                        x[r][j][1] = s[j][2 * r + 1] * t;
                    }
                }
            }
            float vs[NR][NC];  // scales of V as the lane's rows see them
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int r = 0; r < NR; r++) vs[r][n] = scales[stage * NC + n].y;
            if (KS + step * L::UNIT > all_see) {
#pragma unroll
                for (int r = 0; r < NR; r++) {
                    const int see = sees[r] - step * L::UNIT;
#pragma unroll
                    for (int j = 0; j < KS / 8; j++) {
                        if (8 * j + 2 * c4 >= see) x[r][j][0] = -INFINITY;
                        if (8 * j + 2 * c4 + 1 >= see) x[r][j][1] = -INFINITY;
                    }
#pragma unroll
                    for (int n = 0; n < NC; n++)
                        if (16 * n >= see) vs[r][n] = 0.f;  // (a NaN there is no part of the row)
                }
            }
            bool more = false;
#pragma unroll
            for (int r = 0; r < NR; r++) {
#pragma unroll
                for (int j = 0; j < KS / 8; j++) most[r] = fmaxf(most[r], fmaxf(x[r][j][0], x[r][j][1]));
                most[r] = quad_max(most[r]);
                more = more || most[r] > top[r];
            }
            if (__any_sync(0xffffffffu, more)) {
#pragma unroll
                for (int r = 0; r < NR; r++) {
                    const float corr = top[r] == -INFINITY ? 0.f : ex2(top[r] - most[r]);
                    top[r] = most[r];
                    sum[r] *= corr;
                    own.scale(r, corr, c4);
                }
            }
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const float shift = (top[r] == -INFINITY ? 0.f : top[r]) - 14.f;
#pragma unroll
                for (int j = 0; j < KS / 8; j++) {
                    x[r][j][0] = ex2(x[r][j][0] - shift);
                    x[r][j][1] = ex2(x[r][j][1] - shift);
                    sum[r] += x[r][j][0] + x[r][j][1];
                }
            }
            // ---- values ----
            // Scales of V go into the weights, relative to the one that the accumulators are in: that of the 16 keys before, as long as the ratio is
            // between 2 (weights stay in f16's range) and 2^-12.  (Infinities and NaN go into the weights as they are.)
            float fresh[L::PAIRS ? D / 16 : 1][4];
#pragma unroll
            for (int n = 0; n < NC; n++) {
                const float scale = scales[stage * NC + n].y, ref = scale < INFINITY ? fmaxf(scale, 1.17549435e-38f) : 1.f;
                if constexpr (L::PAIRS) {
                    const bool other = n > 0 && (ref > 2.f * v_ref || ref < v_ref * 2.44140625e-4f);
                    if (other) {
#pragma unroll
                        for (int i = 0; i < D / 16; i++)
#pragma unroll
                            for (int e = 0; e < 4; e++) acc[i][0][e] = fmaf(fresh[i][e], v_ref, acc[i][0][e]);
                    }
                    if (n == 0 || other) {
#pragma unroll
                        for (int i = 0; i < D / 16; i++) fresh[i][0] = fresh[i][1] = fresh[i][2] = fresh[i][3] = 0.f;
                        v_ref = ref;
                        v_inv = 1.f / ref;
                    }
                } else if (scale < INFINITY && (ref > 2.f * v_ref || (ref < v_ref * 2.44140625e-4f && ref > v_top * 5.42101086e-20f))) {  // (2^-64: further down sums might leave fp32's range)
                    const float f = v_ref / ref;
#pragma unroll
                    for (int i = 0; i < D / 16; i++)
#pragma unroll
                        for (int r = 0; r < 4 * NR; r++) acc[i][r >> 2][r & 3] *= f;
                    v_ref = ref;
                    v_inv = 1.f / ref;
                    v_top = fmaxf(v_top, ref);
                }
                uint32_t p[2][2];  // rows 0-7 and 8-15, or the high and low parts: tokens 2 c4, 2 c4 + 1 and 8 further on
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    if constexpr (L::PAIRS) {
                        const float w = vs[0][n] * v_inv, y0 = x[0][2 * n + e][0] * w, y1 = x[0][2 * n + e][1] * w;
                        const __half2 high = __floats2half2_rn(y0, y1);
                        const float2 back = __half22float2(high);
                        p[0][e] = *reinterpret_cast<const uint32_t*>(&high);
                        p[1][e] = pack_f16(y0 - back.x, y1 - back.y);
                    } else {
#pragma unroll
                        for (int r = 0; r < NR; r++) {
                            const float w = vs[r][n] * v_inv;
                            p[r][e] = pack_f16(x[r][2 * n + e][0] * w, x[r][2 * n + e][1] * w);
                        }
                    }
                }
                uint32_t v[4][D / 32];
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const uint8_t* src = at + L::K_BYTES + (4 * n + t) * (4 * D) + lane * (D / 8);
                    if constexpr (D == 64) {
                        const uint2 w = *reinterpret_cast<const uint2*>(src);
                        v[t][0] = w.x ^ 0x80808080u;
                        v[t][1] = w.y ^ 0x80808080u;
                    } else {
                        const uint4 w = *reinterpret_cast<const uint4*>(src);
                        v[t][0] = w.x ^ 0x80808080u;
                        v[t][1] = w.y ^ 0x80808080u;
                        v[t][2] = w.z ^ 0x80808080u;
                        v[t][3] = w.w ^ 0x80808080u;
                    }
                }
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    // two tokens side by side, of dims 2 i and 2 i + 1 of the lane's
                    const uint32_t near = __byte_perm(v[0][i / 2], v[1][i / 2], i & 1 ? 0x7362 : 0x5140), far = __byte_perm(v[2][i / 2], v[3][i / 2], i & 1 ? 0x7362 : 0x5140);
                    const uint32_t a0 = two_f16(near, 0x4140), a1 = two_f16(near, 0x4342), a2 = two_f16(far, 0x4140), a3 = two_f16(far, 0x4342);
                    if constexpr (L::PAIRS) {
                        mma_16816(fresh[i], a0, a1, a2, a3, p[1][0], p[1][1]);
                        mma_16816(fresh[i], a0, a1, a2, a3, p[0][0], p[0][1]);
                    } else {
#pragma unroll
                        for (int r = 0; r < NR; r++) mma_16816(acc[i][r], a0, a1, a2, a3, p[r][0], p[r][1]);
                    }
                }
            }
            if constexpr (L::PAIRS) {
#pragma unroll
                for (int i = 0; i < D / 16; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][0][e] = fmaf(fresh[i][e], v_ref, acc[i][0][e]);
            }
        }

        // ---- the four warps' shares: 2 to 0, 3 to 1, 1 to 0 ----
#pragma unroll
        for (int r = 0; r < NR; r++) {
            sum[r] = quad_sum(sum[r]);
            if constexpr (!L::PAIRS) {
#pragma unroll
                for (int i = 0; i < D / 16; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][r][e] *= v_ref;
            }
        }
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
            if (now.taken == now.units) store(own, b, h, tile);
            else own.put(partials + (static_cast<int64_t>(blockIdx.x) * 2 + (first ? 0 : 1)) * SLOT, lane);
        }
        handed = true;
        first = false;
        if (now.unit + now.taken == hi) break;
        move_on(now);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (warp == 2) pair_wait<FREE_0>();  // (no arrival is left open)
    if (warp == 3) pair_wait<FREE_1>();

    // ---- problems that are shared with other CTAs: at most the share's first and last ----
    // first: begun before the share; last: goes on behind it (one and the same, where the share lies within a problem)
    auto finish = [&](const Segment& s) {
        const int64_t begin = s.seq + divide(s.unit - s.seq, s.units) * s.units;
        const unsigned w0 = worker_of(begin), w1 = worker_of(begin + s.units - 1), parts = w1 - w0 + 1;
        __syncthreads();
        if (tid == 0) {
            __threadfence();
            s_at[0] = atomicInc(&counters[w0], w1 - w0) == w1 - w0;  // back to zero with the last one
            __threadfence();
        }
        __syncthreads();
        if (!s_at[0]) return;
        // each warp joins a run of the parts, then the warps as above
        const int64_t second = begin_of(w0) != begin;  // the first CTA's may be its second piece of the line
        const unsigned p0 = parts * warp / 4, p1 = parts * (warp + 1) / 4;
        Share<D, NR> own;
        own.clear();
        for (unsigned p = p0; p < p1; p++) {
            Share<D, NR> x;
            x.get(partials + (static_cast<int64_t>(w0 + p) * 2 + (p == 0 ? second : 0)) * SLOT, lane);
            own.join(x, c4);
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
    Segment head;
    head.b = share_b;
    head.seq = share_seq;
    head.unit = lo;
    look(head);
    const bool head_shared = head.taken != head.units, tail_shared = now.unit != lo && now.taken != now.units;
    if (head_shared) finish(head);
    if (tail_shared) finish(now);
}

}  // namespace paged
}  // namespace rmlk
