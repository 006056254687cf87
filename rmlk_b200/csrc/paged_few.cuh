// Attention of a few query rows per KV head over the paged 8-bit cache: a step of decoding, or of a few drafted tokens.
//
// What bounds it: HBM, each code of the cache read once (a byte per value, against one multiply-add per query row).  So the work is laid out for
// the memory system, and the products go to mma.sync on registers: a tcgen05 tile has 128 rows, of which a step would fill 4 or 8, and wants its operands in
// shared memory as f16, which costs more than the products themselves.
//
// Shares.  The keys of all (sequence, KV head, row tile) problems lie behind one another in units of 4 x KS keys, and the CTAs - as many as are resident
// at once - take equal parts of that line, whatever the lengths of the sequences; the host does not know them.  A CTA writes the result of a problem that is all its
// own, and a partial one (sums, maximum, weights' sum) of a problem that it shares to the workspace; the CTA that finishes last adds them up in their order
// along the keys, so the result does not depend on which one that is.
//
// A warp's step: KS keys (32 of 64 values, 16 of 128).  Each lane copies by cp.async just the bytes that it will read itself, three steps deep; no
// lane waits for another.  The order of a contraction is free, so a lane's 16 consecutive bytes of a key are its operands of four MMAs (four dims to each), and
// bytes become f16 in registers: 0x6400 | (b ^ 0x80) is 1152 + b.
//   scores  S[16 rows x 8 keys]  = Q K^T: fp32 queries as pairs of f16, the high parts in rows 0-7, the low parts (2^11 times their size) in rows 8-15; f16 queries: 16 rows
//   values  O[16 rows x 8 dims] += P V over 16 keys: the accumulator fragment of S is the operand fragment of P as it is.
// Codes are exact in f16.  Each 16 keys' O is formed from zero and added to fp32 sums times their page's scale of V: that keeps any ratio of scales, and
// keeps the MMA's truncating accumulator short.  Weights are 2^14 exp2(s - max): as pairs for fp32, as f16 for f16 results (2^-11 of a weight, as much as the result's own rounding).
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

template <typename T, int D>
struct Few {
    static constexpr bool PAIRS = sizeof(T) == 4;
    static constexpr int ROWS = PAIRS ? 8 : 16;  // query rows of a tile
    static constexpr int NR = ROWS / 8;          // of them a lane's
    static constexpr int KS = 2048 / D;          // keys of a warp's step
    static constexpr int NC = KS / 16;           // groups of 16 keys: one page each
    static constexpr int UNIT = 4 * KS;
    static constexpr int STAGES = 3;
    static constexpr int STEP = 4096;            // bytes of a step: keys, then values
    static constexpr int RING = 4 * STAGES * STEP;
    static constexpr int MERGE = 4 * ROWS * D * 4;  // the warps' sums, in the place of the ring
    static constexpr int BODY = RING > MERGE ? RING : MERGE;
    static constexpr int SMEM = BODY + 4 * STAGES * NC * 8 + 4 * ROWS * 8 + 64;
    static constexpr int PER_SM = 3;
};
constexpr int SLOT_ROWS = 16;
inline size_t few_workspace(int64_t d) { return COUNTERS * 4 + static_cast<size_t>(sm_count()) * 4 * 2 * SLOT_ROWS * (d + 2) * 4; }

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
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
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
// a share of a softmax under another maximum: a share without keys has the maximum -inf and sums of zero (or NaN, which has to stay)
__device__ __forceinline__ float share_weight(float m, float most) { return m == -INFINITY ? 1.f : ex2(m - most); }

template <typename T, int D>
__global__ void __launch_bounds__(128, Few<T, D>::PER_SM) few_kernel(const Cache c, const Batch q, const Attend a, const int tiles, unsigned* counters, float* partials) {
    using L = Few<T, D>;
    constexpr int ROWS = L::ROWS, NR = L::NR, KS = L::KS, NC = L::NC, PIECES = D / 64;
    dep_sync();
    extern __shared__ __align__(16) uint8_t smem[];
    float2* s_scales = reinterpret_cast<float2*>(smem + L::BODY);                  // [warp][stage][NC] scales of K and V
    float* s_top = reinterpret_cast<float*>(smem + L::BODY + 4 * L::STAGES * NC * 8);  // [warp][ROWS]
    float* s_sum = s_top + 4 * ROWS;
    int64_t* s_at = reinterpret_cast<int64_t*>(smem + L::SMEM - 64);  // scan, then where the share begins
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c4 = lane & 3;
    const int64_t table_keys = q.width << c.page_log;
    // keys behind the table have no page: one of them stands for all
    auto keys_of = [&](int b) { return min(static_cast<int64_t>(q.lens[b]), table_keys + 1); };
    auto units_of = [&](int b) { return max((keys_of(b) + L::UNIT - 1) / L::UNIT, int64_t(1)); };  // (a sequence without keys has rows to write all the same)
    const int64_t items = static_cast<int64_t>(c.kv_heads) * tiles;  // problems of a sequence

    // ---- this CTA's share of the line ----
    int64_t total, lo, hi, seq_first;  // seq_first: where sequence b begins on the line
    int b;
    unsigned workers;
    {
        const int per = (q.batch + 127) / 128, b0 = min(tid * per, q.batch), b1 = min(b0 + per, q.batch);
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
        workers = static_cast<unsigned>(min(static_cast<int64_t>(gridDim.x), total));
        if (blockIdx.x >= workers) return;
        lo = total * blockIdx.x / workers;
        hi = total * (blockIdx.x + 1) / workers;
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
        b = static_cast<int>(s_at[0]);
        seq_first = s_at[1];
    }
    auto worker_of = [&](int64_t unit) { return static_cast<unsigned>(((unit + 1) * workers - 1) / total); };

    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * (L::STAGES * L::STEP);
    const uint8_t* ring_ptr = smem + warp * (L::STAGES * L::STEP);
    float2* scales = s_scales + warp * (L::STAGES * NC);
    const int rows = q.each * a.group;

    for (int64_t unit = lo; unit < hi;) {
        const int64_t keys = keys_of(b), units = units_of(b);
        const int64_t item = (unit - seq_first) / units, unit0 = (unit - seq_first) - item * units;
        const int64_t taken = min(units - unit0, hi - unit);
        const int h = static_cast<int>(item / tiles), tile = static_cast<int>(item - static_cast<int64_t>(h) * tiles);
        const int64_t key0 = unit0 * L::UNIT, key1 = min(keys, (unit0 + taken) * L::UNIT);
        const int64_t before = static_cast<int64_t>(q.lens[b]) - q.each;  // keys before the first new token

        // ---- queries: fragments of the scores' MMAs, and what each lane's rows see ----
        uint32_t qf[4 * PIECES][4];
        float factor[NR];
        int64_t sees[NR];
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const int row = tile * ROWS + g + 8 * r, token = row / a.group;
            const bool in = row < rows;
            sees[r] = in ? min(before + token + 1, keys) : 0;
            const T* src = static_cast<const T*>(a.q) + (static_cast<int64_t>(b) * q.each + token) * a.qs + (static_cast<int64_t>(h) * a.group + row - token * a.group) * D + 16 * c4;
            if constexpr (L::PAIRS) {
                float4 x[4 * PIECES];
                uint32_t most = 0;
#pragma unroll
                for (int s = 0; s < 4 * PIECES; s++) {
                    x[s] = in ? *reinterpret_cast<const float4*>(src + (s >> 2) * 64 + (s & 3) * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
                    most = max(max(most, max(finite_abs_bits(x[s].x), finite_abs_bits(x[s].y))), max(finite_abs_bits(x[s].z), finite_abs_bits(x[s].w)));
                }
                most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
                const int e = scale_exponent(most);
                const float up = exp2_int(e);
                factor[r] = a.scale * 1.44269504f * exp2_int(-e);
#pragma unroll
                for (int s = 0; s < 4 * PIECES; s++) {
                    split2(x[s].x * up, x[s].y * up, qf[s][0], qf[s][1]);
                    split2(x[s].z * up, x[s].w * up, qf[s][2], qf[s][3]);
                }
            } else {
                factor[r] = a.scale * 1.44269504f;
#pragma unroll
                for (int s = 0; s < 4 * PIECES; s++) {
                    const uint2 x = in ? *reinterpret_cast<const uint2*>(src + (s >> 2) * 64 + (s & 3) * 4) : make_uint2(0u, 0u);
                    qf[s][r] = x.x;
                    qf[s][2 + r] = x.y;
                }
            }
        }
        const int64_t all_see = max(min(before + 1 + (tile * ROWS) / a.group, keys), int64_t(0));  // keys that every row of the tile sees

        // ---- the warp's steps: keys key0 + (4 i + warp) KS ----
        const int64_t first_key = key0 + warp * KS;
        const int steps = first_key < key1 ? static_cast<int>((key1 - first_key + L::UNIT - 1) / L::UNIT) : 0;
        int page = 0;
        float2 page_scales = make_float2(0.f, 0.f);
        // pages of 32 / NC steps at a time, one per lane
        auto fetch_pages = [&](int step) {
            const int i = step + lane / NC;
            const int64_t key = first_key + static_cast<int64_t>(i) * L::UNIT + (lane % NC) * 16;
            page = 0;
            page_scales = make_float2(0.f, 0.f);
            if (i < steps && key < key1) {
                const int64_t at = key >> c.page_log;
                const int p = at < q.width ? q.table[static_cast<int64_t>(b) * q.width + at] : -1;
                if (p >= 0 && p < c.pages) {
                    page = p;
                    const int64_t block = static_cast<int64_t>(p) * c.kv_heads + h;
                    page_scales = make_float2(c.ks[block], c.vs[block]);
                } else {  // what sees it becomes NaN; page 0 is read in its place
                    page_scales = make_float2(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
                    if (a.status) *a.status = RMLK_ERR_INVALID_ARG;
                }
            }
        };
        auto issue = [&](int step) {
            if (step < steps) {
                if (step % (32 / NC) == 0) fetch_pages(step);
                const int stage = step % L::STAGES, from = (step % (32 / NC)) * NC;
                const uint32_t dst = ring + stage * L::STEP;
                const int64_t key = first_key + static_cast<int64_t>(step) * L::UNIT;
#pragma unroll
                for (int n = 0; n < NC; n++) {
                    const int64_t p = __shfl_sync(0xffffffffu, page, from + n);
                    const int64_t off = ((p * c.kv_heads + h) * c.page + ((key + 16 * n) & (c.page - 1))) * D;
                    const int8_t* ks = c.k + off + g * D + c4 * 16;
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int i = 0; i < PIECES; i++) copy_async<16>(dst + ((2 * n + j) * PIECES + i) * 512 + lane * 16, ks + j * 8 * D + i * 64);
                    const int8_t* vs = c.v + off + 2 * c4 * D + g * (D / 8);
#pragma unroll
                    for (int t = 0; t < 4; t++)
                        copy_async<D / 8>(dst + 2048 + (4 * n + t) * (4 * D) + lane * (D / 8), vs + ((t & 1) + (t >> 1) * 8) * D);
                }
                if (lane >= from && lane < from + NC) scales[stage * NC + lane - from] = page_scales;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };

        float acc[D / 8][2 * NR], top[NR], sum[NR];
#pragma unroll
        for (int i = 0; i < D / 8; i++)
#pragma unroll
            for (int r = 0; r < 2 * NR; r++) acc[i][r] = 0.f;
#pragma unroll
        for (int r = 0; r < NR; r++) {
            top[r] = -INFINITY;
            sum[r] = 0.f;
        }
#pragma unroll
        for (int s = 0; s < L::STAGES - 1; s++) issue(s);
        for (int step = 0; step < steps; step++) {
            __syncwarp();  // the slot that is filled next has been read, its scales too
            issue(step + L::STAGES - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(L::STAGES - 1) : "memory");
            __syncwarp();  // (scales come from other lanes)
            const int stage = step % L::STAGES;
            const uint8_t* at = ring_ptr + stage * L::STEP;
            const int64_t key = first_key + static_cast<int64_t>(step) * L::UNIT;
            // ---- scores ----
            float x[NR][KS / 8][2];
            float most[NR];
#pragma unroll
            for (int r = 0; r < NR; r++) most[r] = top[r];
#pragma unroll
            for (int j = 0; j < KS / 8; j++) {
                float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < PIECES; i++) {
                    const uint4 w = *reinterpret_cast<const uint4*>(at + (j * PIECES + i) * 512 + lane * 16);
                    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t f = word[k] ^ 0x80808080u;
                        const uint32_t(&qa)[4] = qf[4 * i + k];
                        mma_16816(s, qa[0], qa[1], qa[2], qa[3], two_f16(f, 0x4140), two_f16(f, 0x4342));
                    }
                }
                const float ks = scales[stage * NC + j / 2].x;
                if constexpr (L::PAIRS) {
                    const float t = factor[0] * ks;
                    x[0][j][0] = fmaf(s[2], 1.f / SPLIT_LO, s[0]) * t;
                    x[0][j][1] = fmaf(s[3], 1.f / SPLIT_LO, s[1]) * t;
                } else {
#pragma unroll
                    for (int r = 0; r < NR; r++) {
                        const float t = factor[r] * ks;
                        x[r][j][0] = s[2 * r] * t;
                        x[r][j][1] = s[2 * r + 1] * t;
                    }
                }
            }
            float vs[NR][NC];
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int r = 0; r < NR; r++) vs[r][n] = scales[stage * NC + n].y;
            if (key + KS > all_see) {
#pragma unroll
                for (int r = 0; r < NR; r++) {
                    const int see = static_cast<int>(max(min(sees[r] - key, static_cast<int64_t>(KS)), int64_t(0)));
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
#pragma unroll
                    for (int i = 0; i < D / 8; i++) {
                        acc[i][2 * r] *= corr;
                        acc[i][2 * r + 1] *= corr;
                    }
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
#pragma unroll
            for (int n = 0; n < NC; n++) {
                uint32_t p[4];
                if constexpr (L::PAIRS) {
                    split2(x[0][2 * n][0], x[0][2 * n][1], p[0], p[1]);
                    split2(x[0][2 * n + 1][0], x[0][2 * n + 1][1], p[2], p[3]);
                } else {
#pragma unroll
                    for (int r = 0; r < NR; r++) {
                        p[r] = pack_f16(x[r][2 * n][0], x[r][2 * n][1]);
                        p[2 + r] = pack_f16(x[r][2 * n + 1][0], x[r][2 * n + 1][1]);
                    }
                }
                uint32_t v[4][D / 32];
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const uint8_t* src = at + 2048 + (4 * n + t) * (4 * D) + lane * (D / 8);
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
                for (int w = 0; w < D / 32; w++) {
                    // tokens 2 c4, 2 c4 + 1 (and 8 further on) side by side, for each of four dims
                    const uint32_t l01 = __byte_perm(v[0][w], v[1][w], 0x5140), l23 = __byte_perm(v[0][w], v[1][w], 0x7362);
                    const uint32_t h01 = __byte_perm(v[2][w], v[3][w], 0x5140), h23 = __byte_perm(v[2][w], v[3][w], 0x7362);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        float o[4] = {0.f, 0.f, 0.f, 0.f};
                        const uint32_t sel = k & 1 ? 0x4342 : 0x4140;
                        mma_16816(o, p[0], p[1], p[2], p[3], two_f16(k < 2 ? l01 : l23, sel), two_f16(k < 2 ? h01 : h23, sel));
                        float(&d)[2 * NR] = acc[4 * w + k];
                        if constexpr (L::PAIRS) {
                            d[0] = fmaf(fmaf(o[2], 1.f / SPLIT_LO, o[0]), vs[0][n], d[0]);
                            d[1] = fmaf(fmaf(o[3], 1.f / SPLIT_LO, o[1]), vs[0][n], d[1]);
                        } else {
#pragma unroll
                            for (int r = 0; r < NR; r++) {
                                d[2 * r] = fmaf(o[2 * r], vs[r][n], d[2 * r]);
                                d[2 * r + 1] = fmaf(o[2 * r + 1], vs[r][n], d[2 * r + 1]);
                            }
                        }
                    }
                }
            }
        }

        // ---- the four warps' shares ----
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        float* merge = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int r = 0; r < NR; r++) {
            sum[r] = quad_sum(sum[r]);
            const int row = g + 8 * r;
            if (c4 == 0) {
                s_top[warp * ROWS + row] = top[r];
                s_sum[warp * ROWS + row] = sum[r];
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float4* dst = reinterpret_cast<float4*>(merge + (warp * ROWS + row) * D + (2 * c4 + e) * (D / 8));
#pragma unroll
                for (int i = 0; i < D / 32; i++)
                    dst[i] = make_float4(acc[4 * i][2 * r + e], acc[4 * i + 1][2 * r + e], acc[4 * i + 2][2 * r + e], acc[4 * i + 3][2 * r + e]);
            }
        }
        __syncthreads();
        const int64_t item_first = seq_first + item * units;
        const bool whole = taken == units;
        float* slot = partials + (static_cast<int64_t>(blockIdx.x) * 2 + (unit == lo ? 0 : 1)) * (SLOT_ROWS * (D + 2));
        auto put = [&](int row, int col, float4 o, float l) {
            const int at_row = tile * ROWS + row, token = at_row / a.group;
            if (at_row >= rows) return;
            const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing is 0
            T* dst = static_cast<T*>(a.out) + (static_cast<int64_t>(b) * q.each + token) * a.os + (static_cast<int64_t>(h) * a.group + at_row - token * a.group) * D + col;
            if constexpr (L::PAIRS) *reinterpret_cast<float4*>(dst) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
            else *reinterpret_cast<uint2*>(dst) = make_uint2(pack_f16(o.x * inv, o.y * inv), pack_f16(o.z * inv, o.w * inv));
        };
        for (int e = tid; e < ROWS * D / 4; e += 128) {
            const int row = e / (D / 4), col = e % (D / 4) * 4;
            float m = s_top[row], l = 0.f;
#pragma unroll
            for (int w = 1; w < 4; w++) m = fmaxf(m, s_top[w * ROWS + row]);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float f = share_weight(s_top[w * ROWS + row], m);
                const float4 x = *reinterpret_cast<const float4*>(merge + (w * ROWS + row) * D + col);
                l = fmaf(f, s_sum[w * ROWS + row], l);
                o = make_float4(fmaf(f, x.x, o.x), fmaf(f, x.y, o.y), fmaf(f, x.z, o.z), fmaf(f, x.w, o.w));
            }
            if (whole) {
                put(row, col, o, l);
            } else {
                *reinterpret_cast<float4*>(slot + row * D + col) = o;
                if (col == 0) {
                    slot[SLOT_ROWS * D + row] = m;
                    slot[SLOT_ROWS * (D + 1) + row] = l;
                }
            }
        }
        if (!whole) {
            const unsigned w0 = worker_of(item_first), w1 = worker_of(item_first + units - 1);
            __threadfence();
            __syncthreads();
            if (tid == 0) s_at[2] = atomicInc(&counters[w0], w1 - w0) == w1 - w0;  // back to zero with the last one
            __syncthreads();
            if (s_at[2]) {
                __threadfence();
                for (int e = tid; e < ROWS * D / 4; e += 128) {
                    const int row = e / (D / 4), col = e % (D / 4) * 4;
                    auto part = [&](unsigned w) {  // the first one's may be its second piece of the line
                        const bool second = w == w0 && total * w / workers != item_first;
                        return partials + (static_cast<int64_t>(w) * 2 + (second ? 1 : 0)) * (SLOT_ROWS * (D + 2));
                    };
                    float m = -INFINITY, l = 0.f;
                    for (unsigned w = w0; w <= w1; w++) m = fmaxf(m, __ldcg(part(w) + SLOT_ROWS * D + row));
                    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (unsigned w = w0; w <= w1; w++) {
                        const float* p = part(w);
                        const float f = share_weight(__ldcg(p + SLOT_ROWS * D + row), m);
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(p + row * D + col));
                        l = fmaf(f, __ldcg(p + SLOT_ROWS * (D + 1) + row), l);
                        o = make_float4(fmaf(f, x.x, o.x), fmaf(f, x.y, o.y), fmaf(f, x.z, o.z), fmaf(f, x.w, o.w));
                    }
                    put(row, col, o, l);
                }
            }
        }
        __syncthreads();  // the ring and the flags are free again
        unit += taken;
        if (unit - seq_first == units * items && unit < hi) {
            seq_first = unit;
            b++;
        }
    }
}

}  // namespace paged
}  // namespace rmlk
