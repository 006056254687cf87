// Attention of many query rows per KV head over the paged 8-bit cache: prompts, parts of them behind a cached beginning.
//
// A CTA keeps TILES x 128 query rows of one KV head (the rows of the query heads that share it lie behind one another) and walks over the keys that they see in blocks
// of 64.  Both contractions run on tcgen05.mma kind::f16: codes are exact in f16, f16 queries too; fp32 queries and, for fp32 results, weights are two f16 numbers each (the
// second the rounding error of the first), whose products go to the same accumulator.
//   warps 0-3, 4-7   softmax of a tile, one thread to a row: scores out of TMEM, weights into shared memory
//   warps 8-11       codes of K and V from the pages into f16 tiles, two blocks ahead
//   warp 12          one thread issues the MMAs: scores of block j + 1 before the values of block j, so that a softmax never waits for its scores.  (Its instructions are few on
//                    purpose: with 64-bit descriptors and a barrier more for each thing it was the bound, 4700 cycles per block.)
// What bounds it: the exponentials (16 per clock and SM; the products of a block take as long at 128 values per head, half as long at 64) and, around them, the
// softmax warps' issue slots.
// The output sums stay in TMEM.  They are brought under a new maximum only when a row's has grown by more than 2^8 (weights are up to 2^14 then), which after the first
// blocks hardly happens.  For fp32 results they are added to fp32 sums every four blocks: the accumulator truncates, and 256 keys are what its error allows.
// Scales of K go into the scores' factor, scales of V into the weights, relative to the largest that the rows see.  Where scales of V span more than 2^10, or
// something is not finite or has no page, the rows are taken one by one in fp32 (row_in_fp32): slow, and right for everything.
#pragma once

#include "paged.cuh"
#include "paged_few.cuh"
#include "umma_gemm.cuh"

namespace rmlk {
namespace paged {

using umma::fence_proxy_async;
using umma::mbar_arrive;
using umma::mbar_init;
using umma::mbar_wait;
using umma::smem_u32;
using umma::tc_fence_after;
using umma::tc_fence_before;
using umma::tmem_ld_x32;

__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
        "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename T, int D_>
struct Prompt {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int D = D_, HALVES = D / 64;        // tiles of 64 dims: 128-byte rows of f16
    static constexpr int TILES = F32 && D == 128 ? 1 : 2;  // (fp32 results: sums twice, in TMEM)
    static constexpr int PARTS = F32 ? 2 : 1;            // f16 numbers of a query or weight
    static constexpr int KT = 64;                        // keys of a block
    static constexpr int STAGES = 3;
    static constexpr int THREADS = 128 * TILES + 128 + 32;
    static constexpr uint32_t Q_TILE = 128 * 128 * HALVES, P_TILE = 128 * 128, KV_TILE = KT * 128 * HALVES;
    static constexpr uint32_t Q = 0, P = Q + TILES * PARTS * Q_TILE, STAGE = 2 * KV_TILE, KV = P + TILES * PARTS * P_TILE, EXTRA = KV + STAGES * STAGE;  // a stage: K, then V
    static constexpr uint32_t ROW_SCALE = EXTRA, RED = ROW_SCALE + TILES * 512, BARS = RED + 128, TOTAL = BARS + 256 + 1024;
    static constexpr uint32_t O_AT = 256, O_PITCH = 128, KEPT = D == 64 ? 64 : 128;  // TMEM columns: scores [tile][2][64], sums, (fp32) kept sums behind them
    static constexpr int FLUSH = 4;                      // (fp32) blocks per accumulation
    static_assert(TOTAL <= 227 * 1024, "shared memory budget exceeded");
};

// One query row by one warp, a key after the other, in fp32: any scales, NaN for what is not finite and for a key without a page.
template <typename T, int D>
__device__ __noinline__ void row_in_fp32(const Cache& c, const Batch& q, const Attend& a, int b, int64_t row, int h, int64_t sees) {
    const int lane = threadIdx.x & 31, kv = h / a.group;
    constexpr int N = D / 32;
    float x[N], acc[N];
    const T* src = static_cast<const T*>(a.q) + row * a.qs + static_cast<int64_t>(h) * D;
#pragma unroll
    for (int i = 0; i < N; i++) {
        x[i] = static_cast<float>(src[lane + 32 * i]);
        acc[i] = 0.f;
    }
    float top = -INFINITY, sum = 0.f;
    for (int64_t t = 0; t < sees; t++) {
        const int64_t at = t >> c.page_log;
        const int page = at < q.width ? q.table[b * q.width + at] : -1;
        if (page < 0 || page >= c.pages) {
            if (a.status) *a.status = RMLK_ERR_INVALID_ARG;
            sum = __int_as_float(0x7fc00000);
            break;
        }
        const int64_t block = static_cast<int64_t>(page) * c.kv_heads + kv, off = (block * c.page + (t & (c.page - 1))) * D;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) s = fmaf(x[i], static_cast<float>(c.k[off + lane + 32 * i]), s);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= c.ks[block] * (a.scale * 1.44269504f);
        const float v_scale = c.vs[block];
        if (!(s - s == 0.f) || !(fabsf(v_scale) < INFINITY)) sum = __int_as_float(0x7fc00000);
        const float most = fmaxf(top, s), corr = top == -INFINITY ? 0.f : ex2(top - most), e = ex2(s - most);
        top = most;
        sum = fmaf(sum, corr, e);
        const float w = e * v_scale;
#pragma unroll
        for (int i = 0; i < N; i++) acc[i] = fmaf(w, static_cast<float>(c.v[off + lane + 32 * i]), acc[i] * corr);
    }
    T* o = static_cast<T*>(a.out) + row * a.os + static_cast<int64_t>(h) * D;
#pragma unroll
    for (int i = 0; i < N; i++) o[lane + 32 * i] = static_cast<T>(sees <= 0 ? 0.f : acc[i] / sum);
}

// two fp32 operations by one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// D[tmem] (+)= A x B, kind::f16, issued by one thread: the descriptors' lower halves (their addresses) vary, their upper halves are the same for all tiles here.
template <bool ADD>
__device__ __forceinline__ void mma_at(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
    constexpr uint32_t upper = (1024 >> 4) | (1u << 14) | (2u << 29);  // 1 KB between groups of 8 rows, version 1, 128-byte swizzle
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %4};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(upper), "n"(ADD ? 1 : 0)
        : "memory");
}

// 16-byte unit u of row r in a tile of 128-byte rows, 128-byte swizzle
__device__ __forceinline__ uint32_t swizzled(int r, int u) { return static_cast<uint32_t>(r * 128 + ((u ^ (r & 7)) << 4)); }

// eight codes as f16: 0x6400 | (b ^ 0x80) is 1152 + b
__device__ __forceinline__ uint4 eight_f16(uint32_t w0, uint32_t w1) {
    auto two = [](uint32_t flipped, uint32_t selector) {
        const uint32_t biased = __byte_perm(flipped, 0x64646464u, selector), offset = 0x64806480u;
        const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&biased), *reinterpret_cast<const __half2*>(&offset));
        return *reinterpret_cast<const uint32_t*>(&v);
    };
    w0 ^= 0x80808080u;
    w1 ^= 0x80808080u;
    return make_uint4(two(w0, 0x4140), two(w0, 0x4342), two(w1, 0x4140), two(w1, 0x4342));
}

template <typename T, int D>
__global__ void __launch_bounds__(Prompt<T, D>::THREADS, 1) prompt_kernel(const Cache c, const Batch q, const Attend a) {
    using L = Prompt<T, D>;
    constexpr int TILES = L::TILES, HALVES = L::HALVES, PARTS = L::PARTS, KT = L::KT, ROWS = TILES * 128;
    dep_sync();
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* sm = smem_raw + (base - smem_u32(smem_raw));
    float* s_row = reinterpret_cast<float*>(sm + L::ROW_SCALE);
    volatile uint32_t* s_red = reinterpret_cast<volatile uint32_t*>(sm + L::RED);
    const uint32_t bars = base + L::BARS;
    // barriers: keys and values of a stage in place and done with, scores in TMEM, weights in place and done with.  (A place for scores is free again when the
    // weights made of them are there: nobody waits for that apart.)
    auto kv_full = [&](int i) { return bars + 8u * i; };
    auto kv_free = [&](int i) { return bars + 8u * (4 + i); };
    auto s_full = [&](int t, int i) { return bars + 8u * (8 + 2 * t + i); };
    auto p_full = [&](int t) { return bars + 8u * (12 + t); };
    auto p_free = [&](int t) { return bars + 8u * (14 + t); };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + L::BARS + 8 * 16);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + L::BARS + 8 * 16 + 8);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // ---- which rows: sequence by sequence, the tiles that see most first ----
    int b = 0, item = blockIdx.x;
    int64_t first = 0, count = 0;
    if (!q.starts) {
        const int per = (q.each * a.group + ROWS - 1) / ROWS;
        b = item / per;
        item = per - 1 - (item - b * per);
        q.rows(b, first, count);
    } else {
        // a warp looks at 32 sequences at a time (every warp for itself: the same answer)
        bool found = false;
        for (int b0 = 0; b0 < q.batch && !found; b0 += 32) {
            int64_t f = 0, n = 0;
            if (b0 + lane < q.batch) q.rows(b0 + lane, f, n);
            const int own = static_cast<int>((n * a.group + ROWS - 1) / ROWS);
            int upto = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            const uint32_t mask = __ballot_sync(0xffffffffu, item < upto);
            if (mask) {
                const int l = __ffs(mask) - 1;
                b = b0 + l;
                first = __shfl_sync(0xffffffffu, f, l);
                count = __shfl_sync(0xffffffffu, n, l);
                item = __shfl_sync(0xffffffffu, upto, l) - 1 - item;
                found = true;
            } else {
                item -= __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        if (!found) return;
    }
    const int h = blockIdx.y, rows = static_cast<int>(min(count * a.group - static_cast<int64_t>(item) * ROWS, static_cast<int64_t>(ROWS)));  // valid rows from row0 on
    const int64_t row0 = static_cast<int64_t>(item) * ROWS;
    const int64_t table_keys = q.width << c.page_log;
    const int64_t len = q.lens[b], keys = min(len, table_keys + 1), before = len - count;
    // rows of the sequence and head are counted from its first new token on (fewer than 2^31: tokens x 64)
    auto token_of = [&](int64_t row) { return ((row | a.group) >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(row) / static_cast<uint32_t>(a.group)) : row / a.group; };
    auto sees_of = [&](int64_t row) { return min(before + token_of(row) + 1, keys); };
    const int64_t seen = max(sees_of(row0 + rows - 1), int64_t(0));                     // keys that the last row sees

    // ---- the pages that they see: all there, scales finite and not below zero, those of V of one size? ----
    float v_top = 0.f, v_low = INFINITY;
    bool plain = true;
    const int64_t pages = (seen + c.page - 1) >> c.page_log;
    for (int64_t i = tid; i < pages; i += L::THREADS) {
        const int p = i < q.width ? q.table[static_cast<int64_t>(b) * q.width + i] : -1;
        if (p < 0 || p >= c.pages) {
            plain = false;
        } else {
            const int64_t block = static_cast<int64_t>(p) * c.kv_heads + h;
            const float k = c.ks[block], v = c.vs[block];
            plain = plain && k >= 0.f && k < INFINITY && v >= 0.f && v < INFINITY;
            v_top = fmaxf(v_top, v);
            if (v > 7.52316385e-37f) v_low = fminf(v_low, v);  // 2^-120: a block of zeros has the scale 2^-126
        }
    }
    {
        const uint32_t t = __reduce_max_sync(0xffffffffu, __float_as_uint(v_top)), l = __reduce_min_sync(0xffffffffu, __float_as_uint(v_low));
        if (lane == 0) {
            s_red[2 * warp] = t;
            s_red[2 * warp + 1] = l;
        }
        if (tid == 0) {
            for (int i = 0; i < L::STAGES; i++) {
                mbar_init(kv_full(i), 128);
                mbar_init(kv_free(i), 1);
            }
            for (int i = 0; i < 2; i++) {
                mbar_init(s_full(0, i), 1);
                mbar_init(s_full(1, i), 1);
                mbar_init(p_full(i), 128);
                mbar_init(p_free(i), 1);
            }
            *abort_flag = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        plain = __syncthreads_and(plain);
        uint32_t top = 0, low = 0x7f800000u;
        for (int w = 0; w < L::THREADS / 32; w++) {
            top = max(top, s_red[2 * w]);
            low = min(low, s_red[2 * w + 1]);
        }
        v_top = __uint_as_float(top);
        v_low = __uint_as_float(low);
    }
    if (!plain || !(v_low * 1024.f >= v_top) || seen == 0) {
        for (int r = warp; r < rows; r += L::THREADS / 32) {
            const int64_t row = row0 + r;
            const int64_t token = token_of(row);
            row_in_fp32<T, D>(c, q, a, b, first + token, h * a.group + static_cast<int>(row - token * a.group), sees_of(row));
        }
        return;
    }
    if (v_top == 0.f) v_top = 1.f;

    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // blocks of each tile (the second one sees at least as much as the first), and whether it has rows
    const int tiles = rows > 128 ? 2 : 1;
    auto blocks_of = [&](int t) { return static_cast<int>((max(sees_of(row0 + min(rows, 128 * (t + 1)) - 1), int64_t(0)) + KT - 1) / KT); };
    const int blocks0 = blocks_of(0), blocks = tiles == 2 ? blocks_of(1) : blocks0;
    const bool negative = a.scale < 0.f;  // scores' factors are not below zero: the sign goes to the queries

    // ---- queries ----
    if (warp < 4 * TILES) {
        const int t = warp >> 2;
        constexpr int PER = D / 4, AT_ONCE = 32 / PER, BATCH = 8;  // lanes to a row (four values each), rows of a warp at a time, loads on their way
        using Four = typename std::conditional<L::F32, float4, uint2>::type;
        const int c4 = lane % PER;
#pragma unroll 1
        for (int r0 = (warp & 3) * AT_ONCE + lane / PER; r0 < 128; r0 += 4 * AT_ONCE * BATCH) {
            Four raw[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                const int at = t * 128 + r0 + i * 4 * AT_ONCE;
                raw[i] = Four{};
                if (at < rows) {
                    const int64_t row = row0 + at, token = token_of(row);
                    raw[i] = *reinterpret_cast<const Four*>(static_cast<const T*>(a.q) + (first + token) * a.qs + (static_cast<int64_t>(h) * a.group + row - token * a.group) * D + 4 * c4);
                }
            }
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                const int r = r0 + i * 4 * AT_ONCE;
                uint8_t* tile = sm + L::Q + (t * PARTS) * L::Q_TILE + (c4 >> 4) * (128 * 128);
                const uint32_t to = swizzled(r, (c4 & 15) >> 1) + (c4 & 1) * 8;
                if constexpr (L::F32) {
                    float4 x = raw[i];
                    uint32_t most = max(max(finite_abs_bits(x.x), finite_abs_bits(x.y)), max(finite_abs_bits(x.z), finite_abs_bits(x.w)));
#pragma unroll
                    for (int o = PER / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                    const int e = scale_exponent(most);
                    const float up = negative ? -exp2_int(e) : exp2_int(e);
                    if (c4 == 0) s_row[t * 128 + r] = exp2_int(-e);
                    x = make_float4(x.x * up, x.y * up, x.z * up, x.w * up);
                    const __half2 h0 = __floats2half2_rn(x.x, x.y), h1 = __floats2half2_rn(x.z, x.w);
                    const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
                    *reinterpret_cast<uint2*>(tile + to) = make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
                    *reinterpret_cast<uint2*>(tile + L::Q_TILE + to) = make_uint2(pack_f16(x.x - f0.x, x.y - f0.y), pack_f16(x.z - f1.x, x.w - f1.y));
                } else {
                    uint2 x = raw[i];
                    if (negative) x = make_uint2(x.x ^ 0x80008000u, x.y ^ 0x80008000u);
                    *reinterpret_cast<uint2*>(tile + to) = x;
                }
            }
        }
        fence_proxy_async();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    int* status = a.status;

    if (warp < 4 * TILES) {
        // ---------------- softmax ----------------
        const int t = warp >> 2, r = tid & 127, at = t * 128 + r;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + t * 128, o_at = tmem + lanes + L::O_AT + t * L::O_PITCH;
        const int own_blocks = t < tiles ? (t == 0 ? blocks0 : blocks) : 0;
        const int64_t sees = at < rows ? sees_of(row0 + at) : 0;
        // blocks that every row of the tile sees whole
        const int64_t least = t < tiles ? sees_of(row0 + t * 128) : 0;
        const float q_scale = fabsf(a.scale) * 1.44269504f * (L::F32 ? s_row[at] : 1.f);
        const float v_inv = 1.f / v_top;
        float top = -INFINITY, sum = 0.f;
        uint32_t s_phase = 0, p_phase = 0;
        bool ok = true, fresh = true;  // fresh: nothing kept yet (fp32)
        int in_run = 0;                // (fp32) blocks since the sums were last added up
        // scales of 16 keys each: lanes 0-3 look up pages two blocks ahead, scales one
        int page_next = 0;
        float ks_next = 0.f, vs_next = 0.f;
        auto page_of = [&](int j) {
            const int64_t key = static_cast<int64_t>(j) * KT + (lane & 3) * 16;
            page_next = -1;
            if (lane < 4 && key < seen) page_next = q.table[static_cast<int64_t>(b) * q.width + (key >> c.page_log)];
        };
        auto scales_of = [&]() {
            ks_next = vs_next = 0.f;
            if (page_next >= 0) {
                const int64_t block = static_cast<int64_t>(page_next) * c.kv_heads + h;
                ks_next = c.ks[block];
                vs_next = c.vs[block];
            }
        };
        if (own_blocks > 0) {
            page_of(0);
            scales_of();
            page_of(1);
        }
        for (int j = 0; j < own_blocks; j++) {
            float f[4], v[4];
#pragma unroll
            for (int n = 0; n < 4; n++) {
                f[n] = fmaxf(__shfl_sync(0xffffffffu, ks_next, n) * q_scale, 1e-38f);  // (not zero: hidden scores stay -inf)
                v[n] = __shfl_sync(0xffffffffu, vs_next, n) * v_inv;
            }
            scales_of();
            page_of(j + 2);
            const int buf = j & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(s_full(t, buf), s_phase, abort_flag, status));
            if (!ok) break;
            tc_fence_after();
            float s[KT];
            tmem_ld_x32(s_at + buf * 64, *reinterpret_cast<uint32_t(*)[32]>(s));
            tmem_ld_x32(s_at + buf * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
            tmem_wait_ld();
            if (buf) s_phase ^= 1;
            if (static_cast<int64_t>(j + 1) * KT > least) {
                const int see = static_cast<int>(max(min(sees - static_cast<int64_t>(j) * KT, static_cast<int64_t>(KT)), int64_t(0)));
#pragma unroll
                for (int i = 0; i < KT; i++)
                    if (i >= see) s[i] = -INFINITY;
            }
            float most = -INFINITY;
#pragma unroll
            for (int n = 0; n < 4; n++) {
                float m = s[16 * n];
#pragma unroll
                for (int i = 1; i < 16; i++) m = fmaxf(m, s[16 * n + i]);
                most = fmaxf(most, m * f[n]);
            }
            // The maximum that the sums are under moves when it has fallen behind by more than 2^8.
            const bool move = most > top + 8.f || (top == -INFINITY && most > top);
            const float new_top = move ? most : top;
            const float corr = top == -INFINITY ? 0.f : ex2(top - new_top);
            const bool any = __any_sync(0xffffffffu, move && j > 0);
            top = new_top;
            sum *= move ? corr : 1.f;
            const float shift = (top == -INFINITY ? 0.f : top) - 6.f;  // weights are 2^6 exp2(s - top)
            float2 part[2] = {};
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const float2 f2 = make_float2(f[n], f[n]), shift2 = make_float2(-shift, -shift);
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    float2 x = fma2(make_float2(s[16 * n + i], s[16 * n + i + 1]), f2, shift2);
                    x.x = ex2(x.x);
                    x.y = ex2(x.y);
                    part[(i >> 1) & 1] = add2(part[(i >> 1) & 1], x);
                    s[16 * n + i] = x.x;
                    s[16 * n + i + 1] = x.y;
                }
            }
            part[0] = add2(part[0], part[1]);
            sum += part[0].x + part[0].y;
#pragma unroll
            for (int n = 0; n < 4; n++) {
                if (v[n] != 1.f) {
                    const float2 v2 = make_float2(v[n], v[n]);
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float2 x = mul2(make_float2(s[16 * n + i], s[16 * n + i + 1]), v2);
                        s[16 * n + i] = x.x;
                        s[16 * n + i + 1] = x.y;
                    }
                }
            }
            // the values of the block before have been added: their weights' place is free, and the sums can be touched
            if (j > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(p_free(t), p_phase, abort_flag, status));
                if (!ok) break;
                p_phase ^= 1;
                tc_fence_after();
                if constexpr (L::F32) {
                    in_run++;
                    if (any || in_run == L::FLUSH) {
                        const float k = move ? corr : 1.f;
#pragma unroll 1
                        for (int i = 0; i < D; i += 32) {
                            uint32_t o[32], m[32];
                            tmem_ld_x32(o_at + i, o);
                            tmem_ld_x32(o_at + L::KEPT + i, m);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; e++) {
                                m[e] = __float_as_uint((__uint_as_float(o[e]) + (fresh ? 0.f : __uint_as_float(m[e]))) * k);
                                o[e] = 0;
                            }
                            tmem_st_x32(o_at + L::KEPT + i, m);
                            tmem_st_x32(o_at + i, o);
                        }
                        tmem_wait_st();
                        fresh = false;
                        in_run = 0;
                    }
                } else if (any) {
                    const float k = move ? corr : 1.f;
#pragma unroll 1
                    for (int i = 0; i < D; i += 32) {
                        uint32_t o[32];
                        tmem_ld_x32(o_at + i, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * k);
                        tmem_st_x32(o_at + i, o);
                    }
                    tmem_wait_st();
                }
            }
            uint8_t* p = sm + L::P + t * PARTS * L::P_TILE;
#pragma unroll
            for (int u = 0; u < 8; u++) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float y0 = s[8 * u + 2 * e], y1 = s[8 * u + 2 * e + 1];
                    const __half2 w = __floats2half2_rn(y0, y1);
                    hi[e] = *reinterpret_cast<const uint32_t*>(&w);
                    if constexpr (L::F32) {
                        const float2 back = __half22float2(w);
                        lo[e] = pack_f16(y0 - back.x, y1 - back.y);
                    }
                }
                *reinterpret_cast<uint4*>(p + swizzled(r, u)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if constexpr (L::F32) *reinterpret_cast<uint4*>(p + L::P_TILE + swizzled(r, u)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            fence_proxy_async();
            tc_fence_before();
            mbar_arrive(p_full(t));
        }
        // ---- results ----
        if (own_blocks > 0 && ok) ok = __all_sync(0xffffffffu, mbar_wait(p_free(t), p_phase, abort_flag, status));
        tc_fence_after();
        if (at < rows || own_blocks > 0) {
            const float inv = 1.f / sum * v_top;
            const int64_t row = row0 + at, token = token_of(row);
            T* dst = static_cast<T*>(a.out) + (first + token) * a.os + (static_cast<int64_t>(h) * a.group + row - token * a.group) * D;
#pragma unroll 1
            for (int i = 0; i < D; i += 32) {
                uint32_t o[32];
                if (own_blocks > 0) {
                    tmem_ld_x32(o_at + i, o);
                    if constexpr (L::F32) {
                        uint32_t m[32];
                        tmem_ld_x32(o_at + L::KEPT + i, m);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) + (fresh ? 0.f : __uint_as_float(m[e])));
                    } else {
                        tmem_wait_ld();
                    }
                }
                if (at < rows) {
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = __float_as_uint(!ok ? __int_as_float(0x7fc00000) : sees <= 0 ? 0.f : __uint_as_float(o[e]) * inv);
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        if constexpr (L::F32) {
                            *reinterpret_cast<uint4*>(dst + i + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                            *reinterpret_cast<uint4*>(dst + i + e + 4) = make_uint4(o[e + 4], o[e + 5], o[e + 6], o[e + 7]);
                        } else {
                            *reinterpret_cast<uint4*>(dst + i + e) =
                                make_uint4(pack_f16(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), pack_f16(__uint_as_float(o[e + 2]), __uint_as_float(o[e + 3])),
                                           pack_f16(__uint_as_float(o[e + 4]), __uint_as_float(o[e + 5])), pack_f16(__uint_as_float(o[e + 6]), __uint_as_float(o[e + 7])));
                        }
                    }
                }
            }
        }
        tc_fence_before();
    } else if (warp < 4 * TILES + 4) {
        // ---------------- codes to f16 tiles ----------------
        constexpr int PIECES = D / 16, N = KT * PIECES / 128;  // 16-byte pieces of a key; of a block's, a thread's: key first_key + i STEP, always the same piece
        constexpr int STEP = 128 / PIECES;
        const int me = tid - 128 * TILES, own_key = me / PIECES, piece = me % PIECES;
        const int64_t head = static_cast<int64_t>(h) * c.page * D + piece * 16, page_bytes = static_cast<int64_t>(c.kv_heads) * c.page * D;
        const uint32_t tile_at = (piece >> 2) * (KT * 128);
        // Pages are looked up three blocks ahead, codes asked for two ahead.
        int page[N];
        uint4 kx[2][N], vx[2][N];
        auto look_up = [&](int j) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int64_t key = static_cast<int64_t>(j) * KT + own_key + i * STEP;
                page[i] = key < seen ? q.table[static_cast<int64_t>(b) * q.width + (key >> c.page_log)] : -1;
            }
        };
        auto load = [&](int j, uint4 (&kr)[N], uint4 (&vr)[N]) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                kr[i] = vr[i] = make_uint4(0u, 0u, 0u, 0u);  // (keys that no row sees)
                if (page[i] >= 0) {
                    const int slot = (static_cast<int>(j * KT) + own_key + i * STEP) & (c.page - 1);
                    const int64_t off = static_cast<int64_t>(page[i]) * page_bytes + head + slot * D;
                    kr[i] = *reinterpret_cast<const uint4*>(c.k + off);
                    vr[i] = *reinterpret_cast<const uint4*>(c.v + off);
                }
            }
        };
        auto put = [&](uint32_t tile, const uint4 (&x)[N]) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int r = own_key + i * STEP, u = 2 * (piece & 3);
                *reinterpret_cast<uint4*>(sm + tile + tile_at + swizzled(r, u)) = eight_f16(x[i].x, x[i].y);
                *reinterpret_cast<uint4*>(sm + tile + tile_at + swizzled(r, u + 1)) = eight_f16(x[i].z, x[i].w);
            }
        };
        bool ok = true;
        int stage = 0;
        uint32_t phase = 1;  // (the first pass over the stages goes through)
        auto put_block = [&](const uint4 (&kr)[N], const uint4 (&vr)[N]) {
            ok = mbar_wait(kv_free(stage), phase, abort_flag, status);
            if (!ok) return;
            put(L::KV + stage * L::STAGE, kr);
            put(L::KV + stage * L::STAGE + L::KV_TILE, vr);
            fence_proxy_async();
            mbar_arrive(kv_full(stage));
            if (++stage == L::STAGES) {
                stage = 0;
                phase ^= 1;
            }
        };
        look_up(0);
        load(0, kx[0], vx[0]);
        look_up(1);
        load(1, kx[1], vx[1]);
        look_up(2);
        for (int j = 0; j < blocks && ok; j += 2) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                if (j + e < blocks && ok) {
                    put_block(kx[e], vx[e]);
                    load(j + e + 2, kx[e], vx[e]);
                    look_up(j + e + 3);
                }
            }
        }
    } else if (lane == 0) {
        // ---------------- MMAs ----------------
        constexpr uint32_t qk = (1u << 4) | ((KT >> 3) << 17) | ((128 >> 4) << 24), pv = (1u << 4) | (1u << 16) | ((D >> 3) << 17) | ((128 >> 4) << 24);  // (values: keys along the rows)
        // lower halves of the operands' descriptors: address / 16, and for the values 8 KB between blocks of 64 dims
        const uint32_t q_at = (base + L::Q) >> 4 | 1u << 16, k_at = (base + L::KV) >> 4 | 1u << 16, p_at = (base + L::P) >> 4 | 1u << 16,
                       v_at = (base + L::KV + L::KV_TILE) >> 4 | (8192u >> 4) << 16;
        bool ok = true;
        int ask = 0, use = 0;  // stages of the next scores and values
        uint32_t ask_phase = 0;
        auto block_scores = [&](int j) {
            ok = ok && mbar_wait(kv_full(ask), ask_phase, abort_flag, status);
            if (!ok) return;
            tc_fence_after();
            const uint32_t kd = k_at + ask * (L::STAGE >> 4), d = tmem + (j & 1) * 64;
#pragma unroll
            for (int t = 0; t < TILES; t++) {
                if (t == 0 ? j < blocks0 : tiles == 2) {
#pragma unroll
                    for (int part = PARTS - 1; part >= 0; part--)  // the small products first
#pragma unroll
                        for (int half = 0; half < HALVES; half++)
#pragma unroll
                            for (int kk = 0; kk < 4; kk++) {
                                const uint32_t qa = q_at + (((t * PARTS + part) * L::Q_TILE + half * (128 * 128)) >> 4) + kk * 2, kb = kd + ((half * (KT * 128)) >> 4) + kk * 2;
                                if (part < PARTS - 1 || half > 0 || kk > 0) mma_at<true>(d + t * 128, qa, kb, qk);
                                else mma_at<false>(d + t * 128, qa, kb, qk);
                            }
                    umma::commit<1>(s_full(t, j & 1));
                }
            }
            if (++ask == L::STAGES) {
                ask = 0;
                ask_phase ^= 1;
            }
        };
        block_scores(0);
        for (int j = 0; j < blocks && ok; j++) {
            if (j + 1 < blocks) block_scores(j + 1);
            const uint32_t vd = v_at + use * (L::STAGE >> 4);
#pragma unroll
            for (int t = 0; t < TILES; t++) {
                if (t == 0 ? j < blocks0 : tiles == 2) {
                    ok = ok && mbar_wait(p_full(t), j & 1, abort_flag, status);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int part = PARTS - 1; part >= 0; part--)
#pragma unroll
                        for (int kk = 0; kk < 4; kk++) {
                            const uint32_t d = tmem + L::O_AT + t * L::O_PITCH, pa = p_at + (((t * PARTS + part) * L::P_TILE) >> 4) + kk * 2, vb = vd + kk * 128;
                            if (part < PARTS - 1 || kk > 0 || j > 0) mma_at<true>(d, pa, vb, pv);
                            else mma_at<false>(d, pa, vb, pv);
                        }
                    umma::commit<1>(p_free(t));
                }
            }
            if (ok) umma::commit<1>(kv_free(use));
            if (++use == L::STAGES) use = 0;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

}  // namespace paged
}  // namespace rmlk
