// Attention of many query rows per KV head over the paged 8-bit cache: prompts, parts of them behind a cached beginning.
//
// A CTA keeps two tiles (fp32 with 128 values: one) of 128 query rows of one KV head - the rows of the query heads that share it lie behind one another - and walks over the
// keys that they see in blocks of 64.  Both contractions run on tcgen05.mma kind::f16: codes are exact in f16, f16 queries too; fp32 queries and, for fp32 results, weights are two
// f16 numbers each (the second the rounding error of the first), whose products go to the same accumulator.  For f16 results a weight is one f16 number, off by at most 2^-11 of itself,
// while the weights' sum is that of the fp32 ones: the result is off by some 2e-4 before it is rounded, as much as that rounding does; second numbers would add half as many MMAs again.
//   warps 0-3, 4-7   softmax of a tile, one thread to a row: scores out of TMEM, weights back into TMEM in their place, where the values' MMAs take them as their first operand
//   warps 8-11       codes of K and V from the pages into f16 tiles, three of each: the codes are turned once for both tiles
//   warps 12, 13     one thread of each issues the MMAs of the scores, up to two blocks ahead of the softmax, and those of the values
// Where there are fewer such CTAs than SMs, a cluster of 2, 4 or 8 shares the keys: each leaves its sums in its shared memory, in the place of its operands, and joins some of the rows
// over distributed shared memory.
// What was tried, f16, 4 prompts of up to 1024 tokens, 32 heads of 128, behind up to 5000 keys: one thread for all MMAs and the weights through shared memory 445 us (the thread needs some 70
// cycles per MMA: it was the bound); two CTAs of one tile per SM, blocks of 128 keys with the scores behind the values 433 us (half of a CTA's time is MMAs, during which its softmax
// waits), blocks of 64 with the scores ahead 442 us (the codes are turned twice: half of all instructions); as it is 336 us, 0.70 PFLOP/s.
// What bounds it there: instructions (49 % of all issue slots: a score is scaled, compared, exponentiated and packed, a code turned) beside the tensor pipe (36 % of its cycles), which
// wait for one another at the ends of a block.
// 16 prompts of up to 512 tokens, fp32, 32 heads of 64: 90 us.  A CTA has 4 blocks on average, so starting (queries turned into f16 pairs) and storing are half of it; with the pages
// looked at before the queries, not beside them, 95 us.
// The output sums stay in TMEM.  They are brought under a new maximum only when a row's has grown by more than 2^8 (weights are up to 2^14 then), which after the first
// blocks hardly happens.  The accumulator truncates, up to 2^-23 of a sum with every 16 keys (values of one sign over 200000 keys came out 1.4e-3 too small), so they are added to
// fp32 sums every 256 keys for fp32 results, every 4096 for f16.  Those are in TMEM too, where two f16 tiles of 128 values leave no room: up to 16384 keys of a CTA they do without,
// 1.0e-4 of a sum; over more, scores have one place instead of two, and the sums of one half of the values go to the other, those of the other half to shared memory.  4 prompts of 1024
// tokens, 32 heads of 128: over 16000 keys 1.39 ms, over 20000 2.16, where sums that are cut off took 1.71.
// Scales of K go into the scores' factor, scales of V into the weights, relative to the largest that the rows see.  Where scales of V span more than 2^10, some
// are below zero, or something is not finite or has no page, the rows are taken one by one in fp32 (row_in_fp32): right for everything, and
// hundreds of times slower (0.36 us per key and row of 64 values, a row to each of the CTA's warps).  So are, at the end and by themselves, fp32 rows whose values differ in size by so
// much that two f16 numbers lose what the scores need (rows_again).
#pragma once

#include "paged.cuh"
#include "paged_few.cuh"
#include "umma_gemm.cuh"

namespace rmlk {
namespace paged {

using umma::cluster_sync_all;
using umma::fence_proxy_async;
using umma::mapa_shared;
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
    static constexpr int D = D_, HALVES = D / 64;  // tiles of 64 dims: 128-byte rows of f16
    static constexpr int TILES = F32 && D == 128 ? 1 : 2, ROWS = 128 * TILES;  // (fp32 sums twice, in TMEM: room for one tile of 128 values)
    static constexpr int PARTS = F32 ? 2 : 1;              // f16 numbers of a query or weight
    static constexpr int KT = 64, GROUPS = KT / 16;        // keys of a block; 16 of them have a page
    static constexpr int MAKERS = 128, THREADS = ROWS + MAKERS + 64;
    static constexpr int NBUF = 3;                         // blocks of keys, and of values, in shared memory
    static constexpr uint32_t Q_HALF = 128 * 128, Q_TILE = Q_HALF * HALVES, KV_HALF = KT * 128, KV_TILE = KV_HALF * HALVES;
    static constexpr bool FULL = !F32 && D == 128;         // no room in TMEM for fp32 sums beside those of the MMAs
    static constexpr uint32_t Q = 0, K = TILES * PARTS * Q_TILE, V = K + NBUF * KV_TILE, BEHIND = V + NBUF * KV_TILE, HALF_KEPT = BEHIND,
                              ROW_SCALE = FULL ? ROWS * D * 4 : BEHIND, RED = BEHIND + (FULL ? ROWS * 64 * 4 : ROWS * 8), BARS = RED + 128, TOTAL = BARS + 256 + 1024;
    // TMEM columns: for each tile two places for scores (64 columns) and the weights made of them (two keys to a column; fp32: the second numbers behind the first), sums and (fp32)
    // kept sums
    static constexpr uint32_t O_AT = 256, O_PITCH = 128, KEPT = D;
    static constexpr int FLUSH = F32 ? 4 : 64, MOST = 256;  // blocks per accumulation; (FULL) of a CTA that does without
    static_assert(TOTAL <= 227 * 1024, "shared memory budget exceeded");
    static_assert(ROWS * D * 4 <= ROW_SCALE && ROW_SCALE + ROWS * 8 <= RED, "a CTA's sums take the place of its operands");
    static_assert(!FULL || ROW_SCALE + ROWS * 8 <= BEHIND, "");
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

// (fp32) What the second f16 number of a query's values leaves, up to half of f16's least step, may move an exponent by more than 2^-16: 1 / sqrt(12) of a step each and a root of
// their sum of squares, times codes of 128 under the largest scale of K.  Only where scores would be millions, if the row's values were of one size.
template <int D>
__device__ __forceinline__ bool pairs_lose(float step, float k_top, float scale) {
    return 5.9604645e-8f * (D == 64 ? 2.3094011f : 3.2659863f) * 128.f * step * (fabsf(scale) * 1.44269504f * k_top) > 1.52587890625e-5f;
}
// Those of the rows first_row, first_row + every, ... that pairs hold too little of, again.
template <typename T, int D>
__device__ __noinline__ void rows_again(const Cache& c, const Batch& q, const Attend& a, int b, int64_t first, int h, int row0, int rows, int first_row, int every, int before, int keys, float k_top) {
    const int lane = threadIdx.x & 31;
    for (int r = first_row; r < rows; r += every) {
        const int row = row0 + r, token = row / a.group, head = h * a.group + row - token * a.group;
        const T* src = static_cast<const T*>(a.q) + (first + token) * a.qs + static_cast<int64_t>(head) * D;
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < D / 32; i++) most = max(most, finite_abs_bits(static_cast<float>(src[lane + 32 * i])));
        most = __reduce_max_sync(0xffffffffu, most);
        if (most > 0 && pairs_lose<D>(exp2_int(-scale_exponent(most)), k_top, a.scale)) row_in_fp32<T, D>(c, q, a, b, first + token, head, min(before + token + 1, keys));
    }
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

// D[tmem] (+)= A x B, kind::f16, issued by one thread.  Descriptors: their lower halves (addresses) vary, their upper halves are the same for all tiles here.
constexpr uint32_t DESC_UPPER = (1024 >> 4) | (1u << 14) | (2u << 29);  // 1 KB between groups of 8 rows, version 1, 128-byte swizzle
// (shared addresses of a cluster's CTAs hold their rank in the upper bits)
__device__ __forceinline__ uint32_t desc_lower(uint32_t address, uint32_t distance) { return (address & 0x3ffffu) >> 4 | distance << 16; }
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %4};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(DESC_UPPER), "r"(add)
        : "memory");
}
// A from TMEM: lane = row, two consecutive k to a column
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %4};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d), "r"(a_tmem), "r"(b), "r"(idesc), "r"(DESC_UPPER), "r"(add)
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

// The sums of a row that lie beside those of the MMAs: in TMEM, of FULL tiles the upper half of them in shared memory
template <typename T, int D>
struct KeptSums {
    using L = Prompt<T, D>;
    uint32_t o_at, at;
    uint8_t* half;
    int r;

    __device__ __forceinline__ float4* unit(int i) const { return reinterpret_cast<float4*>(half + ((((i - 64) >> 2) ^ (r & 7)) << 4)); }
    __device__ __forceinline__ void get(int i, uint32_t (&m)[32]) const {
        if (L::FULL && i >= 64) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                const float4 x = *unit(i + e);
                m[e] = __float_as_uint(x.x);
                m[e + 1] = __float_as_uint(x.y);
                m[e + 2] = __float_as_uint(x.z);
                m[e + 3] = __float_as_uint(x.w);
            }
        } else {
            tmem_ld_x32(at + i, m);
        }
    }
    __device__ __forceinline__ void put(int i, const uint32_t (&m)[32]) const {
        if (L::FULL && i >= 64) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) *unit(i + e) = make_float4(__uint_as_float(m[e]), __uint_as_float(m[e + 1]), __uint_as_float(m[e + 2]), __uint_as_float(m[e + 3]));
        } else {
            tmem_st_x32(at + i, m);
        }
    }
    // the MMAs' sums go to these, all times `corr`
    __device__ __forceinline__ void add(float corr, bool fresh) const {
#pragma unroll 1
        for (int i = 0; i < D; i += 32) {
            uint32_t o[32], m[32];
            tmem_ld_x32(o_at + i, o);
            get(i, m);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e++) {
                m[e] = __float_as_uint((__uint_as_float(o[e]) + (fresh ? 0.f : __uint_as_float(m[e]))) * corr);
                o[e] = 0;
            }
            put(i, m);
            tmem_st_x32(o_at + i, o);
        }
    }
};
template <typename K>
__device__ __noinline__ void add_seldom(K kept, float corr, bool fresh) { kept.add(corr, fresh); }

// SHARED: a cluster of `cluster` CTAs shares the keys of each tile pair
template <typename T, int D, bool SHARED>
__global__ void __launch_bounds__(Prompt<T, D>::THREADS, 1) prompt_kernel(const Cache c, const Batch q, const Attend a, const int cluster) {
    using L = Prompt<T, D>;
    constexpr int TILES = L::TILES, HALVES = L::HALVES, PARTS = L::PARTS, KT = L::KT, ROWS = L::ROWS, GROUPS = L::GROUPS, NBUF = L::NBUF;
    dep_sync();
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* sm = smem_raw + (base - smem_u32(smem_raw));
    float* s_row = reinterpret_cast<float*>(sm + L::ROW_SCALE);
    volatile uint32_t* s_red = reinterpret_cast<volatile uint32_t*>(sm + L::RED);
    // barriers: keys and values in place and done with; of each tile: scores there and their place free again, weights there, values of a block added
    const uint32_t bars = base + L::BARS;
    auto k_full = [&](int i) { return bars + 8u * i; };
    auto k_free = [&](int i) { return bars + 8u * (NBUF + i); };
    auto v_full = [&](int i) { return bars + 8u * (2 * NBUF + i); };
    auto v_free = [&](int i) { return bars + 8u * (3 * NBUF + i); };
    auto s_full = [&](int t, int i) { return bars + 8u * (4 * NBUF + 2 * t + i); };
    auto s_free = [&](int t, int i) { return bars + 8u * (4 * NBUF + 4 + 2 * t + i); };
    auto p_full = [&](int t) { return bars + 8u * (4 * NBUF + 8 + t); };
    auto o_done = [&](int t) { return bars + 8u * (4 * NBUF + 10 + t); };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + L::BARS + 8 * (4 * NBUF + 12));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + L::BARS + 8 * (4 * NBUF + 13));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // ---- which rows: sequence by sequence, the tiles that see most first ----
    const int splits = SHARED ? cluster : 1;
    const int problem = static_cast<int>(blockIdx.x) / splits, share = static_cast<int>(blockIdx.x) - problem * splits;  // the CTAs of a cluster share the keys
    const int h = problem % c.kv_heads;
    int b = 0, item = problem / c.kv_heads;
    // (CTAs of a cluster see the same and leave here together; should what they read change meanwhile, the others find this one's memory still there)
    auto leave = [&]() {
        if constexpr (SHARED) {
            __syncwarp();
            cluster_sync_all();
            cluster_sync_all();
        }
    };
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
        if (!found) {
            leave();
            return;
        }
    }
    const int rows = static_cast<int>(min(count * a.group - static_cast<int64_t>(item) * ROWS, static_cast<int64_t>(ROWS)));  // valid rows from row0 on
    const int row0 = item * ROWS;
    const int64_t table_keys = q.width << c.page_log;
    // (the table has room for at most 2^30 keys; what lies far below the first is as good as -1)
    const int64_t len = q.lens[b];
    const int keys = static_cast<int>(min(len, table_keys + 1)), before = static_cast<int>(min(max(len - count, -(int64_t(1) << 31) + (1 << 26)), int64_t(1) << 30));
    // rows of the sequence and head are counted from its first new token on
    auto token_of = [&](int row) { return static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(a.group)); };
    auto sees_of = [&](int row) { return min(before + token_of(row) + 1, keys); };
    const int seen = max(sees_of(row0 + rows - 1), 0);  // keys that the last row sees
    const int32_t* table = q.table + static_cast<int64_t>(b) * q.width;

    // this CTA's blocks, from key0 on, and those of each tile: the second one's rows see at least as much as the first one's
    const int all_blocks = (seen + KT - 1) / KT, each_blocks = (all_blocks + splits - 1) / splits, block0 = min(share * each_blocks, all_blocks), key0 = block0 * KT;
    const int blocks = min(each_blocks, all_blocks - block0);
    const int blocks0 = rows > 128 ? min(max((sees_of(row0 + 127) + KT - 1) / KT - block0, 0), blocks) : blocks, blocks1 = rows > 128 ? blocks : 0;
    const bool lean = L::FULL && blocks > L::MOST;  // one place for scores
    // block j's scores: which place, how many came there before
    auto place_of = [&](int j) { return lean ? 0 : j & 1; };
    auto turn_of = [&](int j) { return lean ? j : j >> 1; };
    const bool negative = a.scale < 0.f;  // scores' factors are not below zero: the sign goes to the queries
    int* status = a.status;
    constexpr int OTHERS = L::MAKERS + 64, FIRST = ROWS / 32;  // threads and first warp that are not the softmax's

    // ---- while the softmax's warps bring the queries, the others look at the pages: all there, scales finite and not below zero, those of V of one size? ----
    if (warp >= FIRST) {
        float v_top = 0.f, v_low = INFINITY, k_top = 0.f;
        bool plain = true;
        const int pages = (seen + c.page - 1) >> c.page_log;
        for (int i = tid - ROWS; i < pages; i += OTHERS) {
            const int p = i < q.width ? table[i] : -1;
            if (p < 0 || p >= c.pages) {
                plain = false;
            } else {
                const int64_t block = static_cast<int64_t>(p) * c.kv_heads + h;
                const float k = c.ks[block], v = c.vs[block];
                plain = plain && k >= 0.f && k < INFINITY && v >= 0.f && v < INFINITY;
                k_top = fmaxf(k_top, k);
                v_top = fmaxf(v_top, v);
                if (v > 1.17549435e-38f) v_low = fminf(v_low, v);  // 2^-126: the scale of a block of zeros
            }
        }
        const uint32_t t = __reduce_max_sync(0xffffffffu, __float_as_uint(v_top)), l = __reduce_min_sync(0xffffffffu, __float_as_uint(v_low));
        plain = __all_sync(0xffffffffu, plain);
        if constexpr (L::F32) {
            const uint32_t k = __reduce_max_sync(0xffffffffu, __float_as_uint(k_top));
            if (lane == 0) s_red[2 * (OTHERS / 32) + warp - FIRST] = k;
        }
        if (lane == 0) {
            s_red[2 * (warp - FIRST)] = t;
            s_red[2 * (warp - FIRST) + 1] = plain ? l : 0u;  // (0: no lower end, never of one size)
        }
        if (warp == FIRST + 4) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        if (warp == FIRST + 5 && lane == 0) {
            for (int i = 0; i < NBUF; i++) {
                mbar_init(k_full(i), L::MAKERS);
                mbar_init(k_free(i), 1);
                mbar_init(v_full(i), L::MAKERS);
                mbar_init(v_free(i), 1);
            }
            for (int t = 0; t < 2; t++) {
                for (int i = 0; i < 2; i++) {
                    mbar_init(s_full(t, i), 1);
                    mbar_init(s_free(t, i), 1);
                }
                mbar_init(p_full(t), 128);
                mbar_init(o_done(t), 1);
            }
            *abort_flag = 0;
            s_red[31] = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        asm volatile("bar.sync 2, %0;" ::"n"(OTHERS) : "memory");
    }
    // ---- queries ----
    if (warp < FIRST) {
        const int t = warp >> 2;
        constexpr int PER = D / 4, AT_ONCE = 32 / PER, BATCH = 16;  // lanes to a row (four values each), rows of a warp at a time, loads on their way
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
                    const int row = row0 + at, token = token_of(row);
                    raw[i] = *reinterpret_cast<const Four*>(static_cast<const T*>(a.q) + (first + token) * a.qs + (static_cast<int64_t>(h) * a.group + row - token * a.group) * D + 4 * c4);
                }
            }
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                const int r = r0 + i * 4 * AT_ONCE;
                uint8_t* tile = sm + L::Q + t * PARTS * L::Q_TILE + (c4 >> 4) * L::Q_HALF;
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
    // the queries are there, TMEM and what was seen of the pages; the warps that bring the codes need no queries and go on
    const bool maker = warp >= FIRST && warp < FIRST + 4;
    if (maker) {
        asm volatile("bar.arrive 1, %0;" ::"n"(L::THREADS) : "memory");
    } else {
        tc_fence_before();
        asm volatile("bar.sync 1, %0;" ::"n"(L::THREADS) : "memory");
        tc_fence_after();
    }
    float v_top;
    {
        uint32_t top = 0, low = 0x7f800000u;
        for (int w = 0; w < OTHERS / 32; w++) {
            top = max(top, s_red[2 * w]);
            low = min(low, s_red[2 * w + 1]);
        }
        v_top = __uint_as_float(top);
        if (!(__uint_as_float(low) * 1024.f >= v_top) || low == 0 || seen == 0) {
            for (int r = warp + share * (L::THREADS / 32); r < rows; r += splits * (L::THREADS / 32)) {
                const int row = row0 + r, token = token_of(row);
                row_in_fp32<T, D>(c, q, a, b, first + token, h * a.group + row - token * a.group, sees_of(row));
            }
            if (warp == FIRST + 4) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "n"(512) : "memory");
            leave();
            return;
        }
        if (v_top == 0.f) v_top = 1.f;
    }
    const uint32_t tmem = maker ? 0u : *tmem_slot;

    // (once for each number of places for scores: a choice within the loop took 4 % where most prompts have two)
    auto softmax = [&](auto one_place) {
        constexpr bool ONE = decltype(one_place)::value;
        const int t = warp >> 2, r = tid, own_blocks = t == 0 ? blocks0 : blocks1;
        const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16), at = lanes + t * 128, o_at = lanes + L::O_AT + t * L::O_PITCH;
        const int sees = r < rows ? sees_of(row0 + r) : 0, least = sees_of(row0 + t * 128);  // least: what every row of the tile sees
        const float q_scale = fabsf(a.scale) * 1.44269504f * (L::F32 ? s_row[r] : 1.f);
        // v / v_top: the reciprocal of a number near the lower end of fp32 would be infinite, of 2^64 times it is not
        const float v_up = v_top < 1.f ? 18446744073709551616.f : 1.f, v_inv = 1.f / (v_top * v_up);
        if constexpr (L::F32) {
            float k_top = 0.f;
            for (int w = 0; w < OTHERS / 32; w++) k_top = fmaxf(k_top, __uint_as_float(s_red[2 * (OTHERS / 32) + w]));
            if (pairs_lose<D>(s_row[r], k_top, a.scale)) {
                // what is needed to form such rows again, at the end (kept in registers until then it cost 3 %; every row writes the same)
                const uint32_t note[9] = {static_cast<uint32_t>(b), static_cast<uint32_t>(h), static_cast<uint32_t>(row0), static_cast<uint32_t>(rows), static_cast<uint32_t>(before),
                                          static_cast<uint32_t>(keys), static_cast<uint32_t>(first), static_cast<uint32_t>(first >> 32), __float_as_uint(k_top)};
#pragma unroll
                for (int i = 0; i < 9; i++) s_red[22 + i] = note[i];
                s_red[31] = 1;
            }
        }
        float top = -INFINITY, sum = 0.f;
        bool ok = true, fresh = true;  // fresh: nothing kept yet
        int in_run = 0;                // blocks since the sums were last added up
        constexpr bool KEEPS = !L::FULL || ONE;
        using Kept = KeptSums<T, D>;
        const Kept kept = {o_at, L::FULL ? at + KT : o_at + L::KEPT, L::FULL ? sm + L::HALF_KEPT + r * 256 : nullptr, r};
        // scales of 16 keys each: lanes look up pages two blocks ahead, scales one
        int page_next = 0;
        float ks_next = 0.f, vs_next = 0.f;
        auto page_of = [&](int j) {
            const int key = key0 + j * KT + lane * 16;
            page_next = -1;
            if (lane < GROUPS && key < seen) page_next = table[key >> c.page_log];
        };
        auto scales_of = [&]() {
            ks_next = 0.f;
            vs_next = v_top;
            if (page_next >= 0) {
                const int block = page_next * c.kv_heads + h;
                ks_next = c.ks[block];
                vs_next = c.vs[block];
            }
        };
        page_of(0);
        scales_of();
        page_of(1);
        for (int j = 0; j < own_blocks; j++) {
            // lane n has the scales of 16 keys; f_of: what a row's scores are multiplied by (not zero: hidden scores stay -inf)
            const float ks = ks_next, vs = vs_next * v_up * v_inv;
            auto f_of = [&](int n) { return fmaxf(__shfl_sync(0xffffffffu, ks, n) * q_scale, 1e-38f); };
            const bool even = __all_sync(0xffffffffu, vs == 1.f);  // all scales of V are the largest
            scales_of();
            page_of(j + 2);
            const bool hidden = key0 + (j + 1) * KT > least;
            const int see = sees - key0 - j * KT;
            ok = __all_sync(0xffffffffu, mbar_wait(s_full(t, ONE ? 0 : j & 1), (ONE ? j : j >> 1) & 1, abort_flag, status));
            if (!ok) break;
            tc_fence_after();
            const uint32_t s_at = at + (ONE ? 0 : j & 1) * KT;
            float x[KT];
            tmem_ld_x32(s_at, *reinterpret_cast<uint32_t(*)[32]>(x));
            tmem_ld_x32(s_at + 32, *reinterpret_cast<uint32_t(*)[32]>(x + 32));
            tmem_wait_ld();
            if (hidden) {
#pragma unroll
                for (int i = 0; i < KT; i++)
                    if (i >= see) x[i] = -INFINITY;
            }
            float most = -INFINITY;
#pragma unroll
            for (int n = 0; n < GROUPS; n++) {
                float m = x[16 * n];
#pragma unroll
                for (int i = 1; i < 16; i++) m = fmaxf(m, x[16 * n + i]);
                most = fmaxf(most, m * f_of(n));
            }
            // The maximum that the sums are under moves when it has fallen behind by more than 2^8.
            const bool move = most > top + 8.f || (top == -INFINITY && most > top);
            const float new_top = move ? most : top;
            const float corr = move && top != -INFINITY ? ex2(top - new_top) : move ? 0.f : 1.f;
            const bool any = __any_sync(0xffffffffu, move && j > 0);
            top = new_top;
            sum *= corr;
            const float shift = (top == -INFINITY ? 0.f : top) - 6.f;  // weights are 2^6 exp2(s - top)
            float2 part = make_float2(0.f, 0.f);
            const float2 shift2 = make_float2(-shift, -shift);
#pragma unroll
            for (int n = 0; n < GROUPS; n++) {
                const float f = f_of(n);
#pragma unroll
                for (int i = 16 * n; i < 16 * n + 16; i += 2) {
                    float2 y = fma2(make_float2(x[i], x[i + 1]), make_float2(f, f), shift2);
                    y.x = ex2(y.x);
                    y.y = ex2(y.y);
                    part = add2(part, y);
                    x[i] = y.x;
                    x[i + 1] = y.y;
                }
            }
            sum += part.x + part.y;
            if (!even) {
#pragma unroll
                for (int n = 0; n < GROUPS; n++) {
                    const float v = __shfl_sync(0xffffffffu, vs, n);
#pragma unroll
                    for (int i = 16 * n; i < 16 * n + 16; i++) x[i] *= v;
                }
            }
#pragma unroll
            for (int ch = 0; ch < 2; ch++) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    float(&y)[2] = *reinterpret_cast<float(*)[2]>(x + 32 * ch + 2 * i);
                    w[i] = pack_f16(y[0], y[1]);
                    if constexpr (L::F32) {
                        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                        y[0] -= back.x;
                        y[1] -= back.y;
                    }
                }
                tc::tmem_st_x16(s_at + 16 * ch, w);
                if constexpr (L::F32) {
#pragma unroll
                    for (int i = 0; i < 16; i++) w[i] = pack_f16(x[32 * ch + 2 * i], x[32 * ch + 2 * i + 1]);
                    tc::tmem_st_x16(s_at + 32 + 16 * ch, w);
                }
            }
            // The values of the block before have been added: the sums can be touched.  (And the MMA thread has seen the weights before these: p_full is never two ahead of it.)
            if (j > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(o_done(t), (j - 1) & 1, abort_flag, status));
                if (!ok) break;
                tc_fence_after();
            }
            // ---- the sums under the new maximum; now and then added to those that are kept ----
            if (KEEPS && j > 0 && ((any && (L::F32 || !fresh)) || ++in_run >= L::FLUSH)) {
                if constexpr (L::F32) kept.add(corr, fresh);
                else add_seldom(kept, corr, fresh);
                fresh = false;
                in_run = 0;
            } else if (!L::F32 && any) {
#pragma unroll 1
                for (int i = 0; i < D; i += 32) {
                    uint32_t o[32];
                    tmem_ld_x32(o_at + i, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                    tmem_st_x32(o_at + i, o);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(p_full(t));
        }
        // ---- results ----
        if (ok && own_blocks > 0) ok = __all_sync(0xffffffffu, mbar_wait(o_done(t), (own_blocks - 1) & 1, abort_flag, status));
        tc_fence_after();
        // (the sums of a share go to where the operands of both tiles were)
        if constexpr (SHARED) asm volatile("bar.sync 3, %0;" ::"n"(ROWS) : "memory");
        [[maybe_unused]] const float inv = 1.f / sum;  // (not times v_top: that could leave the normal numbers although the result does not)
        const int row = row0 + r, token = token_of(row);
        [[maybe_unused]] T* dst = static_cast<T*>(a.out) + (first + token) * a.os + (static_cast<int64_t>(h) * a.group + row - token * a.group) * D;
#pragma unroll 1
        for (int i = 0; i < D; i += 32) {
            uint32_t o[32];  // (of a tile without keys: nothing that is looked at)
            tmem_ld_x32(o_at + i, o);
            if (KEEPS && !fresh) {
                uint32_t m[32];
                kept.get(i, m);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) + __uint_as_float(m[e]));
            } else {
                tmem_wait_ld();
            }
            if constexpr (SHARED) {
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const float4 x = make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
                    *reinterpret_cast<float4*>(sm + r * (D * 4) + ((((i + e) >> 2) ^ (r & 7)) << 4)) = own_blocks > 0 ? x : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            } else if (r < rows) {
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = __float_as_uint(!ok ? __int_as_float(0x7fc00000) : sees <= 0 ? 0.f : __uint_as_float(o[e]) * inv * v_top);
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
        if constexpr (SHARED) reinterpret_cast<float2*>(sm + L::ROW_SCALE)[r] = make_float2(top, ok ? sum : __int_as_float(0x7fc00000));
        tc_fence_before();
    };
    if (warp < FIRST) {
        // ---------------- softmax ----------------
        if constexpr (L::FULL) {
            if (lean) softmax(std::true_type{});
            else softmax(std::false_type{});
        } else {
            softmax(std::false_type{});
        }
    } else if (maker) {
        // ---------------- codes to f16 tiles: 16-byte pieces of a key, a thread always the same piece, of keys own_key + i STEP ----------------
        constexpr int PIECES = D / 16, STEP = L::MAKERS / PIECES, N = KT / STEP;
        const int me = tid - ROWS, own_key = me / PIECES, piece = me % PIECES;
        const int64_t head = static_cast<int64_t>(h) * c.page * D + piece * 16, page_bytes = static_cast<int64_t>(c.kv_heads) * c.page * D;
        int page[N];
        uint4 kx[N], vx[N];
        auto look_up = [&](int j) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int key = key0 + j * KT + own_key + i * STEP;
                page[i] = key < seen ? table[key >> c.page_log] : -1;
            }
        };
        auto load = [&](const int8_t* codes, int j, uint4 (&x)[N]) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                x[i] = make_uint4(0u, 0u, 0u, 0u);  // (keys that no row sees)
                if (page[i] >= 0)
                    x[i] = *reinterpret_cast<const uint4*>(codes + static_cast<int64_t>(page[i]) * page_bytes + head + ((key0 + j * KT + own_key + i * STEP) & (c.page - 1)) * D);
            }
        };
        auto put = [&](uint32_t tile, const uint4 (&x)[N]) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int r = own_key + i * STEP, u = 2 * (piece & 3);
                uint8_t* to = sm + tile + (piece >> 2) * L::KV_HALF;
                *reinterpret_cast<uint4*>(to + swizzled(r, u)) = eight_f16(x[i].x, x[i].y);
                *reinterpret_cast<uint4*>(to + swizzled(r, u + 1)) = eight_f16(x[i].z, x[i].w);
            }
            fence_proxy_async();
        };
        look_up(0);
        load(c.k, 0, kx);
        load(c.v, 0, vx);
        look_up(1);
        bool ok = true;
        int i = 0;
        uint32_t phase = 1;  // (the first use of a place goes through)
#pragma unroll 1
        for (int j = 0; j < blocks; j++) {
            ok = mbar_wait(k_free(i), phase, abort_flag, status);
            if (!ok) break;
            put(L::K + i * L::KV_TILE, kx);
            mbar_arrive(k_full(i));
            load(c.k, j + 1, kx);
            ok = mbar_wait(v_free(i), phase, abort_flag, status);
            if (!ok) break;
            put(L::V + i * L::KV_TILE, vx);
            mbar_arrive(v_full(i));
            load(c.v, j + 1, vx);
            look_up(j + 2);
            if (++i == NBUF) {
                i = 0;
                phase ^= 1;
            }
        }
    } else if (warp == FIRST + 4) {
        // ---------------- MMAs of the scores: lower halves of descriptors are address / 16, and for the values the distance between blocks of 64 dims ----------------
        if (lane == 0) {
            constexpr uint32_t qk = (1u << 4) | ((KT >> 3) << 17) | ((128 >> 4) << 24);
            const uint32_t q_desc = desc_lower(base + L::Q, 1), k_desc = desc_lower(base + L::K, 1);
            bool ok = true;
            int i = 0;
            uint32_t phase = 0;
#pragma unroll 1
            for (int j = 0; j < blocks && ok; j++) {
                ok = mbar_wait(k_full(i), phase, abort_flag, status);
                const uint32_t kd = k_desc + i * (L::KV_TILE >> 4), d = tmem + place_of(j) * KT;
#pragma unroll
                for (int t = 0; t < TILES; t++) {
                    if (!ok || j >= (t == 0 ? blocks0 : blocks1)) continue;
                    // the weights of the block before, which lie there, have been read
                    ok = mbar_wait(s_free(t, place_of(j)), (turn_of(j) & 1) ^ 1, abort_flag, status);
                    if (!ok) continue;
                    tc_fence_after();
#pragma unroll
                    for (int part = PARTS - 1; part >= 0; part--)  // the small products first
#pragma unroll
                        for (int half = 0; half < HALVES; half++)
#pragma unroll
                            for (int kk = 0; kk < 4; kk++)
                                mma_ss(d + t * 128, q_desc + (((t * PARTS + part) * L::Q_TILE + half * L::Q_HALF) >> 4) + kk * 2, kd + ((half * L::KV_HALF) >> 4) + kk * 2, qk,
                                       part < PARTS - 1 || half > 0 || kk > 0);
                    umma::commit<1>(s_full(t, place_of(j)));
                }
                if (ok) umma::commit<1>(k_free(i));
                if (++i == NBUF) {
                    i = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (lane == 0) {
        // ---------------- MMAs of the values ----------------
        constexpr uint32_t pv = (1u << 4) | (1u << 16) | ((D >> 3) << 17) | ((128 >> 4) << 24);  // keys along the rows
        const uint32_t v_desc = desc_lower(base + L::V, L::KV_HALF >> 4);
        bool ok = true;
        int i = 0;
        uint32_t phase = 0;
#pragma unroll 1
        for (int j = 0; j < blocks && ok; j++) {
            ok = mbar_wait(v_full(i), phase, abort_flag, status);
            const uint32_t vd = v_desc + i * (L::KV_TILE >> 4);
#pragma unroll
            for (int t = 0; t < TILES; t++) {
                if (!ok || j >= (t == 0 ? blocks0 : blocks1)) continue;
                ok = mbar_wait(p_full(t), j & 1, abort_flag, status);
                if (!ok) continue;
                tc_fence_after();
#pragma unroll
                for (int part = PARTS - 1; part >= 0; part--)
#pragma unroll
                    for (int kk = 0; kk < 4; kk++)
                        mma_ts(tmem + L::O_AT + t * L::O_PITCH, tmem + t * 128 + place_of(j) * KT + part * 32 + kk * 8, vd + kk * 128, pv, part < PARTS - 1 || kk > 0 ? 1u : j > 0);
                umma::commit<1>(o_done(t));
                umma::commit<1>(s_free(t, place_of(j)));
            }
            if (ok) umma::commit<1>(v_free(i));
            if (++i == NBUF) {
                i = 0;
                phase ^= 1;
            }
        }
    }
    if constexpr (SHARED) {
        // ---- the shares' sums, maxima and weights' sums joined, in the keys' order: each CTA of the cluster takes every splits-th row ----
        __syncwarp();
        cluster_sync_all();
        constexpr int UNITS = D / 4, MOST = 8;
        for (int i = tid; i < ROWS / splits * UNITS; i += L::THREADS) {
            const int r = i / UNITS * splits + share, u = i % UNITS;
            if (r >= rows) break;
            const uint32_t of_row = base + L::ROW_SCALE + r * 8, of_sums = base + r * (D * 4) + ((u ^ (r & 7)) << 4);
            float2 part[MOST];  // a share's maximum and its weights' sum
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int p = 0; p < MOST; p++)
                if (p < splits) asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(part[p].x), "=f"(part[p].y) : "r"(mapa_shared(of_row, p)));
#pragma unroll
            for (int p = 0; p < MOST; p++)
                if (p < splits) top = fmaxf(top, part[p].x);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int p = 0; p < MOST; p++)
                if (p < splits) {
                    const float f = part[p].x == -INFINITY ? 1.f : ex2(part[p].x - top);  // (no keys: sums of zero, or NaN, which has to stay)
                    float4 x;
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(mapa_shared(of_sums, p)));
                    sum = fmaf(part[p].y, f, sum);
                    o = make_float4(fmaf(x.x, f, o.x), fmaf(x.y, f, o.y), fmaf(x.z, f, o.z), fmaf(x.w, f, o.w));
                }
            const int row = row0 + r, token = token_of(row);
            const float inv = 1.f / sum;
            o = sees_of(row) <= 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o.x * inv * v_top, o.y * inv * v_top, o.z * inv * v_top, o.w * inv * v_top);
            T* dst = static_cast<T*>(a.out) + (first + token) * a.os + (static_cast<int64_t>(h) * a.group + row - token * a.group) * D + 4 * u;
            if constexpr (L::F32) *reinterpret_cast<float4*>(dst) = o;
            else *reinterpret_cast<uint2*>(dst) = make_uint2(pack_f16(o.x, o.y), pack_f16(o.z, o.w));
        }
        cluster_sync_all();  // (what is read lies in all of them)
    }
    tc_fence_before();
    __syncthreads();
    if (warp == FIRST + 4) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    }
    // (behind the barrier: every row has its first result; where a cluster shares the keys, from this CTA)
    if constexpr (L::F32)
        if (s_red[31]) {
            const int by = SHARED ? cluster : 1, own = SHARED ? static_cast<int>(blockIdx.x) % by : 0;
            rows_again<T, D>(c, q, a, s_red[22], static_cast<int64_t>(s_red[29]) << 32 | s_red[28], s_red[23], s_red[24], s_red[25], own + by * (threadIdx.x >> 5), by * (L::THREADS / 32), s_red[26],
                             s_red[27], __uint_as_float(s_red[30]));
        }
}

}  // namespace paged
}  // namespace rmlk
