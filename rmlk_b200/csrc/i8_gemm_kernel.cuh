// i8_gemm_kernel: out[m][n] = (sum_k x[m][k] w[n][k]) sx[m] sw[n] on tcgen05.mma kind::i8 (see matmul_i8.cu for the overview).
#pragma once

#include "umma_gemm.cuh"

namespace rmlk {
namespace i8 {

using umma::arrive_cluster;
using umma::BN;
using umma::cluster_ctarank;
using umma::cluster_sync_all;
using umma::commit;
using umma::load_2d;
using umma::mapa_shared;
using umma::mbar_arrive;
using umma::mbar_expect_tx;
using umma::mbar_init;
using umma::mbar_wait;
using umma::smem_desc_k128;
using umma::smem_u32;
using umma::tc_fence_after;
using umma::tc_fence_before;
using umma::tmem_ld;

constexpr int KB = 128;  // k per block: one 128-byte row of both tiles

struct Params {
    void* out;
    int64_t M, N, ldo;
    const float *sx, *sw;
    int n_tiles, m_tiles, m_group;  // tiles of CG * 128 channels x MT tokens; token tiles that share a pass over the channels
    int k_blocks;
    int* status;
};

// CG: CTAs per tile (a pair shares 256 channels); MT: tokens per tile; ST: stages; SPLIT: the CTAs of a cluster share the tile's k, add their sums through distributed shared
// memory and each write a part of the tokens
template <int CG, int MT, int ST, bool SPLIT>
struct Layout {
    static constexpr int EPI_WARPS = MT >= 192 ? 16 : 8;
    static constexpr int THREADS = 64 + 32 * EPI_WARPS;  // TMA warp, MMA warp, epilogue warps
    static constexpr int XR = MT / CG;                   // tokens that this CTA loads
    static constexpr uint32_t W_BYTES = BN * KB, X_BYTES = XR * KB, STAGE = W_BYTES + X_BYTES;
    static constexpr int NBUF = SPLIT || MT > 256 ? 1 : 2;
    static constexpr uint32_t COLS = MT * NBUF;
    static constexpr uint32_t TMEM_COLS = COLS <= 32 ? 32 : COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
    static constexpr uint32_t SUMS = ST * STAGE;  // SPLIT: the cluster's sums for the tokens of this CTA, [split][token][channel]
    static constexpr uint32_t BAR_OFFSET = SUMS + (SPLIT ? MT * BN * 4 : 0);
    static_assert(!SPLIT || CG == 1, "");
    static constexpr uint32_t N_BARS = 2 * ST + 2 * NBUF;
    static constexpr uint32_t TOTAL = BAR_OFFSET + 8 * N_BARS + 32 + 1024;
    static_assert(COLS <= 512 && TOTAL <= 227 * 1024, "TMEM or shared memory budget exceeded");
    static_assert(X_BYTES % 1024 == 0, "a swizzled tile starts on a 1 KB boundary");
};

template <int CG>
__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

// sum times the scales of a row and a column.  Their product first where it is a normal number: the sum times one of them alone may leave the range although the
// result does not.
__device__ __forceinline__ float scaled(int sum, float a, float b) {
    const float v = static_cast<float>(sum), t = a * b;
    return fabsf(t) >= 1.17549435e-38f && fabsf(t) < INFINITY ? v * t : v * a * b;
}

struct Tile {
    int n_tile, m_tile;
};
// Passes over all channel tiles with `m_group` token tiles each, so that concurrently running tiles share weights and activations in L2.
__device__ __forceinline__ Tile tile_at(int w, const Params& p) {
    const int per_pass = p.m_group * p.n_tiles, pass = w / per_pass, r = w - pass * per_pass, m_first = pass * p.m_group, rows = min(p.m_group, p.m_tiles - m_first);
    Tile t;
    t.n_tile = r / rows;
    t.m_tile = m_first + r - t.n_tile * rows;
    return t;
}

template <int CG, int MT, int ST, bool OUT16, bool SPLIT>
__global__ void __launch_bounds__(Layout<CG, MT, ST, SPLIT>::THREADS, 1) gemm_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                                                                                    const __grid_constant__ Params p) {
    using L = Layout<CG, MT, ST, SPLIT>;
    using Out = typename std::conditional<OUT16, __half, float>::type;
    dep_trigger();
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bars = base + L::BAR_OFFSET;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (ST + s); };
    auto acc_full = [&](int b) { return bars + 8u * (2 * ST + b); };
    auto acc_empty = [&](int b) { return bars + 8u * (2 * ST + L::NBUF + b); };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + L::BAR_OFFSET + 8 * L::N_BARS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(base_ptr + L::BAR_OFFSET + 8 * L::N_BARS + 8);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 || SPLIT ? cluster_ctarank() : 0;
    const int log_splits = SPLIT ? 31 - __clz(gridDim.y) : 0, splits = 1 << log_splits;  // (a power of two)
    const int first = CG == 2 ? blockIdx.x >> 1 : blockIdx.x, stride = CG == 2 ? gridDim.x >> 1 : gridDim.x;
    const int tiles = p.n_tiles * p.m_tiles;
    const int kb0 = SPLIT ? blockIdx.y * p.k_blocks >> log_splits : 0, nk = SPLIT ? ((blockIdx.y + 1) * p.k_blocks >> log_splits) - kb0 : p.k_blocks;  // (at least one block each)
    const uint32_t in_pair = CG == 2 ? rank : 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; s++) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < L::NBUF; b++) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), CG * L::EPI_WARPS);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(L::TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(L::TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    if constexpr (CG == 2 || SPLIT) cluster_sync_all();  // the pair's barriers exist and both have their TMEM; all CTAs of a cluster are there
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    int sums[SPLIT ? MT / (L::EPI_WARPS / 4) : 1];  // (SPLIT) this warp's sums: MT / 2 tokens of 32 channels
    // (SPLIT) what an epilogue thread writes: tokens at0, at0 + ROWS, ... of the `here` ones of this CTA, m0 + (those << log_splits), of channel n
    constexpr int ROWS = L::EPI_WARPS * 32 / BN, MOST = SPLIT ? MT / 2 / ROWS : 1;
    const Tile own = tile_at(SPLIT ? first : 0, p);
    const int per = MT >> log_splits, channel = (static_cast<int>(threadIdx.x) - 64) & (BN - 1), at0 = (static_cast<int>(threadIdx.x) - 64) / BN;
    const int64_t n = static_cast<int64_t>(own.n_tile) * BN + channel, m0 = static_cast<int64_t>(own.m_tile) * MT + rank;
    const int here = static_cast<int>(min(static_cast<int64_t>(per), (p.M - m0 + splits - 1) >> log_splits));
    float sx[MOST], sw = 0.f;
    if (warp == 0) {
        // ---------------- loads ----------------
        if (lane == 0) {
            const uint32_t pair_bar = CG == 2 ? mapa_shared(bars, 0) : bars;  // the pair's full barriers live in its first CTA
            dep_wait();
            int s = 0, asked = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int w = first; w < tiles && ok; w += stride) {
                const Tile t = tile_at(w, p);
                for (int kb = 0; kb < nk && ok; kb++) {
                    if (asked >= ST) ok = mbar_wait(empty(s), phase ^ 1, abort_flag, p.status);
                    if (!ok) break;
                    asked++;
                    if (in_pair == 0) mbar_expect_tx(full(s), CG * L::STAGE);
                    const uint32_t dst = base + s * L::STAGE, bar = pair_bar + 8u * s;
                    load_2d<CG>(dst, &tmW, (kb0 + kb) * KB, (t.n_tile * CG + static_cast<int>(in_pair)) * BN, bar);
                    load_2d<CG>(dst + L::W_BYTES, &tmX, (kb0 + kb) * KB, t.m_tile * MT + static_cast<int>(in_pair) * L::XR, bar);
                    if (++s == ST) {
                        s = 0;
                        phase ^= 1;
                    }
                }
            }
            if (in_pair == 0)  // (the pair's bytes all arrive here; its CTAs leave together)
                for (int i = max(asked - ST, 0); i < asked; i++) tc::wait_for_copies(full(i % ST), (i / ST) & 1);
        }
    } else if (warp == 1) {
        // ---------------- MMAs: one thread of the pair's first CTA ----------------
        if (lane == 0 && in_pair == 0) {
            dep_wait();  // (a bounded wait that starts before the kernel before this one has ended would count that one's time)
            constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((MT >> 3) << 17) | ((CG * BN >> 4) << 24);  // s8 x s8 -> s32, both k-major
            const uint64_t w_desc0 = smem_desc_k128(base), x_desc0 = smem_desc_k128(base + L::W_BYTES);
            int s = 0, buf = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            for (int w = first; w < tiles && ok; w += stride) {
                ok = mbar_wait(acc_empty(buf), acc_phase ^ 1, abort_flag, p.status);  // its first use passes at once
                for (int kb = 0; kb < nk && ok; kb++) {
                    ok = mbar_wait(full(s), phase, abort_flag, p.status);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t wd = w_desc0 + ((s * L::STAGE) >> 4), xd = x_desc0 + ((s * L::STAGE) >> 4);
#pragma unroll
                    for (int kk = 0; kk < 4; kk++) mma_i8<CG>(tmem + buf * MT, wd + kk * 2, xd + kk * 2, idesc, kb > 0 || kk > 0);  // 32 k: 32 bytes inside the rows
                    commit<CG>(empty(s));
                    if (++s == ST) {
                        s = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                commit<CG>(acc_full(buf));
                if (++buf == L::NBUF) {
                    buf = 0;
                    acc_phase ^= 1;
                }
            }
        }
    } else {
        // ---------------- epilogue: several warps per group of 32 TMEM lanes (= channels), each with its part of the tile's tokens ----------------
        constexpr int HM = MT / (L::EPI_WARPS / 4), STEP = HM < 16 ? HM : 16;
        const int sub = warp & 3, part = (warp - 2) >> 2;
        const uint32_t lane_field = static_cast<uint32_t>(sub * 32) << 16;
        const uint32_t pair_empty = CG == 2 ? mapa_shared(acc_empty(0), 0) : acc_empty(0);
        dep_wait();  // scales and outputs may belong to kernels before this one
        if constexpr (SPLIT) {  // (asked for one by one at the end, the scales of 64 tokens took 4 us)
            if (n < p.N) sw = __ldg(p.sw + n);
#pragma unroll
            for (int i = 0; i < MOST; i++) sx[i] = at0 + i * ROWS < here ? __ldg(p.sx + m0 + ((at0 + i * ROWS) << log_splits)) : 0.f;
        }
        int buf = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        int w = first;
        for (; w < tiles; w += stride) {
            const Tile t = tile_at(w, p);
            const int64_t n = (static_cast<int64_t>(t.n_tile) * CG + in_pair) * BN + sub * 32 + lane;
            const int64_t m_base = static_cast<int64_t>(t.m_tile) * MT + part * HM;
            const bool in = n < p.N;
            const float sw = in && !SPLIT ? __ldg(p.sw + n) : 0.f;
            // (one lane's limit may run out before another's)
            ok = __all_sync(0xffffffffu, mbar_wait(acc_full(buf), acc_phase, abort_flag, p.status));
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tmem + lane_field + buf * MT + part * HM;
            if constexpr (SPLIT) {
#pragma unroll
                for (int j0 = 0; j0 < HM; j0 += STEP) tmem_ld<STEP>(d + j0, reinterpret_cast<uint32_t*>(sums) + j0);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            } else {
                int acc[HM];
#pragma unroll
                for (int j0 = 0; j0 < HM; j0 += STEP) tmem_ld<STEP>(d + j0, reinterpret_cast<uint32_t*>(acc) + j0);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (CG == 2) arrive_cluster(pair_empty + 8u * buf);
                    else mbar_arrive(acc_empty(buf));
                }
                Out* o = static_cast<Out*>(p.out) + m_base * p.ldo + n;
                const int64_t rows = p.M - m_base;
#pragma unroll
                for (int j = 0; j < HM; j++) {
                    if (j < rows && in) *o = static_cast<Out>(scaled(acc[j], __ldg(p.sx + m_base + j), sw));
                    o += p.ldo;
                }
            }
            if (++buf == L::NBUF) {
                buf = 0;
                acc_phase ^= 1;
            }
        }
        if constexpr (!SPLIT) {  // given up: what has not been written is NaN
            for (; w < tiles; w += stride) {
                const Tile t = tile_at(w, p);
                const int64_t n = (static_cast<int64_t>(t.n_tile) * CG + in_pair) * BN + sub * 32 + lane, m_base = static_cast<int64_t>(t.m_tile) * MT + part * HM;
                for (int j = 0; j < HM && m_base + j < p.M; j++)
                    if (n < p.N) static_cast<Out*>(p.out)[(m_base + j) * p.ldo + n] = static_cast<Out>(__int_as_float(0x7fc00000));
            }
        } else if (!ok) {  // the cluster's sums are not all there: all of it gives up
#pragma unroll
            for (int j = 0; j < HM; j++) sums[j] = 0;
            const uint32_t flag = smem_u32(base_ptr + L::BAR_OFFSET + 8 * L::N_BARS + 8);
            for (int r = 0; r < splits; r++) asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(mapa_shared(flag, r)), "r"(1) : "memory");
        }
        if constexpr (SPLIT) {
            // CTA r of the cluster adds up tokens r, r + splits, ...: their sums go to its shared memory
            const int tokens = static_cast<int>(min(p.M - static_cast<int64_t>(tile_at(first, p).m_tile) * MT, static_cast<int64_t>(MT)));
            const uint32_t at = base + L::SUMS + ((static_cast<int>(rank) * (MT >> log_splits)) * BN + sub * 32 + lane) * 4;
#pragma unroll
            for (int j = 0; j < HM; j++) {
                const int token = part * HM + j;
                const uint32_t addr = mapa_shared(at + (token >> log_splits) * (BN * 4), token & (splits - 1));
                if (token < tokens) asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(sums[j]) : "memory");
            }
        }
    }
    if constexpr (SPLIT) {
        __syncwarp();
        cluster_sync_all();
        if (warp >= 2 && n < p.N) {
            const bool given_up = *abort_flag;
            const int* s = reinterpret_cast<const int*>(base_ptr + L::SUMS) + channel;
            int sum[MOST] = {};
#pragma unroll 1
            for (int r = 0; r < splits; r++) {
#pragma unroll
                for (int i = 0; i < MOST; i++)
                    if (at0 + i * ROWS < here) sum[i] += s[(r * per + at0 + i * ROWS) * BN];
            }
            Out* o = static_cast<Out*>(p.out) + n;
#pragma unroll
            for (int i = 0; i < MOST; i++) {
                if (at0 + i * ROWS < here) o[(m0 + ((at0 + i * ROWS) << log_splits)) * p.ldo] = static_cast<Out>(given_up ? __int_as_float(0x7fc00000) : scaled(sum[i], sx[i], sw));
            }
        }
    }
    tc_fence_before();
    if constexpr (CG == 2) cluster_sync_all();  // no CTA of the pair leaves while the other may still signal its barriers or read its tiles
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (CG == 1)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::TMEM_COLS) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::TMEM_COLS) : "memory");
    }
}

}  // namespace i8
}  // namespace rmlk
