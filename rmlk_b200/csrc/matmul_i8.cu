// Products of 8-bit integers with a scale per row of X (token) and per row of W (channel).
//
//   out[m][n] = (sum_k x[m][k] w[n][k]) sx[m] sw[n]
//
// The sum is exact in 32 bits (k <= 131071 and |x w| <= 2^14), so it does not depend on the order of its parts: the sums of CTAs that share a product's k are
// added as they come.
//
// tcgen05.mma kind::i8 behind TMA, laid out as the f16 product is (umma_gemm.cu): a CTA owns 128 channels - the MMA's M, one TMEM lane each - and a tile of MT
// tokens, the MMA's N; a pair of CTAs (cta_group::2) shares 256 channels.  Both operands have k along their rows, 128 bytes to a swizzled row.
// What bounds it: for many tokens the tensor pipe; for few the weights' bytes, which is why a product with fewer tiles than SMs is shared along k by a cluster.
// Measured, m x k x n: 4096 x 4096 x 14336 in f16 181 to 186 us, 2.6 POP/s; 64 x 2048 x 16384 in f32 11.5 us, 3.3 TB/s (a wave of 128 CTAs, 16 blocks of k each: the first bytes and
// the last sums are half of it); 1 x 2048 x 2048 3.7 us.
#include "umma_gemm.h"

#include <algorithm>
#include <mutex>

#include "i8_gemm_kernel.cuh"

namespace rmlk {
namespace i8 {

static bool map_2d(CUtensorMap* map, const void* ptr, int64_t k, int64_t rows, int64_t pitch, uint32_t box_rows) {
    tc::EncodeTiledFn fn = tc::encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
    const cuuint32_t box[2] = {KB, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int CG, int MT, int ST, bool OUT16, bool SPLIT>
static int launch(cudaStream_t st, const CUtensorMap& tmW, const CUtensorMap& tmX, const Params& p, int splits) {
    using L = Layout<CG, MT, ST, SPLIT>;
    auto kernel = gemm_kernel<CG, MT, ST, OUT16, SPLIT>;
    static std::once_flag configured[64];  // the dynamic shared memory limit is raised once per device
    int dev = 0;
    cudaGetDevice(&dev);
    cudaError_t cfg_err = cudaSuccess;
    if (dev >= 0 && dev < 64)
        std::call_once(configured[dev], [&] { cfg_err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL); });
    RMLK_CUDA(cfg_err);
    const int64_t tiles = static_cast<int64_t>(p.n_tiles) * p.m_tiles;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = SPLIT ? dim3(static_cast<unsigned>(tiles), splits) : dim3(static_cast<unsigned>(CG * std::min<int64_t>(tiles, sm_count() / CG)));
    cfg.blockDim = dim3(L::THREADS);
    cfg.dynamicSmemBytes = L::TOTAL;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    unsigned na = 0;
    if (CG == 2 || SPLIT) {
        at[na].id = cudaLaunchAttributeClusterDimension;
        at[na].val.clusterDim.x = CG;
        at[na].val.clusterDim.y = SPLIT ? splits : 1;
        at[na].val.clusterDim.z = 1;
        na++;
    }
    if (dep_launch_enabled()) {
        at[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[na].val.programmaticStreamSerializationAllowed = 1;
        na++;
    }
    cfg.attrs = at;
    cfg.numAttrs = na;
    RMLK_CUDA(cudaLaunchKernelEx(&cfg, kernel, tmW, tmX, p));
    RMLK_CHECK_LAUNCH("i8 gemm_kernel");
    return RMLK_OK;
}

struct Plan {
    int cg, mt, splits;
};

// The shape whose waves cost least, in cycles: an item costs its blocks of k (the MMAs, or the bytes that a CTA has to bring in where those take longer) and what starting and
// storing a tile takes.  k is shared by 2, 4 or 8 CTAs of a cluster where the tiles alone would leave SMs idle; clusters of 4 fill 7/8 of the SMs, those of 8 some 3/4.
// Measured, us alone and shared, m x k x n: 1 x 2048 x 2048 6.7, 3.7 (by 4; by 8, where 16 clusters wait for one another, 6.6); 16 x 4096 x 4096 11.4, 5.6; 64 x 4096 x 4096 11.5, 7.8;
// 561 x 1003 x 777 5.5, 6.2 (not shared).
static Plan plan_for(int64_t m, int64_t n, int64_t k) {
    static const int shapes[][2] = {{1, 16}, {1, 32}, {1, 64}, {1, 128}, {2, 128}, {2, 192}, {2, 256}};
    const int64_t sms = sm_count(), kb = ceil_div64(k, KB);
    Plan best = {1, 16, 1};
    double best_cost = 1e300;
    for (const auto& s : shapes) {
        const int cg = s[0], mt = s[1];
        const int64_t tiles = ceil_div64(n, BN * cg) * ceil_div64(m, mt), slots = sms / cg;
        for (int splits = 1; splits <= 8; splits *= 2) {
            if (splits > 1 && (cg > 1 || mt > 64 || tiles * splits > (splits == 2 ? slots : splits == 4 ? slots * 7 / 8 : slots * 3 / 4) || kb < 2 * splits)) break;
            const double per_block = std::max(2.0 * mt, (BN + mt / cg) * KB / 40.0);
            const double item = ceil_div64(kb, splits) * per_block + 1200 + 6.0 * mt + (splits > 1 ? 1000 + 40.0 * mt : 0.0);
            const double cost = ceil_div64(tiles * splits, slots) * item;
            if (cost < best_cost) {
                best_cost = cost;
                best = {cg, mt, splits};
            }
        }
    }
    return best;
}

template <bool OUT16>
static int dispatch(cudaStream_t st, const Plan& pl, const CUtensorMap& tmW, const CUtensorMap& tmX, const Params& p) {
    if (pl.splits > 1) switch (pl.mt) {
        case 16: return launch<1, 16, 10, OUT16, true>(st, tmW, tmX, p, pl.splits);
        case 32: return launch<1, 32, 8, OUT16, true>(st, tmW, tmX, p, pl.splits);
        default: return launch<1, 64, 7, OUT16, true>(st, tmW, tmX, p, pl.splits);
    }
    if (pl.cg == 1) switch (pl.mt) {
        case 16: return launch<1, 16, 11, OUT16, false>(st, tmW, tmX, p, 1);
        case 32: return launch<1, 32, 10, OUT16, false>(st, tmW, tmX, p, 1);
        case 64: return launch<1, 64, 8, OUT16, false>(st, tmW, tmX, p, 1);
        default: return launch<1, 128, 6, OUT16, false>(st, tmW, tmX, p, 1);
    }
    switch (pl.mt) {
        case 128: return launch<2, 128, 8, OUT16, false>(st, tmW, tmX, p, 1);
        case 192: return launch<2, 192, 7, OUT16, false>(st, tmW, tmX, p, 1);
        default: return launch<2, 256, 6, OUT16, false>(st, tmW, tmX, p, 1);
    }
}

// k = 0: the sums are zero, the scales still count (a NaN makes NaN)
template <typename T>
__global__ void __launch_bounds__(256) empty_kernel(int64_t m, int64_t n, const float* __restrict__ sx, const float* __restrict__ sw, T* __restrict__ out, int64_t ldo) {
    dep_sync();
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < m * n; i += static_cast<int64_t>(gridDim.x) * 256)
        out[i / n * ldo + i % n] = static_cast<T>(scaled(0, sx[i / n], sw[i % n]));
}

}  // namespace i8
}  // namespace rmlk

using namespace rmlk;

extern "C" int rmlk_b200_matmul_i8(rmlk_stream_t stream, int out_dtype, int64_t m, int64_t n, int64_t k, const void* x, int64_t ldx, const float* x_scales, const void* w,
                                   int64_t ldw, const float* w_scales, void* out, int64_t ldo, int* status) {
    if (out_dtype != RMLK_F32 && out_dtype != RMLK_F16) return fail(RMLK_ERR_UNSUPPORTED_DTYPE, "unsupported data type for matmul_i8 (f32, f16)");
    if (m < 0 || n < 0 || k < 0 || m >= (1ll << 24) || n >= (1ll << 24)) return fail(RMLK_ERR_INVALID_ARG, "matmul_i8: bad extent");
    if (k > 131071) return fail(RMLK_ERR_INVALID_ARG, "matmul_i8: k above 131071 may overflow the 32-bit sums");
    if (m == 0 || n == 0) return RMLK_OK;
    if (!x_scales || !w_scales || !out || (k > 0 && (!x || !w))) return fail(RMLK_ERR_INVALID_ARG, "matmul_i8: NULL pointer");
    if (ldx < k || ldw < k || ldo < n || ldx >= (1ll << 40) || ldw >= (1ll << 40)) return fail(RMLK_ERR_INVALID_ARG, "matmul_i8: rows overlap, or lie too far apart");
    if (k > 0 && (ldx % 16 || ldw % 16 || !aligned_to(x, 16) || !aligned_to(w, 16))) return fail(RMLK_ERR_INVALID_ARG, "matmul_i8: rows of codes must lie on 16-byte boundaries");
    if (!aligned_to(x_scales, 4) || !aligned_to(w_scales, 4) || !aligned_to(out, dtype_size(out_dtype))) return fail(RMLK_ERR_INVALID_ARG, "matmul_i8: misaligned pointer");
    const cudaStream_t st = as_stream(stream);
    if (k == 0) {
        const dim3 grid(flat_grid(m * n, 256, 8));
        if (out_dtype == RMLK_F32) launch_dep(i8::empty_kernel<float>, grid, dim3(256), 0, st, m, n, x_scales, w_scales, static_cast<float*>(out), ldo);
        else launch_dep(i8::empty_kernel<__half>, grid, dim3(256), 0, st, m, n, x_scales, w_scales, static_cast<__half*>(out), ldo);
        RMLK_CHECK_LAUNCH("matmul_i8 empty_kernel");
        return RMLK_OK;
    }
    const i8::Plan pl = i8::plan_for(m, n, k);
    CUtensorMap tmW, tmX;
    if (!i8::map_2d(&tmW, w, k, n, ldw, umma::BN) || !i8::map_2d(&tmX, x, k, m, ldx, pl.mt / pl.cg)) return fail(RMLK_ERR_INTERNAL, "matmul_i8: cuTensorMapEncodeTiled failed");
    i8::Params p = {};
    p.out = out;
    p.M = m;
    p.N = n;
    p.ldo = ldo;
    p.sx = x_scales;
    p.sw = w_scales;
    p.n_tiles = static_cast<int>(ceil_div64(n, umma::BN * pl.cg));
    p.m_tiles = static_cast<int>(ceil_div64(m, pl.mt));
    if (static_cast<int64_t>(p.n_tiles) * p.m_tiles >= (1ll << 30)) return fail(RMLK_ERR_INVALID_ARG, "matmul_i8: too many tiles");
    p.m_group = std::min(p.m_tiles, 8);
    p.k_blocks = static_cast<int>(ceil_div64(k, i8::KB));
    p.status = status;
    return out_dtype == RMLK_F32 ? i8::dispatch<false>(st, pl, tmW, tmX, p) : i8::dispatch<true>(st, pl, tmW, tmX, p);
}
