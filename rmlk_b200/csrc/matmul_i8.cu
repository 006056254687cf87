// Products of 8-bit integers with a scale per row of X (token) and per row of W (channel).
//
//   out[m][n] = (sum_k x[m][k] w[n][k]) sx[m] sw[n]
//
// The sum is exact in 32 bits (k <= 131071 and |x w| <= 2^14), so it does not depend on the order of its parts.
#include "common.cuh"

namespace rmlk {
namespace i8 {

__device__ __forceinline__ float scaled(int acc, float a, float b) {
    const float v = static_cast<float>(acc), t = a * b;
    // a b first where it is a normal number: acc times one of them alone may leave the range although the result does not
    return t >= 1.17549435e-38f && t < INFINITY ? v * t : v * a * b;
}

template <typename T>
__global__ void __launch_bounds__(256) tile_kernel(int64_t m, int64_t n, int64_t k, const int8_t* __restrict__ x, int64_t ldx, const float* __restrict__ sx,
                                                   const int8_t* __restrict__ w, int64_t ldw, const float* __restrict__ sw, T* __restrict__ out, int64_t ldo) {
    dep_sync();
    __shared__ int s_x[64][17], s_w[64][17];
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 64, n0 = static_cast<int64_t>(blockIdx.x) * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int64_t k0 = 0; k0 < k; k0 += 64) {
        for (int i = threadIdx.x; i < 64 * 16; i += 256) {
            const int r = i >> 4, c = i & 15;
            int a = 0, b = 0;
            const int64_t kk = k0 + 4 * c, left = k - kk;
            const uint32_t mask = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1;
            if (m0 + r < m && mask) a = *reinterpret_cast<const int*>(x + (m0 + r) * ldx + kk) & mask;
            if (n0 + r < n && mask) b = *reinterpret_cast<const int*>(w + (n0 + r) * ldw + kk) & mask;
            s_x[r][c] = a;
            s_w[r][c] = b;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 16; c++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(s_x[ty + 16 * i][c], s_w[tx + 16 * j][c], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const int64_t r = m0 + ty + 16 * i, c = n0 + tx + 16 * j;
            if (r < m && c < n) out[r * ldo + c] = static_cast<T>(scaled(acc[i][j], sx[r], sw[c]));
        }
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
    if (ldx < k || ldw < k || ldo < n) return fail(RMLK_ERR_INVALID_ARG, "matmul_i8: rows overlap");
    if (k > 0 && (ldx % 16 || ldw % 16 || !aligned_to(x, 16) || !aligned_to(w, 16))) return fail(RMLK_ERR_INVALID_ARG, "matmul_i8: rows of codes must lie on 16-byte boundaries");
    if (!aligned_to(x_scales, 4) || !aligned_to(w_scales, 4) || !aligned_to(out, dtype_size(out_dtype))) return fail(RMLK_ERR_INVALID_ARG, "matmul_i8: misaligned pointer");
    (void)status;
    const dim3 grid(static_cast<unsigned>(ceil_div64(n, 64)), static_cast<unsigned>(ceil_div64(m, 64)));
    if (grid.y > 65535) return fail(RMLK_ERR_INVALID_ARG, "matmul_i8: too many rows");
    if (out_dtype == RMLK_F32)
        launch_dep(i8::tile_kernel<float>, grid, dim3(256), 0, as_stream(stream), m, n, k, static_cast<const int8_t*>(x), ldx, x_scales, static_cast<const int8_t*>(w), ldw,
                   w_scales, static_cast<float*>(out), ldo);
    else
        launch_dep(i8::tile_kernel<__half>, grid, dim3(256), 0, as_stream(stream), m, n, k, static_cast<const int8_t*>(x), ldx, x_scales, static_cast<const int8_t*>(w), ldw,
                   w_scales, static_cast<__half*>(out), ldo);
    RMLK_CHECK_LAUNCH("matmul_i8 tile_kernel");
    return RMLK_OK;
}
