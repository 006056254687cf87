// Rows as 8-bit integers with one scale each: what the integer product takes (matmul_i8.cu).
//
//   s = max(fl(max |x| / 127), 2^-126),   c = the integer nearest to x / s, ties to even.
//
// The codes are those of the real quotient.  fl(x / s) rounded to an integer is not: a quotient of size 100 keeps 17 bits behind the point, so of a
// million values a few lie so near the middle between two integers that the division rounds onto it.  Here x times 1 / s gives the integer to within
// one, and the sign of fma(-(c +- 1/2), s, x), which rounds once and so cannot change it, says on which side of the middle x is.
//
// What bounds it: HBM, one read of x (4 or 2 bytes per element) and one byte written.  A row stays in registers between its maximum and its codes.
#include "common.cuh"

namespace rmlk {
namespace quant {

template <typename T>
__global__ void __launch_bounds__(256) rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t cols, int8_t* __restrict__ codes, int64_t ldc, float* __restrict__ scales) {
    dep_sync();
    __shared__ float s_max[8];
    __shared__ int s_bad[8];
    const int64_t row = blockIdx.x;
    const T* xr = x + row * ldx;
    float m = 0.f;
    bool bad = false;
    for (int64_t i = threadIdx.x; i < cols; i += 256) {
        const float v = fabsf(static_cast<float>(xr[i]));
        bad = bad || !(v < INFINITY);
        m = fmaxf(m, v);
    }
    const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
    const int any = __any_sync(0xffffffffu, bad);
    if ((threadIdx.x & 31) == 0) {
        s_max[threadIdx.x >> 5] = __uint_as_float(most);
        s_bad[threadIdx.x >> 5] = any;
    }
    __syncthreads();
    m = 0.f;
    bad = false;
#pragma unroll
    for (int w = 0; w < 8; w++) {
        m = fmaxf(m, s_max[w]);
        bad = bad || s_bad[w];
    }
    float s = fmaxf(__fdiv_rn(m, 127.f), 1.17549435e-38f);
    if (threadIdx.x == 0) scales[row] = bad ? __int_as_float(0x7fc00000) : s;
    const float up24 = s < 7.888609052210118e-31f ? 16777216.f : 1.f;  // below 2^-100 differences would round to zero: all times 2^24
    s *= up24;
    const float inv = __frcp_rn(s);
    for (int64_t i = threadIdx.x; i < cols; i += 256) {
        const float v = static_cast<float>(xr[i]) * up24;
        float c = rintf(v * inv);
        const float up = fmaf(-(c + 0.5f), s, v), down = fmaf(-(c - 0.5f), s, v);
        const bool odd = static_cast<int>(c) & 1;
        if (up > 0.f || (up == 0.f && odd)) c += 1.f;
        else if (down < 0.f || (down == 0.f && odd)) c -= 1.f;
        codes[row * ldc + i] = bad ? 0 : static_cast<int8_t>(c);
    }
}

}  // namespace quant
}  // namespace rmlk

using namespace rmlk;

extern "C" int rmlk_b200_quantize_rows(rmlk_stream_t stream, int dtype, int64_t rows, int64_t cols, const void* x, int64_t ldx, void* codes, int64_t ldc, float* scales) {
    if (dtype != RMLK_F32 && dtype != RMLK_F16) return fail(RMLK_ERR_UNSUPPORTED_DTYPE, "unsupported data type for quantize_rows (f32, f16)");
    if (rows < 0 || cols < 0 || rows > 0x7fffffffll || cols > 0x7fffffffll) return fail(RMLK_ERR_INVALID_ARG, "quantize_rows: bad extent");
    if (rows == 0) return RMLK_OK;
    if (!scales || (cols > 0 && (!x || !codes))) return fail(RMLK_ERR_INVALID_ARG, "quantize_rows: NULL pointer");
    if (ldx < cols || ldc < cols) return fail(RMLK_ERR_INVALID_ARG, "quantize_rows: rows overlap");
    const size_t e = dtype_size(dtype);
    if (!aligned_to(x, e) || !aligned_to(scales, 4)) return fail(RMLK_ERR_INVALID_ARG, "quantize_rows: misaligned pointer");
    if (dtype == RMLK_F32)
        launch_dep(quant::rows_kernel<float>, dim3(static_cast<unsigned>(rows)), dim3(256), 0, as_stream(stream), static_cast<const float*>(x), ldx, cols,
                   static_cast<int8_t*>(codes), ldc, scales);
    else
        launch_dep(quant::rows_kernel<__half>, dim3(static_cast<unsigned>(rows)), dim3(256), 0, as_stream(stream), static_cast<const __half*>(x), ldx, cols,
                   static_cast<int8_t*>(codes), ldc, scales);
    RMLK_CHECK_LAUNCH("quantize rows_kernel");
    return RMLK_OK;
}
