// Rows as 8-bit integers with one scale each: what the integer product takes (matmul_i8.cu).
//
//   s = max(fl(max |x| / 127), 2^-126),   c = the integer nearest to x / s, ties to even.
//
// The codes are those of the real quotient.  fl(x / s) rounded to an integer is not: a quotient of size 100 keeps 17 bits behind the point, so of a
// million values a few lie so near the middle between two integers that the division rounds onto it.  Here x times 1 / s, off by less than 4e-5, gives the integer, and where it
// lies within 1e-4 of a middle the sign of fma(-(c +- 1/2), s, x), which rounds once and so cannot change it, says on which side x is.
//
// What bounds it: HBM, one read of x (4 or 2 bytes per element) and one byte written.  A row stays in registers between its maximum and its codes: a warp to a row of up to
// 256 values (512 in f16; 1024 in f32 where rows are many), else a CTA; rows off 16-byte boundaries, and longer than a CTA's registers, are read twice.
// [4096, 14336] f16: 37 us, 4.7 TB/s; with a branch for each value instead of each four 64.  [4096, 4096] f16: 13 us, read twice 28.  [16384, 4096] f32: 55 us, 6.1 TB/s.
#include "common.cuh"

namespace rmlk {
namespace quant {

struct RowScale;
__device__ __noinline__ uint32_t exact_codes(RowScale r, float x0, float x1, float x2, float x3);

struct RowScale {
    float s, up, by;  // the scale, times `up`; a value times `by` is the quotient
    bool bad;
    // from the largest magnitude's bits
    __device__ __forceinline__ float set(uint32_t most) {
        bad = most >= 0x7f800000u;
        const float scale = fmaxf(__fdiv_rn(__uint_as_float(most), 127.f), 1.17549435e-38f);
        up = scale < 7.888609052210118e-31f ? 16777216.f : 1.f;  // below 2^-100 differences would round to zero: all times 2^24
        s = scale * up;
        by = __frcp_rn(s) * up;
        return bad ? __int_as_float(0x7fc00000) : scale;
    }
    // the quotient rounded to an integer in the lowest bits, nearly always the right one
    __device__ __forceinline__ float rounded(float x) const { return fmaf(x, by, 12582912.f); }  // 1.5 2^23
    __device__ __forceinline__ bool near_middle(float x, float sum) const { return fabsf(fmaf(x, by, -(sum - 12582912.f))) > 0.4999f; }
    __device__ __forceinline__ int exact(float x) const {
        const float v = x * up;
        float c = rounded(x) - 12582912.f;
        const float above = fmaf(-(c + 0.5f), s, v), below = fmaf(-(c - 0.5f), s, v);
        const bool odd = static_cast<int>(c) & 1;
        if (above > 0.f || (above == 0.f && odd)) c += 1.f;
        else if (below < 0.f || (below == 0.f && odd)) c -= 1.f;
        return static_cast<int>(c);
    }
    __device__ __forceinline__ int code(float x) const {
        const float sum = rounded(x);
        return bad ? 0 : near_middle(x, sum) ? exact(x) : __float_as_int(sum);  // (its lowest byte)
    }
    // four codes as the bytes of a word
    __device__ __forceinline__ uint32_t codes(const float (&x)[4]) const {
        float sum[4];
        bool near = false;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            sum[i] = rounded(x[i]);
            near = near || near_middle(x[i], sum[i]);
        }
        if (near) return exact_codes(*this, x[0], x[1], x[2], x[3]);  // (one word in a thousand)
        const uint32_t w = __byte_perm(__byte_perm(__float_as_uint(sum[0]), __float_as_uint(sum[1]), 0x0040), __byte_perm(__float_as_uint(sum[2]), __float_as_uint(sum[3]), 0x0040), 0x5410);
        return bad ? 0u : w;
    }
};

__device__ __noinline__ uint32_t exact_codes(RowScale r, float x0, float x1, float x2, float x3) {
    return __byte_perm(__byte_perm(r.code(x0), r.code(x1), 0x0040), __byte_perm(r.code(x2), r.code(x3), 0x0040), 0x5410);
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <int GROUP>
__device__ __forceinline__ uint32_t group_max(uint32_t m, uint32_t* s_max) {
    m = __reduce_max_sync(0xffffffffu, m);
    if constexpr (GROUP > 32) {
        if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < GROUP / 32; w++) m = max(m, s_max[w]);
    }
    return m;
}

// Rows on 16-byte boundaries, V values to a 16-byte load; GROUP threads to a row, ITERS loads to a thread.
template <typename T, int GROUP, int ITERS>
__global__ void __launch_bounds__(GROUP > 256 ? GROUP : 256) packs_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int cols, int8_t* __restrict__ codes, int64_t ldc,
                                                                         float* __restrict__ scales) {
    dep_sync();
    constexpr int V = 16 / sizeof(T), CTA = GROUP > 256 ? GROUP : 256;
    __shared__ uint32_t s_max[GROUP / 32];
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (CTA / GROUP) + threadIdx.x / GROUP;
    if (row >= rows) return;  // (a whole warp; where a CTA has one row, never)
    const int me = threadIdx.x % GROUP;
    const T* xr = x + row * ldx;
    Pack<T, V> p[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; i++) {
        const int at = (i * GROUP + me) * V;
        if (at + V <= cols) {
            p[i] = load_pack<T, V>(xr + at);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) p[i].v[e] = at + e < cols ? xr[at + e] : static_cast<T>(0.f);
        }
    }
    uint32_t most = 0;
    if constexpr (sizeof(T) == 2) {  // magnitudes of f16 are in the order of their bits: two at a time
        uint32_t m2 = 0;
#pragma unroll
        for (int i = 0; i < ITERS; i++)
#pragma unroll
            for (int e = 0; e < V; e += 2) m2 = __vmaxu2(m2, reinterpret_cast<const uint32_t&>(p[i].v[e]) & 0x7fff7fffu);
        most = magnitude(__half2float(__ushort_as_half(static_cast<unsigned short>(max(m2 & 0xffffu, m2 >> 16)))));
    } else {
#pragma unroll
        for (int i = 0; i < ITERS; i++)
#pragma unroll
            for (int e = 0; e < V; e++) most = max(most, magnitude(static_cast<float>(p[i].v[e])));
    }
    most = group_max<GROUP>(most, s_max);
    RowScale r;
    const float scale = r.set(most);
    if (me == 0) scales[row] = scale;
#pragma unroll
    for (int i = 0; i < ITERS; i++) {
        const int at = (i * GROUP + me) * V;
        if (at >= cols) continue;
        Pack<int8_t, V> c;
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            const float x[4] = {static_cast<float>(p[i].v[e]), static_cast<float>(p[i].v[e + 1]), static_cast<float>(p[i].v[e + 2]), static_cast<float>(p[i].v[e + 3])};
            reinterpret_cast<uint32_t&>(c.v[e]) = r.codes(x);
        }
        int8_t* to = codes + row * ldc + at;
        if (at + V <= cols) {
            store_pack<int8_t, V>(to, c);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++)
                if (at + e < cols) to[e] = c.v[e];
        }
    }
}

// Any rows: a CTA each, read twice.
template <typename T>
__global__ void __launch_bounds__(256) rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t cols, int8_t* __restrict__ codes, int64_t ldc, float* __restrict__ scales) {
    dep_sync();
    __shared__ uint32_t s_max[8];
    const int64_t row = blockIdx.x;
    const T* xr = x + row * ldx;
    uint32_t most = 0;
    for (int64_t i = threadIdx.x; i < cols; i += 256) most = max(most, magnitude(static_cast<float>(xr[i])));
    most = group_max<256>(most, s_max);
    RowScale r;
    const float scale = r.set(most);
    if (threadIdx.x == 0) scales[row] = scale;
    for (int64_t i = threadIdx.x; i < cols; i += 256) codes[row * ldc + i] = static_cast<int8_t>(r.code(static_cast<float>(xr[i])));
}

template <typename T, int GROUP, int ITERS>
static void packs(cudaStream_t st, const T* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* codes, int64_t ldc, float* scales) {
    constexpr int CTA = GROUP > 256 ? GROUP : 256;
    launch_dep(packs_kernel<T, GROUP, ITERS>, dim3(static_cast<unsigned>(ceil_div64(rows, CTA / GROUP))), dim3(CTA), 0, st, x, ldx, rows, static_cast<int>(cols), codes, ldc, scales);
}

template <typename T>
static void quantize(cudaStream_t st, const T* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* codes, int64_t ldc, float* scales) {
    constexpr int V = 16 / sizeof(T);
    const int64_t loads = ceil_div64(cols, V);
    const bool whole = aligned_to(x, 16) && ldx % V == 0 && aligned_to(codes, V) && ldc % V == 0 && loads <= 512 * 8;
    if (!whole) launch_dep(rows_kernel<T>, dim3(static_cast<unsigned>(rows)), dim3(256), 0, st, x, ldx, cols, codes, ldc, scales);
    else if (loads <= 32) packs<T, 32, 1>(st, x, ldx, rows, cols, codes, ldc, scales);
    else if (loads <= 64) packs<T, 32, 2>(st, x, ldx, rows, cols, codes, ldc, scales);
    else if (V == 4 && loads <= 256 && rows > 2 * sm_count()) packs<T, 32, 8>(st, x, ldx, rows, cols, codes, ldc, scales);  // ([4096, 1024] 5.4 us, with CTAs 6.5; f16, [4096, 2048]: 14.3, with CTAs 8.2)
    else if (loads <= 256) packs<T, 256, 1>(st, x, ldx, rows, cols, codes, ldc, scales);
    else if (loads <= 512) packs<T, 256, 2>(st, x, ldx, rows, cols, codes, ldc, scales);
    else if (loads <= 1024) packs<T, 256, 4>(st, x, ldx, rows, cols, codes, ldc, scales);
    else if (loads <= 2048) packs<T, 512, 4>(st, x, ldx, rows, cols, codes, ldc, scales);
    else packs<T, 512, 8>(st, x, ldx, rows, cols, codes, ldc, scales);
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
    const cudaStream_t st = as_stream(stream);
    if (dtype == RMLK_F32) quant::quantize(st, static_cast<const float*>(x), ldx, rows, cols, static_cast<int8_t*>(codes), ldc, scales);
    else quant::quantize(st, static_cast<const __half*>(x), ldx, rows, cols, static_cast<int8_t*>(codes), ldc, scales);
    RMLK_CHECK_LAUNCH("quantize_rows");
    return RMLK_OK;
}
