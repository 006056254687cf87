// Attention over a paged cache of 8-bit codes (paged.cuh): softmax(scale q k^T) v, k and v = code times the scale of their page and head.
#include <mutex>

#include "paged_few.cuh"

namespace rmlk {
namespace paged {

__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(__half x) { return __half2float(x); }

// One warp per (new token, query head), one key after the other.
template <typename T, int D>
__global__ void __launch_bounds__(128) row_kernel(const Cache c, const Batch q, const Attend a) {
    dep_sync();
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int64_t row = item / a.q_heads;
    const int h = static_cast<int>(item - row * a.q_heads), lane = threadIdx.x & 31, kv = h / a.group;
    if (row >= q.tokens) return;
    int b;
    int64_t first = 0, count = 0;
    if (!q.starts) {
        b = static_cast<int>(row / q.each);
        q.rows(b, first, count);
    } else {
        for (b = 0; b < q.batch; b++) {
            q.rows(b, first, count);
            if (row >= first && row < first + count) break;
        }
        if (b == q.batch) return;
    }
    constexpr int N = D / 32;
    float x[N], acc[N];
    const T* src = static_cast<const T*>(a.q) + row * a.qs + static_cast<int64_t>(h) * D;
#pragma unroll
    for (int i = 0; i < N; i++) {
        x[i] = as_f32(src[lane + 32 * i]);
        acc[i] = 0.f;
    }
    const int64_t see = q.lens[b] - count + row - first + 1;
    float top = -INFINITY, sum = 0.f;
    bool bad = false;
    for (int64_t t = 0; t < see; t++) {
        const int64_t at = t >> c.page_log;
        const int page = at < q.width ? q.table[b * q.width + at] : -1;
        if (page < 0 || page >= c.pages) {
            bad = true;
            break;
        }
        const int64_t block = static_cast<int64_t>(page) * c.kv_heads + kv, off = (block * c.page + (t & (c.page - 1))) * D;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) s = fmaf(x[i], static_cast<float>(c.k[off + lane + 32 * i]), s);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= c.ks[block] * a.scale;
        const float most = s > top || s != s ? s : top, corr = top == -INFINITY ? 0.f : expf(top - most), e = expf(s - most);
        top = most;
        sum = sum * corr + e;
        const float w = e * c.vs[block];
#pragma unroll
        for (int i = 0; i < N; i++) acc[i] = fmaf(w, static_cast<float>(c.v[off + lane + 32 * i]), acc[i] * corr);
    }
    if (bad && a.status && lane == 0) *a.status = RMLK_ERR_INVALID_ARG;
    T* o = static_cast<T*>(a.out) + row * a.os + static_cast<int64_t>(h) * D;
#pragma unroll
    for (int i = 0; i < N; i++) o[lane + 32 * i] = static_cast<T>(bad ? __int_as_float(0x7fc00000) : see <= 0 ? 0.f : acc[i] / sum);
}

template <typename T, int D, int NR>
static int launch_few(cudaStream_t st, const Cache& c, const Batch& s, const Attend& a, void* workspace) {
    using L = Few<T, D, NR>;
    auto kernel = few_kernel<T, D, NR>;
    static std::once_flag configured[64];  // the dynamic shared memory limit is raised once per device
    int dev = 0;
    cudaGetDevice(&dev);
    cudaError_t cfg_err = cudaSuccess;
    if (dev >= 0 && dev < 64) std::call_once(configured[dev], [&] { cfg_err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM); });
    RMLK_CUDA(cfg_err);
    const int rows = s.each * a.group, tiles = (rows + L::ROWS - 1) / L::ROWS;
    RMLK_CUDA(launch_dep(kernel, dim3(static_cast<unsigned>(sm_count() * L::PER_SM)), dim3(128), L::SMEM, st, c, s, a, tiles, static_cast<unsigned*>(workspace),
                         reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + COUNTERS * 4)));
    RMLK_CHECK_LAUNCH("paged_attention few_kernel");
    return RMLK_OK;
}

}  // namespace paged
}  // namespace rmlk

using namespace rmlk;

// Rows of a KV head (new tokens x query heads that share it) up to which few_kernel takes a call.
constexpr int64_t FEW_ROWS = 64;
static bool takes_few(int64_t tokens, int64_t batch, int64_t group, bool ragged) { return !ragged && batch > 0 && tokens / batch * group <= FEW_ROWS; }

extern "C" size_t rmlk_b200_paged_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int ragged) {
    if (kv_heads < 1 || q_heads < kv_heads || !takes_few(tokens, batch, q_heads / kv_heads, ragged != 0)) return 0;
    return paged::few_workspace(head_dim);
}

extern "C" int rmlk_b200_paged_attention(rmlk_stream_t stream, int dtype, const rmlk_paged_cache* cache, int64_t tokens, int64_t batch, int64_t q_heads, const int32_t* starts,
                                         const int32_t* lens, const int32_t* table, int64_t table_width, const void* q, int64_t q_stride, float scale, void* out,
                                         int64_t out_stride, void* workspace, size_t workspace_bytes, int* status) {
    if (dtype != RMLK_F32 && dtype != RMLK_F16) return fail(RMLK_ERR_UNSUPPORTED_DTYPE, "unsupported data type for paged_attention (f32, f16)");
    paged::Cache c;
    paged::Batch s;
    const int rc = paged::take("paged_attention", cache, tokens, batch, starts, lens, table, table_width, c, s);
    if (rc != RMLK_OK) return rc;
    if (q_heads < 1 || q_heads % c.kv_heads || q_heads / c.kv_heads > 64) return fail(RMLK_ERR_INVALID_ARG, "paged_attention: q_heads must be a multiple of kv_heads, up to 64 for each");
    if (tokens == 0 || batch == 0) return RMLK_OK;
    if (!q || !out) return fail(RMLK_ERR_INVALID_ARG, "paged_attention: NULL pointer");
    const int64_t e = static_cast<int64_t>(dtype_size(dtype)), per = 16 / e;
    if (q_stride < q_heads * c.d || out_stride < q_heads * c.d) return fail(RMLK_ERR_INVALID_ARG, "paged_attention: rows overlap");
    if (!aligned_to(q, 16) || !aligned_to(out, 16) || q_stride % per || out_stride % per) return fail(RMLK_ERR_INVALID_ARG, "paged_attention: rows must lie on 16-byte boundaries");
    paged::Attend a = {q, out, q_stride, out_stride, static_cast<int>(q_heads), static_cast<int>(q_heads / c.kv_heads), scale, status};
    if (takes_few(tokens, batch, a.group, starts != nullptr)) {
        if (!workspace || workspace_bytes < paged::few_workspace(c.d) || !aligned_to(workspace, 16))
            return fail(RMLK_ERR_INVALID_ARG, "paged_attention: the workspace is missing, too small or misaligned (rmlk_b200_paged_attention_workspace_bytes)");
        const cudaStream_t st = as_stream(stream);
        const bool one = s.each * a.group <= 8;
        if (dtype == RMLK_F32) {
            if (c.d == 64) return one ? paged::launch_few<float, 64, 1>(st, c, s, a, workspace) : paged::launch_few<float, 64, 2>(st, c, s, a, workspace);
            return one ? paged::launch_few<float, 128, 1>(st, c, s, a, workspace) : paged::launch_few<float, 128, 2>(st, c, s, a, workspace);
        }
        if (c.d == 64) return one ? paged::launch_few<__half, 64, 1>(st, c, s, a, workspace) : paged::launch_few<__half, 64, 2>(st, c, s, a, workspace);
        return one ? paged::launch_few<__half, 128, 1>(st, c, s, a, workspace) : paged::launch_few<__half, 128, 2>(st, c, s, a, workspace);
    }
    const int64_t ctas = ceil_div64(tokens * q_heads, 4);
    if (ctas > 0x7fffffffll) return fail(RMLK_ERR_INVALID_ARG, "paged_attention: too many tokens");
    const dim3 grid(static_cast<unsigned>(ctas));
    if (dtype == RMLK_F32) launch_dep(c.d == 64 ? paged::row_kernel<float, 64> : paged::row_kernel<float, 128>, grid, dim3(128), 0, as_stream(stream), c, s, a);
    else launch_dep(c.d == 64 ? paged::row_kernel<__half, 64> : paged::row_kernel<__half, 128>, grid, dim3(128), 0, as_stream(stream), c, s, a);
    RMLK_CHECK_LAUNCH("paged_attention row_kernel");
    return RMLK_OK;
}
