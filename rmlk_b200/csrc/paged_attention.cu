// Attention over a paged cache of 8-bit codes (paged.cuh): softmax(scale q k^T) v, k and v = code times the scale of their page and head.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "paged_few.cuh"
#include "paged_prompt.cuh"

namespace rmlk {
namespace paged {

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

template <typename T, int D>
static int launch_prompt(cudaStream_t st, const Cache& c, const Batch& s, const Attend& a) {
    using L = Prompt<T, D>;
    auto kernel = prompt_kernel<T, D>;
    static std::once_flag configured[64];  // the dynamic shared memory limit is raised once per device
    int dev = 0;
    cudaGetDevice(&dev);
    cudaError_t cfg_err = cudaSuccess;
    if (dev >= 0 && dev < 64) std::call_once(configured[dev], [&] { cfg_err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL); });
    RMLK_CUDA(cfg_err);
    constexpr int64_t ROWS = L::ROWS;
    const int64_t tokens = s.tokens, batch = s.batch;
    const int64_t items = s.starts ? tokens * a.group / ROWS + std::min(batch, tokens) : batch * ceil_div64(s.each * a.group, ROWS);  // ragged: as many as there can be
    if (items * c.kv_heads > 0x7fffffffll) return fail(RMLK_ERR_INVALID_ARG, "paged_attention: too many tokens");
    RMLK_CUDA(launch_dep(kernel, dim3(static_cast<unsigned>(items * c.kv_heads)), dim3(L::THREADS), L::TOTAL, st, c, s, a));
    RMLK_CHECK_LAUNCH("paged_attention prompt_kernel");
    return RMLK_OK;
}

}  // namespace paged
}  // namespace rmlk

using namespace rmlk;

// Which kernel takes a call: few_kernel shares the keys out over all SMs and reads them once for each 16 query rows; prompt_kernel has a CTA per SM to 128 or 256 rows, which
// walks over all their keys.  With P = batch x kv_heads, few_kernel takes the time of P ceil(rows / 16) tiles spread evenly over the GPU, prompt_kernel that of its CTAs, as many at
// a time as there are SMs.  A CTA takes as long as `cost` tiles of few_kernel on an SM.  Measured with 8 KV heads over 8000 keys, us (few, prompt), B x rows of a KV head:
//   f16 128: 8 x 64 112, 156;  8 x 128 210, 159;  1 x 512 112, 180;  8 x 256 421, 187;  64 x 32 407, 604;  64 x 64 793, 603
//   f32 128: 8 x 64 139, 200;  8 x 128 260, 203;  8 x 256 505, 204;  64 x 32 505, 755;  64 x 64 992, 760
//   f16 64:  8 x 128 128, 136;  8 x 256 246, 175;  64 x 64 478, 511;  64 x 128 944, 512
//   f32 64:  8 x 128 150, 187;  8 x 256 287, 259;  64 x 64 564, 764;  64 x 128 1115, 772
// The new tokens of ragged sequences lie at places that only the device knows: they go to prompt_kernel.
static bool takes_few(bool f32, int64_t tokens, int64_t batch, int64_t kv_heads, int64_t group, int64_t head_dim, bool ragged) {
    if (ragged || batch < 1) return false;
    const double sms = sm_count(), rows = static_cast<double>(tokens / batch) * group, problems = static_cast<double>(batch) * kv_heads;
    const bool pairs = !(f32 && head_dim == 128);  // a CTA of prompt_kernel has two tiles of 128 rows where there are as many
    const double cost = pairs && rows > 128 ? (head_dim == 64 ? 5.5 : 3.1) : (head_dim == 64 ? 4.2 : 2.6);
    return problems * std::ceil(rows / 16.0) <= cost * sms * std::ceil(problems * std::ceil(rows / (pairs ? 256.0 : 128.0)) / sms);
}

extern "C" size_t rmlk_b200_paged_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int ragged) {
    if (kv_heads < 1 || q_heads < kv_heads) return 0;
    const int64_t group = q_heads / kv_heads;
    if (!takes_few(true, tokens, batch, kv_heads, group, head_dim, ragged != 0) && !takes_few(false, tokens, batch, kv_heads, group, head_dim, ragged != 0)) return 0;
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
    if (tokens * (q_heads / c.kv_heads) >= (1ll << 31)) return fail(RMLK_ERR_INVALID_ARG, "paged_attention: too many tokens");
    if (!(scale - scale == 0.f)) return fail(RMLK_ERR_INVALID_ARG, "paged_attention: the scale must be finite");
    if (tokens == 0 || batch == 0) return RMLK_OK;
    if (!q || !out) return fail(RMLK_ERR_INVALID_ARG, "paged_attention: NULL pointer");
    const int64_t e = static_cast<int64_t>(dtype_size(dtype)), per = 16 / e;
    if (q_stride < q_heads * c.d || out_stride < q_heads * c.d) return fail(RMLK_ERR_INVALID_ARG, "paged_attention: rows overlap");
    if (!aligned_to(q, 16) || !aligned_to(out, 16) || q_stride % per || out_stride % per) return fail(RMLK_ERR_INVALID_ARG, "paged_attention: rows must lie on 16-byte boundaries");
    paged::Attend a = {q, out, q_stride, out_stride, static_cast<int>(q_heads), static_cast<int>(q_heads / c.kv_heads), scale, status};
    const cudaStream_t st = as_stream(stream);
    if (takes_few(dtype == RMLK_F32, tokens, batch, c.kv_heads, a.group, c.d, starts != nullptr)) {
        if (!workspace || workspace_bytes < paged::few_workspace(c.d) || !aligned_to(workspace, 16))
            return fail(RMLK_ERR_INVALID_ARG, "paged_attention: the workspace is missing, too small or misaligned (rmlk_b200_paged_attention_workspace_bytes)");
        const bool one = s.each * a.group <= 8;
        if (dtype == RMLK_F32) {
            if (c.d == 64) return one ? paged::launch_few<float, 64, 1>(st, c, s, a, workspace) : paged::launch_few<float, 64, 2>(st, c, s, a, workspace);
            return one ? paged::launch_few<float, 128, 1>(st, c, s, a, workspace) : paged::launch_few<float, 128, 2>(st, c, s, a, workspace);
        }
        if (c.d == 64) return one ? paged::launch_few<__half, 64, 1>(st, c, s, a, workspace) : paged::launch_few<__half, 64, 2>(st, c, s, a, workspace);
        return one ? paged::launch_few<__half, 128, 1>(st, c, s, a, workspace) : paged::launch_few<__half, 128, 2>(st, c, s, a, workspace);
    }
    if (dtype == RMLK_F32) return c.d == 64 ? paged::launch_prompt<float, 64>(st, c, s, a) : paged::launch_prompt<float, 128>(st, c, s, a);
    return c.d == 64 ? paged::launch_prompt<__half, 64>(st, c, s, a) : paged::launch_prompt<__half, 128>(st, c, s, a);
}
