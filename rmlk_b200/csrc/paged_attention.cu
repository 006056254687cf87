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

// CTAs of prompt_kernel where all sequences have as many tokens
static int64_t prompt_ctas(int64_t tokens, int64_t batch, int64_t kv_heads, int64_t group, int64_t rows) { return kv_heads * batch * ceil_div64(ceil_div64(tokens, batch) * group, rows); }
// CTAs of a cluster that share the keys of each of them: as many as leave all clusters room at once, with 256 keys each or more.  Clusters of 4 fill 7/8 of the SMs, those
// of 8 some 3/4 (16 of them, f16, 512 rows over 8000 keys: 78 us, with clusters of 4 61).
// One prompt of 16 tokens, 4 query heads of 128 to each of 8 KV heads, f16: over 8000 keys 28 us, 132 without sharing; over 2000 15 and 38.
static int prompt_splits(int64_t ctas, int64_t most_keys) {
    const int64_t sms = sm_count();
    int splits = 1;
    while (splits < 8 && ctas * 2 * splits <= (splits == 1 ? sms : splits == 2 ? sms * 7 / 8 : sms * 3 / 4) && most_keys >= 512 * splits) splits *= 2;
    return splits;
}

template <typename T, int D, bool SHARED>
static int launch_prompt(cudaStream_t st, const Cache& c, const Batch& s, const Attend& a, int64_t ctas, int splits) {
    using L = Prompt<T, D>;
    auto kernel = prompt_kernel<T, D, SHARED>;
    static std::once_flag configured[64];  // the dynamic shared memory limit is raised once per device
    int dev = 0;
    cudaGetDevice(&dev);
    cudaError_t cfg_err = cudaSuccess;
    if (dev >= 0 && dev < 64) std::call_once(configured[dev], [&] { cfg_err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL); });
    RMLK_CUDA(cfg_err);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas * splits));
    cfg.blockDim = dim3(L::THREADS);
    cfg.dynamicSmemBytes = L::TOTAL;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    unsigned na = 0;
    if (SHARED) {
        at[na].id = cudaLaunchAttributeClusterDimension;
        at[na].val.clusterDim.x = splits;
        at[na].val.clusterDim.y = at[na].val.clusterDim.z = 1;
        na++;
    }
    if (dep_launch_enabled()) {
        at[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[na].val.programmaticStreamSerializationAllowed = 1;
        na++;
    }
    cfg.attrs = at;
    cfg.numAttrs = na;
    RMLK_CUDA(cudaLaunchKernelEx(&cfg, kernel, c, s, a, splits));
    RMLK_CHECK_LAUNCH("paged_attention prompt_kernel");
    return RMLK_OK;
}

template <typename T, int D>
static int prompts(cudaStream_t st, const Cache& c, const Batch& s, const Attend& a) {
    constexpr int64_t ROWS = Prompt<T, D>::ROWS;
    const int64_t even = prompt_ctas(s.tokens, s.batch, c.kv_heads, a.group, ROWS);
    const int64_t ctas = s.starts ? c.kv_heads * (s.tokens * a.group / ROWS + std::min<int64_t>(s.batch, s.tokens)) : even;  // (ragged: as many as there can be)
    const int splits = prompt_splits(even, s.width << c.page_log);
    if (ctas * splits > 0x7fffffffll) return fail(RMLK_ERR_INVALID_ARG, "paged_attention: too many tokens");
    return splits > 1 ? launch_prompt<T, D, true>(st, c, s, a, ctas, splits) : launch_prompt<T, D, false>(st, c, s, a, ctas, 1);
}

}  // namespace paged
}  // namespace rmlk

using namespace rmlk;

// Which kernel takes a call: few_kernel shares the keys out over all SMs and reads them once for each 16 query rows; prompt_kernel has a CTA or a cluster of them to 128 or 256
// rows, which walks over all their keys.  With P = batch x kv_heads, few_kernel takes the time of P ceil(rows / 16) tiles spread evenly over the GPU, prompt_kernel that of
// its CTAs, as many at a time as there are SMs.  A CTA with all keys takes as long as `cost` tiles of few_kernel on an SM.  Measured with 8 KV heads over 8000 keys, us (few,
// prompt), B x rows of a KV head:
//   f16 128: 1 x 64 29, 30;  1 x 256 69, 41;  1 x 512 120, 61;  8 x 64 121, 100;  8 x 128 227, 103;  8 x 256 436, 113;  64 x 32 437, 610;  64 x 64 854, 611
//   f32 128: 1 x 64 32, 36;  1 x 256 82, 64;  8 x 64 147, 113;  8 x 128 278, 118;  8 x 256 538, 204;  64 x 32 537, 752;  64 x 64 1051, 757
//   f16 64:  1 x 64 21, 25;  1 x 256 45, 34;  8 x 64 74, 76;  8 x 128 137, 77;  8 x 256 263, 98;  64 x 64 511, 500;  64 x 128 1006, 503
//   f32 64:  1 x 64 23, 34;  1 x 256 50, 42;  8 x 64 85, 125;  8 x 128 158, 130;  8 x 256 302, 136;  64 x 64 589, 719;  64 x 128 1165, 723
// The rule picks the faster one of each but for f16 64, 64 x 64 (2 %).  It knows the table's width, not the lengths: over 600 keys, for which few_kernel's start and joins count most,
// its choice of few_kernel is up to 1.6 times as slow as the other (f16 64: 64 x 64 95, 60; 8 x 64 20, 14; f16 128: 64 x 32 98, 71), under a table of 8000 or 131072 keys alike.
// The new tokens of ragged sequences lie at places that only the device knows: they go to prompt_kernel.
static bool takes_few(bool f32, int64_t tokens, int64_t batch, int64_t kv_heads, int64_t group, int64_t head_dim, int64_t most_keys, bool ragged) {
    if (ragged || batch < 1) return false;
    const double sms = sm_count(), rows = static_cast<double>(tokens / batch) * group, problems = static_cast<double>(batch) * kv_heads;
    const bool pairs = !(f32 && head_dim == 128);  // a CTA of prompt_kernel has two tiles of 128 rows where there are as many
    const double cost = pairs && rows > 128 ? (head_dim == 64 ? 5.5 : 3.1) : (head_dim == 64 ? 4.2 : 2.6), ctas = problems * std::ceil(rows / (pairs ? 256.0 : 128.0));
    const int splits = ctas > sms ? 1 : paged::prompt_splits(static_cast<int64_t>(ctas), most_keys);
    return problems * std::ceil(rows / 16.0) <= cost * sms * std::ceil(ctas / sms) / splits;
}

extern "C" size_t rmlk_b200_paged_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int ragged) {
    if (kv_heads < 1 || q_heads < kv_heads) return 0;
    const int64_t group = q_heads / kv_heads;
    // (with few keys few_kernel has the most calls: enough for a table of any width)
    if (!takes_few(true, tokens, batch, kv_heads, group, head_dim, 0, ragged != 0) && !takes_few(false, tokens, batch, kv_heads, group, head_dim, 0, ragged != 0)) return 0;
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
    if (takes_few(dtype == RMLK_F32, tokens, batch, c.kv_heads, a.group, c.d, s.width << c.page_log, starts != nullptr)) {
        if (!workspace || workspace_bytes < paged::few_workspace(c.d) || !aligned_to(workspace, 16))
            return fail(RMLK_ERR_INVALID_ARG, "paged_attention: the workspace is missing, too small or misaligned (rmlk_b200_paged_attention_workspace_bytes)");
        // Tiles of 8 or 16 rows; one of 16 takes 1.6 times as long over long contexts, where the keys come from HBM, 1.9 times over short ones.  In tiles of 8, of 16, us: 24 rows (24
        // requests, 4 KV heads, 1500 keys) f16 64 20.5, 25.3, f16 128 28.3, 35.2, f32 64 22.4, 26.3, f32 128 33.0, 40.6; over 8000 keys 56, 60; 87, 95; 64, 68; 109, 115.  16 rows (32 requests,
        // 8 heads, 2000 keys): 31.7, 31.3; 49.8, 47.1; 35.8, 34.1; 60.4, 56.0.  40 rows (2 requests, 8 heads, 20000 keys): 41, 43; 64, 66; 47, 47; 78, 78.
        const int rows = s.each * a.group;
        const bool one = rows <= 8 || (rows > 16 && rows <= 24);
        if (dtype == RMLK_F32) {
            if (c.d == 64) return one ? paged::launch_few<float, 64, 1>(st, c, s, a, workspace) : paged::launch_few<float, 64, 2>(st, c, s, a, workspace);
            return one ? paged::launch_few<float, 128, 1>(st, c, s, a, workspace) : paged::launch_few<float, 128, 2>(st, c, s, a, workspace);
        }
        if (c.d == 64) return one ? paged::launch_few<__half, 64, 1>(st, c, s, a, workspace) : paged::launch_few<__half, 64, 2>(st, c, s, a, workspace);
        return one ? paged::launch_few<__half, 128, 1>(st, c, s, a, workspace) : paged::launch_few<__half, 128, 2>(st, c, s, a, workspace);
    }
    if (dtype == RMLK_F32) return c.d == 64 ? paged::prompts<float, 64>(st, c, s, a) : paged::prompts<float, 128>(st, c, s, a);
    return c.d == 64 ? paged::prompts<__half, 64>(st, c, s, a) : paged::prompts<__half, 128>(st, c, s, a);
}
