// New keys and values into a paged cache of 8-bit codes, the keys rotated on the way; the queries rotated beside them.
//
//   r = x cos[p] + (-x[D/2:], x[:D/2]) sin[p]       (products of fp32 values are exact in fp64; one rounding to fp32)
//   2^e: the least power of two with max |r| <= 127 2^e over the new tokens of a block (page, head), at least the block's present scale
//   code = rne(r 2^-e)
//
// Scales are powers of two because a block fills over many calls: where its scale grows, the codes in it are divided by a power of two, so
// that after any number of steps a code is off by less than one step of the final scale (1/2 + 1/4 + ...); ratios of any size would add half a step
// each time.  It costs up to one bit of the eight (a scale of max / 127 is up to twice as fine).
#include <algorithm>

#include "paged.cuh"

namespace rmlk {
namespace paged {

int take(const char* what, const rmlk_paged_cache* cache, int64_t tokens, int64_t batch, const int32_t* starts, const int32_t* lens, const int32_t* table, int64_t table_width,
         Cache& c, Batch& q) {
    auto bad = [&](const char* why) { return fail(RMLK_ERR_INVALID_ARG, std::string(what) + ": " + why); };
    if (!cache) return bad("NULL cache");
    const int64_t page = cache->page_size, d = cache->head_dim;
    if (page != 16 && page != 32 && page != 64 && page != 128) return bad("page_size must be 16, 32, 64 or 128");
    if (d != 64 && d != 128) return bad("head_dim must be 64 or 128");
    if (cache->pages < 0 || cache->pages >= (1ll << 31) || cache->kv_heads < 1 || cache->kv_heads > 65535 || cache->pages * cache->kv_heads >= (1ll << 31))
        return bad("bad cache extent");
    if (tokens < 0 || tokens >= (1ll << 31) || batch < 0 || batch >= (1ll << 24) || table_width < 0 || table_width >= (1ll << 31) / page) return bad("bad extent");
    if (static_cast<double>(batch) * static_cast<double>(table_width + 1) * static_cast<double>(cache->kv_heads) > 1e13) return bad("bad extent");  // (unit counts times CTAs stay in 63 bits)
    if (tokens > 0 && batch > 0 && !starts && tokens % batch) return bad("without starts, tokens must be a multiple of batch");
    if (tokens > 0 && batch > 0) {
        if (!lens || (!table && table_width > 0)) return bad("NULL pointer");
        if (cache->pages < 1) return bad("a cache without pages");
        if (!cache->k || !cache->v || !cache->k_scales || !cache->v_scales) return bad("NULL pointer in the cache");
        if (!aligned_to(cache->k, 16) || !aligned_to(cache->v, 16) || !aligned_to(cache->k_scales, 4) || !aligned_to(cache->v_scales, 4) || !aligned_to(lens, 4) ||
            !aligned_to(table, 4) || !aligned_to(starts, 4))
            return bad("misaligned pointer");
    }
    c.k = static_cast<int8_t*>(cache->k);
    c.v = static_cast<int8_t*>(cache->v);
    c.ks = cache->k_scales;
    c.vs = cache->v_scales;
    c.pages = static_cast<int>(cache->pages);
    c.kv_heads = static_cast<int>(cache->kv_heads);
    c.page = static_cast<int>(page);
    c.page_log = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7;
    c.d = static_cast<int>(d);
    q.starts = starts;
    q.lens = lens;
    q.table = table;
    q.width = table_width;
    q.tokens = tokens;
    q.batch = static_cast<int>(batch);
    q.each = batch > 0 ? static_cast<int>(tokens / batch) : 0;
    return RMLK_OK;
}

struct Append {
    const void *k, *v, *q;
    int64_t ks, vs, qs, os;  // row strides
    const float *cos, *sin;
    int64_t table_rows;
    int q_heads;
    void* q_out;
    int* status;
};

// one rounding: the products are exact in fp64
__device__ __forceinline__ float rotated(float x, float y, float c, float s) {
    return static_cast<float>(static_cast<double>(x) * c + static_cast<double>(y) * s);
}

// the least 2^e >= 2^-126 with m <= 127 2^e; NaN for a maximum that is not finite
__device__ __forceinline__ float least_scale(uint32_t max_bits) {
    if (max_bits >= 0x7f800000u) return __int_as_float(0x7fc00000);
    int e = static_cast<int>(max_bits >> 23) - 6 + ((max_bits & 0x7fffffu) > 0x7e0000u ? 1 : 0);  // (biased) 1.984375 = 127 / 64
    return __int_as_float(max(e, 1) << 23);
}

__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ float value(const __half* p) { return __half2float(*p); }

// One CTA per (page that a sequence's new tokens fall into, head, K or V).
template <typename T>
__global__ void __launch_bounds__(128) append_kernel(const Cache c, const Batch q, const Append a, int pages_each) {
    dep_sync();
    __shared__ uint32_t s_max[4];
    int b, j;
    int64_t first, count;
    if (!q.starts) {
        b = blockIdx.x / pages_each;
        j = blockIdx.x - b * pages_each;
        q.rows(b, first, count);
    } else {  // sequence by sequence; item i of all
        int i = blockIdx.x;
        for (b = 0; b < q.batch; b++) {
            q.rows(b, first, count);
            const int64_t p0 = q.lens[b] - count;
            const int n = count > 0 && q.lens[b] > 0 ? static_cast<int>(((q.lens[b] - 1) >> c.page_log) - (max(p0, int64_t(0)) >> c.page_log) + 1) : 0;
            if (i < n) break;
            i -= n;
        }
        if (b == q.batch) return;
        j = i;
    }
    const int64_t len = q.lens[b], p0 = len - count;  // the first new token's position, below 0 where it has none
    if (count == 0 || len <= 0) return;
    const int64_t at = (max(p0, int64_t(0)) >> c.page_log) + j;
    const int64_t t0 = max(max(p0, int64_t(0)), at << c.page_log), t1 = min(len, (at + 1) << c.page_log);
    if (t0 >= t1) return;
    const int page = at < q.width ? q.table[b * q.width + at] : -1;
    const int64_t t_end = a.cos ? min(t1, a.table_rows) : t1;  // tokens behind it have no row in the tables
    if (page < 0 || page >= c.pages || t_end < t1) {
        if (a.status && threadIdx.x == 0) *a.status = RMLK_ERR_INVALID_ARG;
        if (page < 0 || page >= c.pages) return;
    }
    const int h = blockIdx.y, half = c.d / 2;
    const bool is_v = blockIdx.z;
    const int slot0 = static_cast<int>(t0 & (c.page - 1)), n = static_cast<int>(t_end - t0);
    if (n <= 0) return;
    const T* src = static_cast<const T*>(is_v ? a.v : a.k) + (first + t0 - p0) * (is_v ? a.vs : a.ks) + static_cast<int64_t>(h) * c.d;
    const int64_t stride = is_v ? a.vs : a.ks;
    const int64_t block = static_cast<int64_t>(page) * c.kv_heads + h;
    int8_t* dst = (is_v ? c.v : c.k) + block * c.page * c.d;
    float* scale = (is_v ? c.vs : c.ks) + block;
    auto get = [&](int r, int i) {
        const T* x = src + r * stride;
        const float own = value(x + i);
        if (is_v || !a.cos) return own;
        const float other = i < half ? -value(x + i + half) : value(x + i - half);
        return rotated(own, other, a.cos[(t0 + r) * c.d + i], a.sin[(t0 + r) * c.d + i]);
    };
    uint32_t m = 0;
    for (int i = threadIdx.x; i < n * c.d; i += 128) m = max(m, __float_as_uint(get(i / c.d, i % c.d)) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
    const float old = slot0 > 0 ? *scale : 0.f;
    __syncthreads();
    m = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
    float s = least_scale(m);
    if (!(s > old)) s = s != s ? s : old;  // (a NaN of either stays)
    if (threadIdx.x == 0) *scale = s;
    if (slot0 > 0 && s > old) {
        const float ratio = old / s;
        for (int i = threadIdx.x; i < slot0 * c.d; i += 128) dst[i] = static_cast<int8_t>(rintf(dst[i] * ratio));
    }
    const float inv = 1.f / s;
    for (int i = threadIdx.x; i < n * c.d; i += 128) dst[slot0 * c.d + i] = s == s ? static_cast<int8_t>(rintf(get(i / c.d, i % c.d) * inv)) : 0;
}

// The queries: one CTA per new token.
template <typename T>
__global__ void __launch_bounds__(128) rotate_kernel(const Cache c, const Batch q, const Append a) {
    dep_sync();
    const int64_t row = blockIdx.x;
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
    const int64_t p = q.lens[b] - count + row - first, at = p >> c.page_log;
    if (p < 0) return;
    const int page = at < q.width ? q.table[b * q.width + at] : -1;
    if (page < 0 || page >= c.pages || p >= a.table_rows) {
        if (a.status && threadIdx.x == 0) *a.status = RMLK_ERR_INVALID_ARG;
        return;
    }
    const int half = c.d / 2;
    const T* x = static_cast<const T*>(a.q) + row * a.qs;
    T* o = static_cast<T*>(a.q_out) + row * a.os;
    for (int i = threadIdx.x; i < a.q_heads * c.d; i += 128) {
        const int e = i % c.d;
        const float other = e < half ? -value(x + i + half) : value(x + i - half);
        o[i] = static_cast<T>(rotated(value(x + i), other, a.cos[p * c.d + e], a.sin[p * c.d + e]));
    }
}

}  // namespace paged
}  // namespace rmlk

using namespace rmlk;

extern "C" int rmlk_b200_paged_append(rmlk_stream_t stream, int dtype, const rmlk_paged_cache* cache, int64_t tokens, int64_t batch, const int32_t* starts, const int32_t* lens,
                                      const int32_t* table, int64_t table_width, const void* k, int64_t k_stride, const void* v, int64_t v_stride, const float* cos,
                                      const float* sin, int64_t table_rows, int64_t q_heads, const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, int* status) {
    if (dtype != RMLK_F32 && dtype != RMLK_F16) return fail(RMLK_ERR_UNSUPPORTED_DTYPE, "unsupported data type for paged_append (f32, f16)");
    paged::Cache c;
    paged::Batch s;
    const int rc = paged::take("paged_append", cache, tokens, batch, starts, lens, table, table_width, c, s);
    if (rc != RMLK_OK) return rc;
    if ((cos == nullptr) != (sin == nullptr) || table_rows < 0) return fail(RMLK_ERR_INVALID_ARG, "paged_append: cos and sin come together");
    if (q && !cos) return fail(RMLK_ERR_INVALID_ARG, "paged_append: queries need the tables");
    if (q && (q_heads < 1 || q_heads > 65535)) return fail(RMLK_ERR_INVALID_ARG, "paged_append: bad extent");
    if (tokens == 0 || batch == 0) return RMLK_OK;
    if (!k || !v || (q && !q_out)) return fail(RMLK_ERR_INVALID_ARG, "paged_append: NULL pointer");
    const int64_t e = static_cast<int64_t>(dtype_size(dtype)), kv = static_cast<int64_t>(c.kv_heads) * c.d, qd = q ? q_heads * c.d : 0;
    if (k_stride < kv || v_stride < kv || (q && (q_stride < qd || q_out_stride < qd))) return fail(RMLK_ERR_INVALID_ARG, "paged_append: rows overlap");
    if (!aligned_to(k, 4 * e) || !aligned_to(v, 4 * e) || !aligned_to(q, 4 * e) || !aligned_to(q_out, 4 * e) || !aligned_to(cos, 16) || !aligned_to(sin, 16) || k_stride % 4 ||
        v_stride % 4 || (q && (q_stride % 4 || q_out_stride % 4)))
        return fail(RMLK_ERR_INVALID_ARG, "paged_append: rows must lie on boundaries of four values");
    paged::Append a = {k, v, q, k_stride, v_stride, q_stride, q_out_stride, cos, sin, table_rows, static_cast<int>(q_heads), q_out, status};
    // pages that the new tokens can fall into: of each sequence one more than their number divided by the page size, rounded up to whole pages
    const int64_t pages_each = (s.each + c.page - 2) / c.page + 1;
    const int64_t items = starts ? tokens / c.page + 2 * std::min<int64_t>(batch, tokens) : batch * pages_each;
    if (items > 0x7fffffffll) return fail(RMLK_ERR_INVALID_ARG, "paged_append: too many tokens");
    const dim3 grid(static_cast<unsigned>(items), c.kv_heads, 2);
    if (dtype == RMLK_F32) launch_dep(paged::append_kernel<float>, grid, dim3(128), 0, as_stream(stream), c, s, a, static_cast<int>(pages_each));
    else launch_dep(paged::append_kernel<__half>, grid, dim3(128), 0, as_stream(stream), c, s, a, static_cast<int>(pages_each));
    RMLK_CHECK_LAUNCH("append_kernel");
    if (q) {
        if (dtype == RMLK_F32) launch_dep(paged::rotate_kernel<float>, dim3(static_cast<unsigned>(tokens)), dim3(128), 0, as_stream(stream), c, s, a);
        else launch_dep(paged::rotate_kernel<__half>, dim3(static_cast<unsigned>(tokens)), dim3(128), 0, as_stream(stream), c, s, a);
        RMLK_CHECK_LAUNCH("rotate_kernel");
    }
    return RMLK_OK;
}
