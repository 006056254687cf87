// New keys and values into a paged cache of 8-bit codes, the keys rotated on the way; the queries rotated beside them.
//
//   r = x cos[p] + (-x[D/2:], x[:D/2]) sin[p]       (keys: in fp64, then rounded to fp32; queries: in fp32)
//   2^e: the least power of two with max |r| <= 127 2^e over the new tokens of a block (page, head), at least the block's present scale
//   code = rne(r 2^-e)
//
// Scales are powers of two because a block fills over many calls: where its scale grows, the codes in it are divided by a power of two, so
// that after any number of steps a code is off by less than one step of the final scale (1/2 + 1/4 + ...); ratios of any size would add half a step
// each time.  It costs up to one bit of the eight (a scale of max / 127 is up to twice as fine).
//
// What bounds it: the floor is HBM's, q, k, v and the tables' rows read and q and the codes written once.  5600 tokens of 32 + 8 + 8 heads of 128, f16: 36 us, 3.7 TB/s, with instructions in
// 62 % of all issue slots and 45 % of the warps there could be.  Keys and values wait in registers for their block's maximum (64 of them with a few spilled, 38 us with the 80 that it would
// take), and the keys' conversions to fp64 and back take their time; queries, most of the bytes, wait for nothing but share the instance and its registers.
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
    if (tokens < 0 || tokens >= (1ll << 31) || batch < 0 || batch >= (1ll << 24) || table_width < 0 || table_width > (1ll << 30) / page)  // (keys and steps past them stay in 31 bits)
        return bad("bad extent");
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
    int q_heads, parts;  // parts of a piece: K of each head, V of each head, queries by four heads
    void* q_out;
    int* status;
    int64_t items;
    int pages_each;  // pages that a sequence's new tokens can fall into, where all have as many
};

// the least 2^e >= 2^-126 with m <= 127 2^e; NaN for a maximum that is not finite
__device__ __forceinline__ float least_scale(uint32_t max_bits) {
    if (max_bits >= 0x7f800000u) return __int_as_float(0x7fc00000);
    const int e = static_cast<int>(max_bits >> 23) - 6 + ((max_bits & 0x7fffffu) > 0x7e0000u ? 1 : 0);  // (biased) 1.984375 = 127 / 64
    return __int_as_float(max(e, 1) << 23);
}

__device__ __forceinline__ float4 four(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 four(const __half* p) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void put_four(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }
__device__ __forceinline__ void put_four(__half* p, float4 x) {
    const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// Keys: four dims of the lower half of a head and the four that go with them, in fp64.  Products of fp32 values are exact there; their sum is rounded to fp64 and that to fp32,
// so that a key's codes do not depend on how the rotation is computed.  (Two roundings: where the sum lies next to the middle of two fp32 numbers, closer than fp64 tells, the result
// may be the other of them.)  (The conversions cost more than the arithmetic, 8 cycles per warp each: with the queries rotated so too they were the
// bound, 55 us for 5600 tokens of 32 + 8 heads of 128.)
struct Rotation {
    double cl[4], sl[4], ch[4], sh[4];
    __device__ __forceinline__ void load(const float* cos, const float* sin, int half) {
        const float4 a = four(cos), b = four(sin), c = four(cos + half), d = four(sin + half);
        cl[0] = a.x, cl[1] = a.y, cl[2] = a.z, cl[3] = a.w;
        sl[0] = b.x, sl[1] = b.y, sl[2] = b.z, sl[3] = b.w;
        ch[0] = c.x, ch[1] = c.y, ch[2] = c.z, ch[3] = c.w;
        sh[0] = d.x, sh[1] = d.y, sh[2] = d.z, sh[3] = d.w;
    }
    __device__ __forceinline__ void turn(float4& low, float4& high) const {
        float l[4] = {low.x, low.y, low.z, low.w}, h[4] = {high.x, high.y, high.z, high.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double x = l[i], y = h[i];
            l[i] = static_cast<float>(x * cl[i] - y * sl[i]);
            h[i] = static_cast<float>(y * ch[i] + x * sh[i]);
        }
        low = make_float4(l[0], l[1], l[2], l[3]);
        high = make_float4(h[0], h[1], h[2], h[3]);
    }
};

__device__ __forceinline__ uint32_t most_of(float4 x) {
    return max(max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu), max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu));
}
// |x inv| <= 127: the lowest byte of x inv + 1.5 2^23, which is rounded to an integer, ties to even
__device__ __forceinline__ uint32_t codes_of(float4 x, float inv) {
    const float up = 12582912.f;
    const uint32_t a = __float_as_uint(fmaf(x.x, inv, up)), b = __float_as_uint(fmaf(x.y, inv, up)), c = __float_as_uint(fmaf(x.z, inv, up)), d = __float_as_uint(fmaf(x.w, inv, up));
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// An item: the new tokens of a sequence that fall into one page, as K or V of one head, or the queries of some heads.  GROUP threads to an item; a thread has four dims of
// the lower half of a head and the four that go with them in the upper half, of every (GROUP / (D / 8))-th token: values stay in registers from their maximum to their codes.
template <typename T, int D, int GROUP, int ITERS>
__global__ void __launch_bounds__(256, ITERS <= 2 ? 4 : 2) append_kernel(const Cache c, const Batch q, const Append a) {
    dep_sync();
    constexpr int PACKS = D / 8, AT_ONCE = GROUP / PACKS, HALF = D / 2;
    __shared__ uint32_t s_max[8];
    const int me = threadIdx.x % GROUP, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * (256 / GROUP) + threadIdx.x / GROUP;
    if (item >= a.items) return;  // (GROUP = 256: never)
    const int64_t piece = item / a.parts;
    const int part = static_cast<int>(item - piece * a.parts);
    // ---- which sequence, which of its pages ----
    int b = 0;
    int64_t j = 0, first = 0, count = 0;
    if (!q.starts) {
        b = static_cast<int>(piece / a.pages_each);
        j = piece - static_cast<int64_t>(b) * a.pages_each;
        q.rows(b, first, count);
    } else {  // a warp looks at 32 sequences at a time (every warp for itself: the same answer)
        int64_t left = piece;
        bool found = false;
        for (int b0 = 0; b0 < q.batch && !found; b0 += 32) {
            int64_t f = 0, n = 0;
            int own = 0;
            if (b0 + lane < q.batch) {
                q.rows(b0 + lane, f, n);
                const int64_t len = q.lens[b0 + lane], p0 = max(len - n, int64_t(0));
                own = n > 0 && len > 0 ? static_cast<int>(((len - 1) >> c.page_log) - (p0 >> c.page_log) + 1) : 0;
            }
            int upto = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            const uint32_t mask = __ballot_sync(0xffffffffu, left < upto);
            if (mask) {
                const int l = __ffs(mask) - 1;
                b = b0 + l;
                j = left - __shfl_sync(0xffffffffu, upto - own, l);
                first = __shfl_sync(0xffffffffu, f, l);
                count = __shfl_sync(0xffffffffu, n, l);
                found = true;
            } else {
                left -= __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        if (!found) return;
    }
    const int64_t len = q.lens[b], p0 = len - count;  // the first new token's position, below 0 where it has none
    if (count == 0 || len <= 0) return;
    const int64_t at = (max(p0, int64_t(0)) >> c.page_log) + j;
    const int64_t t0 = max(max(p0, int64_t(0)), at << c.page_log), t1 = min(len, (at + 1) << c.page_log);
    if (t0 >= t1) return;
    const int page = at < q.width ? q.table[static_cast<int64_t>(b) * q.width + at] : -1;
    const int64_t t_end = a.cos ? min(t1, a.table_rows) : t1;  // tokens behind it have no row in the tables
    const bool lost = page < 0 || page >= c.pages;
    if ((lost || t_end < t1) && a.status && me == 0) *a.status = RMLK_ERR_INVALID_ARG;
    const int n = lost ? 0 : static_cast<int>(max(t_end - t0, int64_t(0)));
    if (n == 0) return;
    const int64_t row = first + t0 - p0;
    const int c4 = me % PACKS * 4, r0 = me / PACKS;

    if (part >= 2 * c.kv_heads) {  // ---- queries: in fp32, one product fused with the sum ----
        constexpr int HEADS = 4;  // loads of so many heads are on their way together
        const int h0 = (part - 2 * c.kv_heads) * HEADS;
        for (int r = r0; r < n; r += AT_ONCE) {
            const float* cos = a.cos + (t0 + r) * D + c4;
            const float* sin = a.sin + (t0 + r) * D + c4;
            const float4 cl = four(cos), ch = four(cos + HALF), sl = four(sin), sh = four(sin + HALF);
            const T* src = static_cast<const T*>(a.q) + (row + r) * a.qs + c4;
            T* dst = static_cast<T*>(a.q_out) + (row + r) * a.os + c4;
            float4 low[HEADS], high[HEADS];
#pragma unroll
            for (int i = 0; i < HEADS; i++)
                if (h0 + i < a.q_heads) {
                    low[i] = four(src + static_cast<int64_t>(h0 + i) * D);
                    high[i] = four(src + static_cast<int64_t>(h0 + i) * D + HALF);
                }
#pragma unroll
            for (int i = 0; i < HEADS; i++)
                if (h0 + i < a.q_heads) {
                    const float4 x = low[i], y = high[i];
                    put_four(dst + static_cast<int64_t>(h0 + i) * D,
                             make_float4(fmaf(x.x, cl.x, -__fmul_rn(y.x, sl.x)), fmaf(x.y, cl.y, -__fmul_rn(y.y, sl.y)), fmaf(x.z, cl.z, -__fmul_rn(y.z, sl.z)), fmaf(x.w, cl.w, -__fmul_rn(y.w, sl.w))));
                    put_four(dst + static_cast<int64_t>(h0 + i) * D + HALF,
                             make_float4(fmaf(y.x, ch.x, __fmul_rn(x.x, sh.x)), fmaf(y.y, ch.y, __fmul_rn(x.y, sh.y)), fmaf(y.z, ch.z, __fmul_rn(x.z, sh.z)), fmaf(y.w, ch.w, __fmul_rn(x.w, sh.w))));
                }
        }
        return;
    }

    // ---- K or V of one head ----
    const bool is_v = part >= c.kv_heads;
    const int h = is_v ? part - c.kv_heads : part, slot0 = static_cast<int>(t0 & (c.page - 1));
    const int64_t stride = is_v ? a.vs : a.ks, block = static_cast<int64_t>(page) * c.kv_heads + h;
    const T* src = static_cast<const T*>(is_v ? a.v : a.k) + row * stride + static_cast<int64_t>(h) * D + c4;
    int8_t* dst = (is_v ? c.v : c.k) + block * c.page * D;
    float* scale = (is_v ? c.vs : c.ks) + block;
    const float old = slot0 > 0 ? *scale : 0.f;
    float4 low[ITERS], high[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; i++) {
        const int r = r0 + i * AT_ONCE;
        low[i] = high[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < n) {
            low[i] = four(src + r * stride);
            high[i] = four(src + r * stride + HALF);
        }
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < ITERS; i++) {
        const int r = r0 + i * AT_ONCE;
        if (!is_v && a.cos && r < n) {
            Rotation turn;
            turn.load(a.cos + (t0 + r) * D + c4, a.sin + (t0 + r) * D + c4, HALF);
            turn.turn(low[i], high[i]);
        }
        m = max(m, max(most_of(low[i]), most_of(high[i])));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if constexpr (GROUP > 32) {
        if (lane == 0) s_max[warp] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < GROUP / 32; w++) m = max(m, s_max[w]);
    } else {
        __syncwarp();  // every lane has read the old scale
    }
    float s = least_scale(m);
    if (!(s > fabsf(old))) s = s != s ? s : fabsf(old);  // (a NaN of either stays)
    if (old < 0.f) s = -s;                               // (the codes that are there keep their sign)
    if (me == 0) *scale = s;
    if (slot0 > 0 && fabsf(s) > fabsf(old)) {  // the codes that are there, under the larger scale
        const float ratio = old / s;
        for (int i = me; i < slot0 * D / 4; i += GROUP) {
            const uint32_t w = reinterpret_cast<uint32_t*>(dst)[i];
            reinterpret_cast<uint32_t*>(dst)[i] = codes_of(make_float4(static_cast<int8_t>(w), static_cast<int8_t>(w >> 8), static_cast<int8_t>(w >> 16), static_cast<int8_t>(w >> 24)), ratio);
        }
    }
    const float inv = s == s ? 1.f / s : 0.f;
#pragma unroll
    for (int i = 0; i < ITERS; i++) {
        const int r = r0 + i * AT_ONCE;
        if (r < n) {
            uint32_t* to = reinterpret_cast<uint32_t*>(dst + (slot0 + r) * D + c4);
            to[0] = s == s ? codes_of(low[i], inv) : 0u;
            to[HALF / 4] = s == s ? codes_of(high[i], inv) : 0u;
        }
    }
}

template <typename T, int D, int GROUP, int ITERS>
static int launch_append(cudaStream_t st, const Cache& c, const Batch& s, const Append& a) {
    const int64_t ctas = ceil_div64(a.items, 256 / GROUP);
    if (ctas > 0x7fffffffll) return fail(RMLK_ERR_INVALID_ARG, "paged_append: too many tokens");
    RMLK_CUDA(launch_dep(append_kernel<T, D, GROUP, ITERS>, dim3(static_cast<unsigned>(ctas)), dim3(256), 0, st, c, s, a));
    RMLK_CHECK_LAUNCH("append_kernel");
    return RMLK_OK;
}

// A warp to an item where its tokens fit one pass of a warp's lanes (64 x 1 tokens, 32 + 8 heads of 64: 4.3 us, with a CTA to each, of which all but a few threads have nothing to do,
// 10.2; 64 x 4: 5.5, 13.6), else a CTA.
template <typename T, int D>
static int dispatch_append(cudaStream_t st, const Cache& c, const Batch& s, const Append& a) {
    if (!s.starts && s.each <= 256 / D) return launch_append<T, D, 32, 1>(st, c, s, a);
    switch (c.page * D / (8 * 256)) {
        case 0: case 1: return launch_append<T, D, 256, 1>(st, c, s, a);
        case 2: return launch_append<T, D, 256, 2>(st, c, s, a);
        case 4: return launch_append<T, D, 256, 4>(st, c, s, a);
        default: return launch_append<T, D, 256, 8>(st, c, s, a);
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
    paged::Append a = {};
    a.k = k;
    a.v = v;
    a.q = q;
    a.ks = k_stride;
    a.vs = v_stride;
    a.qs = q_stride;
    a.os = q_out_stride;
    a.cos = cos;
    a.sin = sin;
    a.table_rows = table_rows;
    a.q_heads = static_cast<int>(q_heads);
    a.q_out = q_out;
    a.status = status;
    a.parts = 2 * c.kv_heads + (q ? static_cast<int>(ceil_div64(q_heads, 4)) : 0);
    // pages that the new tokens can fall into: of each sequence one more than their number less two, divided by the page size
    a.pages_each = (s.each + c.page - 2) / c.page + 1;
    const int64_t pieces = starts ? tokens / c.page + 2 * std::min<int64_t>(batch, tokens) : batch * a.pages_each;
    a.items = pieces * a.parts;
    const cudaStream_t st = as_stream(stream);
    if (dtype == RMLK_F32) return c.d == 64 ? paged::dispatch_append<float, 64>(st, c, s, a) : paged::dispatch_append<float, 128>(st, c, s, a);
    return c.d == 64 ? paged::dispatch_append<__half, 64>(st, c, s, a) : paged::dispatch_append<__half, 128>(st, c, s, a);
}
