"""Plain 64-bit forms of the 8-bit serving operators, for the tests."""
import math

import torch


def quantized(x):
    """codes (float64), scales (float32) of quantize_rows' definition."""
    x = x.double().cpu()
    amax = x.abs().amax(1) if x.shape[1] else torch.zeros(x.shape[0], dtype=torch.float64)
    scales = (amax / 127).float().clamp_min(2.0 ** -126)
    codes = torch.round(x / scales.double()[:, None])
    bad = ~torch.isfinite(amax)
    scales[bad] = math.nan
    codes[bad] = 0
    return codes, scales


def least_scale(amax: float) -> float:
    if not math.isfinite(amax):
        return math.nan
    e = -126
    while amax > 127 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def same_queries(got, want, q):
    """Rotated queries against the exact ones.  The sine's product is rounded in fp32, half a step of it, and the sum, half a step of that; |cos|, |sin| <= 1, so the product is at most
    the largest |q|, the sum twice that: 3 x 2^-24 of it.  want is the fp32 rounding of the exact sum: 2 x 2^-24 more.  f16: both are rounded, 2^-11 of the value each, 2^-25 among
    the subnormal ones."""
    f16 = q.dtype == torch.float16
    got, want, q = got.double().cpu(), want.double().cpu(), q.double().cpu()
    limit = 5 * 2.0 ** -24 * q.abs().amax(-1, keepdim=True) + (2 * 2.0 ** -11 * want.abs() + 2 * 2.0 ** -25 if f16 else 0)
    assert bool(((got - want).abs() <= limit).all()), float((got - want).abs().max())


def rotated(x, cos, sin):
    """x [heads, D], one position's rows of the tables: exact in 64 bits but for the last rounding of the sum, then one rounding to fp32."""
    half = x.shape[-1] // 2
    x = x.double()
    return (x * cos.double() + torch.cat([-x[:, half:], x[:, :half]], 1) * sin.double()).float()


class Cache:
    """What paged_append does to a cache, token group by token group, on the CPU."""

    def __init__(self, cache):
        self.codes = [cache.k.cpu().double(), cache.v.cpu().double()]
        self.scales = [cache.k_scales.cpu().clone(), cache.v_scales.cpu().clone()]
        self.pages, self.heads, self.page, self.d = cache.k.shape

    def append(self, k, v, lens, table, cos=None, sin=None, q=None, starts=None):
        k, v, table = k.cpu(), v.cpu(), table.cpu().tolist()
        lens = lens.cpu().tolist()
        cos, sin = (None, None) if cos is None else (cos.cpu(), sin.cpu())
        batch = len(lens)
        starts = [k.shape[0] // batch * b for b in range(batch + 1)] if starts is None else starts.cpu().tolist()
        out = None if q is None else torch.full(q.shape, math.nan, dtype=q.dtype)
        bad = False
        for b in range(batch):
            n, blocks = starts[b + 1] - starts[b], {}
            for i in range(n):
                p, row = lens[b] - n + i, starts[b] + i
                if p < 0:
                    continue
                page = table[b][p // self.page] if p // self.page < len(table[b]) else -1
                if not 0 <= page < self.pages or (cos is not None and p >= cos.shape[0]):
                    bad = True
                    continue
                kk = k[row].float() if cos is None else rotated(k[row], cos[p], sin[p])
                if q is not None:
                    out[row] = rotated(q[row].cpu(), cos[p], sin[p]).to(q.dtype)
                blocks.setdefault(page, []).append((p % self.page, kk, v[row].float()))
            for page, new in blocks.items():
                first = new[0][0]
                for w in (0, 1):
                    values = torch.stack([t[1 + w] for t in new])  # [tokens, heads, D]
                    for h in range(self.heads):
                        amax = float(values[:, h].abs().max()) if bool(torch.isfinite(values[:, h]).all()) else math.inf
                        scale, old = least_scale(amax), float(self.scales[w][page, h])
                        codes = self.codes[w][page, h]
                        if first:
                            scale = math.nan if math.isnan(scale) or math.isnan(old) else max(scale, old)
                            if scale > old:
                                codes[:first] = torch.round(codes[:first] * (old / scale))
                        self.scales[w][page, h] = scale
                        codes[first: first + len(new)] = 0 if math.isnan(scale) else torch.round(values[:, h].double() / scale)
        return out, bad

    def same(self, cache):
        for w, (codes, scales) in enumerate(((cache.k, cache.k_scales), (cache.v, cache.v_scales))):
            assert torch.equal(scales.cpu().view(torch.int32) & 0x7fffffff, torch.where(torch.isnan(self.scales[w]), scales.cpu(), self.scales[w]).view(torch.int32) & 0x7fffffff)
            assert torch.equal(torch.isnan(scales.cpu()), torch.isnan(self.scales[w]))
            differ = codes.cpu().double() != self.codes[w]
            differ &= ~torch.isnan(self.scales[w])[:, :, None, None]  # codes under the scale NaN stand for nothing
            assert not bool(differ.any()), (w, differ.nonzero()[:5].tolist())


def attention(q, cache, lens, table, scale, starts=None):
    """(out in float64, bound): out [tokens, heads, D], NaN rows where no sequence has the row; bound [tokens, heads, 1], how far an fp32 result may be.

    Scores are sums of D / 16 steps in fp32 that may truncate (2^-23 each), of pairs that hold 22 bits of q against its largest, scaled by two factors and rounded
    in the exponent's argument: (D / 16 + 8) 2^-23 of S = |scale| sum |q| |k|.  A weight is off by that share, twice (its sum too), and by 2^-21 for the
    exponential and its pair; the sums over T keys by 2^-23 for each of T / 16 + 16 steps, twice.  All of it times the largest |v|.
    f16 queries: the weights are rounded to f16, each by at most 2^-11 of itself, and so the sum of w v by at most 2^-11 sum w |v| <= 2^-11 max |v|."""
    page, d, group = cache.k.shape[2], cache.k.shape[3], q.shape[1] // cache.k.shape[1]
    dev = q.device
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=dev)
    bound = torch.zeros(q.shape[0], q.shape[1], 1, dtype=torch.float64, device=dev)
    lens, rows = lens.tolist(), table.tolist()
    batch = len(lens)
    starts = [q.shape[0] // batch * b for b in range(batch + 1)] if starts is None else starts.tolist()
    for b in range(batch):
        n, total = starts[b + 1] - starts[b], lens[b]
        if n == 0:
            continue
        x = q[starts[b]: starts[b + 1]].double()
        if total <= 0:
            out[starts[b]: starts[b + 1]] = 0
            continue
        pages = torch.tensor(rows[b][: -(-total // page)], device=dev)
        k, v = (c[pages].double() * s[pages].double()[..., None, None] for c, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)))
        k, v = (t.permute(1, 0, 2, 3).reshape(cache.k.shape[1], -1, d)[:, :total].repeat_interleave(group, 0) for t in (k, v))  # [heads, tokens, D]
        hidden = torch.arange(total, device=dev) > (total - n + torch.arange(n, device=dev))[:, None]
        s = torch.einsum("nhd,htd->hnt", x, k) * scale
        size = torch.einsum("nhd,htd->hnt", x.abs(), k.abs()) * abs(scale)
        s = s.masked_fill(hidden, -math.inf)
        w = torch.softmax(s, -1)
        w = torch.where(hidden.all(-1)[None, :, None], torch.zeros((), dtype=w.dtype, device=dev), w)
        v_ok = torch.nan_to_num(v, nan=0.0)
        o = torch.einsum("hnt,htd->nhd", w, v_ok)
        poison = torch.einsum("hnt,htd->nhd", (~hidden).double().expand(w.shape), torch.isnan(v).double()) > 0
        out[starts[b]: starts[b + 1]] = torch.where(poison, torch.full_like(o, math.nan), o)
        most = torch.nan_to_num(size.masked_fill(hidden, 0).amax(-1))  # [heads, n]
        share = 2 * (d / 16 + 8) * 2.0 ** -23 * most + 2 * 2.0 ** -21 + 2 * (total / 16 + 16) * 2.0 ** -23
        if q.dtype == torch.float16:
            share = share + 2.0 ** -11
        bound[starts[b]: starts[b + 1]] = (share * v_ok.abs().amax((1, 2))[:, None]).t()[..., None]
    return out, bound


def close(got, want, bound):
    """got against want, within the bound and, for f16 results, their rounding: half a step, 2^-11 of the value, 2^-25 among the subnormal ones."""
    known = ~torch.isnan(want)
    assert torch.equal(torch.isnan(got) & known, torch.zeros_like(known)), "NaN in a row that has a value"
    limit = bound.expand_as(want).clone()
    if got.dtype == torch.float16:
        limit = limit + 2.0 ** -11 * want.abs() + 2.0 ** -25
    err = (got.double() - want).abs()
    over = known & ~(err <= limit)
    assert not bool(over.any()), (float(err[over].max()), float(limit[over].min()), over.nonzero()[:4].tolist())


def make(kv_heads, page, d, lens, dev, gen, spare=3, width=None, spread=2):
    """A cache of random codes and scales (powers of two, `spread` of them), and a table of shuffled pages for sequences of these lengths."""
    from rmlk_b200 import kernels as K
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    table = torch.full((len(lens), width or max(max(counts, default=0), 1)), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at: at + c]
        at += c
    cache = K.paged_cache(pages, kv_heads, page, d, dev)
    for codes, scales in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        codes.copy_((torch.randn(codes.shape, generator=gen) * 36).round().clamp(-127, 127))
        scales.copy_(torch.exp2(torch.randint(-5, -5 + spread, scales.shape, generator=gen).float()))
    return cache, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
