"""Attention over the paged 8-bit cache under scales of any size and sign, against 64 bits (tests/eight_bit.py has the derivation of the bounds)."""
import math

import pytest
import torch

import eight_bit as E

pytestmark = pytest.mark.gpu


def _gen(*seed):
    g = torch.Generator()
    g.manual_seed(sum((i + 1) * 7919 * s for i, s in enumerate(seed)))
    return g


def _make(kv, page, d, lens, dev, gen):
    """As eight_bit.make, but page 0 is a stranger's: no sequence names it, its codes are large and its scales 1."""
    from rmlk_b200 import kernels as K
    cache, table, n = E.make(kv, page, d, lens, dev, gen)
    cache = K.PagedCache(*(torch.cat([torch.full_like(t[:1], 127 if t.dim() == 4 else 1), t]) for t in cache))
    return cache, torch.where(table < 0, table, table + 1).to(torch.int32), n


def _scales(cache, low, high, gen):
    return torch.exp2(torch.randint(low, high, cache.v_scales.shape, generator=gen).float()).to(cache.v_scales.device)


def _attend(q, cache, n, table, d, starts=None):
    from rmlk_b200 import kernels as K
    return K.paged_attention(q, cache, n, table, d ** -0.5, starts=starts), *E.attention(q, cache, n, table, d ** -0.5, starts)


@pytest.mark.parametrize("page,d,each", [(16, 64, 1), (64, 64, 4), (16, 128, 4), (32, 128, 1)])
def test_values_that_are_tiny_throughout(cuda, page, d, each):
    """Scales of V near the lower end of fp32, as paged_append makes them for values below 1e-30, all alike, near one another and far apart: as precise as any others.  The last
    step of a sequence has places without keys, for which page 0 is read."""
    g = _gen(page, d, each)
    cache, table, n = _make(2, page, d, [each + 1, 40, 70, 300, 2983], cuda, g)
    q = torch.randn(5 * each, 6, d, generator=g).to(cuda)
    for low, high in ((-126, -125), (-126, -123), (-122, -102), (-110, -109), (-112, -109), (-104, -102)):
        cache.v_scales.copy_(_scales(cache, low, high, g))
        out, want, bound = _attend(q, cache, n, table, d)
        E.close(out, want, bound)


@pytest.mark.parametrize("page,d,each", [(16, 64, 1), (128, 64, 2), (32, 128, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_values_of_zero_are_zero(cuda, page, d, each, dtype):
    """A cache that paged_append has filled with zeros has the scales 2^-126; whatever page 0 holds, the result is zero to the last bit."""
    from rmlk_b200 import kernels as K
    g = _gen(page, d, each)
    lens = [each, 33, 100, 777]
    cache, table, n = _make(2, page, d, lens, cuda, g)
    k, v = torch.randn(sum(lens), 2, d, generator=g).to(dtype).to(cuda), torch.zeros(sum(lens), 2, d, dtype=dtype, device=cuda)
    K.paged_append(cache, k, v, n, table, starts=torch.tensor([sum(lens[:b]) for b in range(5)], dtype=torch.int32, device=cuda))
    used = table[table >= 0].long()
    assert bool((cache.v_scales[used] == 2.0 ** -126).all())
    out = K.paged_attention(torch.randn(4 * each, 4, d, generator=g).to(dtype).to(cuda), cache, n, table, d ** -0.5)
    assert not bool(out.any())


@pytest.mark.parametrize("d,each,group", [(64, 1, 4), (128, 1, 7), (64, 3, 5), (128, 2, 8), (64, 70, 4), (128, 60, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_scales_below_zero(cuda, d, each, group, dtype):
    """A value is its code times the scale, whatever the sign: all below zero, some of them, of one size and of many; for one token, for a few and for prompts."""
    g = _gen(d, each, group)
    cache, table, n = _make(2, 16, d, [each, each + 17, 200, 1500], cuda, g)
    q = torch.randn(4 * each, 2 * group, d, generator=g).to(dtype).to(cuda)
    for low, high, share in ((-4, -3, 1.0), (-5, -3, 0.5), (-12, 2, 0.5), (-5, -3, 0.02)):
        for part in (cache.v_scales, cache.k_scales):
            part.copy_(_scales(cache, low if part is cache.v_scales else -5, high if part is cache.v_scales else -3, g))
            part.mul_(torch.where(torch.rand(part.shape, generator=g) < share, -1.0, 1.0).to(cuda))
        out, want, bound = _attend(q, cache, n, table, d)
        E.close(out, want, bound)


@pytest.mark.parametrize("d,each,group", [(64, 1, 4), (128, 2, 8), (64, 4, 6), (128, 60, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_scales_that_are_not_finite(cuda, d, each, group, dtype):
    """Infinities of either sign and NaN make NaN of the rows and heads that see a token of their page, and of no others."""
    from rmlk_b200 import kernels as K
    g = _gen(d, each, group, 5)
    lens = [200 + each, 100 + each, 48 + each]
    cache, table, n = _make(2, 16, d, lens, cuda, g)
    q = torch.randn(3 * each, 2 * group, d, generator=g).to(dtype).to(cuda)
    pages = table[0, 2], table[1, 6], table[2, 3]  # seen by all rows of their sequence; by its last ones; by the last one alone or all but the first
    for value in (math.inf, -math.inf, math.nan):
        for of_k in (True, False):
            told = [t.clone() for t in cache]
            for i, page in enumerate(pages):
                told[2 if of_k else 3][page, i % 2] = value
            out = K.paged_attention(q, K.PagedCache(*told), n, table, d ** -0.5)
            for i, page in enumerate(pages):
                told[2 if of_k else 3][page, i % 2] = math.nan
            want, bound = E.attention(q, K.PagedCache(*told), n, table, d ** -0.5)
            assert torch.equal(torch.isnan(out), torch.isnan(want))
            assert bool(torch.isnan(out).any()) and not bool(torch.isnan(out).all())
            E.close(out, want, bound)


@pytest.mark.parametrize("new,total", [([40, 33], [1000, 700]), ([130] * 40, [130 + 9 * i for i in range(40)])])
@pytest.mark.parametrize("d", [64, 128])
def test_prompts_over_values_of_any_size(cuda, new, total, d):
    """Scales of V at both ends of fp32, alike and not, alone and with the keys shared by a cluster.  Nothing but the result itself has to fit: the sum of the weights times the values
    is a thousand times larger, the largest scale over the weights' sum as much smaller."""
    g = _gen(d, len(new))
    cache, table, n = _make(2, 32, d, total, cuda, g)
    starts = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=cuda)
    q = torch.randn(sum(new), 8, d, generator=g).to(cuda)
    for low, high in ((-126, -125), (-126, -119), (-115, -109), (100, 101), (106, 110)):
        cache.v_scales.copy_(_scales(cache, low, high, g))
        out, want, bound = _attend(q, cache, n, table, d, starts)
        E.close(out, want, bound)


@pytest.mark.parametrize("d", [64, 128])
def test_rows_that_see_only_tiny_values(cuda, d):
    """The first rows of a prompt see a page of tiny values, the others one of ordinary values as well: the first keep theirs."""
    g = _gen(d, 3)
    cache, table, n = _make(1, 16, d, [40], cuda, g)
    q = torch.randn(40, 4, d, generator=g).to(cuda)
    for tiny in (2.0 ** -123, 2.0 ** -125):
        cache.v_scales.fill_(0.125)
        cache.v_scales[table[0, 0]] = tiny
        out, _, _ = _attend(q, cache, n, table, d, torch.tensor([0, 40], dtype=torch.int32, device=cuda))
        for i in (0, 5, 15, 16, 39):
            want, bound = E.attention(q[i: i + 1], cache, torch.tensor([i + 1]), table, d ** -0.5)
            E.close(out[i: i + 1], want, bound)


@pytest.mark.parametrize("d,batch,each,total", [(64, 80, 4, 120000), (128, 80, 4, 120000), (128, 80, 2, 120000), (128, 2, 4, 400000), (64, 2, 4, 400000), (128, 80, 4, 16000), (128, 3, 4, 100)])
def test_sums_over_long_prompts_are_not_cut_off(cuda, d, batch, each, total):
    """Values of one sign under many keys: what each MMA cuts off its sum is always of the same sign and would add up.  Results are off by roundings to nearest of either sign
    (weights, results: each at most 2^-11), which in the mean over many results nearly vanish, and by what is cut off: at most 2^-23 for each 16 of 16384 keys, 2^-13.  The mean of
    N results that are off by at most 2^-10 is off by 2^-10 / sqrt(N) with 6 standard deviations' room: 6 x 2^-10 / sqrt(3) / sqrt(N)."""
    from rmlk_b200 import kernels as K
    g = _gen(d, batch, each)
    page, group = 128, 64
    cache, _, _ = E.make(1, page, d, [4 * page], cuda, g)
    cache.v.copy_(cache.v.abs().clamp_min(20))
    table = torch.randint(0, 4, (batch, -(-total // page)), generator=g).to(torch.int32).to(cuda)  # (pages may be named more than once)
    n = torch.full((batch,), total, dtype=torch.int32, device=cuda)
    n[-1] -= 5000 if total > 5000 else 0
    q = torch.randn(batch * each, group, d, generator=g).to(torch.float16).to(cuda)
    starts = torch.arange(0, batch * each + 1, each, dtype=torch.int32, device=cuda)
    out = K.paged_attention(q, cache, n, table, d ** -0.5, starts=starts)
    for b in (0, batch - 1):
        rows = slice(b * each, (b + 1) * each)
        want, _ = E.attention(q[rows], cache, n[b: b + 1], table[b: b + 1], d ** -0.5)
        off = (out[rows].double() - want) / want
        assert float(off.abs().max()) < 2 * 2.0 ** -11 + 2.0 ** -13
        assert abs(float(off.mean())) < 2.0 ** -13 + 6 * 2.0 ** -10 / math.sqrt(3 * off.numel())


@pytest.mark.parametrize("d", [64, 128])
def test_tiles_one_after_the_other(cuda, d):
    """Two f16 tiles over more keys than they take at once, alone and with the keys shared by a cluster: ragged ends, tiles that see different numbers of keys, first rows that see none."""
    from rmlk_b200 import kernels as K
    g = _gen(31, d)
    page, group = 64, 4
    for new, total in (([300, 64, 40], [17000, 33333, 60]), ([65] * 60, [16385 + 37 * i for i in range(60)]), ([20000], [19990]), ([64], [140001])):
        cache, _, _ = E.make(1, page, d, [9 * page], cuda, g)
        table = torch.randint(0, 9, (len(new), -(-max(total) // page)), generator=g).to(torch.int32).to(cuda)
        n = torch.tensor(total, dtype=torch.int32, device=cuda)
        starts = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=cuda)
        q = torch.randn(sum(new), group, d, generator=g).to(torch.float16).to(cuda)
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        out = K.paged_attention(q, cache, n, table, d ** -0.5, starts=starts, status=status)
        assert int(status) == 0
        for b in sorted({0, len(new) // 2, len(new) - 1}):
            rows = slice(int(starts[b]), int(starts[b + 1]))
            if new[b] > 1000:  # some of its rows, as the last ones of shorter sequences
                for i in (0, 11, 5000, 16500, 19999):
                    seen = total[b] - new[b] + i + 1
                    want, bound = E.attention(q[rows][i: i + 1], cache, torch.tensor([seen], device=cuda), table[b: b + 1], d ** -0.5)
                    E.close(out[rows][i: i + 1], want, bound)
            else:
                want, bound = E.attention(q[rows], cache, n[b: b + 1], table[b: b + 1], d ** -0.5)
                E.close(out[rows], want, bound)
