"""Attention over the paged 8-bit cache for queries whose values differ in size, against 64 bits (tests/eight_bit.py has the derivation of the bounds)."""
import pytest
import torch

import eight_bit as E

pytestmark = pytest.mark.gpu


def _gen(*seed):
    g = torch.Generator()
    g.manual_seed(sum((i + 1) * 7919 * s for i, s in enumerate(seed)))
    return g


def _case(d, each, group, dtype, dev, g):
    lens = [each, each + 300, 2000]
    cache, table, n = E.make(2, 32, d, lens, dev, g)
    return cache, table, n, torch.randn(3 * each, 2 * group, d, generator=g)


@pytest.mark.parametrize("d,each,group", [(64, 1, 4), (64, 2, 8), (128, 1, 8), (128, 4, 3), (128, 5, 8), (64, 9, 4)])
@pytest.mark.parametrize("size", [1.0, 4.0, 8.0])
def test_f16_queries_with_an_outlier(cuda, d, each, group, size):
    """A value of 10 to 33 times the others, in a dim that no key has a part in: what the others are, to the last bit of f16, decides the weights."""
    g = _gen(d, each, group, int(size))
    cache, table, n, x = _case(d, each, group, torch.float16, cuda, g)
    cache.k[..., 5] = 0
    for up in (10.0, 16.0, 24.0, 30.0, 33.0, 100.0, 1000.0):
        q = x * size
        q[..., 5] = up * size
        q = q.to(torch.float16).to(cuda)
        from rmlk_b200 import kernels as K
        out = K.paged_attention(q, cache, n, table, d ** -0.5)
        want, bound = E.attention(q, cache, n, table, d ** -0.5)
        E.close(out, want, bound)


@pytest.mark.parametrize("d,each,group", [(64, 1, 4), (128, 2, 3), (128, 1, 16), (64, 5, 5)])
def test_f16_queries_of_two_sizes(cuda, d, each, group):
    """Half of a query's values are far larger than the other half, and keys have no part in their dims; and values that are far smaller in dims that keys alone have a part in."""
    from rmlk_b200 import kernels as K
    g = _gen(d, each, group)
    cache, table, n, x = _case(d, each, group, torch.float16, cuda, g)
    cache.k[..., ::2] = 0
    for large, small, scale in ((20.0, 1.0, 1.0), (300.0, 1.0, 1.0), (10000.0, 1.0, 1.0), (10000.0, 0.01, 100.0), (1000.0, 2.0 ** -14, 2.0 ** 14)):
        q = x * small
        q[..., ::2] = x[..., ::2] * large
        q = q.to(torch.float16).to(cuda)
        out = K.paged_attention(q, cache, n, table, scale * d ** -0.5)
        want, bound = E.attention(q, cache, n, table, scale * d ** -0.5)
        E.close(out, want, bound)


@pytest.mark.parametrize("d", [64, 128])
def test_f16_queries_and_keys_of_any_scale(cuda, d):
    """Whether third digits, or scores in fp32, are called for depends on the keys' scales: pages of different ones in a step."""
    from rmlk_b200 import kernels as K
    g = _gen(d)
    for each, group in ((1, 4), (1, 16), (2, 5)):
        cache, table, n, x = _case(d, each, group, torch.float16, cuda, g)
        for low, high, size in ((-14, -2, 4.0), (-3, 1, 1.0), (-30, -20, 1000.0), (-20, 0, 0.25)):
            cache.k_scales.copy_(torch.exp2(torch.randint(low, high, cache.k_scales.shape, generator=g).float()))
            q = (x * size).to(torch.float16).to(cuda)
            out = K.paged_attention(q, cache, n, table, d ** -0.5)
            want, bound = E.attention(q, cache, n, table, d ** -0.5)
            E.close(out, want, 4 * bound)  # (scores in fp32: D roundings of 2^-24, where the bound counts D / 16 + 8 of 2^-23)


@pytest.mark.parametrize("d,each,group", [(64, 1, 4), (128, 2, 3), (128, 1, 16), (64, 5, 5)])
def test_fp32_queries_of_two_sizes(cuda, d, each, group):
    """As above: the digits of a row lie under its largest value, and keys need not have a part in that."""
    from rmlk_b200 import kernels as K
    g = _gen(d, each, group)
    cache, table, n, x = _case(d, each, group, torch.float32, cuda, g)
    cache.k[..., ::2] = 0
    for large, small, scale in ((20.0, 1.0, 1.0), (300.0, 1.0, 1.0), (1e6, 1.0, 1.0), (1e9, 1e-6, 1e6)):
        q = x * small
        q[..., ::2] = x[..., ::2] * large
        q = q.to(cuda)
        out = K.paged_attention(q, cache, n, table, scale * d ** -0.5)
        want, bound = E.attention(q, cache, n, table, scale * d ** -0.5)
        E.close(out, want, 4 * bound)  # (scores in fp32: D roundings of 2^-24, where the bound counts D / 16 + 8 of 2^-23)


@pytest.mark.parametrize("d,group,new,total", [(64, 4, [70, 40], [500, 900]), (128, 2, [100, 130], [100, 2000]), (64, 3, [130] * 30, [130 + 11 * i for i in range(30)]), (128, 4, [65] * 30, [200] * 30)])
def test_fp32_queries_of_two_sizes_in_prompts(cuda, d, group, new, total):
    """The same for whole prompts, alone and with the keys shared by a cluster, with rows of one size beside them."""
    from rmlk_b200 import kernels as K
    g = _gen(d, group, len(new))
    cache, table, n = E.make(2, 32, d, total, cuda, g)
    cache.k[..., ::2] = 0
    starts = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=cuda)
    x = torch.randn(sum(new), 2 * group, d, generator=g)
    for large, small, scale in ((1e4, 1.0, 1.0), (1e7, 1.0, 1.0), (1e9, 1.0, 1.0), (1e9, 1e-6, 1e6), (1e30, 1.0, 1.0)):
        q = x * small
        q[::3, :, ::2] = x[::3, :, ::2] * large
        out = K.paged_attention(q.to(cuda), cache, n, table, scale * d ** -0.5, starts=starts)
        want, bound = E.attention(q.to(cuda), cache, n, table, scale * d ** -0.5, starts)
        E.close(out, want, 4 * bound)  # (scores in fp32: D roundings of 2^-24, where the bound counts D / 16 + 8 of 2^-23)
