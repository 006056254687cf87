"""The paged 8-bit cache: appending (paged_append.cu) against its definition, code for code, and attention over it (paged_attention.cu) against 64 bits."""
import math

import pytest
import torch

import eight_bit as E

pytestmark = pytest.mark.gpu


def _gen(*seed):
    g = torch.Generator()
    g.manual_seed(sum((i + 1) * 7919 * s for i, s in enumerate(seed)))
    return g


def _tables(rows, d, dev):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(d // 2, dtype=torch.float64) * 2 / d)
    return (f(torch.cat([angle, angle], 1)).float().to(dev) for f in (torch.cos, torch.sin))


def _table(batch, width, pages, g, dev):
    return torch.randperm(pages, generator=g)[: batch * width].view(batch, width).to(torch.int32).to(dev)


# ---- append ----
@pytest.mark.parametrize("page,d,kv,dtype", [(16, 64, 1, torch.float32), (16, 128, 2, torch.float16), (32, 64, 3, torch.float16), (64, 64, 2, torch.float32),
                                             (64, 128, 1, torch.float16), (128, 64, 1, torch.float32), (128, 128, 2, torch.float32)])
def test_append_token_by_token(cuda, page, d, kv, dtype):
    """Sequences that grow over page borders, larger and larger values among the tokens, so that scales grow with codes in the block."""
    from rmlk_b200 import kernels as K
    g = _gen(page, d, kv)
    cos, sin = _tables(3 * page, d, cuda)
    cache = K.paged_cache(20, kv, page, d, cuda)
    cache.k_scales.fill_(1e30)  # what earlier owners left: the first slot begins a block anew
    cache.v_scales.fill_(math.nan)
    cache.k.random_(-127, 127)
    plain = E.Cache(cache)
    table = _table(4, 3, 20, g, cuda)
    before = torch.tensor([0, page - 3, page, 2 * page - 1], dtype=torch.int32)
    first = K.paged_append(cache, *(torch.randn(int(before.sum()), kv, d, generator=g).to(dtype).to(cuda) for _ in range(2)), before.to(cuda), table, cos, sin,
                           starts=torch.cumsum(torch.cat([torch.zeros(1), before]), 0).to(torch.int32).to(cuda))
    assert first is None
    plain = E.Cache(cache)
    for step in range(12):
        lens = (before + 1 + step).to(cuda)
        size = torch.exp(2 * torch.randn(4, 1, 1, generator=g))
        q, k, v = ((torch.randn(4, h, d, generator=g) * size).to(dtype).to(cuda) for h in (kv * 2, kv, kv))
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        out = K.paged_append(cache, k, v, lens, table, cos, sin, q=q, status=status)
        want, bad = plain.append(k, v, lens, table, cos, sin, q)
        E.same_queries(out, want, q)
        assert not bad and int(status) == 0
        plain.same(cache)


@pytest.mark.parametrize("page,d,kv,dtype", [(16, 64, 2, torch.float16), (16, 128, 1, torch.float32), (32, 128, 2, torch.float16), (64, 64, 4, torch.float32), (64, 128, 2, torch.float32),
                                             (128, 64, 2, torch.float16), (128, 128, 1, torch.float16), (128, 128, 2, torch.float32)])
@pytest.mark.parametrize("rotate", [True, False])
def test_append_prompts(cuda, page, d, kv, dtype, rotate):
    """Ragged prompts, with and without a cached beginning, of no token, of one and of several pages; q, k, v as columns of one matrix; rows that
    belong to no sequence and pages that belong to none stay as they were."""
    from rmlk_b200 import kernels as K
    g = _gen(page, d, kv, int(rotate))
    new = [1, 0, page, page + 1, 3 * page - 5, 7, 2 * page]
    old = [0, 5, 0, page - 1, 3, page - 7, page]
    total = [a + b for a, b in zip(new, old)]
    cache, table, lens = E.make(kv, page, d, total, cuda, g)
    starts = torch.tensor([sum(new[:b]) for b in range(8)], dtype=torch.int32)
    tokens = int(starts[-1]) + 5
    size = torch.exp(torch.randn(tokens, 1, 1, generator=g))
    qkv = (torch.randn(tokens, 5 * kv, d, generator=g) * size).to(dtype).to(cuda)
    q, k, v = qkv[:, : 3 * kv], qkv[:, 3 * kv: 4 * kv], qkv[:, 4 * kv:]
    cos, sin = _tables(max(total), d, cuda) if rotate else (None, None)
    q_out = torch.full((tokens, 3 * kv, d), 3.0, dtype=dtype, device=cuda)
    plain = E.Cache(cache)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    K.paged_append(cache, k, v, lens, table, cos, sin, q=q if rotate else None, starts=starts.to(cuda), q_out=q_out if rotate else None, status=status)
    want, bad = plain.append(k, v, lens, table, cos, sin, q if rotate else None, starts)
    assert int(status) == 0 and not bad
    plain.same(cache)
    if rotate:
        E.same_queries(q_out[: int(starts[-1])], want[: int(starts[-1])], q[: int(starts[-1])])
        assert bool((q_out[int(starts[-1]):] == 3).all())


def test_append_again_gives_the_same(cuda):
    from rmlk_b200 import kernels as K
    g = _gen(3)
    cache, table, lens = E.make(2, 32, 64, [40, 70], cuda, g)
    k, v = (torch.randn(20, 2, 64, generator=g).to(cuda) for _ in range(2))
    starts = torch.tensor([0, 15, 20], dtype=torch.int32, device=cuda)
    K.paged_append(cache, k, v, lens, table, starts=starts)
    once = [t.clone() for t in cache]
    K.paged_append(cache, k, v, lens, table, starts=starts)
    assert all(torch.equal(a, b) for a, b in zip(once, cache))


def test_append_values_of_any_size(cuda):
    """Zeros, subnormal and huge values, and infinities and NaN, which poison their block and head and nothing else, until the block is begun anew."""
    from rmlk_b200 import kernels as K
    g = _gen(4)
    for dtype in (torch.float32, torch.float16):
        cache = K.paged_cache(6, 2, 16, 64, cuda)
        plain = E.Cache(cache)
        table = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32, device=cuda)
        for step, size in enumerate((0.0, 1e-42, 1e-20, 1.0, 3e4, 1.0)):
            k, v = ((torch.randn(3, 2, 64, generator=g) * size).to(dtype) for _ in range(2))
            if step == 2:
                k[0, 0, 3], v[1, 1, 63] = math.inf, math.nan
            lens = torch.full((3,), step + 1, dtype=torch.int32, device=cuda)
            K.paged_append(cache, k.to(cuda), v.to(cuda), lens, table)
            plain.append(k, v, lens, table)
            plain.same(cache)
        # (3e4 times some values is infinite in f16: more blocks than the two)
        assert bool(torch.isnan(cache.k_scales[0, 0])) and bool(torch.isnan(cache.v_scales[2, 1]))
        assert dtype == torch.float16 or int(torch.isnan(cache.k_scales).sum()) == int(torch.isnan(cache.v_scales).sum()) == 1
        k, v = ((torch.randn(60, 2, 64, generator=g)).to(dtype).to(cuda) for _ in range(2))
        lens = torch.full((3,), 20, dtype=torch.int32, device=cuda)
        K.paged_append(cache, k, v, lens, table)  # from slot 0 on
        plain.append(k, v, lens, table)
        plain.same(cache)
        assert not bool(torch.isnan(cache.k_scales).any())
    top = torch.full((1, 2, 64), 3.4e38)
    lens = torch.ones(1, dtype=torch.int32, device=cuda)
    K.paged_append(cache, top.to(cuda), -top.to(cuda), lens, table[:1])
    plain.append(top, -top, lens, table[:1])
    plain.same(cache)


def test_append_passes_over_what_has_no_place(cuda):
    """Pages out of range, sequences longer than their row of the table or the rotary tables: those tokens are not stored and the status says so; the others are.
    Lengths below the new tokens, and of zero, leave nothing to store and are no error."""
    from rmlk_b200 import kernels as K
    g = _gen(5)
    cos, sin = _tables(50, 64, cuda)
    for each in (1, 20):
        cache = K.paged_cache(8, 1, 16, 64, cuda)
        plain = E.Cache(cache)
        table = torch.tensor([[0, 1, 2, 9], [-1, 8, 3, -7], [4, 5, 6, 7]], dtype=torch.int32, device=cuda)
        q, k, v = (torch.randn(3 * each, h, 64, generator=g).to(cuda) for h in (2, 1, 1))
        for lens, bad in (([20, 0, 30], False), ([0, 0, 0], False), ([each // 2, 0, 1], False), ([20, 20, 20], True), ([55, 0, 49], True), ([20, 0, 64], True), ([20, 0, 70], True)):
            lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
            status = torch.zeros(1, dtype=torch.int32, device=cuda)
            out = torch.full_like(q, math.nan)
            K.paged_append(cache, k, v, lens, table, cos, sin, q=q, q_out=out, status=status)
            want, told = plain.append(k, v, lens, table, cos, sin, q)
            assert told == bad and int(status) == int(bad)
            assert torch.equal(torch.isnan(out).cpu(), torch.isnan(want))
            E.same_queries(torch.nan_to_num(out), torch.nan_to_num(want), q)
            plain.same(cache)


def test_append_of_nothing(cuda):
    from rmlk_b200 import kernels as K
    cache = K.paged_cache(2, 1, 16, 64, cuda)
    lens, table = torch.zeros(2, dtype=torch.int32, device=cuda), torch.zeros(2, 1, dtype=torch.int32, device=cuda)
    none = torch.empty(0, 1, 64, device=cuda)
    K.paged_append(cache, none, none, lens, table)
    assert K.paged_attention(none, cache, lens, table, 1.0).shape == (0, 1, 64)
    zero = torch.zeros(3, dtype=torch.int32, device=cuda)
    some = torch.full((2, 1, 64), 5.0, device=cuda)
    K.paged_append(cache, some, some, lens, table, starts=zero)
    out = torch.full((2, 1, 64), 5.0, device=cuda)
    K.paged_attention(some, cache, lens, table, 1.0, starts=zero, out=out)
    assert not bool(cache.k.any()) and bool((out == 5).all())


# ---- attention ----
def _attend(q, cache, lens, table, scale, starts=None, **more):
    from rmlk_b200 import kernels as K
    status = torch.zeros(1, dtype=torch.int32, device=q.device)
    out = K.paged_attention(q, cache, lens, table, scale, starts=starts, status=status, **more)
    assert int(status) == 0
    want, bound = E.attention(q, cache, lens, table, scale, starts)
    E.close(out, want, bound)
    return out


# lengths around pages, units of 64 keys and shares of a CTA; new tokens x heads of a group around tiles of 8, 16 and 128 rows
@pytest.mark.parametrize("page,d", [(16, 64), (32, 64), (64, 64), (128, 64), (16, 128), (32, 128), (64, 128), (128, 128)])
@pytest.mark.parametrize("each,group,kv", [(1, 1, 3), (1, 4, 2), (1, 7, 1), (1, 8, 2), (2, 4, 1), (3, 3, 2), (1, 16, 1), (4, 6, 1), (5, 1, 2), (9, 4, 1), (1, 33, 1), (2, 64, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_a_few_tokens(cuda, page, d, each, group, kv, dtype):
    g = _gen(page, d, each, group, kv)
    lens = [each, 0, 1, 2, 15, 16, 17, 63, 64, 65, 100, 127, 128, 129, 500, each + 1]
    cache, table, n = E.make(kv, page, d, lens, cuda, g, width=max(lens) // page + 3)
    q = torch.randn(len(lens) * each, kv * group, d, generator=g).to(dtype).to(cuda)
    _attend(q, cache, n, table, 1 / math.sqrt(d))


@pytest.mark.parametrize("lens", [[1], [64], [5000], [40000, 3], [1, 1, 1, 30001], [9000, 8000, 7000, 6001, 5003]])
@pytest.mark.parametrize("page,d,group,kv,dtype", [(64, 64, 4, 2, torch.float32), (16, 128, 8, 1, torch.float16), (128, 64, 1, 1, torch.float16), (32, 128, 5, 3, torch.float32)])
def test_long_sequences(cuda, lens, page, d, group, kv, dtype):
    g = _gen(len(lens), page, group)
    cache, table, n = E.make(kv, page, d, lens, cuda, g)
    q = torch.randn(len(lens), kv * group, d, generator=g).to(dtype).to(cuda)
    _attend(q, cache, n, table, 1 / math.sqrt(d))
    _attend(3 * q, cache, n, table, -0.2)


@pytest.mark.parametrize("page,d,group,kv,dtype", [(64, 64, 4, 2, torch.float32), (64, 64, 1, 3, torch.float16), (16, 64, 3, 1, torch.float32), (16, 128, 4, 2, torch.float16), (32, 64, 8, 1, torch.float16),
                                                   (32, 128, 6, 1, torch.float32), (128, 64, 33, 1, torch.float16), (128, 128, 2, 2, torch.float32), (64, 128, 64, 1, torch.float32)])
def test_prompts(cuda, page, d, group, kv, dtype):
    """Ragged prompts with and without a cached beginning, of no token, of one, around tiles of 128 rows and blocks of keys; sequences shorter than
    their new tokens, whose first rows see nothing; rows of no sequence stay as they were."""
    g = _gen(page, d, group)
    new = [1, 0, 31, 32, 33, 130, 200, 64, 7, 20, 3, 97]
    total = [1, 10, 31, 40, 33 + 500, 130, 1000, 64, 3, 0, 700, 97 + 64]
    cache, table, lens = E.make(kv, page, d, total, cuda, g, width=max(total) // page + 2)
    starts = torch.tensor([sum(new[:b]) for b in range(13)], dtype=torch.int32, device=cuda)
    tokens = sum(new) + 3
    q = torch.randn(tokens, kv * group, d, generator=g).to(dtype).to(cuda)
    out = torch.full_like(q, 9.0)
    got = _attend(q, cache, lens, table, 1 / math.sqrt(d), starts, out=out)
    assert got is out and bool((out[-3:] == 9).all())
    assert not bool(out[starts[8]: starts[8] + 4].any()) and not bool(out[starts[9]: starts[10]].any())
    one = K_uniform(q, cache, lens, table, d, starts, new, total)
    for a, b in one:
        # the same row by another way through the kernels: each within the bound of the exact one
        E.close(a, b[0], b[1])


def K_uniform(q, cache, lens, table, d, starts, new, total):
    """The last token of each sequence that has one, as a call of one token per sequence."""
    from rmlk_b200 import kernels as K
    have = [b for b, n in enumerate(new) if n]
    last = [int(starts[b + 1]) - 1 for b in have]
    x, n, t = q[last].contiguous(), lens[have].contiguous(), table[have].contiguous()
    yield K.paged_attention(x, cache, n, t, 1 / math.sqrt(d)), E.attention(x, cache, n, t, 1 / math.sqrt(d))


@pytest.mark.parametrize("new,total", [([40], [5000]), ([300], [300]), ([1, 20], [3000, 513]), ([9, 0, 3], [2000, 0, 1]), ([130, 257], [1500, 4000]), ([33], [20])])
@pytest.mark.parametrize("page,d,group,kv,dtype", [(16, 64, 4, 1, torch.float32), (64, 128, 1, 2, torch.float32), (32, 64, 8, 1, torch.float16), (128, 128, 6, 1, torch.float16)])
def test_few_prompts_share_their_keys(cuda, new, total, page, d, group, kv, dtype):
    """So few that clusters of CTAs share the keys of each: shares that see nothing of the keys or only for some rows, sequences of a share or less."""
    g = _gen(page, d, len(new), total[0])
    cache, table, lens = E.make(kv, page, d, total, cuda, g, width=5000 // page + 1)
    starts = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=cuda)
    q = torch.randn(sum(new) + 1, kv * group, d, generator=g).to(dtype).to(cuda)
    out = torch.full_like(q, 9.0)
    _attend(q, cache, lens, table, 1 / math.sqrt(d), starts, out=out)
    assert bool((out[-1] == 9).all())
    _attend(4 * q, cache, lens, table, -0.3, starts)
    table[:, 0] = table[0, 0].clone()  # the same beginning for all
    _attend(q, cache, lens, table, 1 / math.sqrt(d), starts)


def test_shared_keys_of_any_scale(cuda):
    """Poisoned blocks, scales of V of any size, queries that are not finite: where clusters share the keys, too."""
    from rmlk_b200 import kernels as K
    for d, dtype in ((64, torch.float32), (128, torch.float16)):
        g = _gen(21, d)
        cache, table, n = E.make(2, 64, d, [3000, 900], cuda, g)
        starts = torch.tensor([0, 100, 140], dtype=torch.int32, device=cuda)
        q = torch.randn(140, 8, d, generator=g).to(dtype).to(cuda)
        q[7, 3, 5], q[120, 0, 0] = math.nan, math.inf
        out = K.paged_attention(q, cache, n, table, d ** -0.5, starts=starts)
        want, bound = E.attention(q.nan_to_num(0.0, 0.0), cache, n, table, d ** -0.5, starts)
        want[7, 3], want[120, 0] = math.nan, math.nan
        assert torch.equal(torch.isnan(out), torch.isnan(want))
        E.close(out, want, bound)
        q = torch.randn(140, 8, d, generator=g).to(dtype).to(cuda)
        for spread in ((-60, 40), (-9, 0)):
            cache.v_scales.copy_(torch.exp2(torch.randint(*spread, cache.v_scales.shape, generator=g).float()))
            if spread[0] > -20 or dtype == torch.float32:
                _attend(q, cache, n, table, d ** -0.5, starts)
        cache.v_scales.fill_(0.125)
        cache.k_scales[table[0, 46], 1] = math.nan  # tokens 2944 .. 2999, of which the first 44 are seen by all rows
        out = K.paged_attention(q, cache, n, table, d ** -0.5, starts=starts)
        cache.k_scales[table[0, 46], 1] = 0.125
        want, bound = E.attention(q, cache, n, table, d ** -0.5, starts)
        want[44:100, 4:] = math.nan
        assert torch.equal(torch.isnan(out), torch.isnan(want))
        E.close(out, want, bound)


def test_queries_are_rotated_in_place(cuda):
    from rmlk_b200 import kernels as K
    g = _gen(22)
    cos, sin = _tables(100, 64, cuda)
    for dtype, new in ((torch.float32, 1), (torch.float16, 40)):
        cache, table, lens = E.make(2, 16, 64, [90, 50, 41], cuda, g)
        q, k, v = (torch.randn(3 * new, h, 64, generator=g).to(dtype).to(cuda) for h in (6, 2, 2))
        want = K.paged_append(cache, k, v, lens, table, cos, sin, q=q)
        got = K.paged_append(cache, k, v, lens, table, cos, sin, q=q, q_out=q)
        assert got is q and torch.equal(q, want)


def test_rows_that_lie_apart(cuda):
    from rmlk_b200 import kernels as K
    g = _gen(6)
    for dtype in (torch.float32, torch.float16):
        for each in (1, 40):
            lens = [100, 50, 77]
            cache, table, n = E.make(2, 32, 64, lens, cuda, g)
            wide = torch.randn(3 * each, 10, 64, generator=g).to(dtype).to(cuda)
            place = torch.full((3 * each, 9, 64), 4.0, dtype=dtype, device=cuda)
            _attend(wide[:, 2:8], cache, n, table, 0.125, out=place[:, 1:7])
            assert bool((place[:, 0] == 4).all()) and bool((place[:, 7:] == 4).all())


def test_what_lies_behind_the_last_token(cuda):
    """Codes of the rest of a page and pages that no row sees, their scales NaN and infinite, have no part in the result; nor have table entries
    behind the last page."""
    from rmlk_b200 import kernels as K
    g = _gen(7)
    for page in (16, 64, 128):
        for each, lens in ((1, [page + 3, 5, 2 * page, 300]), (50, [page + 50, 50, 2 * page + 60, 300])):
            cache, table, n = E.make(2, page, 64, lens, cuda, g, width=40)
            q = torch.randn(4 * each, 8, 64, generator=g).to(cuda)
            a = _attend(q, cache, n, table, 0.125)
            used = set()
            for b, m in enumerate(lens):
                for j in range(-(-m // page)):
                    p = int(table[b, j])
                    used.add(p)
                    end = min(page, m - j * page)
                    cache.k[p, :, end:], cache.v[p, :, end:] = 127, -128
            for p in set(range(cache.k.shape[0])) - used:
                cache.k_scales[p], cache.v_scales[p] = math.nan, math.inf
            table[table < 0] = 2 ** 31 - 1
            assert torch.equal(_attend(q, cache, n, table, 0.125), a)


def test_poisoned_blocks_and_scales_of_any_size(cuda):
    """A NaN scale makes NaN of the rows and heads that see a token of that page, and of no others; scales from 2^-126 to 2^100, zero among them."""
    from rmlk_b200 import kernels as K
    g = _gen(8)
    for d in (64, 128):
        for each in (1, 70):
            lens = [200, 200, 200]
            cache, table, n = E.make(2, 16, d, lens, cuda, g)
            q = torch.randn(3 * each, 4, d, generator=g).to(cuda)
            bad_k, bad_v = int(table[0, 3]), int(table[1, 12])  # positions 48 .. 63; 192 .. 207, of which 192 .. 199 are there
            cache.k_scales[bad_k, 0] = math.nan
            cache.v_scales[bad_v, 1] = math.nan
            out = K.paged_attention(q, cache, n, table, d ** -0.5)
            want, bound = E.attention(q, cache, n, table, d ** -0.5)
            assert torch.equal(torch.isnan(out), torch.isnan(want))
            E.close(out, want, bound)
            assert bool(torch.isnan(out[each - 1, :2]).all()) and not bool(torch.isnan(out[each - 1, 2:]).any())
            for spread in ((-126, 100), (-40, 40), (-20, 20)):
                cache, table, n = E.make(2, 16, d, lens, cuda, g)
                cache.v_scales.copy_(torch.exp2(torch.randint(*spread, cache.v_scales.shape, generator=g).float()))
                cache.v_scales[table[2, 1].long()] = 0
                _attend(q, cache, n, table, d ** -0.5)


def test_small_values_are_not_lost_beside_large_ones(cuda):
    """A page whose values are 2^30 times those of the others, under weights of exp(-100): the rest decides the result and keeps its precision."""
    from rmlk_b200 import kernels as K
    g = _gen(9)
    for each in (1, 40):
        for dtype, rel in ((torch.float32, 2e-6), (torch.float16, 2.5e-3)):
            lens = [160, 160]
            cache, table, n = E.make(1, 16, 64, lens, cuda, g)
            cache.k_scales.fill_(2.0 ** -5)
            cache.k[..., 0] = 64  # a component that is 2 for all ...
            for b in range(2):
                p = int(table[b, 2 + b])
                cache.k[p, ..., 0] = -127
                cache.k_scales[p] = 0.4  # ... but one page
                cache.v_scales[p] = 2.0 ** 25
            q = torch.randn(2 * each, 3, 64, generator=g).to(dtype).to(cuda)
            q[..., 0] = 20
            out = K.paged_attention(q, cache, n, table, 0.125)
            want, _ = E.attention(q, cache, n, table, 0.125)
            assert float((out.double() - want).norm() / want.norm()) < rel


def test_queries_of_any_size(cuda):
    from rmlk_b200 import kernels as K
    g = _gen(10)
    for each in (1, 40):
        cache, table, n = E.make(2, 64, 64, [90, 300], cuda, g)
        q = torch.randn(2 * each, 8, 64, generator=g).to(cuda)
        for up in (1e-30, 1e-3, 1e4, 1e30):
            _attend(q * up, cache, n, table, 0.125 / up)
        big = q.clone()
        big[0, 0, 0] = math.nan
        big[0, 1, 5] = math.inf
        out = K.paged_attention(big, cache, n, table, 0.125)
        assert bool(torch.isnan(out[0, :2]).all()) and not bool(torch.isnan(out[0, 2:]).any()) and not bool(torch.isnan(out[1:]).any())
        zero = _attend(torch.zeros_like(q), cache, n, table, 0.125)
        assert torch.equal(zero[each - 1, 0], zero[each - 1, 1])
        _attend(q, cache, n, table, 0.0)


def test_queries_with_outliers(cuda):
    """A few values of a query are far larger than the rest, in dims that keys have no part in or the same in all: the rest decides the weights.

    D fp32 roundings of 2^-24 each in a score, where the bound of `attention` counts D / 16 + 8 of 2^-23: at most 4 times that for D = 128."""
    from rmlk_b200 import kernels as K
    g = _gen(24)
    for d, group, dtype in ((64, 4, torch.float32), (128, 3, torch.float16), (128, 16, torch.float32), (64, 9, torch.float16)):
        for each in (1, 2, 300):
            lens = [each + 500, each, 5000]
            cache, table, n = E.make(2, 32, d, lens, cuda, g)
            cache.k[..., 3], cache.k[..., 17] = 0, 0
            for up in (3.0, 40.0, 1000.0, 30000.0):
                q = torch.randn(3 * each, 2 * group, d, generator=g).to(dtype).to(cuda)
                q[1::2, :, 3], q[:, 1::2, 17] = up, -up
                out = K.paged_attention(q, cache, n, table, d ** -0.5)
                want, bound = E.attention(q, cache, n, table, d ** -0.5)
                E.close(out, want, 4 * bound)


def test_pages_out_of_range(cuda):
    """A row that sees a token without a valid page is NaN and the status says so; the others have their values."""
    from rmlk_b200 import kernels as K
    g = _gen(11)
    for each in (1, 40):
        lens = [100, 100, 100, 170]
        cache, table, n = E.make(2, 32, 64, lens, cuda, g, width=6)
        good = table.clone()
        table[1, 3], table[3, 0] = 10 ** 6, -5
        n[3] = 32 * 6 + 20  # longer than its row of the table
        n[2] = 30 + each
        q = torch.randn(4 * each, 4, 64, generator=g).to(cuda)
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        out = K.paged_attention(q, cache, n, table, 0.125, status=status)
        assert int(status) == 1
        torch.cuda.synchronize()
        want, bound = E.attention(q, cache, torch.tensor([100, 100, 30 + each, 170], device=cuda), good, 0.125)
        sees = torch.arange(each, device=cuda) + 100 - each >= 96
        assert torch.equal(torch.isnan(out[each: 2 * each]).all(2).all(1), sees) and bool(torch.isnan(out[3 * each:]).all())
        want[each: 2 * each][sees] = math.nan
        want[3 * each:] = math.nan
        E.close(out, want, bound)
        assert not bool(torch.isnan(out[:each]).any())


def test_workspaces(cuda):
    """One workspace for calls of every size one after the other, results that do not depend on it, and its counters zero again."""
    from rmlk_b200 import kernels as K
    g = _gen(12)
    calls = []
    for batch, each, kv, group, d, most in ((1, 1, 1, 4, 64, 20000), (40, 1, 2, 4, 64, 900), (3, 4, 1, 6, 128, 5000), (200, 1, 1, 1, 64, 100), (2, 2, 1, 16, 128, 3000)):
        lens = [1 + (i * 7919) % most for i in range(batch)]
        lens[0] = most
        cache, table, n = E.make(kv, 64, d, lens, cuda, g)
        calls.append((torch.randn(batch * each, kv * group, d, generator=g).to(cuda), cache, n, table, d ** -0.5))
    own = [K.paged_attention(*c) for c in calls]
    need = max((K.paged_attention_workspace(c[0], c[1], c[3].shape[0]) for c in calls), key=lambda t: t.numel())
    for order in (calls, calls[::-1], calls):
        for c in order:
            out = K.paged_attention(*c, workspace=need)
            assert torch.equal(out, own[[x is c for x in calls].index(True)])
    if need.numel() > 16:
        with pytest.raises(K.RmlkError, match="workspace"):
            K.paged_attention(*calls[0], workspace=need[:16])


def test_graphs_and_streams(cuda):
    """A captured step replayed as its lengths grow: append and attention read lengths and pages on the device."""
    from rmlk_b200 import kernels as K
    g = _gen(13)
    cache, table, _ = E.make(2, 16, 64, [64, 64, 64], cuda, g)
    lens = torch.tensor([10, 0, 30], dtype=torch.int32, device=cuda)
    cos, sin = _tables(64, 64, cuda)
    q, k, v = (torch.zeros(3, h, 64, device=cuda) for h in (8, 2, 2))
    work = K.paged_attention_workspace(q, cache, 3)

    def step():
        x = K.paged_append(cache, k, v, lens, table, cos, sin, q=q)
        return K.paged_attention(x, cache, lens, table, 0.125, workspace=work)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    plain = E.Cache(cache)
    for i in range(25):
        lens += torch.tensor([1, 1 if i > 5 else 0, 1], dtype=torch.int32, device=cuda)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        want, _ = plain.append(k, v, lens, table, cos, sin, q)
        plain.same(cache)
        written = ~torch.isnan(want).any(2)
        x = K.paged_append(cache, k, v, lens, table, cos, sin, q=q)
        E.same_queries(x.cpu()[written], want[written], q.cpu()[written])
        x = torch.nan_to_num(x.masked_fill(~written.to(cuda)[..., None], 0.0))
        want, bound = E.attention(x, cache, lens, table, 0.125)
        E.close(out, want, bound)


def test_calls_side_by_side(cuda):
    """Single tokens, a few prompts (clusters) and many, captured each on a stream of its own and replayed at the same time over one cache, with a workspace each."""
    from rmlk_b200 import kernels as K
    g = _gen(23)
    calls = []
    lens = [700, 90, 2000, 1, 300, 512]
    cache, table, n = E.make(2, 32, 64, lens, cuda, g)
    for new in ([1] * 6, [40, 7, 64, 1, 90, 33], [700, 90, 1500, 1, 300, 512]):
        starts = torch.tensor([sum(new[:b]) for b in range(7)], dtype=torch.int32, device=cuda) if max(new) > 1 else None
        q = torch.randn(sum(new), 8, 64, generator=g).to(torch.float16).to(cuda)
        calls.append((q, cache, n, table, 0.125, starts, torch.empty_like(q), K.paged_attention_workspace(q, cache, 6, starts is not None)))
    alone = [K.paged_attention(*c).clone() for c in calls]
    torch.cuda.synchronize()
    streams, graphs = [torch.cuda.Stream() for _ in calls], []
    for s, c in zip(streams, calls):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            K.paged_attention(*c)
            K.paged_attention(*c)
        graphs.append(graph)
    for c in calls:
        c[6].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for c, want in zip(calls, alone):
        assert torch.equal(c[6], want)


def test_a_decoder_layer(cuda):
    """A prompt and a few steps as a program runs them: quantised projections, append, attention, output projection; against the same
    in 64 bits on the codes and scales that the operators left."""
    from rmlk_b200 import kernels as K
    g = _gen(14)
    hidden, kv, group, d, page, batch = 256, 2, 4, 64, 16, 3
    heads = kv * group
    w_qkv = K.quantize_weight((torch.randn(hidden, (heads + 2 * kv) * d, generator=g) / 16).to(cuda))
    w_o = K.quantize_weight((torch.randn(heads * d, hidden, generator=g) / 22).to(cuda))
    cos, sin = _tables(200, d, cuda)
    cache = K.paged_cache(60, kv, page, d, cuda)
    table = _table(batch, 12, 60, g, cuda)
    plain = E.Cache(cache)
    lens = torch.zeros(batch, dtype=torch.int32, device=cuda)
    for new in ([33, 1, 90], None, None, [1, 5, 40], None):
        counts = torch.tensor(new or [1] * batch, dtype=torch.int32)
        starts = torch.cumsum(torch.cat([torch.zeros(1), counts]), 0).to(torch.int32).to(cuda) if new else None
        lens += counts.to(cuda)
        x = torch.randn(int(counts.sum()), hidden, generator=g).to(cuda)
        qkv = K.matmul_i8(*K.quantize_rows(x), *w_qkv).view(-1, heads + 2 * kv, d)
        q = K.paged_append(cache, qkv[:, heads: heads + kv], qkv[:, heads + kv:], lens, table, cos, sin, q=qkv[:, :heads], starts=starts)
        y = K.paged_attention(q, cache, lens, table, d ** -0.5, starts=starts)
        out = K.matmul_i8(*K.quantize_rows(y.view(-1, heads * d)), *w_o)
        plain_q, _ = plain.append(qkv[:, heads: heads + kv], qkv[:, heads + kv:], lens, table, cos, sin, qkv[:, :heads], starts)
        E.same_queries(q, plain_q, qkv[:, :heads])
        plain.same(cache)
        want, bound = E.attention(q, cache, lens, table, d ** -0.5, starts)
        E.close(y, want, bound)
        codes, scales = E.quantized(y.view(-1, heads * d))
        want = (codes @ w_o[0].cpu().double().T) * scales.double()[:, None] * w_o[1].cpu().double()
        assert bool(((out.cpu().double() - want).abs() <= 3.001 * 2.0 ** -24 * want.abs()).all())


def test_a_cache_beyond_32_bit_offsets(cuda):
    """Pages whose codes lie more than 2^31 bytes into the cache."""
    from rmlk_b200 import kernels as K
    g = _gen(15)
    kv, page, d = 8, 128, 128
    pages = 2 ** 31 // (kv * page * d) + 40
    cache = K.paged_cache(pages, kv, page, d, cuda)
    table = torch.tensor([[pages - 1, pages - 3, pages - 2], [pages - 20, 0, pages - 7]], dtype=torch.int32, device=cuda)
    lens = torch.tensor([300, 270], dtype=torch.int32, device=cuda)
    k, v = (torch.randn(2 * 200, kv, d, generator=g).to(cuda) for _ in range(2))
    K.paged_append(cache, k, v, lens, table)
    lens1 = lens + 1
    k1, v1 = (torch.randn(2, kv, d, generator=g).to(cuda) for _ in range(2))
    K.paged_append(cache, k1, v1, lens1, table)
    used = table.flatten().tolist()
    small = K.PagedCache(*(t[table.flatten().long()] for t in cache))
    plain = E.Cache(K.paged_cache(6, kv, page, d, cuda))
    near = torch.arange(6, dtype=torch.int32, device=cuda).view(2, 3)
    plain.append(k, v, lens, near)
    plain.append(k1, v1, lens1, near)
    plain.same(small)
    assert len(set(used)) == 6
    for each in (1, 100):
        q = torch.randn(2 * each, 2 * kv, d, generator=g).to(cuda)
        out = K.paged_attention(q, cache, lens1, table, d ** -0.5)
        want, bound = E.attention(q, small, lens1, near, d ** -0.5)
        E.close(out, want, bound)
