"""Rows as 8-bit integers (quantize.cu) and products of them (matmul_i8.cu) against 64 bits."""
import math

import pytest
import torch

from eight_bit import quantized

pytestmark = pytest.mark.gpu


def _gen(*seed):
    g = torch.Generator()
    g.manual_seed(sum((i + 1) * 7919 * s for i, s in enumerate(seed)))
    return g


def _same(codes, scales, x):
    """Codes and scales as the definition has them; a row with an infinity (a wide row in f16 may hold one) has the scale NaN."""
    want, s = quantized(x)
    assert torch.equal(torch.isnan(scales.cpu()), torch.isnan(s)) and torch.equal(torch.nan_to_num(scales.cpu()), torch.nan_to_num(s))
    assert torch.equal(codes.cpu().double(), want)


# widths around 16-byte units and the width that a CTA of any kind covers, one row and many
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (2, 15), (5, 16), (7, 17), (300, 64), (2, 1003), (64, 2048), (3, 4100), (2, 14336), (2, 20001), (1000, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows(cuda, rows, cols, dtype):
    from rmlk_b200 import kernels as K
    g = _gen(rows, cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))).to(dtype)
    codes, scales = K.quantize_rows(x.to(cuda))
    _same(codes, scales, x)
    assert codes.stride(0) % 16 == 0 or rows == 1


def test_rows_that_lie_apart_or_start_anywhere(cuda):
    from rmlk_b200 import kernels as K
    g = _gen(5)
    store = torch.randn(9, 700, generator=g).to(cuda)
    for dtype in (torch.float32, torch.float16):
        for first, cols in ((0, 640), (1, 640), (3, 333), (4, 1)):
            x = store.to(dtype)[:, first: first + cols]
            place = torch.full((9, 801), 99, dtype=torch.int8, device=cuda)
            codes, _ = K.quantize_rows(x, codes=place[:, 5: 5 + cols])
            want, _ = quantized(x)
            assert torch.equal(codes.cpu().double(), want)
            assert bool((place[:, :5] == 99).all()) and bool((place[:, 5 + cols:] == 99).all())


def test_codes_next_to_the_middle(cuda):
    """Values whose quotient lies on, just above and just below the middle between two integers, for scales of every size."""
    from rmlk_b200 import kernels as K
    rows = []
    for e in (-149, -130, -126, -120, -101, -100, -60, 0, 60, 118, 120):
        for mantissa in (1.0, 1.1, 1.5, 1.9999):
            top = torch.tensor(mantissa * 127 * 2.0 ** e, dtype=torch.float64).float()
            if not bool(torch.isfinite(top)):
                continue
            s = max(float((top.double() / 127).float()), 2.0 ** -126)
            mid = torch.tensor([(c + 0.5) * s for c in range(-127, 127)], dtype=torch.float64).float()
            around = [mid, torch.nextafter(mid, torch.full_like(mid, math.inf)), torch.nextafter(mid, torch.full_like(mid, -math.inf))]
            x = torch.cat(around + [top.view(1), -top.view(1)])
            rows.append(x.clamp(-top, top))
    x = torch.stack(rows)
    codes, scales = K.quantize_rows(x.to(cuda))
    _same(codes, scales, x)


def test_rows_of_zeros_infinities_and_nans(cuda):
    from rmlk_b200 import kernels as K
    x = torch.randn(7, 65)
    x[1] = 0
    x[2, 64] = math.inf
    x[3, 0] = -math.inf
    x[4, 33] = math.nan
    x[5] = 3.4e38
    for dtype in (torch.float32, torch.float16):
        codes, scales = K.quantize_rows(x.to(dtype).to(cuda))
        _same(codes, scales, x.to(dtype))


def test_no_rows_and_no_columns(cuda):
    from rmlk_b200 import kernels as K
    codes, scales = K.quantize_rows(torch.empty(0, 8, device=cuda))
    assert codes.shape == (0, 8) and scales.shape == (0,)
    codes, scales = K.quantize_rows(torch.empty(3, 0, device=cuda))
    assert codes.shape == (3, 0) and scales.tolist() == [2.0 ** -126] * 3
    out = K.matmul_i8(codes, scales, torch.empty(5, 0, dtype=torch.int8, device=cuda), torch.ones(5, device=cuda))
    assert out.tolist() == [[0.0] * 5] * 3
    assert K.matmul_i8(torch.empty(0, 16, dtype=torch.int8, device=cuda), torch.empty(0, device=cuda), torch.empty(4, 16, dtype=torch.int8, device=cuda),
                       torch.ones(4, device=cuda)).shape == (0, 4)


def _codes(g, rows, k, dev, low=-128):
    store = torch.full((rows, (k + 15) // 16 * 16 + 16), 77, dtype=torch.int8)  # what lies behind a row's codes is no part of it
    store[:, :k] = torch.randint(low, 128, (rows, k), generator=g).to(torch.int8)
    return store.to(dev)[:, :k]


def _close(out, x, sx, w, sw):
    want = (x.double() @ w.double().T) * (sx.double()[:, None] * sw.double())
    # the sum exact; its conversion, the product of the scales and that with the sum: a rounding each.  f16: one more, or half its least step
    limit = 3.001 * 2.0 ** -24 * want.abs() if out.dtype == torch.float32 else 1.001 * 2.0 ** -11 * want.abs() + 2.0 ** -25
    err = (out.double() - want).abs()
    assert bool((err <= limit).all()), (float(err.max()), (err > limit).nonzero()[:4].tolist())


# rows around the sizes at which another kernel or tile takes over; channels and depths on and off 16, 64, 128
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 5, 17), (1, 128, 64), (1, 2048, 2048), (2, 130, 127), (3, 1000, 4096), (5, 64, 16), (8, 2048, 1003), (9, 777, 256), (16, 128, 128),
                                   (17, 129, 129), (31, 300, 2047), (32, 512, 8192), (33, 96, 640), (64, 2048, 2048), (65, 1003, 777), (100, 16, 31), (128, 4097, 512), (129, 128, 100),
                                   (200, 700, 1500), (256, 1024, 1024), (257, 255, 4096), (511, 513, 515), (1000, 2000, 300), (2049, 384, 128), (300, 20000, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_product(cuda, m, n, k, dtype):
    from rmlk_b200 import kernels as K
    g = _gen(m, n, k)
    x, w = _codes(g, m, k, cuda), _codes(g, n, k, cuda)
    sx, sw = (torch.exp(torch.randn(r, generator=g)).to(cuda) / (40 if dtype == torch.float16 else 1) / math.sqrt(k) for r in (m, n))
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = K.matmul_i8(x, sx, w, sw, dtype=dtype, status=status)
    _close(out, x, sx, w, sw)
    assert int(status) == 0
    place = torch.full((m + 1, n + 8), 7.0, dtype=dtype, device=cuda)  # rows of the result that lie apart
    K.matmul_i8(x, sx, w, sw, dtype=dtype, out=place[:m, :n])
    assert torch.equal(place[:m, :n], out) and bool((place[m:] == 7).all()) and bool((place[:, n:] == 7).all())


@pytest.mark.parametrize("m,n,k", [(1, 64, 131071), (4, 128, 131071), (40, 130, 131071), (300, 256, 65537)])
def test_sums_at_the_edge_of_32_bits(cuda, m, n, k):
    """All codes -128: 131071 products of 2^14 are 2^31 - 2^14."""
    from rmlk_b200 import kernels as K
    ld = (k + 15) // 16 * 16
    x, w = (torch.full((r, ld), -128, dtype=torch.int8, device=cuda)[:, :k] for r in (m, n))
    out = K.matmul_i8(x, torch.ones(m, device=cuda), w, torch.ones(n, device=cuda))
    assert out.unique().tolist() == [float(torch.tensor(k * 2 ** 14, dtype=torch.int64).float())]


def test_scales_of_any_size(cuda):
    """Scales whose product is ordinary although the sum times one of them is not; zeros, infinities and NaN in scales."""
    from rmlk_b200 import kernels as K
    g = _gen(9)
    for m in (2, 40, 300):
        x, w = _codes(g, m, 200, cuda), _codes(g, 33, 200, cuda)
        for a, b in ((1e37, 1e-37), (1e-37, 1e37), (1e-30, 1e-30), (1.0, 0.0)):
            sx, sw = torch.full((m,), a, device=cuda), torch.full((33,), b, device=cuda)
            out = K.matmul_i8(x, sx, w, sw)
            want = (x.double() @ w.double().T) * sx.double()[:, None] * sw.double()
            assert bool(((out.double() - want).abs() <= 2.0 ** -22 * want.abs() + 2.0 ** -149).all())
        sx, sw = torch.ones(m, device=cuda), torch.ones(33, device=cuda)
        sx[1], sw[2] = math.nan, math.inf
        out = K.matmul_i8(x, sx, w, sw)
        assert bool(torch.isnan(out[1]).all()) and bool(torch.isfinite(out[0, :2]).all()) and not bool(torch.isfinite(out[:, 2]).any())


def test_both_together_as_a_layer_uses_them(cuda):
    """x w with w quantised once ([k, n], as the other products take it) and x on the way: the error is that of the codes."""
    from rmlk_b200 import kernels as K
    g = _gen(11)
    x, w = torch.randn(37, 500, generator=g).to(cuda), (torch.randn(500, 260, generator=g) / 22).to(cuda)
    wc, ws = K.quantize_weight(w)
    assert wc.shape == (260, 500)
    out = K.matmul_i8(*K.quantize_rows(x), wc, ws)
    want = x.double() @ w.double()
    # each factor is off by half a step of its scale, largest / 254
    sx, sw = x.abs().amax(1).double() / 254, w.abs().amax(0).double() / 254
    limit = 1.001 * (sx[:, None] * w.double().abs().sum(0) + x.double().abs().sum(1)[:, None] * sw + 500 * sx[:, None] * sw)
    assert bool(((out.double() - want).abs() <= limit).all())
    assert float((out.double() - want).norm() / want.norm()) < 0.02


def test_streams_and_graphs(cuda):
    from rmlk_b200 import kernels as K
    g = _gen(13)
    x, w = torch.randn(20, 512, generator=g).to(cuda), _codes(g, 384, 512, cuda)
    sw = torch.ones(384, device=cuda)
    want = K.matmul_i8(*K.quantize_rows(x), w, sw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.matmul_i8(*K.quantize_rows(x), w, sw)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = K.matmul_i8(*K.quantize_rows(x), w, sw)
    x.copy_(torch.randn(20, 512, generator=g))
    for _ in range(3):
        graph.replay()
    assert torch.equal(got, K.matmul_i8(*K.quantize_rows(x), w, sw))


def test_operands_beyond_32_bit_offsets(cuda):
    from rmlk_b200 import kernels as K
    m, n, k = 65600, 64, 32768  # x: 2.15 GB
    x = torch.zeros(m, k, dtype=torch.int8, device=cuda)
    x[-3:] = torch.randint(-128, 128, (3, k), device=cuda)
    w = torch.randint(-128, 128, (n, k), device=cuda).to(torch.int8)
    sx, sw = torch.ones(m, device=cuda), torch.ones(n, device=cuda)
    out = K.matmul_i8(x, sx, w, sw)
    _close(out[-3:], x[-3:], sx[-3:], w, sw)
    assert not bool(out[:-3].any())
    del out
    values = torch.zeros(m, k, dtype=torch.float16, device=cuda)
    values[-1] = torch.randn(k, device=cuda)
    codes, scales = K.quantize_rows(values, codes=x)
    want, s = quantized(values[-1:])
    assert torch.equal(codes[-1:].cpu().double(), want) and torch.equal(scales[-1:].cpu(), s) and not bool(codes[:-1].any())
