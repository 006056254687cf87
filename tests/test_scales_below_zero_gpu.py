"""Scales below zero in the 8-bit operators that take scales from their caller: integer products, and appending to blocks that have one."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_products_under_scales_of_any_sign_and_size(cuda):
    """The product of the two scales is an ordinary number although the sum times one of them is not."""
    from rmlk_b200 import kernels as K
    g = torch.Generator()
    g.manual_seed(2)
    for m in (2, 40, 300):
        x, w = (torch.randint(-128, 128, (r, 208), generator=g).to(torch.int8).to(cuda) for r in (m, 33))
        for a, b in ((1e37, -1e-37), (-1e37, 1e-37), (-1e37, -1e-37), (-1e-37, 1e37), (-0.5, 0.25)):
            sx, sw = torch.full((m,), a, device=cuda), torch.full((33,), b, device=cuda)
            out = K.matmul_i8(x, sx, w, sw)
            want = (x.double() @ w.double().T) * sx.double()[:, None] * sw.double()
            assert bool(((out.double() - want).abs() <= 3.001 * 2.0 ** -24 * want.abs()).all())


@pytest.mark.parametrize("new", [1, 5])
@pytest.mark.parametrize("d", [64, 128])
def test_append_to_blocks_under_scales_below_zero(cuda, d, new):
    """The tokens that are there keep their values to half a step of the block's scale (to the last bit where that stays), the new ones are within half a step of theirs; the scale
    is the least that holds both, with the sign that it had."""
    from rmlk_b200 import kernels as K
    g = torch.Generator()
    g.manual_seed(d + new)
    for size, old in ((100.0, -0.25), (0.5, -4.0), (100.0, 0.25), (30.0, -0.25)):
        cache = K.paged_cache(3, 2, 16, d, cuda)
        for t in (cache.k, cache.v):
            t.copy_(torch.randint(-127, 128, t.shape, generator=g))
        cache.k_scales.fill_(old)
        cache.v_scales.fill_(old)
        before = [t.clone() for t in cache]
        k, v = (torch.randn(new, 2, d, generator=g).to(cuda) * size for _ in range(2))
        table = torch.tensor([[2]], dtype=torch.int32, device=cuda)
        K.paged_append(cache, k, v, torch.tensor([6 + new], dtype=torch.int32, device=cuda), table)
        for codes, scales, was, was_scale, fresh in ((cache.k, cache.k_scales, before[0], before[2], k), (cache.v, cache.v_scales, before[1], before[3], v)):
            assert torch.equal(codes[:2], was[:2]) and torch.equal(scales[:2], was_scale[:2]) and torch.equal(codes[2, :, 6 + new:], was[2, :, 6 + new:])
            need = torch.exp2(torch.ceil(torch.log2(fresh.double().abs().amax((0, 2)) / 127)))
            step = scales[2].double()
            assert torch.equal(step.abs(), torch.maximum(need, torch.full_like(need, abs(old)))) and bool((step.sign() == (1 if old > 0 else -1)).all())
            kept = (was[2, :, :6].double() * old - codes[2, :, :6].double() * step[:, None, None]).abs()
            assert bool((kept <= torch.where(step.abs() > abs(old), step.abs() / 2, 0.0)[:, None, None]).all())
            got = codes[2, :, 6: 6 + new].double() * step[:, None, None]
            assert bool(((got - fresh.double().permute(1, 0, 2)).abs() <= step.abs()[:, None, None] / 2).all())
