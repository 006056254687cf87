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
