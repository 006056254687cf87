"""Products whose launch overlaps the end of a kernel that runs for long: their bounded waits count their own time alone."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


class Long:
    """A call that keeps a few CTAs busy for some 2 s: a prompt over so many keys whose scales of V lie so far apart that its rows go one key after the
    other.  The next kernel of the stream is scheduled meanwhile."""

    def __init__(self, dev):
        from rmlk_b200 import kernels as K
        g = torch.Generator()
        g.manual_seed(1)
        self.keys = 2000000
        self.cache = K.paged_cache(4, 1, 128, 64, dev)
        self.cache.k.copy_(torch.randint(-100, 100, self.cache.k.shape, generator=g))
        self.cache.v.copy_(torch.randint(-100, 100, self.cache.v.shape, generator=g))
        self.cache.k_scales.fill_(2.0 ** -7)
        self.cache.v_scales.copy_(torch.tensor([[1.0], [2.0 ** -20], [1.0], [1.0]]))
        self.table = torch.randint(0, 4, (1, -(-self.keys // 128)), generator=g).to(torch.int32).to(dev)
        self.lens = torch.full((1,), self.keys, dtype=torch.int32, device=dev)
        self.starts = torch.tensor([0, 4], dtype=torch.int32, device=dev)
        self.q = torch.randn(4, 64, 64, generator=g).to(dev)

    def __call__(self):
        from rmlk_b200 import kernels as K
        return K.paged_attention(self.q, self.cache, self.lens, self.table, 0.125, starts=self.starts)


# one CTA to a tile, k shared by a cluster, pairs of CTAs
@pytest.mark.parametrize("m,n,k", [(100, 20000, 256), (3, 512, 2048), (2048, 2048, 512)])
def test_products_of_codes(cuda, m, n, k):
    from rmlk_b200 import kernels as K
    g = torch.Generator()
    g.manual_seed(m)
    x, w = (torch.randint(-128, 128, (r, k), generator=g).to(torch.int8).to(cuda) for r in (m, n))
    sx, sw = torch.ones(m, device=cuda), torch.ones(n, device=cuda)
    want = (x.double() @ w.double().T).float()  # (sums below 2^24 or rounded once)
    before, status, out = Long(cuda), torch.zeros(1, dtype=torch.int32, device=cuda), torch.empty(m, n, device=cuda)
    K.matmul_i8(x, sx, w, sw, out=out)  # (the first launch of a kernel would wait until it is loaded)
    out.fill_(math.nan)
    torch.cuda.synchronize()
    before()
    K.matmul_i8(x, sx, w, sw, out=out, status=status)
    assert torch.equal(out, want) and int(status) == 0


@pytest.mark.parametrize("m,n,k,dtype", [(64, 2048, 2048, torch.float16), (512, 1024, 512, torch.float16), (512, 2048, 512, torch.float32)])
def test_products(cuda, m, n, k, dtype):
    """Whole numbers that every step of the product holds exactly."""
    from rmlk_b200 import kernels as K
    g = torch.Generator()
    g.manual_seed(m)
    x, w = (torch.randint(-2, 3, s, generator=g).to(dtype).to(cuda) for s in ((m, k), (k, n)))
    want = (x.double() @ w.double()).to(dtype)
    before, out = Long(cuda), torch.empty(m, n, dtype=dtype, device=cuda)
    K.matmul(x, w, out=out)  # (the first launch of a kernel would wait until it is loaded)
    out.fill_(math.nan)
    torch.cuda.synchronize()
    before()
    K.matmul(x, w, out=out)
    assert torch.equal(out, want)
