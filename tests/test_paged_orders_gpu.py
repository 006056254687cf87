"""Attention over the paged 8-bit cache for batches in any order and tables far wider than their sequences."""
import pytest
import torch

import eight_bit as E

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [0, 2048])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
@pytest.mark.parametrize("d,dtype", [(64, torch.float32), (128, torch.float16), (128, torch.float32)])
def test_any_order_under_any_table(cuda, width, order, d, dtype):
    """Prompts, drafts and single tokens; few sequences, whose keys a cluster shares where the table has room for many, and more of them."""
    from rmlk_b200 import kernels as K
    g = torch.Generator()
    g.manual_seed(d + width)
    for batch, each in ((3, None), (24, None), (24, 1), (24, 5), (3, 40)):
        pairs = [(each or 1 + (i * 37) % 150, 7 + (i * 331) % 900) for i in range(batch)]
        pairs.sort(reverse=order == "falling") if order != "mixed" else None
        new, total = [a for a, _ in pairs], [a + b for a, b in pairs]
        cache, table, n = E.make(2, 32, d, total, cuda, g, width=max(width, -(-max(total) // 32)))
        starts = None if each else torch.tensor([sum(new[:b]) for b in range(batch + 1)], dtype=torch.int32, device=cuda)
        q = torch.randn(sum(new), 8, d, generator=g).to(dtype).to(cuda)
        out = K.paged_attention(q, cache, n, table, d ** -0.5, starts=starts)
        want, bound = E.attention(q, cache, n, table, d ** -0.5, starts)
        E.close(out, want, bound)
