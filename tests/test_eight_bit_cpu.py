"""What the 8-bit serving operators refuse: decided on the host before anything is launched, so without a GPU."""
import ctypes

import pytest
import torch

F16, F32, I32 = 0, 1, 3
A = 1 << 20  # an address that is never read


def _lib():
    from rmlk_b200._lib import last_error, lib
    return lib(), last_error


def _quantize(dtype=F32, rows=4, cols=32, x=A, ldx=32, codes=A, ldc=32, scales=A):
    return _lib()[0].rmlk_b200_quantize_rows(None, dtype, rows, cols, x, ldx, codes, ldc, scales)


def _matmul(dtype=F32, m=4, n=8, k=32, x=A, ldx=32, sx=A, w=A, ldw=32, sw=A, out=A, ldo=8):
    return _lib()[0].rmlk_b200_matmul_i8(None, dtype, m, n, k, x, ldx, sx, w, ldw, sw, out, ldo, None)


def _cache(pages=4, kv=2, page=16, d=64, k=A, v=A, ks=A, vs=A):
    from rmlk_b200.kernels import _PagedCacheC
    return _PagedCacheC(pages, kv, page, d, k, v, ks, vs)


def _append(cache=None, dtype=F32, tokens=3, batch=3, starts=None, lens=A, table=A, width=2, k=A, lk=128, v=A, lv=128, cos=A, sin=A, rows=32, qh=4, q=A, lq=256, qo=A, lo=256, **c):
    cache = _cache(**c) if cache is None else cache
    return _lib()[0].rmlk_b200_paged_append(None, dtype, ctypes.addressof(cache) if cache else None, tokens, batch, starts, lens, table, width, k, lk, v, lv, cos, sin, rows, qh, q, lq, qo,
                                            lo, None)


def _attend(cache=None, dtype=F32, tokens=3, batch=3, qh=4, starts=None, lens=A, table=A, width=2, q=A, lq=256, out=A, lo=256, work=A, size=1 << 30, scale=0.125, **c):
    cache = _cache(**c) if cache is None else cache
    return _lib()[0].rmlk_b200_paged_attention(None, dtype, ctypes.addressof(cache) if cache else None, tokens, batch, qh, starts, lens, table, width, q, lq, scale, out, lo, work, size,
                                               None)


@pytest.mark.parametrize("call,bad", [
    (_quantize, [dict(rows=-1), dict(cols=-1), dict(rows=1 << 31), dict(cols=1 << 31), dict(x=0), dict(codes=0), dict(scales=0), dict(ldx=31), dict(ldc=31), dict(x=A + 2), dict(scales=A + 1)]),
    (_matmul, [dict(m=-1), dict(n=-1), dict(k=-1), dict(k=131072, ldx=131072, ldw=131072), dict(m=1 << 24), dict(n=1 << 24, ldo=1 << 24), dict(x=0), dict(w=0), dict(sx=0), dict(sw=0),
               dict(out=0), dict(ldx=16), dict(ldw=16), dict(ldo=7), dict(ldx=33), dict(ldw=40), dict(x=A + 8), dict(w=A + 1), dict(sx=A + 2), dict(sw=A + 1), dict(out=A + 2)]),
    (_append, [dict(cache=0), dict(page=8), dict(page=48), dict(page=256), dict(d=32), dict(d=96), dict(d=256), dict(pages=-1), dict(pages=1 << 31), dict(kv=0), dict(kv=65536), dict(tokens=-1),
               dict(batch=-1), dict(tokens=4), dict(width=-1), dict(width=1 << 28), dict(lens=0), dict(table=0), dict(k=0), dict(v=0), dict(ks=0), dict(vs=0), dict(lk=127), dict(lv=127), dict(lk=130),
               dict(k=A + 8), dict(v=A + 4), dict(cos=None), dict(sin=None), dict(cos=None, sin=None), dict(rows=-1), dict(qh=0), dict(qo=0), dict(lq=255), dict(lo=255), dict(q=A + 4),
               dict(qo=A + 8), dict(lens=A + 2), dict(table=A + 1), dict(starts=A + 2), dict(cos=A + 4)]),
    (_attend, [dict(cache=0), dict(page=8), dict(page=256), dict(d=96), dict(pages=-1), dict(kv=0), dict(qh=3), dict(qh=0), dict(qh=130, lq=130 * 64, lo=130 * 64), dict(tokens=4), dict(tokens=-3),
               dict(width=-1), dict(lens=0), dict(table=0), dict(q=0), dict(out=0), dict(lq=255), dict(lo=252), dict(lq=258), dict(lo=257), dict(q=A + 8), dict(out=A + 4), dict(lens=A + 1),
               dict(pages=0), dict(scale=float("inf")), dict(scale=float("nan")), dict(work=0), dict(work=A + 8), dict(size=0), dict(size=1 << 15), dict(starts=A + 2),
               dict(tokens=1 << 30, batch=1 << 30, qh=8, lq=512, lo=512)]),
])
def test_refused(call, bad):
    for case in bad:
        assert call(**case) == 1, case
        assert _lib()[1]().split(":")[0] in ("quantize_rows", "matmul_i8", "paged_append", "paged_attention"), case
    assert call(dtype=I32) == 2
    assert call(dtype=2) == 2  # f64


def test_nothing_to_do_is_no_error():
    assert _quantize(rows=0, x=0, codes=0, scales=0) == 0
    assert _matmul(m=0, x=0, sx=0, out=0) == 0 and _matmul(n=0, w=0, sw=0, out=0) == 0
    assert _append(tokens=0, k=0, v=0, q=0, qo=0) == 0 and _append(tokens=0, batch=0, lens=0, table=0) == 0
    assert _attend(tokens=0, q=0, out=0) == 0 and _attend(tokens=0, batch=0, lens=0, table=0) == 0


def test_bindings_refuse_before_the_call():
    from rmlk_b200 import kernels as K
    x = torch.zeros(4, 32)
    for call in (lambda: K.quantize_rows(x), lambda: K.quantize_rows(x[0]), lambda: K.quantize_weight(x), lambda: K.matmul_i8(x, x[0], x, x[0]),
                 lambda: K.matmul_i8(x.to(torch.int8), x[:, 0], x[:, :16].to(torch.int8), x[:, 0])):
        with pytest.raises(ValueError):
            call()
    cache = K.paged_cache(2, 1, 16, 64, "cpu")
    lens, table = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    q = torch.zeros(1, 1, 64)
    with pytest.raises(ValueError):
        K.paged_append(cache, q, q, lens, table)
    with pytest.raises(ValueError):
        K.paged_attention(q, cache, lens, table, 1.0)


def test_workspace_sizes():
    L = _lib()[0]
    size = L.rmlk_b200_paged_attention_workspace_bytes
    for d in (64, 128):
        assert size(64, 64, 32, 8, d, 0) > 0 == size(64, 64, 32, 8, d, 1)
        assert size(1, 1, 8, 8, d, 0) == size(64, 64, 32, 8, d, 0)  # one will do for all calls of a head_dim
        assert size(1 << 16, 8, 32, 8, d, 0) == 0  # whole prompts need none
        assert size(0, 0, 32, 8, d, 0) == size(5, 0, 32, 8, d, 0) == size(4, 4, 8, 0, d, 0) == size(4, 4, 4, 8, d, 0) == 0
