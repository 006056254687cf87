"""Serving a decoder in 8 bits: the operators that a layer is made of, through the framework's public entry points.

Three kinds of cases:

* "product": activations quantised with a scale per token, multiplied in 8-bit integers with weights that have a scale per channel
  (`quantize_rows`, `matmul_i8`);
* "append": the keys and values of new tokens rotated and put into a paged cache of 8-bit codes that has one power-of-two scale per page
  and head, the queries rotated in the same call (`paged_append`);
* "attend": attention over such a cache, for one token per sequence, for a few, and for whole prompts (`paged_attention`).

`listed()` has twelve fixed cases, `draw(rng)` gives more of the same ranges.  The cache's codes are whole numbers that a kernel and the plain
form have to agree on to the last one; they are returned as they lie in the cache, with the scales that give them their values.
"""
import math

import torch

own = False

F16, F32 = "f16", "f32"
TORCH = {F16: torch.float16, F32: torch.float32}
SIZE = {F16: 2, F32: 4}
TINY = 2.0 ** -126


def listed():
    return [
        # one projection for the one token of a single request: the smallest call, all latency
        {"name": "product-1x2048x2048", "kind": "product", "m": 1, "k": 2048, "n": 2048, "dtype": F32},
        # gate and up laid side by side, one token of each of 64 requests
        {"name": "product-64x2048x16384", "kind": "product", "m": 64, "k": 2048, "n": 16384, "dtype": F32},
        # sizes that fit no tile: three short prompts, a width off every power of two
        {"name": "product-561x1003x777", "kind": "product", "m": 561, "k": 1003, "n": 777, "dtype": F32},
        # the up projection of a larger model over a long prompt, half precision around it: the heaviest call
        {"name": "product-4096x4096x14336", "kind": "product", "m": 4096, "k": 4096, "n": 14336, "dtype": F16},
        # one token of each of 64 requests goes into the cache
        {"name": "append-64x1", "kind": "append", "batch": 64, "tokens": 1, "ragged": False, "context": 700, "kv_heads": 8, "group": 4, "head_dim": 64, "page": 64,
         "dtype": F32},
        # prompts of different lengths, some behind a cached beginning
        {"name": "append-16x512", "kind": "append", "batch": 16, "tokens": 512, "ragged": True, "context": 200, "kv_heads": 8, "group": 4, "head_dim": 128, "page": 32,
         "dtype": F16},
        # one request, a short context
        {"name": "attend-1x1-512", "kind": "attend", "batch": 1, "tokens": 1, "ragged": False, "context": 512, "kv_heads": 8, "group": 4, "head_dim": 64, "page": 64,
         "dtype": F32},
        # a full serving batch, contexts of different lengths
        {"name": "attend-64x1-1000", "kind": "attend", "batch": 64, "tokens": 1, "ragged": False, "context": 1000, "kv_heads": 8, "group": 4, "head_dim": 64, "page": 64,
         "dtype": F32},
        # few requests with long contexts: the work is shared out along them
        {"name": "attend-3x1-50001", "kind": "attend", "batch": 3, "tokens": 1, "ragged": False, "context": 50001, "kv_heads": 8, "group": 8, "head_dim": 128, "page": 16,
         "dtype": F16},
        # four drafted tokens of each request are looked at in one step
        {"name": "attend-24x4-2000", "kind": "attend", "batch": 24, "tokens": 4, "ragged": False, "context": 2000, "kv_heads": 4, "group": 6, "head_dim": 128, "page": 32,
         "dtype": F16},
        # prompts of different lengths
        {"name": "attend-16x512-0", "kind": "attend", "batch": 16, "tokens": 512, "ragged": True, "context": 0, "kv_heads": 8, "group": 4, "head_dim": 64, "page": 64,
         "dtype": F32},
        # parts of long prompts, the beginnings of which are in the cache
        {"name": "attend-4x1024-5000", "kind": "attend", "batch": 4, "tokens": 1024, "ragged": True, "context": 5000, "kv_heads": 8, "group": 4, "head_dim": 128, "page": 128,
         "dtype": F16},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(2.0 ** rng.uniform(math.log2(lo), math.log2(hi))))))


def draw(rng):
    kind = rng.choice(["product", "append", "attend", "attend"])
    most = work(listed()[3 if kind == "product" else -1])["flops"]
    while True:
        case = _drawn(rng, kind)
        if work(case)["flops"] <= most:
            return case


def _drawn(rng, kind):
    dtype = rng.choice([F32, F16])
    if kind == "product":
        return {"kind": kind, "m": _log_int(rng, 1, 4096), "k": _log_int(rng, 128, 8192), "n": _log_int(rng, 128, 16384), "dtype": dtype}
    heads = {"kv_heads": rng.choice([1, 2, 4, 8]), "group": rng.choice([1, 2, 3, 4, 6, 8]), "head_dim": rng.choice([64, 128]), "page": rng.choice([16, 32, 64, 128]),
             "dtype": dtype}
    if kind == "append":
        ragged = rng.random() < 0.5
        return {"kind": kind, "batch": _log_int(rng, 1, 16 if ragged else 128), "tokens": _log_int(rng, 2, 512) if ragged else 1, "ragged": ragged,
                "context": _log_int(rng, 1, 1000), **heads}
    if rng.random() < 0.6:
        batch = _log_int(rng, 1, 64)
        return {"kind": kind, "batch": batch, "tokens": rng.choice([1, 1, 1, 2, 4]), "ragged": False, "context": _log_int(rng, 1, min(50000, 150000 // batch)), **heads}
    return {"kind": kind, "batch": _log_int(rng, 1, 8), "tokens": _log_int(rng, 8, 1024), "ragged": True, "context": rng.choice([0, _log_int(rng, 1, 4000)]), **heads}


# ---- sizes that follow from a case ----
def _lengths(case):
    """New tokens and cached tokens before them of each sequence: the case's figures for the first, less for those behind it."""
    b, t, c = case["batch"], case["tokens"], case["context"]
    new = [max(1, t - i * t * 2 // (3 * b)) if case["ragged"] else t for i in range(b)]
    if case["kind"] == "attend" and not case["ragged"]:  # the context includes the new tokens
        before = [max(0, c - t - i * c // (2 * b)) for i in range(b)]
    else:
        before = [c - i * c // (2 * b) for i in range(b)]
    return new, before


def _pairs(case):
    """Pairs of a query token and a cached token that it sees."""
    return sum(n * c + n * (n + 1) // 2 for n, c in zip(*_lengths(case)))


def work(case):
    e = SIZE[case["dtype"]]
    if case["kind"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": e * m * k + k * n + 4 * n + e * m * n, "flops": 2 * m * k * n}
    new, before = _lengths(case)
    heads, d = case["kv_heads"] * (case["group"] + 2), case["head_dim"]
    q = sum(new) * case["kv_heads"] * case["group"] * d * e
    if case["kind"] == "append":
        # q, k, v and the rows of the tables in; rotated q and codes out; a scale per block and head in and out
        kv = sum(new) * case["kv_heads"] * d * 2
        blocks = sum((c + n - 1) // case["page"] - c // case["page"] + 1 for n, c in zip(new, before))
        return {"bytes": 2 * q + kv * (e + 1) + sum(new) * d * 8 + blocks * case["kv_heads"] * 16, "flops": 3 * sum(new) * heads * d}
    total = sum(n + c for n, c in zip(new, before))
    blocks = sum(-(-(n + c) // case["page"]) for n, c in zip(new, before))
    return {"bytes": 2 * q + total * case["kv_heads"] * d * 2 + blocks * case["kv_heads"] * 8, "flops": 4 * _pairs(case) * case["kv_heads"] * case["group"] * d}


# ---- inputs ----
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = TORCH[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["kind"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        # a few channels are larger than the others, as in the activations of trained models
        x = (randn(m, k) * torch.exp(0.5 * randn(k))).to(dtype)
        w = randn(n, k) * torch.exp(0.3 * randn(n, 1)) / math.sqrt(k)
        # the weights as a program keeps them: quantised once, rows on 16-byte boundaries
        scales = w.abs().amax(1) / 127
        codes = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :k]
        codes.copy_(torch.round(w / scales[:, None]))
        return {"case": case, "x": x, "codes": codes, "scales": scales}

    new, before = _lengths(case)
    total = [n + c for n, c in zip(new, before)]
    batch, kv, group, d, page = case["batch"], case["kv_heads"], case["group"], case["head_dim"], case["page"]
    counts = [-(-t // page) for t in total]
    pages, width = sum(counts) + 3, max(counts) + 1  # a few pages belong to no sequence, the last one among them
    order = torch.randperm(pages - 1, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at: at + c]
        at += c
    tokens = sum(new)
    s = {"case": case, "table": table, "lens": torch.tensor(total, dtype=torch.int32, device="cuda"), "starts": None}
    if case["ragged"]:
        s["starts"] = torch.tensor([sum(new[:b]) for b in range(batch + 1)], dtype=torch.int32, device="cuda")
    s["most_new"], s["most"] = max(new), max(total)
    for name in ("k", "v"):
        scales = torch.exp2(torch.randint(-6, -3, (pages, kv), device="cuda", generator=gen).float())
        values = randn(pages, kv, page, d)
        s[name + "_scales"] = scales
        s[name + "_codes"] = torch.round(values / scales[:, :, None, None]).clamp(-127, 127).to(torch.int8)
    if case["kind"] == "append":
        # queries, keys and values side by side in the result of one product; tables for every position
        qkv = (randn(tokens, (group + 2) * kv, d) * torch.exp(0.5 * randn((group + 2) * kv, 1))).to(dtype)
        s["q"], s["new_k"], s["new_v"] = qkv[:, : group * kv], qkv[:, group * kv: (group + 1) * kv], qkv[:, (group + 1) * kv:]
        angle = torch.arange(max(total), device="cuda", dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(d // 2, device="cuda", dtype=torch.float64) * 2 / d)
        angle = torch.cat([angle, angle], 1)
        s["cos"], s["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
    else:
        s["q"] = randn(tokens, group * kv, d).to(dtype)
        s["scale"] = 1 / math.sqrt(d)
        s["workspace"] = torch.zeros(32 << 20, dtype=torch.uint8, device="cuda")  # a program has one for its largest call
    return s


# ---- one pass ----
def run(state):
    kind = state["case"]["kind"]
    if kind == "product":
        return _run_product(state)
    return _run_append(state) if kind == "append" else _run_attend(state)


def _run_product(s):
    x = s["x"]
    if own:
        from rmlk_b200 import kernels as K
        codes, scales = K.quantize_rows(x)
        return K.matmul_i8(codes, scales, s["codes"], s["scales"], dtype=x.dtype)
    scales = (x.float().abs().amax(1, keepdim=True) / 127).clamp_min(TINY)
    codes = torch.round(x.double() / scales.double())  # in 64 bits: quotients next to the middle between two codes
    sums = codes.float() @ s["codes"].float().T
    return (sums * scales * s["scales"]).to(x.dtype)


def _places(s):
    """Sequence, position, page and slot of each new token."""
    case, lens = s["case"], s["lens"].long()
    batch, tokens = case["batch"], s["q"].shape[0]
    row = torch.arange(tokens, device="cuda")
    if s["starts"] is None:
        new = torch.full_like(lens, tokens // batch)
        seq = row // (tokens // batch)
        first = seq * (tokens // batch)
    else:
        starts = s["starts"].long()
        new = starts[1:] - starts[:-1]
        seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
        first = starts[seq]
    pos = lens[seq] - new[seq] + row - first
    return seq, row - first, pos, new


def _cache(K, s):
    return K.PagedCache(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"])


def _rotated(x, cos, sin):
    """x cos + (-upper half, lower half) sin; the products of 32-bit values are exact in 64 bits, the sum is rounded once."""
    x, cos, sin = x.double(), cos.double(), sin.double()
    low, high = x.chunk(2, -1)
    return (x * cos + torch.cat([-high, low], -1) * sin).float()


def _least_scale(amax):
    """The least power of two, not below 2^-126, of which 127 times is not below amax; NaN where amax is not finite."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa 2^exponent, 1/2 <= mantissa < 1
    e = exponent - 7 + (mantissa > 127 / 128).int()
    scale = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), TINY).clamp_min(TINY)
    return torch.where(torch.isfinite(amax), scale, math.nan)


def _run_append(s):
    case = s["case"]
    if own:
        from rmlk_b200 import kernels as K
        c = _cache(K, s)
        q = K.paged_append(c, s["new_k"], s["new_v"], s["lens"], s["table"], cos=s["cos"], sin=s["sin"], q=s["q"], starts=s["starts"])
        return {"q": q, "k": c.k, "v": c.v, "k_scales": c.k_scales, "v_scales": c.v_scales}
    seq, _, pos, new = _places(s)
    page, batch = case["page"], case["batch"]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    out = {"q": _rotated(s["q"], cos, sin).to(s["q"].dtype)}
    # the pages that a sequence's new tokens fall into; places without one point to the last page, which belongs to nobody
    before = s["lens"].long() - new
    j = before[:, None] // page + torch.arange((s["most_new"] - 1) // page + 2, device="cuda")
    valid = j <= ((s["lens"].long() - 1) // page)[:, None]
    spare = s["k_scales"].shape[0] - 1
    pages = torch.where(valid, torch.gather(s["table"].long(), 1, j.clamp_max(s["table"].shape[1] - 1)), spare)
    kept = torch.where(valid, (before[:, None] - j * page).clamp(0, page), page)  # tokens that were there before
    page_of, slot = torch.gather(s["table"].long()[seq], 1, (pos // page)[:, None])[:, 0], pos % page
    kept_slots = torch.arange(page, device="cuda") < kept[:, :, None]
    out["k"], out["k_scales"] = _put(s["k_codes"], s["k_scales"], _rotated(s["new_k"], cos, sin), pages, valid, kept_slots, page_of, slot)
    out["v"], out["v_scales"] = _put(s["v_codes"], s["v_scales"], s["new_v"].float(), pages, valid, kept_slots, page_of, slot)
    return out


def _put(codes, scales, value, pages, valid, kept_slots, page_of, slot):
    """The values of the new tokens, [tokens, heads, D], into the cache."""
    amax = torch.zeros_like(scales).index_reduce_(0, page_of, value.abs().amax(2), "amax")
    keeps = kept_slots.any(2)[:, :, None]
    old = scales[pages]
    grown = torch.maximum(torch.where(keeps, old, 0.0), _least_scale(amax[pages]))
    grown = torch.where(valid[:, :, None], grown, old)
    ratio = torch.where(keeps, old / grown, 1.0)
    block = codes[pages]
    codes[pages] = torch.where(kept_slots[:, :, None, :, None], torch.round(block.float() * ratio[..., None, None]).to(torch.int8), block)
    scales[pages] = grown
    codes[page_of, :, slot] = torch.round(value / scales[page_of][:, :, None]).to(torch.int8)
    return codes, scales


def _run_attend(s):
    case = s["case"]
    if own:
        from rmlk_b200 import kernels as K
        return K.paged_attention(s["q"], _cache(K, s), s["lens"], s["table"], s["scale"], starts=s["starts"], workspace=s["workspace"])
    seq, row, pos, new = _places(s)
    batch, kv, group, d, page = case["batch"], case["kv_heads"], case["group"], case["head_dim"], case["page"]
    wide = -(-s["most"] // page)
    pages = s["table"][:, :wide].long().clamp_min(0)

    def dense(name):
        x = s[name + "_codes"][pages].float() * s[name + "_scales"][pages][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(batch, kv, wide * page, d)  # [sequence, head, token, value]

    # queries padded to the longest sequence's
    q = torch.zeros(batch, s["most_new"], kv, group, d, device="cuda")
    q[seq, row] = s["q"].float().view(-1, kv, group, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(batch, kv, group * s["most_new"], d)
    scores = (q @ dense("k").transpose(2, 3) * s["scale"]).view(batch, kv, group, s["most_new"], wide * page)
    at = (s["lens"].long() - new)[:, None] + torch.arange(s["most_new"], device="cuda")
    hidden = torch.arange(wide * page, device="cuda") > at[:, :, None]
    scores = scores.masked_fill(hidden[:, None, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    sums = weights.sum(-1)
    out = (weights.view(batch, kv, group * s["most_new"], wide * page) @ dense("v")).view(batch, kv, group, s["most_new"], d) / sums[..., None]
    return out.permute(0, 3, 1, 2, 4)[seq, row].reshape(-1, kv * group, d).to(s["q"].dtype)


# ---- the definition in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "product":
        x = s["x"].double()
        scale = (x.abs().max(1).values / 127).float().double().clamp(min=TINY)
        return (x / scale[:, None]).round() @ s["codes"].double().t() * (scale[:, None] * s["scales"].double())
    new, before = _lengths(case)
    page, kv, group, d = case["page"], case["kv_heads"], case["group"], case["head_dim"]
    table = s["table"].tolist()
    if case["kind"] == "append":
        if sum(new) > 20000:
            return None
        cos, sin = s["cos"].double(), s["sin"].double()
        half, outs = d // 2, []
        rotated = []
        for x in (s["q"].double(), s["new_k"].double()):
            y, at = torch.empty_like(x), 0
            for n, c in zip(new, before):
                a, b = x[at: at + n, :, :half], x[at: at + n, :, half:]
                co, si = cos[c: c + n, None], sin[c: c + n, None]
                y[at: at + n, :, :half] = a * co[..., :half] - b * si[..., :half]
                y[at: at + n, :, half:] = b * co[..., half:] + a * si[..., half:]
                at += n
            rotated.append(y)
        outs = {"q": rotated[0]}
        for name, x in (("k", rotated[1].float().double()), ("v", s["new_v"].double())):
            codes, scales, at = s[name + "_codes"].double(), s[name + "_scales"].double(), 0
            for b, (n, c) in enumerate(zip(new, before)):
                for j in range(c // page, (c + n - 1) // page + 1):
                    p, lo, hi = table[b][j], max(c, j * page), min(c + n, (j + 1) * page)
                    fresh = x[at + lo - c: at + hi - c].permute(1, 0, 2)
                    amax = fresh.abs().amax((1, 2))
                    need = torch.exp2(torch.ceil(torch.log2(amax / 127))).clamp(min=TINY)
                    keep = lo - j * page
                    scale = torch.maximum(scales[p], need) if keep else need
                    if keep:
                        codes[p, :, :keep] = (codes[p, :, :keep] * (scales[p] / scale)[:, None, None]).round()
                    codes[p, :, keep: keep + hi - lo] = (fresh / scale[:, None, None]).round()
                    scales[p] = scale
                at += n
            outs[name], outs[name + "_scales"] = codes.to(torch.int8), scales
        return outs
    out, at = torch.empty(sum(new), kv * group, d, dtype=torch.float64, device="cuda"), 0
    for b, (n, c) in enumerate(zip(new, before)):
        pages = torch.tensor(table[b][: -(-(n + c) // page)], device="cuda")
        for h in range(kv):
            k, v = ((s[x + "_codes"][pages, h].double() * s[x + "_scales"][pages, h].double()[:, None, None]).reshape(-1, d)[: n + c] for x in "kv")
            for g in range(group):
                w = s["q"][at: at + n, h * group + g].double() @ k.t() * s["scale"]
                w = torch.softmax(w + torch.full((n, n + c), -math.inf, dtype=torch.float64, device="cuda").triu(c + 1), 1)
                out[at: at + n, h * group + g] = w @ v
        at += n
    return out
