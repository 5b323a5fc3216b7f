"""GPU: rotary positions, the paged cache in three forms, attention of new tokens over it - against plain 64-bit restatements.

Tolerances are bounds, put together before the first run from what the kernels round: a result in T is off by half a step of T
(eps / 2 of its value), probabilities that are rounded to T before they meet the values add eps / 2 of sum p |v|, and fp32
arithmetic adds at most (number of terms) * 2^-23 of the sum of the terms' magnitudes."""
import itertools
import math

import pytest
import torch

import framefusion_amd as ffa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0 ** -23


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(dtype, want):
    """Half a step of `dtype` at the value `want`: eps / 2 of it, and below the smallest normal number `tiny`, where steps no longer
    shrink, half of tiny * eps (float16: 2^-14 * 2^-10 / 2 = 2^-25)."""
    return half_step(dtype) * want.abs().clamp(min=torch.finfo(dtype).tiny)


def within(got, want, tol):
    """|got - want| <= tol everywhere, NaN where and only where NaN is wanted."""
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    bad = ~((got - want).abs() <= tol) & ~torch.isnan(want)
    assert not bad.any(), (int(bad.sum()), float((got - want).abs()[bad].max()), float((tol + torch.zeros_like(want))[bad].min()))


# ------------------------------------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape,interleaved,half", [((1, 1), False, 64), ((3, 1, 37), False, 64), ((2, 5), True, 16), ((1, 0), False, 8), ((1, 1001), False, 3)])
def test_tables(dtype, shape, interleaved, half):
    gen = torch.Generator(device=DEV).manual_seed(half)
    pos = torch.randint(-5, 1 << 20, shape, generator=gen, device=DEV)
    if pos.numel() > 3:
        pos.view(-1)[:4] = torch.tensor([0, 1, 2**31 - 1, -2**31])
    inv, _ = ffa.rotary_frequencies(2 * half, 1e6, {"rope_type": "linear", "factor": 1.5})
    inv, factor = inv.to(DEV), 1.25
    cos, sin = ffa.rotary_tables(pos, inv, dtype=DT[dtype], factor=factor, interleaved=interleaved)
    a = pos.double()[..., None] * inv
    a = a.repeat_interleave(2, -1) if interleaved else torch.cat((a, a), -1)
    # 64 bits: three roundings of a phase of |pos * inv| radians; fp32: the rest of a turn (2^-26 turns), sine and cosine (4 ulp), the factor
    phase = a.abs() * 4 * 2.0 ** -53
    for got, want in ((cos, torch.cos(a) * factor), (sin, torch.sin(a) * factor)):
        assert got.dtype == DT[dtype]
        within(got, want, factor * (2 * phase + 2 * math.pi * 2.0 ** -25 + 6 * U) + rounding(DT[dtype], want))


def rotated(x, cos, sin, interleaved, transpose=False):
    rot = cos.shape[-1]
    y = x.clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    c1, c2, s1, s2 = cos[..., a], cos[..., b], sin[..., a], sin[..., b]
    if transpose:
        y[..., a], y[..., b] = x[..., a] * c1 + x[..., b] * s2, x[..., b] * c2 - x[..., a] * s1
    else:
        y[..., a], y[..., b] = x[..., a] * c1 - x[..., b] * s1, x[..., b] * c2 + x[..., a] * s2
    return y


def magnitudes(x, cos, sin, interleaved):
    """An upper bound of |x1 c1| + |x2 s| for either sine of the pair."""
    rot = cos.shape[-1]
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y, s = x.clone(), torch.maximum(sin[..., a], sin[..., b])
    y[..., a], y[..., b] = x[..., a] * cos[..., a] + x[..., b] * s, x[..., b] * cos[..., b] + x[..., a] * s
    return y


ROTARY = [  # B, L, H, H_kv, dh, rot, sections, interleaved
    (1, 1, 28, 4, 128, 128, None, False), (2, 7, 4, 2, 64, 64, None, True), (1, 65, 14, 2, 64, 32, None, False), (3, 5, 3, 1, 40, 24, None, True),
    (1, 33, 8, 2, 128, 128, (16, 24, 24), False), (2, 3, 4, 4, 36, 12, (1, 2, 3), False), (1, 1001, 8, 8, 256, 256, None, False), (1, 9, 6, 2, 10, 6, None, False),
    (2, 4, 70, 70, 32, 32, (5, 5, 6), False), (1, 4, 2, 1, 1024, 1000, None, False), (1, 0, 4, 2, 64, 64, None, False)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("case", ROTARY)
@pytest.mark.parametrize("layout", ["heads", "tokens", "sliced"])
def test_apply_rotary(dtype, case, layout):
    B, L, H, kv, dh, rot, sections, interleaved = case
    T = DT[dtype]
    gen = torch.Generator(device=DEV).manual_seed(L)

    def act(heads):
        if layout == "heads":
            return torch.randn(B, heads, L, dh, generator=gen, device=DEV).to(T)
        if layout == "tokens":
            return torch.randn(B, L, heads, dh, generator=gen, device=DEV).to(T).transpose(1, 2)
        return torch.randn(B, L, heads + 1, dh + 1, generator=gen, device=DEV).to(T)[:, :, 1:, :dh].transpose(1, 2)   # rows on odd addresses
    q, k = act(H), act(kv)
    for table_type in {T, torch.float32}:
        shape = ((3,) if sections else ()) + (B if L != 65 else 1, L, rot)
        cos, sin = (torch.randn(shape, generator=gen, device=DEV).to(table_type) for _ in range(2))
        c, s = cos.double(), sin.double()
        if sections:
            axis = torch.arange(3).repeat_interleave(torch.tensor(sections)).repeat(2)
            c, s = (torch.stack([t[axis[i], ..., i] for i in range(rot)], -1) for t in (c, s))
        for transpose in (False, True):
            out = ffa.apply_rotary(q, k, cos, sin, sections=sections, interleaved=interleaved, transpose=transpose)
            for got, x in zip(out, (q, k)):
                want = rotated(x.double(), c[:, None], s[:, None], interleaved, transpose)
                assert got.dtype == T
                # two products of fp32 and their sum, each channel's own and its partner's
                most = magnitudes(x.double().abs(), c[:, None].abs(), s[:, None].abs(), interleaved)
                within(got, want, rounding(T, want) + 3 * U * most)


def test_apply_rotary_gradient_against_formula_and_differences():
    gen = torch.Generator(device=DEV).manual_seed(3)
    for interleaved, sections, rot in ((False, None, 32), (True, None, 24), (False, (4, 6, 6), 32)):
        q, k = (torch.randn(2, h, 5, 32, generator=gen, device=DEV) for h in (4, 2))
        cos, sin = (torch.randn(((3,) if sections else ()) + (2, 5, rot), generator=gen, device=DEV) for _ in range(2))
        how = dict(sections=sections, interleaved=interleaved)
        a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
        y, z = ffa.apply_rotary(a, b, cos, sin, **how)
        dy, dz = torch.randn_like(y), torch.randn_like(z)
        ga, gb = torch.autograd.grad((y, z), (a, b), (dy, dz), create_graph=True)
        fa, fb = ffa.apply_rotary(dy, dz, cos, sin, transpose=True, **how)
        assert torch.equal(ga, fa) and torch.equal(gb, fb)
        # the operator is linear: a difference of any width has the gradient's slope.  16 products of magnitude about 1 each side
        for x, g, d in ((0, ga, dy), (1, gb, dz)):
            step = torch.randn_like(g)
            plus = ffa.apply_rotary(q + step if x == 0 else q, k + step if x == 1 else k, cos, sin, **how)[x].double()
            minus = ffa.apply_rotary(q - step if x == 0 else q, k - step if x == 1 else k, cos, sin, **how)[x].double()
            slope = ((plus - minus) / 2 * d.double()).sum()
            terms = ((plus.abs() + minus.abs()) * d.double().abs()).sum() * 4 + (g.double() * step.double()).abs().sum()
            assert abs(float(slope - (g.double() * step.double()).sum())) <= 4 * U * float(terms)
        # the second derivative: the gradient of <R^T dy, w> in dy is R w
        w = torch.randn_like(ga)
        a2, b2 = q.clone().requires_grad_(), k.clone().requires_grad_()
        dy2 = dy.clone().requires_grad_()
        g2, = torch.autograd.grad(ffa.apply_rotary(a2, b2, cos, sin, **how)[0], a2, dy2, create_graph=True)
        back, = torch.autograd.grad(g2, dy2, w)
        assert torch.equal(back, ffa.apply_rotary(w, torch.zeros_like(k), cos, sin, **how)[0])
    # only one input needs a gradient
    a = q.clone().requires_grad_()
    y, z = ffa.apply_rotary(a, k, cos, sin, sections=(4, 6, 6))
    assert torch.autograd.grad(y.sum(), a)[0].shape == q.shape


def test_apply_rotary_under_capture():
    """A differentiable call is refused while a graph is captured; the gradient by name is captured and replays."""
    q, k = torch.randn(1, 4, 6, 64, device=DEV), torch.randn(1, 2, 6, 64, device=DEV)
    cos, sin = torch.randn(1, 6, 64, device=DEV), torch.randn(1, 6, 64, device=DEV)
    ffa.apply_rotary(q, k, cos, sin)
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            with pytest.raises(ffa.FrameFusionHipError, match="capture"):
                ffa.apply_rotary(q.detach().requires_grad_(), k, cos, sin)
            out = ffa.apply_rotary(q, k, cos, sin, transpose=True)
    for _ in range(3):
        q.normal_(), k.normal_()
        g.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, ffa.apply_rotary(q, k, cos, sin, transpose=True)):
            assert torch.equal(got, want)


def test_backward_under_capture_is_refused(monkeypatch):
    q, k = torch.randn(1, 4, 6, 64, device=DEV, requires_grad=True), torch.randn(1, 2, 6, 64, device=DEV)
    cos, sin = torch.randn(1, 6, 64, device=DEV), torch.randn(1, 6, 64, device=DEV)
    y, _ = ffa.apply_rotary(q, k, cos, sin)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(ffa.FrameFusionHipError, match="capture"):
        torch.autograd.grad(y.sum(), q)


def test_apply_rotary_of_expanded_inputs():
    """One head shown to several (stride 0): the gradient of the shared one is the sum over them."""
    one = torch.randn(2, 1, 5, 32, device=DEV, requires_grad=True)
    k = torch.randn(2, 2, 5, 32, device=DEV)
    cos, sin = torch.randn(1, 5, 32, device=DEV), torch.randn(1, 5, 32, device=DEV)
    y, _ = ffa.apply_rotary(one.expand(-1, 3, -1, -1), k, cos, sin)
    whole = one.detach().repeat(1, 3, 1, 1).requires_grad_()
    z, _ = ffa.apply_rotary(whole, k, cos, sin)
    assert torch.equal(y, z)
    dy = torch.randn_like(y)
    got, want = torch.autograd.grad(y, one, dy)[0], torch.autograd.grad(z, whole, dy)[0].double().sum(1, keepdim=True)
    within(got, want, 4 * U * torch.autograd.grad(ffa.apply_rotary(whole, k, cos, sin)[0], whole, dy)[0].double().abs().sum(1, keepdim=True))


# ---------------------------------------------------------------------------------------------------- the cache
LIMIT = {"fp8": (448.0, 1.875, -6, 3), "fp4": (6.0, 1.5, 0, 1)}


def stored(x, store, dtype):
    """What a block-quantised row stands for, from the definition in 64 bits."""
    if store is None:
        return x.double()
    top, cap, low, bits = LIMIT[store]
    limit = cap * 2.0 ** (15 if dtype == torch.float16 else 127)
    v = x.double().unflatten(-1, (-1, 32))
    nan = ~torch.isfinite(v).all(-1, keepdim=True)
    v = torch.where(nan, 0.0, v).clamp(-limit, limit)
    big = v.abs().amax(-1, keepdim=True)
    e = torch.full_like(big, -100)
    for k in range(-99, 129):                       # the smallest exponent whose top covers the block
        e = torch.where(big > top * 2.0 ** (k - 1), float(k), e)
    y = v * torch.exp2(-e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** low))) - bits)
    return torch.where(nan, math.nan, torch.round(y / step) * step * torch.exp2(e)).flatten(-2)


def awkward(shape, dtype, gen):
    """Values where quantising can go wrong: every magnitude, ties, borders of the scale, zeros, the type's limits."""
    x = torch.randn(shape, generator=gen, device=DEV) * torch.exp2(torch.randint(-9, 9, shape[:-1] + (1,), generator=gen, device=DEV).float())
    rows = x.view(-1, shape[-1])
    info = torch.finfo(dtype)
    grid = torch.randint(-64, 65, rows[0::5].shape, generator=gen, device=DEV) / 16
    rows[0::5] = grid                                                   # ties of both grids
    special = [0.0, -0.0, info.max, -info.max, info.tiny, -info.tiny, info.tiny / 4, 448.0, 449.0, 448.5, 6.0, 6.03125, 5.0, 3.5, 7.0, -7.0, 1.75, 1.7578125]
    if rows.shape[0] > 12:
        rows[6] = torch.tensor(special, device=DEV).repeat(rows.shape[1] // len(special) + 1)[: rows.shape[1]]
        rows[7] = 0
        rows[8] = info.max
        rows[9] = info.tiny
        rows[10, :3] = torch.tensor([448.0, 0.5 ** 9, 0.5 ** 10], device=DEV)
        rows[11] = torch.exp2(torch.arange(rows.shape[1], device=DEV).float() % 32 - 20)
    return x.to(dtype)


def batch(B, width, pages, gen, holes=True):
    """A table of `width` pages a sequence in mixed order, some entries without a page."""
    assert pages >= B * width
    table = torch.randperm(pages, generator=gen, device=DEV)[: B * width].to(torch.int32).view(B, width).contiguous()
    if holes and width > 2:
        table[-1, -1] = -1
        table[0, 1] = pages if B > 1 else table[0, 1]
    return table


def places(table, start, n, pages, page):
    """[(b, t, page, row)] of every position that has a place."""
    out = []
    t = table.tolist()
    for b, s in enumerate(start.tolist()):
        if s < 0:
            continue
        for i in range(n):
            p = s + i
            if p // page < len(t[b]) and 0 <= t[b][p // page] < pages:
                out.append((b, i, t[b][p // page], p % page))
    return out


CACHES = [  # B, heads, n, dh, page, width, start
    (1, 4, 1, 128, 64, 2, [63]), (2, 2, 37, 64, 16, 5, [0, 15]), (3, 1, 50, 256, 48, 4, [90, -1, 47]), (2, 3, 5, 32, 32, 1, [30, 100]),
    (1, 8, 130, 128, 128, 3, [127]), (2, 2, 20, 96, 16, 3, [3, 2**31 - 5]), (4, 16, 2, 160, 16, 2, [0, 14, 15, 16])]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("store", [None, "fp8", "fp4"])
@pytest.mark.parametrize("case", CACHES)
def test_write_and_read(dtype, store, case):
    B, heads, n, dh, page, width, start = case
    T = DT[dtype]
    gen = torch.Generator(device=DEV).manual_seed(n)
    pages = B * width + 2
    cache = ffa.new_cache(pages, page, heads, dh, T, store, device=DEV)
    ffa.cache_write(cache, awkward((1, heads, pages * page, dh), T, gen), awkward((1, heads, pages * page, dh), T, gen),
                    torch.arange(pages, dtype=torch.int32, device=DEV)[None], torch.zeros(1, dtype=torch.int32, device=DEV))
    before = [None if t is None else t.clone() for t in cache]
    table, start = batch(B, width, pages, gen), torch.tensor(start, dtype=torch.int32, device=DEV)
    k = awkward((B, n, heads, dh), T, gen).transpose(1, 2)              # as a projection leaves it
    v = awkward((B, heads, n, dh + 1), T, gen)[..., 1:]                 # rows on odd addresses
    if n > 3:
        k[0, 0, 1, 3], k[0, 0, 2, 31], v[-1, -1, 3, 0] = math.nan, math.inf, -math.inf
    ffa.cache_write(cache, k, v, table, start)
    where = places(table, start, n, pages, page)
    want_k, want_v = (torch.zeros(B, heads, n, dh, dtype=torch.float64, device=DEV) for _ in range(2))
    qk, qv = stored(k, store, T), stored(v, store, T)
    untouched = torch.ones(pages, page, dtype=torch.bool, device=DEV)
    for b, i, p, r in where:
        want_k[b, :, i], want_v[b, :, i] = qk[b, :, i], qv[b, :, i]
        untouched[p, r] = False
    for read_as in {T, torch.float32} if store else {T}:
        got = ffa.cache_read(cache, table, start, n, dtype=read_as)
        for g, w in zip(got, (want_k, want_v)):
            w = w.to(read_as)
            assert g.dtype == read_as and torch.equal(torch.isnan(g), torch.isnan(w))
            assert torch.equal(torch.nan_to_num(g, nan=0.0, posinf=1.0, neginf=-1.0), torch.nan_to_num(w, nan=0.0, posinf=1.0, neginf=-1.0))
    for t, old in zip(cache, before):                                    # rows without a new token are as they were
        if t is not None:
            a, o = (x.view(torch.uint8).transpose(1, 2)[untouched] for x in (t, old))
            assert torch.equal(a, o)


def test_every_code_reads_as_what_it_stands_for():
    """All e4m3 and e2m1 codes under scales from the smallest to the largest, and the two special scale bytes."""
    for store, width in (("fp8", 256), ("fp4", 128)):
        cache = ffa.new_cache(1, 256, 1, 256, torch.float32, store, device=DEV)
        cache.keys.view(torch.uint8)[:] = (torch.arange(width, device=DEV) % 256).to(torch.uint8)
        cache.values.view(torch.uint8)[:] = (torch.arange(width, device=DEV) * 2 + 1).to(torch.uint8)
        scales = torch.arange(256, device=DEV).to(torch.uint8)[:, None].expand(256, 8)
        cache.key_scales[0, 0], cache.value_scales[0, 0] = scales, scales
        table, start = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
        for got, codes in zip(ffa.cache_read(cache, table, start, 256, dtype=torch.float32), (cache.keys, cache.values)):
            b = codes.view(torch.uint8)[0, 0].long()
            if store == "fp4":
                b = torch.stack((b % 16, b // 16), -1).flatten(-2)
                m, e, sign = b % 2, b // 2 % 4, b // 8
                v = torch.where(e == 0, m / 2.0, (1 + m / 2.0) * torch.exp2(e.double() - 1))
            else:
                m, e, sign = b % 8, b // 8 % 16, b // 128
                v = torch.where(e == 0, m / 512.0, (1 + m / 8.0) * torch.exp2(e.double() - 7))
                v = torch.where((e == 15) & (m == 7), math.nan, v)
            v = torch.where(sign == 1, -v, v)
            byte = torch.arange(256, device=DEV).double()[:, None]
            want = v * torch.where(byte == 255, math.nan, torch.where(byte == 0, 0.0, torch.exp2(byte - 127)))
            want = want.float()                          # (the largest scales pass fp32's range: infinity)
            assert torch.equal(torch.isnan(got[0, 0]), torch.isnan(want)) and torch.equal(got[0, 0].nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("store,dtype,dh", [(None, torch.bfloat16, 128), (None, torch.float32, 32), ("fp8", torch.bfloat16, 64), ("fp4", torch.float16, 32), ("fp4", torch.bfloat16, 96)])
def test_keep(store, dtype, dh):
    page, heads, width, m = 48, 3, 16, 600
    gen = torch.Generator(device=DEV).manual_seed(dh)
    lists = [[], [0, 1, 2], [3], [0, 2, 3, 7, 8, 90], list(range(1, 601)), sorted(torch.randperm(620, generator=gen, device=DEV)[:300].tolist()),
             [4, 5, 5, 6], [6, 2], [1, 40, 10**6, 10**6 + 1], [0, 1, 300]]
    B = len(lists)
    starts = [17, 5, 47, 40, 100, 63, 0, 2, 30, -1]
    pages = B * width + 1
    cache = ffa.new_cache(pages, page, heads, dh, dtype, store, device=DEV)
    for t in cache:
        if t is not None:
            t.view(torch.uint8).random_(0, 127, generator=gen)
    table = batch(B, width, pages, gen, holes=False)
    table[3, 2] = -1                     # start 40, entry 90 lies on page 2: the list ends there
    accepted = torch.full((B, m), -1, dtype=torch.int32, device=DEV)
    for b, x in enumerate(lists):
        accepted[b, : len(x)] = torch.tensor(x, dtype=torch.int32)
    want = [None if t is None else t.clone() for t in cache]
    end = [0, 3, 1, 5, 600, 300, 2, 1, 2, 0]
    for b in range(B):
        src = [(table[b, (starts[b] + x) // page], (starts[b] + x) % page) for x in lists[b][: end[b]]]
        dst = [(table[b, (starts[b] + i) // page], (starts[b] + i) % page) for i in range(end[b])]
        for w, t in zip(want, cache):
            if t is not None and src:
                sp, sr = (torch.stack([torch.as_tensor(s[i], device=DEV) for s in src]).long() for i in (0, 1))
                dp, dr = (torch.stack([torch.as_tensor(s[i], device=DEV) for s in dst]).long() for i in (0, 1))
                ok = dp >= 0
                w.view(torch.uint8)[dp[ok], :, dr[ok]] = t.view(torch.uint8)[sp[ok], :, sr[ok]]
    ffa.cache_keep(cache, table, torch.tensor(starts, dtype=torch.int32, device=DEV), accepted)
    for w, t in zip(want, cache):
        if t is not None:
            assert torch.equal(w.view(torch.uint8), t.view(torch.uint8))


# ------------------------------------------------------------------------------------------------ the attention
def reference(q, k, v, start, mask, scale, present):
    """64-bit attention over dense keys [B, kv, S, dh] and the bound of its error: (out, tolerance without the output's rounding)."""
    B, H, n, dh = q.shape
    kv, S = k.shape[1], k.shape[2]
    G = H // kv
    out, tol = torch.zeros(B, H, n, dh, dtype=torch.float64, device=q.device), torch.zeros(B, H, n, dh, dtype=torch.float64, device=q.device)
    T = q.dtype
    for b in range(B):
        s = int(start[b])
        if s < 0:
            continue
        at = torch.arange(S, device=q.device)
        see = (at < s)[None].repeat(n, 1)
        new = torch.ones(n, n, dtype=torch.bool, device=q.device).tril() if mask is None else mask[b] if mask.ndim == 3 else mask
        inside = max(0, min(n, S - s))
        see[:, s:s + inside] = new[:, :inside]
        see &= present[b][None]
        for h in range(H):
            kk, vv = k[b, h // G].double(), v[b, h // G].double()
            clean_k, clean_v = torch.nan_to_num(kk, nan=0.0, posinf=0.0, neginf=0.0), torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0)
            nan_k, nan_v = ~torch.isfinite(kk), ~torch.isfinite(vv)
            x = q[b, h].double() @ clean_k.T * scale
            x = torch.where((nan_k.any(-1))[None] & see, math.nan, x).masked_fill(~see, -math.inf)
            any_ = see.any(-1)
            p = torch.softmax(x, -1)
            p = torch.where(any_[:, None], p, 0.0)
            o = p.masked_fill(~see, 0.0) @ clean_v
            poison = (see.double() @ nan_v.double()) > 0
            o = torch.where(poison | torch.isnan(p).any(-1, keepdim=True), math.nan, o)
            o = torch.where(any_[:, None], o, 0.0)
            out[b, h] = o
            # scores: dh terms in fp32, scaled and shifted; each weight is off by that share, its exponential by 4 ulp; the sums
            # have S terms; the weights are rounded to T (not in fp32)
            off = (q[b, h].double().abs() @ clean_k.T.abs() * abs(scale)).masked_fill(~see, 0.0).amax(-1, keepdim=True) * (dh + 4) * U
            spread = p.masked_fill(~see, 0.0).nan_to_num() @ clean_v.abs()
            tol[b, h] = spread * (4 * off + (S + 16) * U + (0 if T == torch.float32 else half_step(T)))
    return out, tol


def attention_case(dtype, store, dh, kv, G, n, page, starts, mask=None, seed=0, scale=None, holes=False, mutate=None, width=None):
    T = DT[dtype]
    gen = torch.Generator(device=DEV).manual_seed(seed + dh * 7 + n)
    B = len(starts)
    width = width or max(1, -(-(max(starts) + n) // page))
    pages = B * width + 2
    cache = ffa.new_cache(pages, page, kv, dh, T, store, device=DEV)
    # everything that is not written holds NaN
    for t in cache:
        if t is not None and (store is None or t.dtype == torch.uint8 and t.shape[-1] == dh // 32):
            t.fill_(math.nan if store is None else 255)
    table, start = batch(B, width, pages, gen, holes), torch.tensor(starts, dtype=torch.int32, device=DEV)
    S = width * page
    k, v = (torch.randn(B, kv, S, dh, generator=gen, device=DEV).to(T) for _ in range(2))
    k[:, :, :, : dh // 8] *= 3
    if mutate:
        mutate(k, v)
    zero = torch.zeros(B, dtype=torch.int32, device=DEV)
    for b, s in enumerate(starts):                               # each sequence exactly as long as it is
        if s >= 0:
            end = min(s + n, S)
            ffa.cache_write(cache, k[b:b + 1, :, :end], v[b:b + 1, :, :end], table[b:b + 1], zero[:1])
    q = (torch.randn(B, n, kv * G, dh, generator=gen, device=DEV) * 0.8).to(T).transpose(1, 2)
    dense_k, dense_v = stored(k, store, T), stored(v, store, T)
    present = torch.zeros(B, S, dtype=torch.bool, device=DEV)
    for b, _, p, r in places(table, zero, S, pages, page):
        present[b, _] = True
    got = ffa.cache_attention(q, cache, table, start, mask=mask, scale=scale)
    want, tol = reference(q, dense_k, dense_v, starts, mask, dh ** -0.5 if scale is None else scale, present)
    assert got.dtype == T and got.transpose(1, 2).is_contiguous()
    within(got, want, tol + rounding(T, want))
    again = ffa.cache_attention(q, cache, table, start, mask=mask, scale=scale)
    assert torch.equal(got.view(torch.int16 if T != torch.float32 else torch.int32), again.view(torch.int16 if T != torch.float32 else torch.int32))
    return got


def tree(n, B, seed, empty=()):
    gen = torch.Generator().manual_seed(seed)
    m = torch.zeros(B, n, n, dtype=torch.bool)
    for b in range(B):
        for i in range(n):
            parent = int(torch.randint(-1, i, (1,), generator=gen)) if i else -1
            if parent >= 0:
                m[b, i] = m[b, parent]
            m[b, i, i] = True
        for i in empty:
            m[b, i] = False
    return m.to(DEV)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("store", [None, "fp8", "fp4"])
@pytest.mark.parametrize("dh", [32, 64, 128, 256])
def test_attention_types_and_heads(dtype, store, dh):
    attention_case(dtype, store, dh, 2, 4, 1, 32, [77, 0, 31, -1])
    attention_case(dtype, store, dh, 1, 5, 6, 16, [130, 3])
    attention_case(dtype, store, dh, 1, 5, 40, 16, [130, 3, -1])                            # more rows than one wave or workgroup holds
    attention_case(dtype, store, dh, 2, 4, 65, 48, [290])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("store", ["fp8", "fp4"])
@pytest.mark.parametrize("dh,n,G", [(32, 1, 2), (64, 3, 2), (128, 1, 7), (256, 2, 3), (64, 60, 3), (128, 61, 3), (256, 60, 3), (32, 70, 2)])
def test_attention_over_blocks_of_nan(dtype, store, dh, n, G):
    """A NaN that was written into the earlier tokens is one block of NaN: as a key it reaches every output of its head, as a value its own
    32 channels; as a new token's value only those of the tokens that see it."""
    T = DT[dtype]
    ctx, bad = 77, 40
    gen = torch.Generator(device=DEV).manual_seed(dh + n)
    k, v = (torch.randn(1, 3, ctx + n, dh, generator=gen, device=DEV).to(T) for _ in range(2))
    k[0, 0, bad, 5] = math.nan
    v[0, 1, bad, dh - 1] = math.inf
    v[0, 2, ctx + n - 1, 0] = math.nan
    cache = ffa.new_cache(16, 16, 3, dh, T, store, device=DEV)
    table, start = torch.randperm(16, generator=gen, device=DEV).to(torch.int32)[None].contiguous(), torch.tensor([ctx], dtype=torch.int32, device=DEV)
    ffa.cache_write(cache, k, v, table, torch.zeros_like(start))
    q = torch.randn(1, 3 * G, n, dh, generator=gen, device=DEV).to(T)
    got = ffa.cache_attention(q, cache, table, start)[0].unflatten(0, (3, G))
    assert torch.isnan(got[0]).all()
    assert torch.isnan(got[1][..., dh - 32:]).all() and torch.isfinite(got[1][..., : dh - 32]).all()
    assert torch.isfinite(got[2][:, : n - 1]).all() and torch.isfinite(got[2][..., 32:]).all() and torch.isnan(got[2][:, n - 1, :32]).all()


def test_attention_of_infinite_values_that_only_some_see():
    """A value of infinity (its key finite): infinity for the tokens that see it, nothing for the others."""
    for dtype, n, kv, G in (("bf16", 9, 2, 3), ("bf16", 64, 1, 3), ("fp32", 9, 2, 3)):
        gen = torch.Generator(device=DEV).manual_seed(n)
        T = DT[dtype]
        cache = ffa.new_cache(8, 32, kv, 64, T, None, device=DEV)
        table, start = torch.arange(8, dtype=torch.int32, device=DEV)[None], torch.tensor([50], dtype=torch.int32, device=DEV)
        k, v = (torch.randn(1, kv, 50 + n, 64, generator=gen, device=DEV).to(T) for _ in range(2))
        v[:, :, 52, 3], v[:, :, 55, 3], v[:, :, 55, 9] = math.inf, -math.inf, -math.inf
        ffa.cache_write(cache, k, v, table, torch.zeros_like(start))
        q = torch.randn(1, kv * G, n, 64, generator=gen, device=DEV).to(T)
        got = ffa.cache_attention(q, cache, table, start, mask=torch.eye(n, dtype=torch.bool, device=DEV))
        odd = torch.zeros(n, 64, dtype=torch.bool, device=DEV)
        odd[2, 3] = odd[5, 3] = odd[5, 9] = True
        assert (got[0, :, 2, 3] == math.inf).all() and (got[0, :, 5, 3] == -math.inf).all() and (got[0, :, 5, 9] == -math.inf).all()
        assert torch.isfinite(got[0][:, ~odd]).all()
        causal = ffa.cache_attention(q, cache, table, start)
        assert torch.isfinite(causal[0, :, :2]).all() and (causal[0, :, 2:5, 3] == math.inf).all() and torch.isnan(causal[0, :, 5:, 3]).all()
        assert (causal[0, :, 5:, 9] == -math.inf).all() and torch.isfinite(causal[0][:, :, 10:]).all()



@pytest.mark.parametrize("store", [None, "fp8", "fp4"])
@pytest.mark.parametrize("kv,G,n,page,starts", [
    (4, 7, 1, 64, [4043]), (1, 1, 1, 16, [0]), (1, 1, 1, 16, [15, 16, 17, 1, 0, -1]), (2, 8, 3, 48, [700, 95]), (3, 1, 33, 64, [1, 127]),
    (1, 16, 17, 128, [1000]), (1, 40, 2, 64, [200, 64]), (2, 2, 129, 64, [5, 260]), (8, 8, 1, 64, [513, 65, 2049]), (1, 3, 257, 16, [0])])
def test_attention_lengths(store, kv, G, n, page, starts):
    attention_case("bf16", store, 128 if n < 100 else 64, kv, G, n, page, starts)


@pytest.mark.parametrize("dtype,store", [("bf16", None), ("fp16", "fp8"), ("fp32", "fp4"), ("bf16", "fp4")])
@pytest.mark.parametrize("n,starts,empty", [(5, [60, 0, 3], ()), (16, [0, 0], (0, 7)), (61, [300, 15], (2, 60)), (2, [63, 64], (0, 1)), (40, [0], range(40)), (100, [77], (50,))])
def test_attention_trees(dtype, store, n, starts, empty):
    """Trees of drafted tokens; rows whose mask leaves nothing see the context alone - or, where there is none, nothing: zeros."""
    m = tree(n, len(starts), n, empty)
    got = attention_case(dtype, store, 64, 2, 3, n, 16, starts, mask=m)
    for b, s in enumerate(starts):
        if s == 0 and len(list(empty)):
            assert not got[b][:, list(empty)].any()
    attention_case(dtype, store, 64, 1, 2, n, 16, starts, mask=m[0])             # one mask for all


def test_attention_leaves_out_what_is_stored_in_masked_places():
    """NaN and infinities in drafted tokens that some tokens see and others do not: only those that see them are hit."""
    for dtype, dh in itertools.product(DT, (64, 128)):
        for n, s, bad in ((9, 40, (3, 6)), (33, 0, (0, 20)), (64, 129, (1, 63))):
            def poison(k, v):
                v[:, :, s + bad[0], 5] = math.nan
                v[:, :, s + bad[1], 7] = math.inf if dtype != "fp16" else -math.inf
                k[:, :, s + bad[1], 2] = math.nan
            m = torch.eye(n, dtype=torch.bool, device=DEV)
            got = attention_case(dtype, None, dh, 2, 3, n, 16, [s], mask=m, mutate=poison)
            clean = [i for i in range(n) if i not in bad]
            assert torch.isfinite(got[0][:, clean]).all()
            attention_case(dtype, None, dh, 2, 3, n, 16, [s], mutate=poison)                # causal: all behind them are hit


def test_attention_with_pages_missing_and_tables_too_short():
    attention_case("bf16", "fp8", 128, 2, 4, 3, 16, [100, 90], holes=True)
    attention_case("fp16", None, 64, 2, 4, 40, 32, [200, 31, 95], holes=True)
    attention_case("bf16", None, 64, 1, 2, 5, 16, [46, 100, 48, 44], width=3)               # new tokens past the table's end
    attention_case("fp32", "fp8", 64, 1, 2, 5, 16, [2**31 - 6, 10], width=3)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5, 30.0])
def test_attention_scales(scale):
    """A flat softmax, a negative scale, one so large that a single key carries everything."""
    attention_case("bf16", None, 64, 2, 2, 4, 16, [300, 33], scale=scale)
    attention_case("fp32", "fp8", 64, 2, 2, 4, 16, [300, 33], scale=scale)


@pytest.mark.parametrize("dtype,store,ctx", [("bf16", "fp4", 70001), ("bf16", None, 20011), ("fp32", None, 9001)])
def test_attention_long(dtype, store, ctx):
    attention_case(dtype, store, 64, 1, 2, 2, 128, [ctx, ctx // 3])


def test_empty_calls():
    cache = ffa.new_cache(4, 16, 2, 64, torch.bfloat16, "fp8", device=DEV)
    start = torch.zeros(2, dtype=torch.int32, device=DEV)
    for width in (0, 2):
        table = torch.full((2, width), -1, dtype=torch.int32, device=DEV)               # no place at all
        x = torch.randn(2, 2, 3, 64, device=DEV).bfloat16()
        ffa.cache_write(cache, x, x, table, start)
        assert not any(t.view(torch.uint8).any() for t in cache)
        assert not ffa.cache_read(cache, table, start, 3)[0].any()
        for n in (3, 70):
            assert not ffa.cache_attention(torch.randn(2, 4, n, 64, device=DEV).bfloat16(), cache, table, start).any()
        ffa.cache_keep(cache, table, start, torch.tensor([[1], [2]], dtype=torch.int32, device=DEV))
    none = ffa.new_cache(0, 16, 2, 64, torch.bfloat16, None, device=DEV)
    table = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    for n in (1, 70):
        assert not ffa.cache_attention(torch.randn(2, 4, n, 64, device=DEV).bfloat16(), none, table, start).any()
    assert ffa.cache_attention(torch.randn(2, 4, 0, 64, device=DEV).bfloat16(), cache, table, start).shape == (2, 4, 0, 64)
    assert ffa.cache_read(cache, table, start, 0)[0].shape == (2, 2, 0, 64)
    table, start = torch.zeros(0, 3, dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV)
    assert ffa.cache_attention(torch.randn(0, 4, 1, 64, device=DEV).bfloat16(), cache, table, start).shape == (0, 4, 1, 64)
    with pytest.raises(ffa.FrameFusionHipError):
        ffa.cache_attention(torch.randn(2, 4, 1, 64, device=DEV).bfloat16(), cache, torch.zeros(2, 3, dtype=torch.int32, device=DEV),
                            torch.zeros(2, dtype=torch.int32, device=DEV), scale=math.nan)


def test_cache_without_heads_is_refused():
    x = torch.zeros(2, 0, 16, 64, device=DEV).bfloat16()
    table, start = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(ffa.FrameFusionHipError, match="0 heads"):
        ffa.cache_attention(torch.randn(1, 4, 1, 64, device=DEV).bfloat16(), (x, x, None, None), table, start)
    with pytest.raises(ffa.FrameFusionHipError):
        ffa.cache_keep((x, x, None, None), table, start, torch.ones(1, 1, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("n,G", [(1, 2), (70, 2)])
@pytest.mark.parametrize("first", [True, False])
def test_attention_small_weights_in_fp16(n, G, first):
    """One key with nearly all the weight and 20 000 others of 2^-23 to 2^-27 of it each, whose values are what comes out.  A weight keeps
    2^-12 of itself, or what lies 2^-32 below the largest: rounded to fp16 as it stands it would be off by 2^-25."""
    dh, ctx = 64, 20000
    gen = torch.Generator(device=DEV).manual_seed(n)
    k, v = torch.zeros(1, 1, ctx + n, dh, device=DEV), torch.zeros(1, 1, ctx + n, dh, device=DEV)
    top = 0 if first else ctx - 1
    k[..., 0] = -(23 + 4 * torch.rand(ctx + n, generator=gen, device=DEV))             # score in octaves below the top one's 0
    v[:] = 500 + 100 * torch.randn(v.shape, generator=gen, device=DEV)
    k[0, 0, top], v[0, 0, top] = 0, 0
    k, v = k.half(), v.half()
    cache = ffa.new_cache(160, 128, 1, dh, torch.float16, None, device=DEV)
    table, start = torch.arange(160, dtype=torch.int32, device=DEV)[None], torch.tensor([ctx], dtype=torch.int32, device=DEV)
    ffa.cache_write(cache, k, v, table, torch.zeros_like(start))
    q = torch.zeros(1, G, n, dh, device=DEV).half()
    q[..., 0] = 1
    got = ffa.cache_attention(q, cache, table, start, scale=math.log(2))
    x = k[0, 0, :, 0].double() * math.log(2)
    for i in (0, n - 1):
        p = torch.softmax(x[: ctx + i + 1], 0)
        want = p @ v[0, 0, : ctx + i + 1].double()
        tol = (p @ v[0, 0, : ctx + i + 1].double().abs()) * (half_step(torch.float16) + (ctx + n + 200) * U) + (ctx + n) * 2.0 ** -33 * 1000
        for g in range(G):
            within(got[0, g, i], want, tol + rounding(torch.float16, want))


@pytest.mark.parametrize("store", ["fp8", "fp4"])
@pytest.mark.parametrize("n", [3, 130])
def test_fp16_attention_over_values_beyond_its_range(store, n):
    """A cache written as bf16 and read as fp16: a value that passes fp16's range is an infinity for the tokens that see it, and nothing to
    the others."""
    cache = ffa.new_cache(16, 16, 1, 64, torch.bfloat16, store, device=DEV)
    table, start = torch.arange(16, dtype=torch.int32, device=DEV)[None], torch.tensor([20], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(1, 1, 20 + n, 64, device=DEV).bfloat16() for _ in range(2))
    v[0, 0, 21, 5], v[0, 0, 21, 6] = 3e6, -3e6
    ffa.cache_write(cache, k, v, table, torch.zeros_like(start))
    q = torch.randn(1, 1, n, 64, device=DEV).half()
    got = ffa.cache_attention(q, cache, table, start, mask=torch.eye(n, dtype=torch.bool, device=DEV))[0, 0]
    assert got[1, 5] == math.inf and got[1, 6] == -math.inf
    got[1, 5:7] = 0
    assert torch.isfinite(got).all()


def test_many_sequences():
    """More sequences than a wave has lanes, and than there are workgroups over the keys: ragged, padded, empty ones among them."""
    gen = torch.Generator().manual_seed(7)
    for B, longest, n in ((150, 300, 1), (70, 900, 3), (300, 40, 2)):
        starts = torch.randint(-1, longest, (B,), generator=gen).tolist()
        starts[3], starts[64] = 0, longest
        attention_case("bf16", "fp8", 32, 1, 2, n, 16, starts)
    attention_case("bf16", None, 32, 1, 2, 66, 16, torch.randint(-1, 200, (70,), generator=gen).tolist(), mask=None)


def test_attention_beyond_32_bit_offsets():
    """Pages whose bytes lie past 4 GiB of each tensor (and whose elements pass 2^31)."""
    page, kv, dh = 64, 8, 128
    pages = (5 << 30) // (page * kv * dh * 2)
    keys, values = (torch.empty(pages, kv, page, dh, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    cache = (keys, values, None, None)
    gen = torch.Generator(device=DEV).manual_seed(1)
    table = torch.tensor([[pages - 1, 3, pages - 2, pages // 2]], dtype=torch.int32, device=DEV)
    start = torch.tensor([200], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(1, kv, 203, dh, generator=gen, device=DEV).bfloat16() for _ in range(2))
    ffa.cache_write(cache, k, v, table, torch.zeros_like(start))
    assert torch.equal(keys[pages - 1, :, :5], k[0, :, :5]) and torch.equal(values[pages - 2, :, 63], v[0, :, 191])
    got_k, got_v = ffa.cache_read(cache, table, torch.zeros_like(start), 203)
    assert torch.equal(got_k, k) and torch.equal(got_v, v)
    q = torch.randn(1, kv, 3, dh, generator=gen, device=DEV).bfloat16()
    want, tol = reference(q, k, v, [200], None, dh ** -0.5, torch.ones(1, 203, dtype=torch.bool, device=DEV))
    within(ffa.cache_attention(q, cache, table, start), want, tol + rounding(torch.bfloat16, want))
    ffa.cache_keep(cache, table, start, torch.tensor([[2]], dtype=torch.int32, device=DEV))
    assert torch.equal(ffa.cache_read(cache, table, start, 1)[0], k[:, :, 202:203])


# ------------------------------------------------------------------------------------- streams, graphs, a run of them
def test_two_captured_graphs_side_by_side():
    """Two graphs of the same calls on two streams at once, replayed with eager work between: every replay equals the eager result."""
    gen = torch.Generator(device=DEV).manual_seed(9)
    kv, G, dh, page, n = 2, 4, 128, 64, 3
    sets = []
    for i, ctx in enumerate((5000, 3001)):
        width = -(-(ctx + n) // page)
        cache = ffa.new_cache(width, page, kv, dh, torch.bfloat16, "fp8", device=DEV)
        table = torch.randperm(width, generator=gen, device=DEV).to(torch.int32)[None].contiguous()
        start = torch.zeros(1, dtype=torch.int32, device=DEV)
        k, v = (torch.randn(1, kv, ctx, dh, generator=gen, device=DEV).bfloat16() for _ in range(2))
        ffa.cache_write(cache, k, v, table, start)
        start.fill_(ctx)
        q = torch.randn(1, kv * G, n, dh, generator=gen, device=DEV).bfloat16()
        new = [torch.randn(1, kv, n, dh, generator=gen, device=DEV).bfloat16() for _ in range(2)]
        sets.append((cache, table, start, q, new, torch.cuda.Stream(), torch.cuda.CUDAGraph()))

    def step(cache, table, start, q, new):
        ffa.cache_write(cache, new[0], new[1], table, start)
        return ffa.cache_attention(q, cache, table, start)
    outs = []
    for cache, table, start, q, new, side, graph in sets:
        step(cache, table, start, q, new)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            outs.append(step(cache, table, start, q, new))
    for _ in range(4):
        for s in sets:
            s[3].normal_(generator=gen), s[4][0].normal_(generator=gen), s[4][1].normal_(generator=gen)
        torch.cuda.synchronize()
        for s in sets:
            with torch.cuda.stream(s[5]):
                s[6].replay()
        torch.cuda.synchronize()
        for s, out in zip(sets, outs):
            assert torch.equal(out, step(*s[:5]))
    torch.cuda.synchronize()


def test_a_run_of_them():
    """A prompt, single tokens and two rounds of drafted trees: the cached path follows dense 64-bit attention over the rotated tokens."""
    torch.manual_seed(4)
    H, kv, dh, page, T = 8, 2, 64, 16, torch.bfloat16
    inv, factor = ffa.rotary_frequencies(dh, 1e6, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64})
    inv = inv.to(DEV)
    for store in (None, "fp8"):
        cache = ffa.new_cache(40, page, kv, dh, T, store, device=DEV)
        table = torch.randperm(40, device=DEV).to(torch.int32)[:30][None].contiguous()
        dense_k, dense_v = (torch.zeros(1, kv, 0, dh, device=DEV, dtype=torch.float64) for _ in range(2))
        held = 0
        for n, mask, accepted in ((101, None, None), (1, None, None), (7, tree(7, 1, 5)[0], [0, 2, 5]), (1, None, None), (12, tree(12, 1, 6)[0], [1])):
            q, k, v = (torch.randn(1, n, h, dh, device=DEV).to(T).transpose(1, 2) for h in (H, kv, kv))
            pos = held + (torch.arange(n, device=DEV)[None] if mask is None else mask.sum(-1)[None] - 1)
            cos, sin = ffa.rotary_tables(pos, inv, dtype=torch.float32, factor=factor)
            q, k = ffa.apply_rotary(q, k, cos, sin)
            start = torch.tensor([held], dtype=torch.int32, device=DEV)
            ffa.cache_write(cache, k, v, table, start)
            got = ffa.cache_attention(q, cache, table, start, mask=mask)
            all_k, all_v = torch.cat((dense_k, stored(k, store, T)), 2), torch.cat((dense_v, stored(v, store, T)), 2)
            want, tol = reference(q, all_k, all_v, [held], mask, dh ** -0.5, torch.ones(1, held + n, dtype=torch.bool, device=DEV))
            within(got, want, tol + rounding(T, want))
            take = list(range(n)) if accepted is None else accepted
            if accepted is not None:
                ffa.cache_keep(cache, table, start, torch.tensor([accepted + [-1]], dtype=torch.int32, device=DEV))
            rows = torch.tensor(list(range(held)) + [held + i for i in take], device=DEV)
            dense_k, dense_v = all_k[:, :, rows], all_v[:, :, rows]
            held += len(take)
            read_k, read_v = ffa.cache_read(cache, table, torch.zeros_like(start), held, dtype=torch.float32 if store else None)
            assert torch.equal(read_k.double(), dense_k) and torch.equal(read_v.double(), dense_v)
