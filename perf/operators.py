"""The cached-decoding operators as they are measured: position tables and rotation, the quantised paged cache, attention of new
tokens over it, keeping accepted drafts.  `run` computes each in elementary torch operations, or (`own`) through the package.

A cache is four tensors: keys, values [pages, kv heads, page, dh] and, for the 8- and 4-bit forms, a scale byte for each 32
channels of each row, [pages, kv heads, page, dh / 32] (value = code * 2^(byte - 127), byte 255: the block is NaN).  The 8-bit form
holds e4m3 codes, the 4-bit form two e2m1 codes a byte, the even channel in the low half.  A table row lists a sequence's pages.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
MOST = {"bf16": 127, "fp16": 15, "fp32": 127}          # exponent of the type's largest power of two
DEV = "cuda"


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # position tables of a long M-RoPE prefill (three axes, video positions beyond the trained range, stretched by 4)
        dict(name="tables_mrope", op="tables", L=36898, axes=3, rot=128, base=1e6, stretch=4.0, layout="half", dtype="bf16", far=1000000),
        # q and k of one decoding step of 32 sequences, 64 / 8 heads
        dict(name="rotary_step", op="rotary", B=32, L=1, H=64, G=8, dh=128, rot=128, axes=1, layout="half", dtype="bf16", grad=False),
        # q and k of a 64-frame prefill with M-RoPE sections, forwards and backwards
        dict(name="rotary_mrope_train", op="rotary", B=1, L=12507, H=28, G=7, dh=128, rot=128, axes=3, layout="half", dtype="bf16", grad=True),
        # one token of 32 sequences written in 8 bits and read back
        dict(name="cache_step_8bit", op="cache", B=32, n=1, kv=8, dh=128, page=64, before=4043, store="fp8", dtype="bf16"),
        # the keys and values of a whole prefill, 8 bits
        dict(name="cache_prefill_8bit", op="cache", B=1, n=13474, kv=4, dh=128, page=64, before=0, store="fp8", dtype="bf16"),
        # a padded batch of chunks of odd length behind what is there, 4 bits, small heads and pages
        dict(name="cache_chunks_4bit", op="cache", B=16, n=517, kv=2, dh=64, page=16, before=901, store="fp4", dtype="fp16"),
        # one token over a reduced prefill: the smallest call, latency counts
        dict(name="attend_single_8bit", op="attend", B=1, n=1, H=28, G=7, dh=128, page=64, longest=4043, store="fp8", dtype="bf16", tree=False),
        # one token of 32 sequences of ragged length, 64 / 8 heads
        dict(name="attend_batch_8bit", op="attend", B=32, n=1, H=64, G=8, dh=128, page=64, longest=36898, store="fp8", dtype="bf16", tree=False),
        # trees of 61 drafted tokens over an unreduced prefill, 16-bit cache
        dict(name="attend_tree", op="attend", B=4, n=61, H=28, G=7, dh=128, page=64, longest=13474, store="none", dtype="bf16", tree=True),
        # one token over a very long context in 4 bits
        dict(name="attend_long_4bit", op="attend", B=1, n=1, H=28, G=7, dh=128, page=128, longest=262141, store="fp4", dtype="bf16", tree=False),
        # the accepted path of one small tree in each of 28 layers, layers as the batch
        dict(name="keep_layers", op="keep", B=28, n=8, kv=4, dh=128, page=64, before=4043, store="none", dtype="bf16"),
        # the accepted paths of wide trees, 64 sequences, 8 bits
        dict(name="keep_batch_8bit", op="keep", B=64, n=61, kv=8, dh=128, page=64, before=2049, store="fp8", dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "rotary", "cache", "attend", "attend", "keep"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    dh = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 48, 64, 128])
    store = rng.choice(["none", "fp8", "fp8", "fp4"])
    kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 5, 7, 8])
    if op == "tables":
        return dict(op=op, L=_spread(rng, 1, 36898), axes=rng.choice([1, 3]), rot=rng.choice([32, 64, 128]), base=rng.choice([1e4, 1e6]),
                    stretch=rng.choice([1.0, 4.0]), layout=rng.choice(["half", "interleaved"]), dtype=dtype, far=_spread(rng, 64, 1000000))
    if op == "rotary":
        B = _spread(rng, 1, 32)
        rot = rng.choice([dh, dh, dh // 2])
        axes = rng.choice([1, 1, 3])
        return dict(op=op, B=B, L=_spread(rng, 1, max(1, 4000000 // (B * kv * (group + 1) * dh))), H=kv * group, G=group, dh=dh, rot=rot, axes=axes,
                    layout="half" if axes == 3 else rng.choice(["half", "interleaved"]), dtype=dtype, grad=rng.random() < 0.4)
    if op == "cache":
        B = _spread(rng, 1, 32)
        return dict(op=op, B=B, n=_spread(rng, 1, max(1, 6000000 // (B * kv * dh))), kv=kv, dh=dh, page=page, before=rng.randrange(0, 700), store=store, dtype=dtype)
    if op == "attend":
        B = _spread(rng, 1, 16)
        tree = rng.random() < 0.5
        n = _spread(rng, 2, 64) if tree else rng.choice([1, 1, 1, 5, 33])
        return dict(op=op, B=B, n=n, H=kv * group, G=group, dh=dh, page=page, longest=_spread(rng, 1, max(2, min(100000, 40000000 // (B * kv * dh)))),
                    store=store, dtype=dtype, tree=tree)
    return dict(op=op, B=_spread(rng, 1, 64), n=_spread(rng, 1, 61), kv=kv, dh=dh, page=page, before=rng.randrange(0, 2100), store=store, dtype=dtype)


# ------------------------------------------------------------------------------------------------------- inputs
def _frequencies(rot, base, stretch):
    """(frequencies, factor on cosine and sine) of positions stretched for long contexts: slow pairs are divided by `stretch`, fast
    ones left, with a ramp between 32 and 1 turns over 32768 positions; the factor is 1 + 0.1 ln(stretch)."""
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if stretch == 1.0:
        return inv, 1.0
    turns = 32768 * inv / (2 * math.pi)
    keep = ((turns.log2() - 0.0) / 5.0).clamp(0, 1)
    return inv / stretch * (1 - keep) + inv * keep, 1.0 + 0.1 * math.log(stretch)


def _sections(rot):
    a = rot // 8
    b = (rot // 2 - a) // 2
    return (a, b, rot // 2 - a - b)


def _activations(gen, shape, dtype):
    """Heads of keys / values: normal values, a few channels eight times as large."""
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)
    gain = torch.where(torch.rand(shape[-1], generator=gen, device=DEV) < 0.04, 8.0, 1.0)
    return (x * gain).to(DT[dtype])


def _grid8(y):
    return y.to(torch.float8_e4m3fn)


def _grid4(y):
    """Codes 0..15 of the nearest e2m1 values, ties to the even code."""
    a = y.abs()
    v = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2)).clamp(max=6)
    code = torch.where(v < 2, v * 2, torch.where(v < 4, v + 2, v / 2 + 4))
    return code.to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)


def _quantise(x, store, dtype):
    """[.., dh] -> (codes, scale bytes)."""
    blocks = x.float().unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(blocks).all(-1, keepdim=True)
    top, half, cap = (1.75, 8, 1.875) if store == "fp8" else (1.5, 2, 1.5)
    limit = cap * 2.0 ** MOST[dtype]
    blocks = torch.where(bad, torch.zeros_like(blocks), blocks).clamp(-limit, limit)
    m, ex = torch.frexp(blocks.abs().amax(-1, keepdim=True))
    e = (ex - 1 - half + (2 * m > top)).clamp(min=-100)
    y = torch.ldexp(blocks, -e).flatten(-2)
    scales = torch.where(bad, 255, e + 127).squeeze(-1).to(torch.uint8)
    if store == "fp8":
        return _grid8(y), scales
    c = _grid4(y)
    return c[..., 0::2] | (c[..., 1::2] << 4), scales


E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _values(codes, scales):
    """float32 values of stored rows."""
    if scales is None:
        return codes.float()
    if codes.dtype == torch.uint8:
        both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
        v = torch.tensor(E2M1, device=codes.device)[both.int()]
    else:
        v = codes.float()
    s = torch.where(scales == 255, torch.nan, torch.exp2(scales.float() - 127))
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def _storage(case, gen, rows):
    """(cache, pages): enough pages in mixed order for `rows` tokens a sequence, filled as a running program's are."""
    B, kv, dh, page = case["B"], case.get("kv") or case["H"] // case["G"], case["dh"], case["page"]
    width = -(-rows // page)
    count = B * width + 3
    order = torch.randperm(count, generator=gen, device=DEV)[: B * width].to(torch.int32).view(B, width)
    shape = (count, kv, page, dh)
    if case["store"] == "none":
        return (_activations(gen, shape, case["dtype"]), _activations(gen, shape, case["dtype"]), None, None), order
    parts = []
    for _ in range(2):
        codes = torch.empty(shape if case["store"] == "fp8" else shape[:3] + (dh // 2,),
                            dtype=torch.float8_e4m3fn if case["store"] == "fp8" else torch.uint8, device=DEV)
        scales = torch.empty(shape[:3] + (dh // 32,), dtype=torch.uint8, device=DEV)
        step = max(1, 64000000 // (kv * page * dh))
        for at in range(0, count, step):
            n = min(step, count - at)
            codes[at:at + n], scales[at:at + n] = _quantise(_activations(gen, (n,) + shape[1:], case["dtype"]), case["store"], case["dtype"])
        parts.append((codes, scales))
    return (parts[0][0], parts[1][0], parts[0][1], parts[1][1]), order


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    pick = torch.Generator().manual_seed(int(seed))
    s = {"case": case, "dtype": DT[case["dtype"]]}
    op = case["op"]
    if op == "tables":
        inv, factor = _frequencies(case["rot"], case["base"], case["stretch"])
        shape = (3, 1, case["L"]) if case["axes"] == 3 else (1, case["L"])
        pos = torch.randint(0, case["far"] + 1, shape, generator=gen, device=DEV)
        s.update(positions=pos.sort(-1).values, inv=inv.to(DEV), factor=factor)
    elif op == "rotary":
        B, L, H, kv, dh, rot = case["B"], case["L"], case["H"], case["H"] // case["G"], case["dh"], case["rot"]
        # as the projections leave them: [B, L, heads, dh], seen head by head
        for name, heads in (("q", H), ("k", kv), ("dq", H), ("dk", kv)):
            if name in ("q", "k") or case["grad"]:
                s[name] = torch.randn((B, L, heads, dh), generator=gen, device=DEV).to(DT[case["dtype"]]).transpose(1, 2)
        pos = torch.randint(0, 40000, (3, B, L) if case["axes"] == 3 else (B, L), generator=gen, device=DEV).double()
        ang = pos[..., None] * _frequencies(rot, 1e6, 1.0)[0].to(DEV)
        ang = torch.cat((ang, ang), -1) if case["layout"] == "half" else ang.repeat_interleave(2, -1)
        s.update(cos=ang.cos().to(s["dtype"]), sin=ang.sin().to(s["dtype"]), sections=_sections(rot) if case["axes"] == 3 else None)
    elif op == "cache":
        s["cache"], s["pages"] = _storage(case, gen, case["before"] + case["n"])
        start = torch.randint(0, case["before"] + 1, (case["B"],), generator=pick)
        start[0] = case["before"]
        if case["B"] > 3:
            start[2] = -1                                      # a padding row of the batch
        s["start"] = start.to(torch.int32).to(DEV)
        kv_shape = (case["B"], case["n"], case["kv"], case["dh"])
        s["k"], s["v"] = (_activations(gen, kv_shape, case["dtype"]).transpose(1, 2) for _ in range(2))
    elif op == "attend":
        B, n, H, dh = case["B"], case["n"], case["H"], case["dh"]
        s["cache"], s["pages"] = _storage(case, gen, case["longest"] + n)
        length = torch.randint(case["longest"] // 2, case["longest"] + 1, (B,), generator=pick)
        length[0] = case["longest"]
        if B > 3:
            length[1], length[2] = 0, -1                       # nothing before the new tokens; a padding row of the batch
        s["length"] = length.to(torch.int32).to(DEV)
        s["q"] = (torch.randn((B, n, H, dh), generator=gen, device=DEV) * 0.7).to(s["dtype"]).transpose(1, 2)
        s["mask"] = None
        if case["tree"]:
            depth = torch.zeros(B, n, n, dtype=torch.bool)
            for b in range(B):
                for i in range(n):
                    parent = int(torch.randint(-1, i, (1,), generator=pick)) if i else -1
                    if parent >= 0:
                        depth[b, i] = depth[b, parent]
                    depth[b, i, i] = True
            s["mask"] = depth.to(DEV)
    else:
        s["cache"], s["pages"] = _storage(case, gen, case["before"] + case["n"])
        start = torch.randint(0, case["before"] + 1, (case["B"],), generator=pick)
        start[0] = case["before"]
        s["start"] = start.to(torch.int32).to(DEV)
        taken = torch.full((case["B"], case["n"]), -1, dtype=torch.int32)
        for b in range(case["B"]):
            count = int(torch.randint(0, case["n"] + 1, (1,), generator=pick)) if b else case["n"] // 2 + 1
            taken[b, :count] = torch.randperm(case["n"], generator=pick)[:count].sort().values.to(torch.int32)
        s["taken"] = taken.to(DEV)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _slots(pages, start, n, page):
    """(page, row in the page, inside) of positions start .. start + n - 1 of each sequence."""
    at = start.long()[:, None] + torch.arange(n, device=start.device)
    ok = (start.long()[:, None] >= 0) & (at < pages.shape[1] * page)
    at = torch.where(ok, at, 0)
    return pages.long().gather(1, at // page), at % page, ok


def _tables(s):
    c = s["case"]
    ang = s["positions"].double()[..., None] * s["inv"]
    ang = torch.cat((ang, ang), -1) if c["layout"] == "half" else ang.repeat_interleave(2, -1)
    return (ang.cos() * s["factor"]).to(s["dtype"]), (ang.sin() * s["factor"]).to(s["dtype"])


def _other(x, layout, rot):
    """The other member of each pair, the first one negated."""
    if layout == "half":
        return torch.cat((-x[..., rot // 2:rot], x[..., :rot // 2]), -1)
    p = x[..., :rot].unflatten(-1, (-1, 2))
    return torch.stack((-p[..., 1], p[..., 0]), -1).flatten(-2)


def _rotated(x, cos, sin, c, back=False):
    y = x.float()
    rot = c["rot"]
    if back:
        turned = y[..., :rot] * cos - _other(y[..., :rot] * sin, c["layout"], rot)
    else:
        turned = y[..., :rot] * cos + _other(y, c["layout"], rot) * sin
    return torch.cat((turned, y[..., rot:]), -1).to(x.dtype)


def _rotary(s):
    c = s["case"]
    cos, sin = s["cos"].float(), s["sin"].float()
    if c["axes"] == 3:
        axis = torch.arange(3, device=cos.device).repeat_interleave(torch.tensor(s["sections"], device=cos.device)).repeat(2)
        cos, sin = (t.gather(0, axis.expand(1, *t.shape[1:])).squeeze(0) for t in (cos, sin))
    cos, sin = cos[:, None], sin[:, None]
    out = [_rotated(s["q"], cos, sin, c), _rotated(s["k"], cos, sin, c)]
    if c["grad"]:
        out += [_rotated(s["dq"], cos, sin, c, True), _rotated(s["dk"], cos, sin, c, True)]
    return out


def _put(store, rows, slots):
    p, r, ok = slots
    if store is not None:
        flat = store.view(torch.uint8) if store.dtype == torch.float8_e4m3fn else store
        rows = rows.view(torch.uint8) if rows.dtype == torch.float8_e4m3fn else rows
        flat[p[ok], :, r[ok]] = rows.transpose(1, 2)[ok]


def _got(store, slots):
    p, r, _ = slots
    return None if store is None else (store.view(torch.uint8)[p, :, r].view(store.dtype) if store.dtype == torch.float8_e4m3fn else store[p, :, r])


def _read_one(codes, scales, slots, dtype):
    v = _values(_got(codes, slots), _got(scales, slots))                           # [B, n, heads, dh]
    return torch.where(slots[2][..., None, None], v, 0.0).to(dtype).transpose(1, 2)


def _read(cache, slots, dtype):
    return [_read_one(cache[0], cache[2], slots, dtype), _read_one(cache[1], cache[3], slots, dtype)]


def _cache(s):
    c, cache = s["case"], s["cache"]
    slots = _slots(s["pages"], s["start"], c["n"], c["page"])
    if c["store"] == "none":
        parts = (s["k"], s["v"], None, None)
    else:
        (kc, ks), (vc, vs) = _quantise(s["k"], c["store"], c["dtype"]), _quantise(s["v"], c["store"], c["dtype"])
        parts = (kc, vc, ks, vs)
    _put(cache[0], parts[0], slots), _put(cache[1], parts[1], slots), _put(cache[2], parts[2], slots), _put(cache[3], parts[3], slots)
    return _read(cache, slots, s["dtype"])


def _attend(s):
    c, cache = s["case"], s["cache"]
    B, n, H, dh, kv = c["B"], c["n"], c["H"], c["dh"], c["H"] // c["G"]
    k, v = (_values(codes[s["pages"].long()], None if scales is None else scales[s["pages"].long()]).permute(0, 2, 1, 3, 4).flatten(2, 3)
            for codes, scales in ((cache[0], cache[2]), (cache[1], cache[3])))     # [B, kv, positions, dh]
    q = s["q"].float().reshape(B, kv, c["G"] * n, dh) * dh ** -0.5
    scores = (q @ k.transpose(-1, -2)).view(B, kv, c["G"], n, -1)
    at = torch.arange(k.shape[2], device=q.device)
    length = s["length"].long()[:, None, None]
    new = at - length                                                              # [B, 1, positions]
    mask = s["mask"] if s["mask"] is not None else torch.ones(n, n, dtype=torch.bool, device=q.device).tril().expand(B, n, n)
    drafted = mask.gather(2, new.clamp(0, n - 1).expand(B, n, -1)) & (new >= 0) & (new < n)
    seen = ((at < length) | drafted) & (length >= 0)
    scores = torch.where(seen[:, None, None], scores, -torch.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    v = torch.where(seen.any(1)[:, None, :, None], v, 0.0)
    return (p.view(B, kv, c["G"] * n, -1) @ v).view(B, H, n, dh).to(s["dtype"])


def _keep(s):
    c, cache = s["case"], s["cache"]
    slots = _slots(s["pages"], s["start"], c["n"], c["page"])
    from_row = torch.where(s["taken"] >= 0, s["taken"].long(), torch.arange(c["n"], device=s["taken"].device))
    source = (slots[0].gather(1, from_row), slots[1].gather(1, from_row), slots[2])
    parts = [None if t is None else _got(t, source).transpose(1, 2) for t in cache]
    _put(cache[0], parts[0], slots), _put(cache[1], parts[1], slots), _put(cache[2], parts[2], slots), _put(cache[3], parts[3], slots)
    return _read(cache, slots, s["dtype"])


def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        import framefusion_amd as ffa
        if op == "tables":
            return ffa.rotary_tables(s["positions"], s["inv"], dtype=s["dtype"], factor=s["factor"], interleaved=c["layout"] == "interleaved")
        if op == "rotary":
            how = dict(sections=s["sections"], interleaved=c["layout"] == "interleaved")
            if not c["grad"]:
                return ffa.apply_rotary(s["q"], s["k"], s["cos"], s["sin"], **how)
            q, k = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
            out = ffa.apply_rotary(q, k, s["cos"], s["sin"], **how)
            return [t.detach() for t in out] + list(torch.autograd.grad(out, (q, k), (s["dq"], s["dk"])))
        if op == "cache":
            ffa.cache_write(s["cache"], s["k"], s["v"], s["pages"], s["start"])
            return ffa.cache_read(s["cache"], s["pages"], s["start"], c["n"], dtype=s["dtype"])
        if op == "attend":
            return ffa.cache_attention(s["q"], s["cache"], s["pages"], s["length"], mask=s["mask"])
        ffa.cache_keep(s["cache"], s["pages"], s["start"], s["taken"])
        return ffa.cache_read(s["cache"], s["pages"], s["start"], c["n"], dtype=s["dtype"])
    return {"tables": _tables, "rotary": _rotary, "cache": _cache, "attend": _attend, "keep": _keep}[op](s)


# ------------------------------------------------------------------------------------------------------ the work
def _row_bytes(case):
    """Bytes of one head's key (or value) of one token in the cache."""
    if case["store"] == "none":
        return case["dh"] * SIZE[case["dtype"]]
    return case["dh"] * (8 if case["store"] == "fp8" else 4) // 8 + case["dh"] // 32


def work(case):
    op, e = case["op"], SIZE[case["dtype"]]
    if op == "tables":
        n = case["axes"] * case["L"]
        return {"bytes": n * (8 + 2 * case["rot"] * e) + case["rot"] * 4, "flops": n * case["rot"] // 2 * 4}
    if op == "rotary":
        heads, times = case["H"] + case["H"] // case["G"], 2 if case["grad"] else 1
        n = case["B"] * case["L"]
        return {"bytes": n * (times * 2 * heads * case["dh"] + 2 * case["axes"] * case["rot"]) * e, "flops": times * 3 * n * heads * case["rot"]}
    if op == "cache":
        rows = 2 * case["B"] * case["n"] * case["kv"]
        return {"bytes": rows * (2 * case["dh"] * e + _row_bytes(case)) + case["B"] * 4, "flops": rows * case["dh"] * 4}
    if op == "attend":
        # prepare() takes lengths between half the longest and the longest; the work is priced at their mean
        held = case["B"] * (0.75 * case["longest"] + case["n"]) if case["B"] > 1 else case["longest"] + case["n"]
        if case["B"] > 3:
            held *= (case["B"] - 2) / case["B"]
        kv = case["H"] // case["G"]
        return {"bytes": int(2 * held * kv * _row_bytes(case) + 2 * case["B"] * case["n"] * case["H"] * case["dh"] * e),
                "flops": int(4 * case["n"] * case["H"] * case["dh"] * held)}
    rows = 2 * case["B"] * case["n"] * case["kv"]
    return {"bytes": int(rows * (_row_bytes(case) * 1.5 + case["dh"] * e)), "flops": rows * case["dh"]}


# ------------------------------------------------------------------------------ the definitions, in 64 bits
def _exact_block(x, store, dtype):
    """A block of 32 numbers -> the numbers that its codes stand for."""
    cap = (1.875 if store == "fp8" else 1.5) * 2.0 ** MOST[dtype]
    x = x.double().unflatten(-1, (-1, 32))
    nan = ~torch.isfinite(x).all(-1, keepdim=True)
    x = torch.where(nan, 0.0, x).clamp(-cap, cap)
    top = 448.0 if store == "fp8" else 6.0
    big = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(big.clamp(min=1e-300) / top)).clamp(min=-100)
    e = torch.where(big > top * torch.exp2(e), e + 1, torch.where((big <= top * torch.exp2(e - 1)) & (e > -100), e - 1, e))
    y = x / torch.exp2(e)
    low, bits = (-6, 3) if store == "fp8" else (0, 1)
    lead = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** low)))
    step = torch.exp2(lead - bits)
    return torch.where(nan, torch.nan, torch.round(y / step) * step * torch.exp2(e)).flatten(-2)


def _exact_rows(cache, which, pages):
    codes, scales = cache[which][pages], None if cache[2 + which] is None else cache[2 + which][pages]
    if scales is None:
        return codes.double()
    b = codes.view(torch.uint8).long()
    if codes.dtype == torch.uint8:
        b = torch.stack((b % 16, b // 16), -1).flatten(-2)
        mant, expo, sign = b % 2, b // 2 % 4, b // 8
        v = torch.where(expo == 0, mant * 0.5, (1 + mant * 0.5) * torch.exp2(expo.double() - 1))
    else:
        mant, expo, sign = b % 8, b // 8 % 16, b // 128
        v = torch.where(expo == 0, mant / 512.0, (1 + mant / 8.0) * torch.exp2(expo.double() - 7))
    v = torch.where(sign == 1, -v, v)
    return (v.unflatten(-1, (-1, 32)) * torch.exp2(scales.double() - 127)[..., None]).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "tables":
        a = s["positions"].double().unsqueeze(-1) * s["inv"]
        pick = torch.arange(case["rot"], device=DEV)
        a = a[..., pick % (case["rot"] // 2) if case["layout"] == "half" else pick // 2]
        return torch.cos(a) * s["factor"], torch.sin(a) * s["factor"]
    if op == "rotary":
        rot, i = case["rot"], torch.arange(case["rot"] // 2, device=DEV)
        first, second = (i, i + rot // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
        cos, sin = s["cos"].double(), s["sin"].double()
        if case["axes"] == 3:
            a, b, _ = s["sections"]
            which = (i >= a).long() + (i >= a + b).long()
            pairs = [t[which, :, :, col].permute(1, 2, 0) for t in (cos, sin) for col in (first, second)]
        else:
            pairs = [t[..., col] for t in (cos, sin) for col in (first, second)]
        c1, c2, s1, s2 = (t.unsqueeze(1) for t in pairs)
        out = []
        for name in ("q", "k"):
            x = s[name].double()
            y = x.clone()
            y[..., first] = x[..., first] * c1 - x[..., second] * s1
            y[..., second] = x[..., second] * c2 + x[..., first] * s2
            out.append(y)
        for name in ("dq", "dk") if case["grad"] else ():
            x = s[name].double()
            y = x.clone()
            y[..., first] = x[..., first] * c1 + x[..., second] * s2
            y[..., second] = x[..., second] * c2 - x[..., first] * s1
            out.append(y)
        return out
    if op == "cache":
        out = []
        for name in ("k", "v"):
            x = s[name].double() if case["store"] == "none" else _exact_block(s[name], case["store"], case["dtype"])
            out.append(torch.where((s["start"] >= 0)[:, None, None, None], x, 0.0))
        return out
    if op == "keep":
        out = []
        for which in (0, 1):
            got = []
            for b in range(case["B"]):
                rows = _exact_rows(s["cache"], which, s["pages"][b].long()).transpose(0, 1).flatten(1, 2)      # [heads, positions, dh]
                at = int(s["start"][b])
                rows = rows[:, at:at + case["n"]].clone()
                take = s["taken"][b][s["taken"][b] >= 0].long()
                rows[:, : len(take)] = rows[:, take]
                got.append(rows)
            out.append(torch.stack(got))
        return out
    if 4.0 * case["n"] * case["H"] * case["dh"] * case["B"] * case["longest"] > 1e13:
        return None
    B, n, H, dh = case["B"], case["n"], case["H"], case["dh"]
    out = torch.zeros(B, H, n, dh, dtype=torch.float64, device=DEV)
    for b in range(B):
        L = int(s["length"][b])
        if L < 0:
            continue
        k, v = (_exact_rows(s["cache"], w, s["pages"][b].long()).transpose(0, 1).flatten(1, 2)[:, : L + n] for w in (0, 1))
        see = torch.ones(n, L + n, dtype=torch.bool, device=DEV)
        see[:, L:] = torch.tril(see[:, L:]) if s["mask"] is None else s["mask"][b]
        for h in range(H):
            score = s["q"][b, h].double() @ k[h // case["G"]].T / math.sqrt(dh)
            out[b, h] = torch.softmax(score.masked_fill(~see, -torch.inf), -1) @ v[h // case["G"]]
    return out
