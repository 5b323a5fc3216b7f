"""GPU: the attention over the paged cache where a wave goes through many blocks of keys: its loads ahead, page numbers two steps ahead, two
buffers, a maximum that moves while outputs are held, every way for the last step to end.

Bounds are those of test_gpu_cached_decoding.reference (the same formula, all heads of a sequence at once)."""
import math

import pytest
import torch

import framefusion_amd as ffa
from framefusion_amd import _lib
from tests.test_gpu_cached_decoding import DEV, DT, U, half_step, rounding, stored, tree, within

pytestmark = pytest.mark.gpu


def steps_of(dtype, store, dh, kv, G, n, page, width, starts):
    """(blocks of keys that a workgroup with a full share goes through, whether sequences are split), from the workspace that the library
    asks for: [kv heads, rows, slots] partial rows, and slots = shares + sequences."""
    B, rows = len(starts), n * G
    many = dtype != "fp32" and rows > 128
    code = {"fp32": 0, "bf16": 1, "fp16": 2}[dtype]
    a = _lib.CACHE_ATTENTION.pack(4096, 4096, *((0, 0) if store is None else (4096, 4096)), 64, 64,
                                  {None: code, "fp8": _lib.STORE_E4M3, "fp4": _lib.STORE_E2M1}[store], B * width + 2, kv, page, dh, width, B, n, code,
                                  4096, 4096, 0, 0, 0, kv * G, *[dh] * 6, 0, 0.1, 0)
    need = _lib.load().ff_cache_attention_workspace_bytes(a)
    blocks = [-(-(s + n) // (64 if many else 128)) for s in starts]
    if need == 0:
        return max(blocks), False
    slots = (need - 8 * B) // (4 * (dh + 2)) // (kv * rows)
    return -(-sum(blocks) // (slots - (B if B > 1 else 0))), True


def run(dtype, store, dh, kv, G, n, page, starts, mask=None, least=3, split=True, seed=0, scale=None):
    T, B = DT[dtype], len(starts)
    gen = torch.Generator(device=DEV).manual_seed(seed + dh + 1000 * n)
    width = -(-(max(starts) + n) // page)
    each, is_split = steps_of(dtype, store, dh, kv, G, n, page, width, starts)
    assert each >= least and is_split == split, (each, is_split)
    S, pages = width * page, B * width + 2
    cache = ffa.new_cache(pages, page, kv, dh, T, store, device=DEV)
    for t in cache:                                                           # what is not written holds NaN
        if t is not None and (store is None or t.shape[-1] == dh // 32):
            t.fill_(math.nan if store is None else 255)
    table = torch.randperm(pages, generator=gen, device=DEV)[: B * width].to(torch.int32).view(B, width).contiguous()
    start, zero = torch.tensor(starts, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    k, v = (torch.randn(B, kv, S, dh, generator=gen, device=DEV) for _ in range(2))
    # a third of the heads flat over the context, a third with scores that climb 12 over it (17 octaves: the maximum keeps moving), a third that fall
    slope = torch.tensor([0.0, 1.0, -1.0], device=DEV)[torch.arange(kv, device=DEV) % 3]
    k[..., 0] = slope[None, :, None] * 12 * math.sqrt(dh) / 1.5 * torch.arange(S, device=DEV) / max(starts)
    k, v = k.to(T), v.to(T)
    for b, s in enumerate(starts):
        ffa.cache_write(cache, k[b:b + 1, :, :s + n], v[b:b + 1, :, :s + n], table[b:b + 1], zero)
    q = torch.randn(B, n, kv * G, dh, generator=gen, device=DEV) * 1.5         # scores of deviation 1.5: no key carries everything, none is nothing
    q[..., 0] = 1.5
    q = q.to(T).transpose(1, 2)
    got = ffa.cache_attention(q, cache, table, start, mask=mask)
    torch.cuda.synchronize()
    dense_k, dense_v = stored(k, store, T).double(), stored(v, store, T).double()
    new = torch.ones(n, n, dtype=torch.bool, device=DEV).tril() if mask is None else mask
    for b, s in enumerate(starts):
        kk, vv = dense_k[b, :, :s + n].contiguous(), dense_v[b, :, :s + n].contiguous()
        qq = q[b].double().reshape(kv, G * n, dh)
        see = torch.cat((torch.ones(n, s, dtype=torch.bool, device=DEV), new[b] if new.ndim == 3 else new), 1).repeat(G, 1)
        kt = kk.transpose(1, 2).contiguous()
        x = (torch.matmul(qq, kt) * dh ** -0.5).masked_fill(~see, -math.inf)
        p = torch.softmax(x, -1)
        want = torch.matmul(p, vv).view(kv * G, n, dh)
        off = (torch.matmul(qq.abs(), kt.abs()) * dh ** -0.5).masked_fill(~see, 0.0).amax(-1, keepdim=True) * (dh + 4) * U
        tol = torch.matmul(p, vv.abs()) * (4 * off + (s + n + 16) * U + (0 if dtype == "fp32" else half_step(T)))
        within(got[b], want, tol.view(kv * G, n, dh) + rounding(T, want))
    again = ffa.cache_attention(q, cache, table, start, mask=mask)
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("store", [None, "fp8", "fp4"])
@pytest.mark.parametrize("dh", [32, 64, 128, 256])
def test_few_rows(dtype, store, dh):
    """One tile of 16 rows a wave, and more rows than that (two tiles where they are built); sequences split over workgroups."""
    run(dtype, store, dh, 64, 1, 1, 64, [5003, 2689, 131], least=4)
    run(dtype, store, dh, 64, 2, 9, 16, [4300, 2177, 700], mask=tree(9, 3, dh), least=3)
    run(dtype, store, dh, 48, 2, 20, 48, [6100], least=3)                        # one sequence: shares known before the lengths are


@pytest.mark.parametrize("dtype,store", [("bf16", None), ("bf16", "fp8"), ("fp16", "fp4"), ("fp16", None), ("fp32", None), ("fp32", "fp8")])
@pytest.mark.parametrize("dh", [32, 64, 128, 256])
def test_few_rows_of_whole_sequences(dtype, store, dh):
    """Sequences enough that none is split: a workgroup goes through all of its keys; lengths that end in every place of a tile."""
    run(dtype, store, dh, 256, 1, 1, 16, [1500, 1027, 512, 511, 385, 900, 128, 1], least=8, split=False)
    run(dtype, store, dh, 256, 2, 10, 32, [700, 300, 260, 129, 60, 31, 480, 640], least=5, split=False)


@pytest.mark.parametrize("ctx", [767, 768, 769, 783, 784, 799, 800, 895, 896])
def test_every_end_of_the_last_step(ctx):
    for dtype, store, dh in (("bf16", "fp8", 128), ("fp32", None, 64), ("fp16", None, 32)):
        run(dtype, store, dh, 256, 1, 1, 16, [ctx] * 8, least=6, split=False, seed=ctx)
    run("bf16", "fp4", 64, 64, 2, 65, 16, [ctx] * 8, least=8, split=False, seed=ctx)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("store", [None, "fp8", "fp4"])
@pytest.mark.parametrize("dh", [32, 64, 128, 256])
def test_many_rows(dtype, store, dh):
    """Trees and chunks of more than 128 rows, split over workgroups, and sequences enough that none is."""
    run(dtype, store, dh, 4, 7, 61, 64, [4099, 4500, 2050, 64], mask=tree(61, 4, dh), least=4)
    run(dtype, store, dh, 16, 3, 45, 16, [3000], least=3)
    run(dtype, store, dh, 64, 3, 45, 48, [700, 513, 64, 300, 447, 448, 449, 1, 640, 127, 10, 580, 333, 200, 690, 100], mask=tree(45, 16, dh), least=8, split=False)
