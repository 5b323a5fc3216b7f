"""CPU: what the cached-decoding operators refuse, where a position lies in the paged cache, frequencies of stretched positions."""
import ctypes as C
import os
import random
import shutil
import subprocess

import numpy as np
import pytest
import torch

import framefusion_amd as ffa
from framefusion_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ERR_ARG, ERR_ALIGN, ERR_UNSUPPORTED = -1, -2, -3


def test_structures_match_the_library():
    lib = _lib.load()
    for which, cls, fmt in ((6, _lib.FFRotary, _lib.ROTARY), (7, _lib.FFCache, _lib.CACHE), (8, _lib.FFCacheRows, _lib.CACHE_ROWS),
                            (9, _lib.FFCacheAttention, _lib.CACHE_ATTENTION)):
        assert lib.ff_abi_sizeof(which) == C.sizeof(cls) == fmt.size


# ---- the C entries look at every argument before anything is launched ---------------------------------------------------
CACHE = dict(keys=4096, values=8192, key_scales=0, value_scales=0, table=64, start=64, store=1, n_pages=4, kv_heads=2, page_size=64, dh=64,
             table_width=2, B=1, n=3, dtype=1)
ROWS = dict(k=4096, v=4096, k_batch=64, k_head=64, k_token=64, v_batch=64, v_head=64, v_token=64, stream=0)
ATT = dict(q=4096, out=4096, mask=0, ws=0, ws_bytes=0, H=4, q_batch=64, q_head=64, q_token=64, o_batch=64, o_head=64, o_token=64, mask_batch=0,
           scale=0.1, stream=0)


def pack(fmt, *parts, **change):
    values = {}
    for p in parts:
        values.update(p)
    assert set(change) <= set(values)
    values.update(change)
    return fmt.pack(*values.values())


@pytest.mark.parametrize("change,want", [
    (dict(keys=0), ERR_ARG), (dict(table=0), ERR_ARG), (dict(start=0), ERR_ARG), (dict(dtype=7), ERR_ARG), (dict(store=0), ERR_ARG),
    (dict(store=5), ERR_ARG), (dict(store=8), ERR_ARG), (dict(store=4, key_scales=64), ERR_ARG), (dict(n_pages=-1), ERR_ARG), (dict(kv_heads=0), ERR_ARG),
    (dict(B=-1), ERR_ARG), (dict(n=-1), ERR_ARG), (dict(dh=0), ERR_ARG), (dict(page_size=0), ERR_ARG), (dict(table_width=-1), ERR_ARG),
    (dict(keys=4100), ERR_ALIGN), (dict(values=4104), ERR_ALIGN), (dict(dh=48), ERR_UNSUPPORTED), (dict(dh=288), ERR_UNSUPPORTED),
    (dict(page_size=40), ERR_UNSUPPORTED), (dict(page_size=1 << 17), ERR_UNSUPPORTED), (dict(n_pages=1 << 31), ERR_UNSUPPORTED),
    (dict(table_width=1 << 26), ERR_UNSUPPORTED), (dict(B=1 << 20, n=1 << 20), ERR_UNSUPPORTED), (dict(B=1 << 40), ERR_UNSUPPORTED),
    (dict(kv_heads=5000), ERR_UNSUPPORTED)])
def test_cache_arguments_are_refused(change, want):
    lib = _lib.load()
    assert lib.ff_cache_write(pack(_lib.CACHE_ROWS, CACHE, ROWS, **change)) == want
    assert lib.ff_cache_read(pack(_lib.CACHE_ROWS, CACHE, ROWS, **change)) == want
    assert lib.ff_cache_keep(pack(_lib.CACHE, CACHE, **change), 64, 2, None) == want
    assert lib.ff_cache_attention(pack(_lib.CACHE_ATTENTION, CACHE, ATT, **change)) == want
    assert lib.ff_cache_attention_workspace_bytes(pack(_lib.CACHE_ATTENTION, CACHE, ATT, **change)) == 0


def test_call_arguments_are_refused():
    lib = _lib.load()
    for change, want in ((dict(k=0), ERR_ARG), (dict(v=0), ERR_ARG), (dict(k=4104), ERR_ALIGN), (dict(k_token=36), ERR_ALIGN), (dict(v_batch=4), ERR_ALIGN)):
        assert lib.ff_cache_write(pack(_lib.CACHE_ROWS, CACHE, ROWS, **change)) == want
        assert lib.ff_cache_read(pack(_lib.CACHE_ROWS, CACHE, ROWS, **change)) == want
    for change, want in ((dict(q=0), ERR_ARG), (dict(out=0), ERR_ARG), (dict(H=3), ERR_ARG), (dict(H=0), ERR_ARG), (dict(mask_batch=-1), ERR_ARG),
                         (dict(scale=float("nan")), ERR_ARG), (dict(scale=float("-inf")), ERR_ARG), (dict(q=4104), ERR_ALIGN), (dict(q_head=4), ERR_ALIGN), (dict(dh=96), ERR_UNSUPPORTED), (dict(H=1 << 17), ERR_UNSUPPORTED)):
        assert lib.ff_cache_attention(pack(_lib.CACHE_ATTENTION, CACHE, ATT, **change)) == want
    assert lib.ff_cache_keep(pack(_lib.CACHE, CACHE), None, 2, None) == ERR_ARG
    assert lib.ff_cache_keep(pack(_lib.CACHE, CACHE), 64, -1, None) == ERR_ARG
    for fn in (lib.ff_cache_write, lib.ff_cache_read, lib.ff_cache_attention, lib.ff_rotary_apply):
        assert fn(None) == ERR_ARG
    # nothing to do is no error
    for change in (dict(B=0), dict(n=0)):
        assert lib.ff_cache_write(pack(_lib.CACHE_ROWS, CACHE, ROWS, **change)) == 0
        assert lib.ff_cache_attention(pack(_lib.CACHE_ATTENTION, CACHE, ATT, **change)) == 0
    assert lib.ff_cache_keep(pack(_lib.CACHE, CACHE), None, 0, None) == 0


def test_rotary_arguments_are_refused():
    lib = _lib.load()
    rot = dict(q=4096, k=4096, q_out=4096, k_out=4096, cos=64, sin=64, dtype=1, table_dtype=1, B=1, L=2, H=4, H_kv=2, dh=64, rot=64, q_batch=0, q_head=64,
               q_token=256, k_batch=0, k_head=64, k_token=128, qo_batch=0, qo_head=64, qo_token=256, ko_batch=0, ko_head=64, ko_token=128, t_axis=0,
               t_batch=0, t_token=64, sec0=0, sec1=0, interleaved=0, transpose=0, stream=0)
    for change in (dict(q=0), dict(k_out=0), dict(cos=0), dict(dtype=3), dict(table_dtype=2), dict(rot=63), dict(rot=66), dict(rot=0), dict(B=-1), dict(L=-1),
                   dict(sec0=-1), dict(sec0=20, sec1=20), dict(sec0=8, sec1=8, interleaved=1)):
        assert lib.ff_rotary_apply(pack(_lib.ROTARY, rot, **change)) == ERR_ARG, change
    for change in (dict(dh=1 << 13), dict(H=1 << 16), dict(B=1 << 20, L=1 << 20)):
        assert lib.ff_rotary_apply(pack(_lib.ROTARY, rot, **change)) == ERR_UNSUPPORTED, change
    assert lib.ff_rotary_apply(pack(_lib.ROTARY, rot, L=0)) == 0
    assert lib.ff_rotary_tables(None, 1, 64, 4, 1.0, 0, 1, 64, 64, None) == ERR_ARG
    assert lib.ff_rotary_tables(64, 1, 64, 0, 1.0, 0, 1, 64, 64, None) == ERR_ARG
    assert lib.ff_rotary_tables(64, 1, 64, 4, 1.0, 0, 9, 64, 64, None) == ERR_ARG
    assert lib.ff_rotary_tables(64, 1, 64, 5000, 1.0, 0, 1, 64, 64, None) == ERR_UNSUPPORTED
    assert lib.ff_rotary_tables(64, 0, 64, 4, 1.0, 0, 1, 64, 64, None) == 0


# ---- the Python entries --------------------------------------------------------------------------------------------------
def cpu_cache(store=None, dtype=torch.bfloat16, pages=3, page=16, heads=2, dh=64):
    return ffa.new_cache(pages, page, heads, dh, dtype, store, device="cpu")


def test_new_cache_shapes_and_refusals():
    for store, width in ((None, 64), ("fp8", 64), ("fp4", 32)):
        c = cpu_cache(store)
        assert c.keys.shape == c.values.shape == (3, 2, 16, width)
        assert (c.key_scales is None) == (store is None)
        if store:
            assert c.key_scales.shape == c.value_scales.shape == (3, 2, 16, 2) and c.key_scales.dtype == torch.uint8
    for bad in (dict(page_size=8), dict(page_size=24), dict(head_dim=80), dict(head_dim=512), dict(kv_heads=0), dict(pages=-1), dict(store="fp6"),
                dict(dtype=torch.float64)):
        with pytest.raises(ffa.FrameFusionHipError):
            ffa.new_cache(**{**dict(pages=3, page_size=16, kv_heads=2, head_dim=64, device="cpu"), **bad})


def test_python_refusals_without_a_gpu():
    table, start = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 2, 5, 64, dtype=torch.bfloat16)
    q = torch.zeros(2, 4, 5, 64, dtype=torch.bfloat16)
    c = cpu_cache()
    calls = [
        lambda: ffa.cache_write(c, x.float(), x.float(), table, start),                      # the cache's type alone
        lambda: ffa.cache_write(c, x, x[:, :1], table, start),
        lambda: ffa.cache_write(c, x[..., :32], x[..., :32], table, start),
        lambda: ffa.cache_write(c, x[0], x[0], table, start),
        lambda: ffa.cache_write(c, x, x.half(), table, start),
        lambda: ffa.cache_write(c, x.clone().requires_grad_(), x, table, start),
        lambda: ffa.cache_write(c, x, x, table.long(), start),
        lambda: ffa.cache_write(c, x, x, table, start.long()),
        lambda: ffa.cache_write(c, x, x, table, start[:1]),
        lambda: ffa.cache_write(c, x, x, table.t().contiguous().t(), start),
        lambda: ffa.cache_write(c._replace(values=c.values[:, :1]), x, x, table, start),
        lambda: ffa.cache_write(c._replace(keys=c.keys.transpose(1, 2)), x, x, table, start),
        lambda: ffa.cache_write(cpu_cache("fp8")._replace(key_scales=None), x, x, table, start),
        lambda: ffa.cache_write(cpu_cache("fp4")._replace(value_scales=torch.zeros(1, dtype=torch.uint8)), x, x, table, start),
        lambda: ffa.cache_write((1, 2, 3, 4), x, x, table, start),
        lambda: ffa.cache_write(c[:3], x, x, table, start),
        lambda: ffa.cache_write(c, None, x, table, start),
        lambda: ffa.cache_write(c, x, x, None, start),
        lambda: ffa.cache_read(c, table, start, 4, dtype="bf16"),
        lambda: ffa.cache_attention(q, c, table, start, mask=3),
        lambda: ffa.cache_read(c, table, start, -1),
        lambda: ffa.cache_read(c, table, start, 4, dtype=torch.float32),
        lambda: ffa.cache_keep(c, table, start, torch.zeros(2, 3)),
        lambda: ffa.cache_keep(c, table, start, torch.zeros(1, 3, dtype=torch.int32)),
        lambda: ffa.cache_attention(q[:, :3], c, table, start),
        lambda: ffa.cache_attention(q[0], c, table, start),
        lambda: ffa.cache_attention(q[:1], c, table, start),
        lambda: ffa.cache_attention(q, c, table, start, mask=torch.ones(5, 4, dtype=torch.bool)),
        lambda: ffa.cache_attention(q, c, table, start, mask=torch.ones(5, 5)),
        lambda: ffa.cache_attention(q.clone().requires_grad_(), c, table, start),
        lambda: ffa.cache_attention(torch.zeros(2, 4, 5, 96), cpu_cache(dtype=torch.float32, dh=96), table, start),
    ]
    for at, call in enumerate(calls):
        with pytest.raises(ffa.FrameFusionHipError):
            call()
            pytest.fail(f"call {at} was not refused")
    with pytest.raises(TypeError):
        ffa.cache_attention(q, c, table, start, scale="half")
    with pytest.raises(TypeError):
        ffa.cache_read(c, table, start, 2.5)
    # what is right but for the device says so
    for call in (lambda: ffa.cache_write(c, x, x, table, start), lambda: ffa.cache_attention(q, c, table, start),
                 lambda: ffa.cache_read(c, table, start, 4), lambda: ffa.cache_keep(c, table, start, torch.zeros(2, 3, dtype=torch.int32))):
        with pytest.raises(ffa.FrameFusionHipError, match="MI355X only"):
            call()


def test_a_cache_is_a_tuple_or_a_list():
    """The tensors of an iterator would be gone before the launch."""
    x, table, start = torch.zeros(2, 2, 5, 64), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    c = cpu_cache(dtype=torch.float32, dh=64)
    for cache in (iter(c), (t for t in c), {t: 0 for t in range(4)}, None):
        with pytest.raises(ffa.FrameFusionHipError, match="four tensors"):
            ffa.cache_write(cache, x, x, table, start)
    for cache in (c, list(c), tuple(c)):
        with pytest.raises(ffa.FrameFusionHipError, match="MI355X only"):
            ffa.cache_write(cache, x, x, table, start)


def test_rotary_refusals_without_a_gpu():
    q, k = torch.zeros(1, 4, 5, 32), torch.zeros(1, 2, 5, 32)
    t, t3 = torch.zeros(1, 5, 32), torch.zeros(3, 1, 5, 32)
    for call in (lambda: ffa.apply_rotary(q[0], k, t, t), lambda: ffa.apply_rotary(q, k[:, :, :4], t, t), lambda: ffa.apply_rotary(q, k.half(), t, t),
                 lambda: ffa.apply_rotary(q.double(), k.double(), t, t), lambda: ffa.apply_rotary(q, k, t, t[..., :16]), lambda: ffa.apply_rotary(q, k, t3, t3),
                 lambda: ffa.apply_rotary(q, k, t, t, sections=(4, 6, 6)), lambda: ffa.apply_rotary(q, k, t3, t3, sections=(4, 6, 5)),
                 lambda: ffa.apply_rotary(q, k, t3, t3, sections=(0, 8, 8)), lambda: ffa.apply_rotary(q, k, t3, t3, sections=(4, 6, 6), interleaved=True),
                 lambda: ffa.apply_rotary(q, k, t[:, :4], t[:, :4]), lambda: ffa.apply_rotary(q, k, t.half(), t.half()),
                 lambda: ffa.apply_rotary(q[..., :16], k[..., :16], t, t), lambda: ffa.apply_rotary(q, k, t[..., :31], t[..., :31]),
                 lambda: ffa.apply_rotary(q, k, t.clone().requires_grad_(), t),
                 lambda: ffa.rotary_tables(torch.zeros(1, 3), torch.zeros(4, dtype=torch.float64)),
                 lambda: ffa.rotary_tables(torch.zeros(1, 3, dtype=torch.int64), torch.zeros(4)),
                 lambda: ffa.rotary_tables(torch.zeros(1, 3, dtype=torch.int64), torch.zeros(4, dtype=torch.float64), dtype=torch.float64)):
        with pytest.raises(ffa.FrameFusionHipError) as e:
            call()
        assert "MI355X only" not in str(e.value)
    with pytest.raises(ffa.FrameFusionHipError, match="MI355X only"):
        ffa.apply_rotary(q, k, t, t)


# ---- where a position lies (csrc/ff_place.h, compiled for the host) ------------------------------------------------------
@pytest.fixture(scope="module")
def place(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("place")
    src, so = d / "place.cpp", d / "place.so"
    src.write_text('#include "ff_place.h"\nextern "C" int64_t row(const int32_t* t, int64_t w, int64_t n, int ps, int kv, int h, int64_t p) '
                   '{ return ff::cache_row(t, w, n, ps, kv, h, p); }\n')
    subprocess.run([gxx, "-O1", "-shared", "-fPIC", "-Wall", "-Werror", "-I", os.path.join(ROOT, "framefusion_amd", "csrc"), str(src), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.row.restype = C.c_int64
    lib.row.argtypes = [C.c_void_p, C.c_int64, C.c_int64, C.c_int, C.c_int, C.c_int, C.c_int64]
    return lambda table, n, ps, kv, h, p: lib.row(table.ctypes.data, len(table), n, ps, kv, h, p)


def test_positions_and_bad_pages(place):
    rng = random.Random(5)
    for _ in range(300):
        ps, kv, n, w = rng.choice([16, 48, 64, 65536]), rng.choice([1, 2, 8]), rng.randrange(1, 9), rng.randrange(0, 7)
        table = np.array([rng.choice([rng.randrange(n), rng.randrange(n), -1, n, 2**31 - 1, -2**31]) for _ in range(w)] + [0], dtype=np.int32)[:w]
        for _ in range(20):
            p, h = rng.choice([rng.randrange(-3, w * ps + 3), -2**40, 2**40, 2**32]), rng.randrange(kv)
            got = place(table, n, ps, kv, h, p)
            if p < 0 or p >= w * ps or not 0 <= table[p // ps] < n:
                assert got == -1
            else:
                assert got == (int(table[p // ps]) * kv + h) * ps + p % ps
    # rows beyond 32 bits
    table = np.array([0, 2_000_000], dtype=np.int32)
    assert place(table, 2_000_001, 64, 64, 63, 127) == (2_000_000 * 64 + 63) * 64 + 63


# ---- frequencies ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("scaling", [
    None, {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
    {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096, "beta_fast": 24, "beta_slow": 2, "attention_factor": 1.5},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}])
@pytest.mark.parametrize("dim,base", [(128, 1e6), (64, 1e4), (32, 5e5)])
def test_frequencies_against_transformers(scaling, dim, base):
    """The installed transformers computes the same in float32: pair for pair within its own rounding."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    inv, factor = ffa.rotary_frequencies(dim, base, scaling)
    assert inv.dtype == torch.float64 and inv.shape == (dim // 2,)
    if scaling is None:
        assert factor == 1.0 and torch.equal(inv, base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim))
        return
    cfg = LlamaConfig(hidden_size=dim * 2, num_attention_heads=2, head_dim=dim, max_position_embeddings=131072,
                      rope_parameters={**scaling, "rope_theta": base})
    want, want_factor = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, "cpu")
    # float32 there: the power (exponents up to ln(1e6) = 14 carry 14 * 2^-24 into the value), the blend and its index arithmetic
    assert torch.allclose(inv, want.double(), rtol=2e-5, atol=0)
    assert abs(factor - want_factor) < 1e-6


def test_ntk_keeps_the_fastest_pair_and_slows_the_last():
    inv, _ = ffa.rotary_frequencies(64, 1e4)
    got, factor = ffa.rotary_frequencies(64, 1e4, {"rope_type": "ntk", "factor": 8.0})
    assert factor == 1.0 and got[0] == 1.0 and abs(got[-1] * 8 / inv[-1] - 1) < 1e-12
    for bad in (dict(dim=7), dict(dim=0), dict(dim=64, scaling={"rope_type": "what", "factor": 2.0}), dict(dim=64, scaling={"rope_type": "linear", "factor": 0.0}),
                dict(dim=2, scaling={"rope_type": "ntk", "factor": 2.0})):
        with pytest.raises(ffa.FrameFusionHipError):
            ffa.rotary_frequencies(**bad)
