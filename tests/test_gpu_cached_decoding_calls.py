"""GPU: the cached-decoding calls under what PyTorch wraps around a call - forward-mode derivatives, lazily negated tensors."""
import pytest
import torch
from torch.autograd import forward_ad

import framefusion_amd as ffa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sections,interleaved", [(None, False), (None, True), ((4, 6, 6), False)])
def test_the_rotation_carries_tangents(dtype, sections, interleaved):
    """The rotation is linear: its tangent is the same call on the tangent, bit for bit."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    q, k = torch.randn(2, 4, 7, 32, generator=gen, device=DEV).to(dtype), torch.randn(2, 2, 7, 32, generator=gen, device=DEV).to(dtype)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    cos, sin = (torch.randn(((3,) if sections else ()) + (2, 7, 32), generator=gen, device=DEV) for _ in range(2))
    how = dict(sections=sections, interleaved=interleaved)
    for transpose in (False, True):
        with forward_ad.dual_level():
            got = [forward_ad.unpack_dual(y) for y in ffa.apply_rotary(forward_ad.make_dual(q, dq), forward_ad.make_dual(k, dk), cos, sin, transpose=transpose, **how)]
        for y, x, t in zip(got, ffa.apply_rotary(q, k, cos, sin, transpose=transpose, **how), ffa.apply_rotary(dq, dk, cos, sin, transpose=transpose, **how)):
            assert torch.equal(y.primal, x) and torch.equal(y.tangent, t)


# ---- values that PyTorch keeps beside the memory: the negative bit, zeros without memory
def negated(t):
    """A tensor of t's values whose memory holds -t."""
    n = torch._neg_view(-t)
    assert n.is_neg() and torch.equal(n, t)
    return n


def decoding_inputs(dtype=torch.bfloat16):
    gen = torch.Generator(device=DEV).manual_seed(5)
    cache = ffa.new_cache(8, 16, 2, 64, dtype, None, device=DEV)
    table, start = torch.randperm(8, generator=gen, device=DEV).to(torch.int32)[None, :6].contiguous(), torch.tensor([37], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(1, 2, 37, 64, generator=gen, device=DEV).to(dtype) for _ in range(2))
    ffa.cache_write(cache, k, v, table, torch.zeros_like(start))
    return cache, table, start, *(torch.randn(1, h, 5, 64, generator=gen, device=DEV).to(dtype) for h in (4, 2, 2))


def test_negated_rotary_inputs():
    gen = torch.Generator(device=DEV).manual_seed(6)
    q, k = torch.randn(1, 4, 5, 64, generator=gen, device=DEV), torch.randn(1, 2, 5, 64, generator=gen, device=DEV)
    cos, sin = torch.randn(1, 5, 64, generator=gen, device=DEV), torch.randn(1, 5, 64, generator=gen, device=DEV)
    want = ffa.apply_rotary(q, k, cos, sin)
    for at in range(4):
        args = [q, k, cos, sin]
        args[at] = negated(args[at])
        for got, w in zip(ffa.apply_rotary(*args), want):
            assert not got.is_neg() and torch.equal(got, w)
    # as they come about: the imaginary part of a conjugate
    z = torch.complex(q, -q)
    assert z.conj().imag.is_neg()
    assert torch.equal(ffa.apply_rotary(z.conj().imag, k, cos, sin)[0], want[0])
    pos, inv = torch.arange(9, device=DEV)[None], torch.rand(8, generator=gen, device=DEV, dtype=torch.float64)
    for got, w in zip(ffa.rotary_tables(negated(pos), negated(inv)), ffa.rotary_tables(pos, inv)):
        assert torch.equal(got, w)


def test_negated_cache_inputs():
    cache, table, start, q, k, v = decoding_inputs()
    ffa.cache_write(cache, k, v, table, start)
    want, held = ffa.cache_attention(q, cache, table, start), [t.clone() for t in cache[:2]]
    assert torch.equal(ffa.cache_attention(negated(q), cache, table, start), want)
    assert torch.equal(ffa.cache_attention(q, cache, negated(table), negated(start)), want)
    ffa.cache_write(cache, torch.zeros_like(k), torch.zeros_like(v), table, start)
    ffa.cache_write(cache, negated(k), negated(v), negated(table), negated(start))
    assert all(torch.equal(t, h) for t, h in zip(cache, held))
    for got, w in zip(ffa.cache_read(cache, negated(table), negated(start), 5), ffa.cache_read(cache, table, start, 5)):
        assert torch.equal(got, w)
    ffa.cache_keep(cache, table, start, negated(torch.tensor([[1, 3]], dtype=torch.int32, device=DEV)))
    assert torch.equal(ffa.cache_read(cache, table, start, 2)[0], k[:, :, [1, 3]])


def test_zeros_without_memory():
    zero = lambda t: torch._efficientzerotensor(t.shape, dtype=t.dtype, device=DEV)
    cache, table, start, q, k, v = decoding_inputs()
    mask = torch.zeros(5, 5, dtype=torch.bool, device=DEV)
    ffa.cache_write(cache, k, v, table, start)
    assert torch.equal(ffa.cache_attention(q, cache, table, start, mask=zero(mask)), ffa.cache_attention(q, cache, table, start, mask=mask))
    assert torch.equal(ffa.cache_attention(zero(q), cache, table, start), ffa.cache_attention(torch.zeros_like(q), cache, table, start))
    ffa.cache_write(cache, zero(k), zero(v), table, start)
    assert not any(t.any() for t in ffa.cache_read(cache, table, start, 5))
    cos = torch.ones(1, 5, 64, device=DEV).bfloat16()
    for got, x in zip(ffa.apply_rotary(q, zero(k), cos, zero(cos)), (q, torch.zeros_like(k))):
        assert torch.equal(got, x)


# ---- infinities among earlier tokens' values
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 9, 64])
def test_an_infinite_value_of_an_earlier_token(dtype, n):
    """All new tokens see it: infinity in its channel, NaN where two of other signs meet, nothing elsewhere.  (Scores of deviation
    1/4: no weight is small beside another.)"""
    gen = torch.Generator(device=DEV).manual_seed(n)
    cache = ffa.new_cache(8, 32, 2, 64, dtype, None, device=DEV)
    table, start = torch.arange(8, dtype=torch.int32, device=DEV)[None], torch.tensor([150], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(1, 2, 150 + n, 64, generator=gen, device=DEV).to(dtype) for _ in range(2))
    k[:, :, [7, 140]] = 0                                                   # score 0: their weight is not small beside any other's
    v[:, :, 7, 3], v[:, :, 140, 9] = float("inf"), float("-inf")
    v[:, :, 7, 20], v[:, :, 140, 20] = float("inf"), float("-inf")
    ffa.cache_write(cache, k, v, table, torch.zeros_like(start))
    q = (torch.randn(1, 6, n, 64, generator=gen, device=DEV) * 0.25).to(dtype)
    got = ffa.cache_attention(q, cache, table, start)[0]
    assert (got[..., 3] == float("inf")).all() and (got[..., 9] == float("-inf")).all() and torch.isnan(got[..., 20]).all()
    rest = [i for i in range(64) if i not in (3, 9, 20)]
    assert torch.isfinite(got[..., rest]).all()
