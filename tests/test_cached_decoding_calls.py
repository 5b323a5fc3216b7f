"""CPU: the cached-decoding calls under what PyTorch wraps around a call - forward-mode derivatives, lazily negated tensors, tracers.

Refusals stand before the check of the device.  Where a call would reach a kernel, the host module is replaced by the formula."""
import pytest
import torch
from torch.autograd import forward_ad

import framefusion_amd as ffa
from framefusion_amd import _lib


def cache_and_rows(store=None, dtype=torch.bfloat16):
    cache = ffa.new_cache(3, 16, 2, 64, dtype, store, device="cpu")
    table, start = torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    return cache, torch.randn(1, 2, 5, 64).to(dtype), torch.randn(1, 4, 5, 64).to(dtype), table, start


class Formula:
    """The half-layout rotation, in place of the host module."""

    def rotary(self, query, key, cos, sin, sections, interleaved, transpose):
        assert sections is None and not interleaved
        half = cos.shape[-1] // 2
        sign = -1.0 if transpose else 1.0
        return tuple(x.detach() * cos[:, None] + sign * torch.cat((-x.detach()[..., half:], x.detach()[..., :half]), -1) * sin[:, None] for x in (query, key))


@pytest.fixture
def formula(monkeypatch):
    monkeypatch.setattr(_lib, "host", lambda: Formula())


def rotary_inputs():
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(1, 4, 5, 8, generator=g), torch.randn(1, 2, 5, 8, generator=g)
    angle = torch.randn(1, 5, 4, generator=g).repeat(1, 1, 2)
    return q, k, angle.cos(), angle.sin()


# ---- forward-mode derivatives
def test_the_rotation_carries_tangents(formula):
    """The rotation is linear: its tangent is the rotation of the tangent (bit for bit: the same call)."""
    q, k, cos, sin = rotary_inputs()
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    want = ffa.apply_rotary(dq, dk, cos, sin)
    with forward_ad.dual_level():
        got = [forward_ad.unpack_dual(y) for y in ffa.apply_rotary(forward_ad.make_dual(q, dq), forward_ad.make_dual(k, dk), cos, sin)]
        for y, x, t in zip(got, ffa.apply_rotary(q, k, cos, sin), want):
            assert torch.equal(y.primal, x) and torch.equal(y.tangent, t)
        # one of the two has a tangent: the other's is nothing or zeros
        y, z = ffa.apply_rotary(forward_ad.make_dual(q, dq), k, cos, sin)
        assert torch.equal(forward_ad.unpack_dual(y).tangent, want[0])
        rest = forward_ad.unpack_dual(z).tangent
        assert rest is None or not rest.any()
        with torch.no_grad():                                                # (forward mode has a switch of its own)
            y, _ = ffa.apply_rotary(forward_ad.make_dual(q, dq), k, cos, sin)
            assert torch.equal(forward_ad.unpack_dual(y).tangent, want[0])
        # forward over backward: the tangent of the gradient R^T g is R^T of g's tangent
        x = q.clone().requires_grad_()
        g, dg = torch.randn_like(q), torch.randn_like(q)
        y, _ = ffa.apply_rotary(x, k, cos, sin)
        grad, = torch.autograd.grad(y, x, forward_ad.make_dual(g, dg), create_graph=True)
        assert torch.equal(forward_ad.unpack_dual(grad).tangent, ffa.apply_rotary(dg, k, cos, sin, transpose=True)[0])
        y, _ = ffa.apply_rotary(x, k, cos, sin)
        grad, = torch.autograd.grad(y, x, forward_ad.make_dual(g, dg))                # (the backward graph is not kept: its tangent is)
        assert torch.equal(forward_ad.unpack_dual(grad).tangent, ffa.apply_rotary(dg, k, cos, sin, transpose=True)[0])
        with pytest.raises(ffa.FrameFusionHipError, match="constants"):
            ffa.apply_rotary(forward_ad.make_dual(q, dq), k, forward_ad.make_dual(cos, cos), sin)


def test_what_has_no_gradient_refuses_tangents_and_caches_that_want_one():
    cache, x, q, table, start = cache_and_rows()
    accepted = torch.zeros(1, 1, dtype=torch.int32)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        tables = torch.zeros(1, 5, 64, dtype=torch.bfloat16)
        calls = [lambda: ffa.cache_write(cache, dual(x), x, table, start), lambda: ffa.cache_write(cache, x, dual(x), table, start),
                 lambda: ffa.cache_attention(dual(q), cache, table, start), lambda: ffa.cache_attention(q, cache._replace(keys=dual(cache.keys)), table, start),
                 lambda: ffa.cache_read(cache._replace(values=dual(cache.values)), table, start, 4), lambda: ffa.apply_rotary(q, x, dual(tables), tables),
                 lambda: ffa.rotary_tables(torch.zeros(1, 3, dtype=torch.int64), dual(torch.ones(4, dtype=torch.float64)))]
        for at, call in enumerate(calls):
            with torch.no_grad(), pytest.raises(ffa.FrameFusionHipError, match="gradient"):
                call()
                pytest.fail(f"call {at} was not refused")
    wants = cache._replace(keys=cache.keys.clone().requires_grad_())
    for call in (lambda: ffa.cache_write(wants, x, x, table, start), lambda: ffa.cache_read(wants, table, start, 4), lambda: ffa.cache_keep(wants, table, start, accepted),
                 lambda: ffa.cache_attention(q, wants, table, start)):
        with pytest.raises(ffa.FrameFusionHipError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(ffa.FrameFusionHipError, match="MI355X only"):
            call()


# ---- values that PyTorch keeps beside the memory
def test_a_cache_lies_in_memory():
    cache, x, q, table, start = cache_and_rows("fp8")
    for bad in (cache._replace(key_scales=torch._neg_view(cache.key_scales)), cache._replace(value_scales=torch._efficientzerotensor(cache.value_scales.shape, dtype=torch.uint8))):
        with pytest.raises(ffa.FrameFusionHipError, match="in memory"):
            ffa.cache_write(bad, x, x, table, start)
    cache, x, q, table, start = cache_and_rows()
    for bad in (cache._replace(keys=torch._neg_view(cache.keys)), cache._replace(values=torch._efficientzerotensor(cache.values.shape, dtype=torch.bfloat16))):
        for call in (lambda: ffa.cache_write(bad, x, x, table, start), lambda: ffa.cache_attention(q, bad, table, start), lambda: ffa.cache_read(bad, table, start, 2)):
            with pytest.raises(ffa.FrameFusionHipError, match="in memory"):
                call()


# ---- tracers
def calls_of_all_kinds():
    cache, x, q, table, start = cache_and_rows()
    cos = torch.zeros(1, 5, 64, dtype=torch.bfloat16)
    return [lambda a: ffa.apply_rotary(q + a, x, cos, cos), lambda a: ffa.rotary_tables(torch.zeros(1, 3, dtype=torch.int64), torch.ones(4, dtype=torch.float64) + a),
            lambda a: ffa.cache_attention(q + a, cache, table, start), lambda a: ffa.cache_write(cache, x + a, x, table, start),
            lambda a: ffa.cache_read(cache, table, start, 4), lambda a: ffa.cache_keep(cache, table, start, torch.zeros(1, 1, dtype=torch.int32))]


def test_a_tracer_is_refused():
    """It would record the outputs' allocation alone."""
    from torch.fx.experimental.proxy_tensor import make_fx
    zero = torch.zeros(())
    for call in calls_of_all_kinds():
        with pytest.raises(ffa.FrameFusionHipError, match="traced"):
            torch.jit.trace(call, (zero,), check_trace=False)
        with pytest.raises(ffa.FrameFusionHipError, match="traced"):
            make_fx(call)(zero)
    q, k, cos, sin = rotary_inputs()
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(ffa.FrameFusionHipError, match="traced"):
            make_fx(lambda q, k, cos, sin: ffa.apply_rotary(q, k, cos, sin), tracing_mode=mode)(q, k, cos, sin)


def test_a_mode_that_only_looks_on_is_none():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    for call in calls_of_all_kinds():
        with Watch(), pytest.raises(ffa.FrameFusionHipError, match="MI355X only"):
            call(torch.zeros(()))


def test_tensors_without_memory_are_refused():
    cache, x, q, table, start = cache_and_rows()
    meta = torch.ones(5, 5, dtype=torch.bool, device="meta")
    with pytest.raises(ffa.FrameFusionHipError, match="memory"):
        ffa.cache_attention(q, cache, table, start, mask=meta)
