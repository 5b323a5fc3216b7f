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
