"""-m gpu: what the documentation of the 8-bit activations states of their error, and what packing a restored activation gives."""
import pytest
import torch

import orbitssm_b200 as ob

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _groups(dtype):
    """Rows of 32 whose largest element runs over every exponent, at the mantissas where the step changes."""
    g = torch.Generator().manual_seed(0)
    tops = torch.tensor([1.0, 1.25, 1.9765625, 1.984375, 1.9921875 - 2.0 ** -20, 1.9921875, 1.99609375], dtype=torch.float64)
    e = torch.arange(-149, 128, dtype=torch.float64)
    top = (tops[:, None] * torch.exp2(e)).reshape(-1, 1)
    x = (2.0 * torch.rand(top.shape[0], 32, generator=g, dtype=torch.float64) - 1.0) * top
    x[:, 5:6] = top
    x[:, 6] = top[:, 0] / 127.5                                              # half a step where the step is largest against the top
    return x.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_error_is_within_what_is_stated(dtype):
    x = _groups(dtype)
    p = ob.pack_activation(x)
    y = ob.unpack_activation(p)
    top = x.double().abs().amax(-1, keepdim=True)
    at_end = p.exponent.view(-1, 1) == 249                                   # the step 2^122
    lim = torch.where(at_end, 2.0 ** 122, (top / 127.5).clamp(min=2.0 ** -127))
    err = (y.double() - x.double()).abs()
    assert bool((err <= lim).all()) and bool(torch.isfinite(y).all())
    normal = ~at_end & (p.exponent.view(-1, 1) > 1)
    # 1/128 of the largest is not enough: 127.5 takes steps of 2
    assert bool(((err > top / 128) & normal).any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_packing_again_gives_the_same_bytes_below_the_largest_step(dtype):
    p = ob.pack_activation(_groups(dtype))
    y = ob.unpack_activation(p)
    again = ob.pack_activation(y)
    assert torch.equal(ob.unpack_activation(again), y)
    below = p.exponent.view(-1) < 249
    assert torch.equal(again.q[below], p.q[below]) and torch.equal(again.exponent[below], p.exponent[below]) and not bool(below.all())
