"""-m gpu: block operators on tensors of more than 2^31 elements: the last rows are what a call on them alone gives."""
import pytest
import torch

import orbitssm_b200 as ob
from orbitssm_b200 import ops

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


@pytest.fixture(autouse=True)
def _leave_no_cache():
    yield
    torch.cuda.empty_cache()


def _fill(*shape, dtype=BF, seed=0):
    """Random values, a block of 2^24 repeated (quick to make), the last one anew."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = torch.empty(shape, device=DEV, dtype=dtype)
    flat, n = t.view(-1), 1 << 24
    block = torch.randn(n, generator=g, device=DEV).to(dtype)
    for a in range(0, flat.numel(), n):
        m = min(n, flat.numel() - a)
        flat[a:a + m] = block[:m]
    flat[-n:] = torch.randn(n, generator=g, device=DEV).to(dtype)
    return t


@pytest.mark.parametrize("D", [1024, 1000])
def test_pack_past_31_bits(D):
    x = _fill((1 << 31) // D + 77, D)
    assert x.numel() > 1 << 31
    p = ob.pack_activation(x)
    last = ob.pack_activation(x[-100:])
    assert torch.equal(p.q[-100:], last.q) and torch.equal(p.exponent[-100:], last.exponent)
    y = ob.unpack_activation(p)
    assert torch.equal(y[-100:], ob.unpack_activation(last)) and torch.equal(y[:100], ob.unpack_activation(ob.pack_activation(x[:100])))


@pytest.mark.parametrize("D", [1024, 1001])
def test_block_norm_past_31_bits(D):
    x = _fill((1 << 31) // D + 77, D)
    w = torch.linspace(0.5, 1.5, D, device=DEV)
    with torch.no_grad():
        r, n = ob.block_norm(x, x, gate=x, scale=w, post_weight=w, pre_weight=w)
        for rows in (slice(0, 50), slice(-50, None)):
            a, b = ob.block_norm(x[rows], x[rows], gate=x[rows], scale=w, post_weight=w, pre_weight=w)
            assert torch.equal(r[rows], a) and torch.equal(n[rows], b)
    del r, n
    t = x.requires_grad_(True)
    r, n = ob.block_norm(t, t.detach(), pre_weight=w)
    g, = torch.autograd.grad((r, n), t, (x.detach(), x.detach()))
    z = x.detach()[-50:].clone().requires_grad_(True)
    r, n = ob.block_norm(z, z.detach(), pre_weight=w)
    h, = torch.autograd.grad((r, n), z, (z.detach(), z.detach()))
    assert torch.equal(g[-50:], h)


@pytest.mark.parametrize("widths", [(128, 128), (100, 100)])
def test_linear_attention_past_31_bits(widths):
    Dk, Dv = widths
    H = 16
    L = (1 << 31) // (H * Dk) + 333
    q = _fill(1, L, H, Dk)
    ld = torch.full((H,), -2.0, device=DEV)              # after 300 tokens nothing of what was before is left
    with torch.no_grad():
        y, s = ob.linear_attention(q, q, q, ld, return_state=True)
        tail = q[:, -500:]
        z, u = ob.linear_attention(tail, tail, tail, ld, return_state=True)
    # the chunks of the two calls begin at other tokens: two results, each within the roundings of its operands and its output
    big, m = ob.linear_attention(tail.abs().float(), tail.abs().float(), tail.abs().float(), ld, return_state=True)
    assert bool(((y[:, -100:].double() - z[:, -100:].double()).abs() <= 4 * 2.0 ** -8 * big[:, -100:].double()).all())
    assert bool(((s.double() - u.double()).abs() <= 1000 * 2.0 ** -24 * m.double()).all())
    ops.check_device_status()


def test_step_past_31_bits():
    B, H, D = 8200, 16, 128
    s = _fill(B, H, D, D, dtype=torch.float32)
    assert s.numel() > 1 << 31
    q = _fill(B, H, D)
    ld = torch.linspace(-1.0, -0.1, H, device=DEV)
    y0, s0 = ob.linear_attention_step(q[-3:], q[-3:], q[-3:], ld, s[-3:])
    y, new = ob.linear_attention_step(q, q, q, ld, s, out_state=s)
    assert new is s and torch.equal(y[-3:], y0) and torch.equal(s[-3:], s0)
