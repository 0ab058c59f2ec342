"""-m gpu: replaced and wrapped modules in a stack of joining blocks, on the kernels."""
import pytest
import torch

import orbitssm_b200 as ob

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Half(torch.nn.Module):
    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x):
        return 0.5 * self.inner(x)


@pytest.mark.parametrize("amp", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_stack_of_other_norms_and_gates(dtype, amp):
    torch.manual_seed(0)
    mix = lambda: ob.LinearAttention(ob.LinearAttentionConfig(64, 2, span_min=4.0, span_max=64.0))  # noqa: E731
    stack = ob.BlockStack.from_mixers([mix() for _ in range(2)], 64, post_norm=True, gate=True, residual_scale=0.5)
    stack.norm_f = torch.nn.LayerNorm(64)
    stack.layers[1].norm = torch.nn.LayerNorm(64)
    stack.layers[0].post_norm = torch.nn.LayerNorm(64)
    stack.layers[1].gate_proj = Half(stack.layers[1].gate_proj)
    stack = stack.to(DEV).to(dtype)
    x = torch.randn(2, 30, 64, device=DEV, dtype=dtype)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=amp):
        y = stack(x)
        r = x
        for b in stack.layers:
            n = b.norm(r)
            r = r + b.scale * b.post_norm(b.mixer(n)) * torch.sigmoid(b.gate_proj(n))
        want = stack.norm_f(r)
    half = dtype == torch.bfloat16 or amp
    # the same products; between them two blocks of at most 16 roundings of the activations' type each
    assert float((y.double() - want.double()).detach().norm() / want.double().norm().detach()) < 32 * (2.0 ** -8 if half else 2.0 ** -24) * 4
    y.float().square().sum().backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in stack.parameters())
