"""-m gpu: stacks whose block inputs wait in eight bits, beside what else a training program does with a block."""
import pytest
import torch

import orbitssm_b200 as ob
from orbitssm_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def mixer(d=64, heads=2):
    return ob.LinearAttention(ob.LinearAttentionConfig(d, heads, span_min=4.0, span_max=64.0))


def stack_of(n=2, dtype=torch.float32, **kw):
    torch.manual_seed(3)
    return ob.BlockStack.from_mixers([mixer() for _ in range(n)], 64, **kw).to(DEV).to(dtype).set_checkpoint("int8")


@pytest.mark.parametrize("kw", [dict(), dict(post_norm=True, gate=True, residual_scale=0.5)])
def test_a_hook_of_a_parameter_runs_once(kw):
    stack = stack_of(**kw)
    x = torch.randn(2, 40, 64, device=DEV)

    def grads():
        stack.zero_grad(set_to_none=True)
        stack(x).square().sum().backward()
        return [p.grad.clone() for p in stack.parameters()]

    want, calls = grads(), []
    for p in stack.parameters():
        p.register_hook(lambda g: calls.append(0) or 0.5 * g)
    got = grads()
    assert len(calls) == len(want) and all(torch.equal(a, 0.5 * b) for a, b in zip(got, want))
    ops.check_device_status()
