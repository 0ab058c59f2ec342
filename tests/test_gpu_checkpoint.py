"""-m gpu: stacks whose block inputs wait in eight bits, beside what else a training program does with a block."""
import pytest
import torch

import orbitssm_b200 as ob
from conftest import load_golden
from orbitssm_b200 import ops
from orbitssm_b200.block_ops import checkpoint_block

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


class DropMixer(torch.nn.Module):
    """A mixer of plain modules that draws from the GPU's generator."""

    def __init__(self, d=64):
        super().__init__()
        self.lin = torch.nn.Linear(d, d)

    def forward(self, x):
        return torch.nn.functional.dropout(self.lin(x), 0.5, self.training)


@pytest.mark.parametrize("kw", [dict(), dict(residual_scale=1.0)])
def test_a_mixer_that_draws_random_numbers(kw):
    torch.manual_seed(4)
    block = ob.BlockStack.from_mixers([DropMixer()], 64, **kw).to(DEV).layers[0]
    x = torch.randn(4, 30, 64, device=DEV)
    seen = []
    block.mixer.register_forward_hook(lambda m, i, o: seen.append(o.detach().clone()))
    y = checkpoint_block(block, x)
    after = torch.cuda.get_rng_state()
    g, = torch.autograd.grad(y.sum(), block.mixer.lin.bias)
    assert torch.equal(torch.cuda.get_rng_state(), after)
    assert bool((seen[0] == 0).any()) and torch.equal(g, (2.0 * (seen[0] != 0)).sum((0, 1)))    # whole numbers: exact


def test_a_block_that_draws_is_not_captured():
    def stack(training):
        torch.manual_seed(4)
        return ob.BlockStack.from_mixers([DropMixer()], 64).to(DEV).set_checkpoint("int8").train(training)

    x = torch.randn(4, 30, 64, device=DEV)
    with pytest.raises(ob.CaptureError, match="draws random numbers"):
        ob.GraphedStep(stack(True), x, x)
    quiet = stack(False)                                                 # the same block, drawing nothing in this mode
    step = ob.GraphedStep(quiet, x, x)
    with torch.no_grad():
        assert torch.equal(step(x, x), quiet(x))
    fresh = stack(False)
    with torch.cuda.graph(torch.cuda.CUDAGraph()), pytest.raises(RuntimeError, match="before the capture"):
        fresh(x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_outputs_with_and_without_the_checkpoint(dtype):
    torch.manual_seed(6)
    x = torch.randn(2, 70, 64, device=DEV, dtype=dtype)
    plain = ob.BlockStack.from_mixers([mixer() for _ in range(3)], 64).to(DEV).to(dtype)
    want = plain(x).detach()
    assert torch.equal(plain.set_checkpoint("int8")(x).detach(), want)
    # a joining block: the final norm is taken from the stream before or after its rounding.  That moves every element by u at most,
    # relative to itself, so the root of the mean square by u as well, and either result is rounded once: 4 u, and terms of u^2
    joined = ob.BlockStack.from_mixers([mixer()], 64, post_norm=True, gate=True, residual_scale=0.5).to(DEV).to(dtype)
    want = joined(x).detach().double()
    got = joined.set_checkpoint("int8")(x).detach().double()
    u = torch.finfo(dtype).eps / 2
    # (float32: the sum of the 64 squares and the product with the weight add their own roundings, fewer than 64)
    assert bool(((got - want).abs() <= (4.1 * u + 64 * 2.0 ** -24) * want.abs()).all())


def test_the_two_runs_of_a_block_may_take_either_host_way():
    stack = stack_of(post_norm=True, gate=True, residual_scale=0.5)
    x = torch.randn(2, 40, 64, device=DEV)

    def grads(timed_first, timed_second):
        stack.zero_grad(set_to_none=True)
        try:
            ops.set_timing([] if timed_first else None)                  # a timed region takes the Python way
            y = stack(x)
            ops.set_timing([] if timed_second else None)
            y.square().sum().backward()
        finally:
            ops.set_timing(None)
        return [p.grad.clone() for p in stack.parameters()]

    want = grads(False, False)
    for a, b in ((True, False), (False, True), (True, True)):
        assert all(torch.equal(g, w) for g, w in zip(grads(a, b), want))


def _other_mixer(name):
    if name == "hybrid":
        return ob.HybridMambaSSM(ob.HybridMambaConfig(**load_golden("hm_small")["config"]))
    if name == "ssd":
        return ob.SSDMimoSSM(ob.mamba2_config(64, d_state=16, d_head=16))
    if name == "ssd tiles":
        return ob.SSDMimoSSM(ob.mamba2_config(128, d_state=128, d_head=64))
    return mixer(128)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [dict(), dict(post_norm=True, residual_scale=0.5)])
@pytest.mark.parametrize("name", ["ssd", "ssd tiles", "hybrid", "linear"])
def test_gradients_at_inputs_that_eight_bits_hold_are_the_blocks_own(name, kw, dtype):
    """Whole numbers up to 127 are restored as they were: gradients, hooks or not, have to be those of the block without a checkpoint."""
    torch.manual_seed(7)
    m = _other_mixer(name)
    stack = ob.BlockStack.from_mixers([m], m.d_model, **kw).to(DEV).to(dtype)
    x = torch.randint(-127, 128, (2, 150, m.d_model), device=DEV).to(dtype)
    dy = torch.randn(x.shape, device=DEV).to(dtype)

    def run(block):
        for p in stack.parameters():
            p.grad = None
        xx = x.clone().requires_grad_(True)
        block(xx).backward(dy)
        return [xx.grad, *[p.grad for p in stack.layers[0].parameters()]]

    got, want = run(lambda t: checkpoint_block(stack.layers[0], t)), run(stack.layers[0])
    assert all((a is None) == (b is None) and (a is None or torch.equal(a, b)) for a, b in zip(got, want, strict=True))
    ops.check_device_status()
