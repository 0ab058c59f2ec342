"""CPU: the autograd side of 8-bit activation checkpoints, with the two kernels replaced by copies, so that a checkpointed block has
to give what the block gives without one, bit for bit."""
import pytest
import torch
import torch.nn as nn

from orbitssm_b200 import block_ops


@pytest.fixture(autouse=True)
def copies(monkeypatch):
    monkeypatch.setattr(block_ops, "pack_activation",
                        lambda x: block_ops.PackedActivation(x.detach().clone(), x.new_zeros(1, dtype=torch.uint8), x.dtype))
    monkeypatch.setattr(block_ops, "unpack_activation", lambda p, dtype=None: p.q.clone())


def _block(seed=0):
    torch.manual_seed(seed)
    return nn.Sequential(nn.Linear(8, 8), nn.Tanh(), nn.Linear(8, 8)).double()


def _x(seed=1):
    return torch.randn(3, 8, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).requires_grad_(True)


def _grads(block, checkpointed, x):
    params = list(block.parameters())
    for t in (x, *params):
        t.grad = None
    y = block_ops.checkpoint_block(block, x) if checkpointed else block(x)
    (y * torch.arange(8.0, dtype=y.dtype)).sum().backward()
    return [y.detach(), x.grad, *[p.grad for p in params]]


def _same(block, x):
    return all(torch.equal(a, b) for a, b in zip(_grads(block, True, x), _grads(block, False, x), strict=True))


def test_gradients_are_the_blocks_own():
    assert _same(_block(), _x())


def test_hooks_of_parameters_run_once():
    block, x = _block(), _x()
    calls = []
    block[0].weight.register_hook(lambda g: calls.append(0) or 0.5 * g)
    block[2].bias.register_post_accumulate_grad_hook(lambda p: calls.append(1))
    assert _same(block, x) and sorted(calls) == [0, 0, 1, 1]            # once with the checkpoint, once without
    block[0].weight.register_hook(lambda g: None)
    g, = torch.autograd.grad(block_ops.checkpoint_block(block, x).sum(), block[0].weight)
    want, = torch.autograd.grad(block(x).sum(), block[0].weight)
    assert torch.equal(g, want)


def test_hooks_of_modules_inside_the_block_run_in_the_backward_pass_once():
    block, x = _block(), _x()
    calls = []
    block[1].register_full_backward_hook(lambda m, gi, go: calls.append(0))
    assert _same(block, x) and calls == [0, 0]


def test_a_parameter_that_the_block_reaches_by_another_way_keeps_its_gradient():
    block, x = _block(), _x()

    class Outer(nn.Module):
        def __init__(self):
            super().__init__()
            self.inner = block
            self.kept = [block[2].weight]                                # not looked up in the module at the time of the call

        def forward(self, x):
            return self.inner[1](x @ self.kept[0].t())

    assert _same_or_none(Outer(), x)


def _same_or_none(block, x):
    return all((a is None) == (b is None) and (a is None or torch.equal(a, b))
               for a, b in zip(_grads(block, True, x), _grads(block, False, x), strict=True))


def test_a_change_of_a_parameter_before_the_backward_pass_is_refused():
    block, x = _block(), _x()
    y = block_ops.checkpoint_block(block, x)
    with torch.no_grad():
        block[0].weight.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    frozen = _block()
    frozen[2].weight.requires_grad_(False)                               # the second run would read it as well
    y = block_ops.checkpoint_block(frozen, x)
    with torch.no_grad():
        frozen[2].weight.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_kept_graph_is_walked_twice_and_the_input_may_change():
    block, x = _block(), _x()
    want = _grads(block, False, x)[1]
    x2 = x.detach().clone().requires_grad_(True)
    h = x2 * 1.0
    y = (block_ops.checkpoint_block(block, h) * torch.arange(8.0, dtype=torch.float64)).sum()
    h.data.zero_()                                                       # what waits for the backward pass is the packed copy
    for _ in range(2):
        g, = torch.autograd.grad(y, x2, retain_graph=True)
        assert torch.equal(g, want)


def test_nothing_is_recorded_without_a_gradient():
    block, x = _block(), _x()
    with torch.no_grad():
        assert not block_ops.checkpoint_block(block, x).requires_grad
    for p in block.parameters():
        p.requires_grad_(False)
    assert not block_ops.checkpoint_block(block, x.detach()).requires_grad


class Drop(nn.Module):
    """A mixer's dropout, by the function: nothing in the module tells that it draws."""

    def __init__(self, p=0.5):
        super().__init__()
        self.lin, self.p = nn.Linear(8, 8).double(), p

    def forward(self, x):
        return nn.functional.dropout(self.lin(x), self.p, self.training)


def test_random_numbers_are_drawn_again_as_they_were():
    torch.manual_seed(5)
    block, x = Drop(), torch.randn(64, 8, dtype=torch.float64, requires_grad=True)
    y = block_ops.checkpoint_block(block, x)
    after = torch.get_rng_state()
    gb, gx = torch.autograd.grad(y.sum(), (block.lin.bias, x))
    assert torch.equal(torch.get_rng_state(), after)                     # the backward pass leaves the generator as it was
    kept = (y.detach() != 0).double()
    assert torch.equal(gb, (2.0 * kept).sum(0))
    assert torch.allclose(gx, (2.0 * kept) @ block.lin.weight.detach(), rtol=1e-14, atol=0)


def test_blocks_that_run_context_parallel_are_refused_whenever_they_were_made_so():
    import orbitssm_b200 as ob

    class Mix(nn.Module):
        def __init__(self):
            super().__init__()
            self.inner = nn.Linear(8, 8)

        def forward(self, x):
            raise AssertionError("the block ran")

    stack = ob.BlockStack.from_mixers([Mix(), Mix()], 8).set_checkpoint("int8")
    stack.layers[1].mixer._cp = object()                                 # what set_context_parallel leaves on a mixer
    with pytest.raises(ValueError, match="context-parallel"):
        stack(torch.zeros(2, 3, 8))
    stack.layers[1].mixer._cp, stack.layers[0].mixer.inner._cp = None, object()
    with pytest.raises(ValueError, match="context-parallel"):
        stack(torch.zeros(2, 3, 8))
    with pytest.raises(ValueError, match="context-parallel"):
        stack.set_checkpoint("int8")
    assert stack.set_checkpoint(None).checkpoint is None


def test_a_block_whose_second_run_takes_another_course_is_refused():
    class Fickle(nn.Module):
        def __init__(self):
            super().__init__()
            self.lin, self.calls = nn.Linear(8, 8).double(), 0

        def forward(self, x):
            self.calls += 1
            return torch.tanh(self.lin(x)) if self.calls == 1 else self.lin(x)

    y = block_ops.checkpoint_block(Fickle(), _x())
    with pytest.raises(RuntimeError, match="saved other tensors"):
        y.sum().backward()


def test_what_a_checkpointed_run_keeps_goes_with_its_graph():
    import gc
    import weakref
    block, x = _block(), _x()
    kept = []
    fetch = block_ops._Checkpoint.fetch
    gc.disable()                                                         # by reference counts alone
    try:
        block_ops._Checkpoint.fetch = lambda self, i: kept.append(weakref.ref(self)) or fetch(self, i)
        y = block_ops.checkpoint_block(block, x)
        y.sum().backward()
        assert kept and all(r() is None for r in kept)                   # (y is still there: its graph has given up what it saved)
    finally:
        block_ops._Checkpoint.fetch = fetch
        gc.enable()


def test_checkpoints_inside_a_checkpointed_block():
    from torch.utils.checkpoint import checkpoint

    class Outer(nn.Module):
        def __init__(self, how):
            super().__init__()
            self.a, self.b, self.how = _block(1), _block(2), how

        def forward(self, x):
            if self.how == "torch":
                return self.b(checkpoint(self.a, x, use_reentrant=False))
            return self.b(block_ops.checkpoint_block(self.a, x))

    for how in ("torch", "own"):
        assert _same(Outer(how), _x())


def test_a_step_of_two_blocks_with_a_shared_parameter_and_an_accumulated_gradient():
    a, x = _block(1), _x()
    want = None
    for checkpointed in (False, True):
        for p in a.parameters():
            p.grad = None
        for _ in range(2):                                               # gradients add up over two passes
            y = x
            for _ in range(2):                                           # the block twice in a row
                y = block_ops.checkpoint_block(a, y) if checkpointed else a(y)
            y.sum().backward()
        got = [p.grad.clone() for p in a.parameters()]
        want = got if want is None else want
    assert all(torch.equal(g, w) for g, w in zip(got, want))
