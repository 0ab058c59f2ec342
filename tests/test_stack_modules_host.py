"""CPU: a stack of joining blocks calls the modules that stand in it wherever they are not the plain ones whose arithmetic the join kernel
does itself.  The kernels are replaced by their formulas, so that every stack has to agree with its modules called one by one."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import orbitssm_b200 as ob
from orbitssm_b200 import model, ops

D = 8


class Mix(nn.Module):
    """A mixer of plain modules with the State contract's calls."""

    def __init__(self):
        super().__init__()
        self.lin = nn.Linear(D, D)

    def forward(self, x, state=None, return_state=False):
        y = torch.tanh(self.lin(x))
        return (y, state) if return_state else y

    def step(self, x_t, state):
        return self.forward(x_t), state

    def init_state(self, n, **kw):
        return None


def rms(x, w, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w


def formula(x, h, *, gate=None, scale=None, post_weight=None, pre_weight=None, eps=1e-5):
    u = h if post_weight is None else rms(h, post_weight, eps)
    m = u if gate is None else u * torch.sigmoid(gate)
    r = x + (m if scale is None else scale * m)
    return r, None if pre_weight is None else rms(r, pre_weight, eps)


class PlainProject:
    @staticmethod
    def apply(x, residual, pad, bias, off, *weights):
        return F.linear(x, torch.cat(weights))


class PlainGateNorm:
    @staticmethod
    def apply(y, z, w, eps, slot=None):
        return rms(y, w, eps)


@pytest.fixture(autouse=True)
def formulas(monkeypatch):
    monkeypatch.setattr(model, "block_norm", formula)
    monkeypatch.setattr(ops, "ProjectFn", PlainProject)
    monkeypatch.setattr(ops, "GateNormFn", PlainGateNorm)


def make(**kw):
    torch.manual_seed(0)
    kw = dict(post_norm=True, gate=True, residual_scale=0.5) | kw
    stack = ob.BlockStack.from_mixers([Mix() for _ in range(3)], D, **kw).double()
    with torch.no_grad():
        for p in stack.parameters():
            p.add_(0.2 * torch.randn_like(p))
    return stack


def one_by_one(stack, x):
    for b in stack.layers:
        if type(b).forward is not ob.ResidualBlock.forward:
            x = b(x)
            continue
        n = b.norm(x)
        h = b.mixer(n)
        if b.post_norm is not None:
            h = b.post_norm(h)
        if b.gate_proj is not None:
            h = h * torch.sigmoid(b.gate_proj(n))
        x = x + (h if b.scale is None else b.scale * h)
    return stack.norm_f(x)


def check(stack):
    x = torch.randn(2, 5, D, dtype=torch.float64)
    want = one_by_one(stack, x)
    assert torch.allclose(stack(x), want, rtol=1e-12, atol=1e-12)
    assert torch.allclose(stack(x, return_state=True)[0], want, rtol=1e-12, atol=1e-12)
    assert torch.allclose(stack.step(x[:, 0], [None] * 3)[0], want[:, 0], rtol=1e-12, atol=1e-12)


class OtherNorm(model.RMSNorm):
    def forward(self, x):
        return 2.0 * super().forward(x)


class Wrapped(nn.Module):
    """A projection under another one's name, as adapters are put in; it still shows the weight of the one inside."""

    def __init__(self, inner):
        super().__init__()
        self.inner, self.weight = inner, inner.weight

    def forward(self, x):
        return 0.5 * self.inner(x)


def swap_final(s): s.norm_f = nn.LayerNorm(D).double()
def swap_final_subclass(s): s.norm_f = OtherNorm(D).double()
def swap_next(s): s.layers[1].norm = nn.LayerNorm(D).double()
def swap_post(s): s.layers[1].post_norm = nn.LayerNorm(D).double()
def swap_post_subclass(s): s.layers[1].post_norm = OtherNorm(D).double()
def wrap_gate(s): s.layers[0].gate_proj = Wrapped(s.layers[0].gate_proj)
def bias_gate(s): s.layers[0].gate_proj = nn.Linear(D, D).double()
def scaled_gate(s): nn.utils.parametrizations.weight_norm(s.layers[0].gate_proj)
def own_forward(s): s.layers[2].norm.forward = lambda x: 3.0 * x
def other_eps(s): s.layers[1].norm.eps = 0.5
def final_eps(s): s.norm_f.eps = 0.5


CHANGES = [lambda s: None, swap_final, swap_final_subclass, swap_next, swap_post, swap_post_subclass, wrap_gate, bias_gate, scaled_gate,
           own_forward, other_eps, final_eps]


@pytest.mark.parametrize("change", CHANGES, ids=lambda f: f.__name__.strip("<>"))
@pytest.mark.parametrize("kw", [dict(), dict(post_norm=False), dict(gate=False, residual_scale=None)], ids=("all", "no_post", "post"))
def test_replaced_and_wrapped_modules_are_called(change, kw):
    if "post" in change.__name__ and not kw.get("post_norm", True) or "gate" in change.__name__ and not kw.get("gate", True):
        pytest.skip("the block has no such module")
    stack = make(**kw)
    change(stack)
    check(stack)


@pytest.mark.parametrize("name", ["norm", "post_norm", "gate_proj", "mixer"])
def test_hooks_of_a_blocks_modules_are_called(name):
    for make_hook in (lambda m: m.register_forward_hook(lambda m, i, o: 2.0 * o), lambda m: m.register_forward_pre_hook(lambda m, i: (i[0] + 1.0,))):
        stack = make()
        make_hook(getattr(stack.layers[1], name))
        check(stack) if name != "mixer" else stack(torch.zeros(1, 2, D, dtype=torch.float64))


def test_a_hook_of_every_module_is_called():
    stack, seen = make(), []
    handle = nn.modules.module.register_module_forward_hook(lambda m, i, o: seen.append(m))
    try:
        stack(torch.zeros(1, 2, D, dtype=torch.float64))
    finally:
        handle.remove()
    for b in stack.layers:
        assert all(any(m is s for s in seen) for m in (b, b.norm, b.post_norm, b.gate_proj, b.mixer))
    assert any(s is stack.norm_f for s in seen)


def test_a_block_of_its_own_forward_is_called():
    class Doubled(ob.ResidualBlock):
        def forward(self, x, state=None, return_state=False):
            y = 2.0 * x
            return (y, state) if return_state else y

        def step(self, x_t, state=None):
            return 2.0 * x_t, state

    stack = make()
    stack.layers[1] = Doubled(Mix(), D, post_norm=True).double()
    check(stack)


def test_a_stack_pickled_before_blocks_could_join_still_runs():
    stack = make(post_norm=False, gate=False, residual_scale=None)
    for b in stack.layers:
        del b.__dict__["joins"]
        for name in ("post_norm", "gate_proj", "scale"):                  # attributes that such a block does not have
            b.__dict__.pop(name, None), b._modules.pop(name, None), b._parameters.pop(name, None)
    del stack.__dict__["checkpoint"]
    x = torch.randn(2, 5, D, dtype=torch.float64)
    want = x
    for b in stack.layers:
        want = want + b.mixer(b.norm(want))
    want = stack.norm_f(want)
    assert torch.equal(stack(x), want) and torch.equal(stack(x, return_state=True)[0], want)
    assert torch.allclose(stack.step(x[:, 0], [None] * 3)[0], want[:, 0], rtol=1e-12, atol=1e-12)
