"""-m gpu: the block operators under forward-mode differentiation and `torch.jit.trace`: served or refused by name, never wrong in
silence."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import orbitssm_b200 as ob

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _args(L=20):
    g = torch.Generator(device=DEV).manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    return rnd(2, L, 2, 8), rnd(2, L, 2, 8), rnd(2, L, 2, 16), torch.tensor([-0.1, -0.2], device=DEV), rnd(2, 2, 16, 8), rnd(5, 24), rnd(24)


def _dual(t):
    return fwd.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused_by_name(grad):
    q, k, v, ld, s, x, w = _args()
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        for i in range(4):
            a = [_dual(t) if j == i else t for j, t in enumerate((q, k, v, s))]
            with pytest.raises(RuntimeError, match="jvp"):
                ob.linear_attention(*a[:3], ld, a[3])
            with pytest.raises(ValueError, match="gradients are not served"):
                ob.linear_attention_step(*(t[:, 0] for t in a[:3]), ld, a[3])
        with pytest.raises(ValueError, match="constant of the layer"):
            ob.linear_attention(q, k, v, _dual(ld))
        with pytest.raises(ValueError, match="constant of the layer"):
            ob.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], _dual(ld), s)
        for i in range(5):
            a = [_dual(t) if j == i else t for j, t in enumerate((x, x, x, w, w))]
            with pytest.raises(RuntimeError, match="jvp"):
                ob.block_norm(a[0], a[1], gate=a[2], scale=a[3], pre_weight=a[4])
        # tensors that carry no tangent are served inside the level as outside of it
        y, new = ob.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s)
        z, m = ob.linear_attention(q[:, :1], k[:, :1], v[:, :1], ld, s, return_state=True)
        n = ob.block_norm(x, x, pre_weight=w)[1]
    assert torch.equal(new, m) and torch.equal(y, z[:, 0]) and torch.equal(n, ob.block_norm(x, x, pre_weight=w)[1])


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_a_trace_holds_the_operators_or_is_refused():
    q, k, v, ld, s, x, w = _args()

    def attention(q, k, v, s):
        return ob.linear_attention(q, k, v, ld, s, return_state=True)

    def norm(x, h):
        return ob.block_norm(x, h, gate=h, pre_weight=w)

    for fn, a in ((attention, (q, k, v, s)), (norm, (x, x * 2))):
        traced = torch.jit.trace(fn, a)
        b = tuple(t + 1.0 for t in a)
        for got, want in zip(traced(*b), fn(*b)):
            assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="linear_attention_step: cannot be recorded"):
        torch.jit.trace(lambda q, k, v, s: ob.linear_attention_step(q, k, v, ld, s), (q[:, 0], k[:, 0], v[:, 0], s))
    with pytest.raises(RuntimeError, match="pack_activation: cannot be recorded"):
        torch.jit.trace(lambda x: ob.unpack_activation(ob.pack_activation(x)), (x,))
    p = ob.pack_activation(x)
    with pytest.raises(RuntimeError, match="unpack_activation: cannot be recorded"):
        torch.jit.trace(lambda q: ob.unpack_activation(ob.PackedActivation(q, p.exponent, x.dtype)), (p.q,))


def test_without_the_host_call_module_the_results_are_the_same_bits(monkeypatch):
    from orbitssm_b200 import _lib
    q, k, v, ld, s, x, w = _args(200)

    def run():
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v, s, x, w)]
        y, new = ob.linear_attention(*leaves[:3], ld, leaves[3], return_state=True)
        r, n = ob.block_norm(leaves[4], leaves[4], gate=leaves[4], pre_weight=leaves[5])
        out = [y, new, r, n, *torch.autograd.grad((y.sum() + new.sum() + (r * n).sum()), leaves)]
        with torch.no_grad():
            return out + [*ob.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s), ob.unpack_activation(ob.pack_activation(x))]

    want = run()
    monkeypatch.setattr(_lib, "_host", _lib._PythonSide())
    assert all(torch.equal(a, b) for a, b in zip(run(), want, strict=True))


def test_a_new_state_written_over_an_operand_is_refused():
    q, k, v, ld, s, _, _ = _args(1)
    arena = torch.zeros(4096, device=DEV)
    state = arena[:s.numel()].view(s.shape)
    for i, (name, t) in enumerate((("q", q), ("k", k), ("v", v))):
        ops = [q[:, 0], k[:, 0], v[:, 0]]
        ops[i] = arena[s.numel() - 4:][:t.numel()].view(t[:, 0].shape)
        with pytest.raises(ValueError, match="out_state overlaps q, k, v or log_decay"):
            ob.linear_attention_step(*ops, ld, s, out_state=state)
        ops[i] = arena[s.numel():][:t.numel()].view(t[:, 0].shape)        # beside it: served
        _, new = ob.linear_attention_step(*ops, ld, s, out_state=state)
        assert new is state and bool(torch.isfinite(new).all())
    with pytest.raises(ValueError, match="out_state overlaps q, k, v or log_decay"):
        ob.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], arena[5:7], s, out_state=state)
