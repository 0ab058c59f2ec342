"""-m gpu: the `LinearAttention` mixer, blocks whose norms, gate and residual scale are one kernel, and stacks that keep their
blocks' inputs in eight bits: as a user runs them, together, against plain float64 modules.

Float32 tolerances: a result is a chain of products over at most 256 terms each (u = 2^-24), through two blocks of about eight
such steps whose conditioning the norms keep near one: 16 * 256 * u < 2.5e-4 of the result's norm."""
import pytest
import torch
import torch.nn.functional as F

import orbitssm_b200 as ob
from orbitssm_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = 2.5e-4


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def mixer(d=64, heads=2, **kw):
    return ob.LinearAttention(ob.LinearAttentionConfig(d, heads, span_min=4.0, span_max=64.0, **kw))


def ref_mixer(m, prm, x, state=None):
    """The layer in float64 from its parameters `prm` (name -> tensor)."""
    B, L, _ = x.shape
    H, Dk, Dv = m.H, m.Dk, m.Dv
    q, k, v, z = (F.linear(x, prm[n + "_proj.weight"]) for n in ("q", "k", "v", "gate"))
    q, k, v = q.view(B, L, H, Dk), k.view(B, L, H, Dk), v.view(B, L, H, Dv)
    a = torch.exp(m.log_decay.double().to(x.device))[:, None, None]
    S = x.new_zeros(B, H, Dv, Dk) if state is None else state
    ys = []
    for t in range(L):
        S = a * S + v[:, t, :, :, None] * k[:, t, :, None, :]
        ys.append(torch.einsum("bhvk,bhk->bhv", S, q[:, t]) * Dk ** -0.5)
    y = torch.stack(ys, 1).flatten(2) * F.silu(z)
    if m.config.out_norm:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + m.config.norm_eps) * prm["norm.weight"]
    return F.linear(y, prm["out_proj.weight"]), S


def ref_block(b, prm, x):
    rms = lambda t, w, eps: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps) * w  # noqa: E731
    n = rms(x, prm["norm.weight"], b.norm.eps)
    h, _ = ref_mixer(b.mixer, {k[6:]: v for k, v in prm.items() if k.startswith("mixer.")}, n)
    if b.post_norm is not None:
        h = rms(h, prm["post_norm.weight"], b.post_norm.eps)
    if b.gate_proj is not None:
        h = h * torch.sigmoid(F.linear(n, prm["gate_proj.weight"]))
    return x + (h if b.scale is None else prm["scale"] * h)


def ref_stack(stack, prm, x):
    for i, b in enumerate(stack.layers):
        x = ref_block(b, {k[len(f"layers.{i}."):]: v for k, v in prm.items() if k.startswith(f"layers.{i}.")}, x)
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + stack.norm_f.eps) * prm["norm_f.weight"]


def params64(mod):
    return {n: p.detach().double().requires_grad_(True) for n, p in mod.named_parameters()}


def jitter(mod, seed=0):
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for p in mod.parameters():
            if p.dim() == 1:
                p.add_(0.2 * torch.randn(p.shape, generator=g).to(p.device))
    return mod


@pytest.mark.parametrize("kw", [dict(), dict(d_key=24, d_value=40), dict(out_norm=False)])
def test_layer_and_its_continuation(kw):
    torch.manual_seed(0)
    m = jitter(mixer(**kw).to(DEV))
    x, dy = torch.randn(2, 150, 64, device=DEV), torch.randn(2, 150, 64, device=DEV)
    s0 = m.init_state(2, device=DEV, h_init=torch.randn(2, *m.hidden_state_shape(), device=DEV))
    for c in s0.values():
        c.requires_grad_(True)
    xx = x.clone().requires_grad_(True)
    y, st = m(xx, state=s0, return_state=True)
    ds = torch.randn_like(st["hidden_state"])
    ((y * dy).sum() + (st["hidden_state"] * ds).sum()).backward()
    prm, xr, sr = params64(m), x.double().requires_grad_(True), s0["hidden_state"].detach().double().requires_grad_(True)
    yr, Sr = ref_mixer(m, prm, xr, sr)
    ((yr * dy.double()).sum() + (Sr * ds.double()).sum()).backward()
    assert rel(y, yr) < TOL and rel(st["hidden_state"], Sr) < TOL
    assert rel(xx.grad, xr.grad) < TOL and rel(s0["hidden_state"].grad, sr.grad) < TOL
    for n, p in m.named_parameters():
        assert rel(p.grad, prm[n].grad) < TOL, n
    with torch.no_grad():                                # in two halves, and token by token
        a, s = m(x[:, :70], state={k: v.detach() for k, v in s0.items()}, return_state=True)
        b, s = m(x[:, 70:140], state=s, return_state=True)
        steps = []
        for t in range(140, 150):
            o, s = m.step(x[:, t], s)
            steps.append(o)
        whole = torch.cat([a, b, torch.stack(steps, 1)], 1)
    assert rel(whole, y) < TOL and rel(s["hidden_state"], st["hidden_state"]) < TOL


def test_layer_gradients_land_in_the_projection_gradient():
    """bfloat16 at a tensor-core geometry: the operator writes into strided column ranges and gives what separate tensors give."""
    torch.manual_seed(1)
    m = mixer(128, 2).to(DEV).to(torch.bfloat16)
    x = torch.randn(2, 300, 128, device=DEV, dtype=torch.bfloat16)
    dy = torch.randn_like(x)

    def run(break_slots):
        m.zero_grad()
        xx = x.clone().requires_grad_(True)
        if break_slots:
            old = ops.GradArena.view
            ops.GradArena.view = lambda self, i, like: None
        try:
            m(xx).backward(dy)
        finally:
            if break_slots:
                ops.GradArena.view = old
        return [xx.grad] + [p.grad.clone() for p in m.parameters()]

    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)
    ops.check_device_status()


BLOCKS = [dict(post_norm=True), dict(gate=True), dict(residual_scale=0.3), dict(post_norm=True, gate=True, residual_scale=0.7)]


@pytest.mark.parametrize("kw", BLOCKS)
def test_stack_of_joined_blocks(kw):
    torch.manual_seed(2)
    stack = jitter(ob.BlockStack.from_mixers([mixer() for _ in range(2)], 64, **kw)).to(DEV)
    x, dy = torch.randn(2, 90, 64, device=DEV), torch.randn(2, 90, 64, device=DEV)
    xx = x.clone().requires_grad_(True)
    y = stack(xx)
    y.backward(dy)
    prm, xr = params64(stack), x.double().requires_grad_(True)
    yr = ref_stack(stack, prm, xr)
    yr.backward(dy.double())
    assert rel(y, yr) < TOL and rel(xx.grad, xr.grad) < TOL
    for n, p in stack.named_parameters():
        assert rel(p.grad, prm[n].grad) < TOL, n
    with torch.no_grad():
        ys, st = stack(x[:, :60], return_state=True)
        out = [ys]
        for t in range(60, 90):
            o, st = stack.step(x[:, t], st)
            out.append(o[:, None])
    assert rel(torch.cat(out, 1), y) < TOL
    one = stack.layers[0]                                # a block by itself gives what it gives in the stack
    with torch.no_grad():
        want = ref_block(one, {k[9:]: v for k, v in prm.items() if k.startswith("layers.0.")}, x.double())
        assert rel(one(x), want) < TOL


def test_joined_blocks_beside_plain_ones_and_other_mixers():
    torch.manual_seed(3)
    ssd = ob.SSDMimoSSM(ob.mamba2_config(64, d_state=16, d_head=16))
    blocks = [ob.ResidualBlock(mixer(), 64, post_norm=True), ob.ResidualBlock(mixer(), 64), ob.ResidualBlock(ssd, 64, gate=True, residual_scale=0.5)]
    stack = ob.BlockStack(blocks, 64).to(DEV)
    x = torch.randn(2, 50, 64, device=DEV)
    with torch.no_grad():
        y = x
        for b in blocks:
            y = b(y)
        want = stack.norm_f(y)
        assert rel(stack(x), want) < TOL
        got, _ = stack(x, return_state=True)
        assert rel(got, want) < TOL


def test_hooks_of_joined_blocks_and_norms_are_called():
    torch.manual_seed(3)
    stack = ob.BlockStack.from_mixers([mixer() for _ in range(3)], 64, post_norm=True, gate=True, residual_scale=0.5).to("cuda")
    x = torch.randn(2, 40, 64, device="cuda")
    with torch.no_grad():
        want = stack(x)
        seen = []
        handles = [m.register_forward_hook(lambda m, i, o, n=n: seen.append(n)) for n, m in
                   (("block 1", stack.layers[1]), ("norm 2", stack.layers[2].norm), ("final", stack.norm_f))]
        got = stack(x)
        assert seen == ["block 1", "norm 2", "final"]
        # norms of the rounded stream instead of the unrounded one: three roundings of float32 of a stream that three blocks pass
        assert rel(got, want) < 64 * 2.0 ** -24
        y, state = stack(x, return_state=True)
        assert rel(y, want) < 64 * 2.0 ** -24 and seen == ["block 1", "norm 2", "final"] * 2
        stack.step(x[:, 0], state)
        for h in handles:
            h.remove()
        assert torch.equal(stack(x), want)


def test_autocast_keeps_a_float32_stream():
    torch.manual_seed(4)
    stack = ob.BlockStack.from_mixers([mixer(128, 2) for _ in range(2)], 128, post_norm=True, gate=True, residual_scale=0.5).to(DEV)
    x = torch.randn(2, 200, 128, device=DEV)
    want = stack(x)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = stack(x)
    # activations, weights and each mixer's output are rounded to bfloat16 (2^-8) about ten times a block
    assert y.dtype == torch.float32 and rel(y, want) < 20 * 2.0 ** -8


@pytest.mark.parametrize("kw", [dict(), dict(post_norm=True, gate=True, residual_scale=0.7)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_checkpointed_stack(kw, dtype):
    """Outputs do not change; the gradients are those of the blocks run at their restored inputs."""
    torch.manual_seed(5)
    stack = jitter(ob.BlockStack.from_mixers([mixer(128, 2) for _ in range(3)], 128, **kw)).to(DEV).to(dtype)
    x, dy = torch.randn(2, 140, 128, device=DEV, dtype=dtype), torch.randn(2, 140, 128, device=DEV, dtype=dtype)
    with torch.no_grad():
        ins = [x]
        for b in stack.layers:
            ins.append(b(ins[-1]))
        plain = stack.norm_f(ins[-1])
    stack.set_checkpoint("int8")
    xx = x.clone().requires_grad_(True)
    y = stack(xx)
    assert torch.equal(y, plain)
    y.backward(dy)
    last = ins[-1].clone().requires_grad_(True)
    g, = torch.autograd.grad(stack.norm_f(last), last, dy)
    for b, i in zip(reversed(stack.layers), reversed(range(len(stack.layers)))):
        xi = ob.unpack_activation(ob.pack_activation(ins[i])).requires_grad_(True)
        ps = list(b.parameters())
        gx, *gp = torch.autograd.grad(b(xi), [xi] + ps, g)
        for p, want in zip(ps, gp):
            assert torch.equal(p.grad, want)
        g = gx
    assert torch.equal(xx.grad, g)
    with torch.no_grad():
        assert rel(stack(x), plain) < (TOL if dtype == torch.float32 else 2.0 ** -6)


def test_checkpoint_with_frozen_parts_and_changed_parameters():
    torch.manual_seed(6)
    stack = ob.BlockStack.from_mixers([mixer() for _ in range(2)], 64).to(DEV).set_checkpoint("int8")
    for p in stack.layers[0].parameters():
        p.requires_grad_(False)
    stack.layers[1].mixer.q_proj.weight.requires_grad_(False)
    x = torch.randn(1, 40, 64, device=DEV)
    stack(x).sum().backward()                            # nothing before the second block wants a gradient
    assert stack.layers[0].mixer.out_proj.weight.grad is None and stack.layers[1].mixer.q_proj.weight.grad is None
    assert stack.layers[1].mixer.k_proj.weight.grad is not None
    y = stack(x)
    with torch.no_grad():
        stack.layers[1].mixer.k_proj.weight.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = stack(x.requires_grad_(True))
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second-order"):
        g.sum().backward()


def test_checkpoint_keeps_less():
    torch.manual_seed(7)
    stack = ob.BlockStack.from_mixers([mixer(256, 2) for _ in range(4)], 256).to(DEV)
    x = torch.randn(4, 2048, 256, device=DEV, requires_grad=True)

    def held(mode):
        stack.set_checkpoint(mode)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = stack(x)
        torch.cuda.synchronize()
        n = torch.cuda.memory_allocated() - before
        y.sum().backward()
        stack.zero_grad(set_to_none=True)
        x.grad = None
        return n

    n = x.numel()
    whole, packed = held(None), held("int8")
    # three float32 tensors at least for the norm (input, output of the stack, its rstd) beside 33/32 byte an element and block
    assert packed < 4 * n * 33 / 32 + 2 * 4 * n + (1 << 20) and packed < whole / 4


def test_captured_training_and_decode_steps():
    torch.manual_seed(8)
    stack = ob.BlockStack.from_mixers([mixer(128, 2) for _ in range(2)], 128, post_norm=True, gate=True, residual_scale=0.5)
    stack = stack.to(DEV).to(torch.bfloat16).set_checkpoint("int8")
    x = torch.randn(2, 260, 128, device=DEV, dtype=torch.bfloat16)
    dy = torch.randn_like(x)
    step = ob.GraphedStep(stack, x, dy)
    for seed in (1, 2):
        g = torch.Generator(device=DEV).manual_seed(seed)
        x = torch.randn(x.shape, generator=g, device=DEV).to(x.dtype)
        dy = torch.randn(x.shape, generator=g, device=DEV).to(x.dtype)
        y = step(x, dy).clone()
        got = [step.x_grad.clone()] + [p.grad.clone() for p in stack.parameters()]
        for p in stack.parameters():
            p.grad = None
        xx = x.clone().requires_grad_(True)
        yy = stack(xx)
        yy.backward(dy)
        assert torch.equal(y, yy)
        for a, b in zip(got, [xx.grad] + [p.grad for p in stack.parameters()]):
            assert torch.equal(a, b)
        del yy
    dec = ob.GraphedDecode(stack, 3)
    st = stack.init_state(3, device=DEV)
    for _ in range(4):
        x_t = torch.randn(3, 128, device=DEV, dtype=torch.bfloat16)
        with torch.no_grad():
            want, st = stack.step(x_t, st)
        assert torch.equal(dec(x_t), want)
    for a, b in zip(dec.state, st):
        assert torch.equal(a["hidden_state"], b["hidden_state"])
    ops.check_device_status()


def test_operators_on_another_stream_and_two_graphs_at_once():
    g = torch.Generator(device=DEV).manual_seed(9)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    q, k, v = (rnd(1, 3000, 2, 64).to(torch.bfloat16) for _ in range(3))       # long enough for a split sequence
    ld, s0 = torch.tensor([-0.01, -0.2], device=DEV), rnd(1, 2, 64, 64)
    x = rnd(500, 256)
    w = rnd(256)

    def run():
        y, s = ob.linear_attention(q, k, v, ld, s0, return_state=True)
        r, n = ob.block_norm(x, x, gate=x, scale=w, post_weight=w, pre_weight=w)
        return y, s, r, n, ob.unpack_activation(ob.pack_activation(x))

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = run()
        graphs.append((gr, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for (gr, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
