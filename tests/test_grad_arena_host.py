"""CPU: the gradient buffer of a fused projection belongs to the gradient once it is handed on."""
import torch

from orbitssm_b200 import ops


class Writes(torch.autograd.Function):
    """A consumer of a column range whose backward pass writes its input's gradient in place, as the kernels do."""

    @staticmethod
    def forward(ctx, x, arena, index):
        ctx.arena, ctx.index = arena, index
        return 2.0 * x

    @staticmethod
    def backward(ctx, dy):
        view = ctx.arena.view(ctx.index, dy)
        view.copy_(2.0 * dy)
        return view, None, None


def test_a_kept_graph_holds_no_gradient_buffer_and_gives_new_ones():
    proj = torch.randn(2, 3, 8, requires_grad=True)
    arena = ops.GradArena()
    a, b = ops.SplitColumnsFn.apply(proj, arena, 4, 4)
    y = (Writes.apply(a, arena, 0) * torch.arange(4.0)).sum() + (3.0 * b).sum()
    want = torch.cat([2.0 * torch.arange(4.0).expand(2, 3, 4), torch.full((2, 3, 4), 3.0)], -1)
    first, = torch.autograd.grad(y, proj, retain_graph=True)
    assert torch.equal(first, want) and arena.buf is None
    first.zero_()                                                        # the caller's own
    second, = torch.autograd.grad(y, proj, retain_graph=True)
    assert torch.equal(second, want) and not bool(first.any()) and second.data_ptr() != first.data_ptr()
