"""Residual containers around a mixer: `ResidualBlock` (``x + mixer(norm(x))``) and `BlockStack` (blocks, then a final
RMSNorm), with per-layer State lists (reference: src/orbit_ssm/model.py:51-118 and 150-255).  The pre-norms run on
this package's gate + RMSNorm kernels with no gate (one kernel forward, one backward plus the weight-gradient column
sum).  A block may also norm its mixer's output, gate it and scale it before the residual add; such a block's post-norm, gate,
scale, add and the norm of whatever comes next are one kernel (`block_norm`).  A stack may keep each block's input in eight bits
and run the block again in the backward pass (`BlockStack.set_checkpoint`).  Only mixer-only blocks (``d_mlp = 0``) are built.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import ops
from .block_ops import block_norm, checkpoint_block
from .config import as_execution


class RMSNorm(nn.Module):
    """``weight * x * rsqrt(mean(x^2) + eps)`` in the input dtype, fp32 accumulation and fp32 weight (reference:
    src/orbit_ssm/layers/norms.py:10-58, the ``fused=True`` form the backbone norms use)."""

    def __init__(self, d, eps=1e-5):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(d))

    def forward(self, x):
        return ops.GateNormFn.apply(x, None, self.weight, self.eps)


def _listened(m):
    """Does somebody listen to calls of the module (its hooks, or hooks of every module)?"""
    own = m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks
    return bool(own) or nn.modules.module._has_any_global_hook()


def _plain(m, cls):
    """Is `m` an ordinary `cls` whose arithmetic a kernel may do from its parameters?  (A subclass, a wrapper, another module in its place
    and one that is listened to are called.)"""
    return type(m) is cls and "forward" not in m.__dict__ and not _listened(m)


class ResidualBlock(nn.Module):
    """``x + mixer(norm(x))``; with `post_norm`, `gate` or `residual_scale`

        n = norm(x),   x + scale * post_norm(mixer(n)) * sigmoid(gate_proj(n))

    (the factors that were asked for).  `residual_scale`: the initial value of a learned [d_model] vector."""

    def __init__(self, mixer, d_model, d_mlp=0, *, post_norm=False, gate=False, residual_scale=None):
        super().__init__()
        if d_mlp:
            raise NotImplementedError("ResidualBlock: the SwiGLU sublayer (d_mlp > 0) is outside this package")
        self.norm = RMSNorm(d_model)
        self.mixer = mixer
        self.d_mlp = 0
        out_proj = getattr(mixer, "out_proj", None)
        if isinstance(out_proj, nn.Linear):
            out_proj.weight._normalize_w_num_layers = True       # residual-out tag (reference: layers/init.py:118-160)
        #: the mixer's output joins the residual stream through `block_norm`
        self.joins = bool(post_norm or gate or residual_scale is not None)
        self.post_norm = RMSNorm(d_model) if post_norm else None
        self.gate_proj = nn.Linear(d_model, d_model, bias=False) if gate else None
        self.scale = None if residual_scale is None else nn.Parameter(torch.full((d_model,), float(residual_scale)))

    n_residuals = 1
    joins = False                        # (a block that was pickled before there were any has no such entry)

    def join(self, x, n, h, next_norm=None):
        """(x + scale * post_norm(h) * sigmoid(gate_proj(n)), next_norm of it | None) in one kernel."""
        gate, io = None, h.dtype
        if self.gate_proj is not None:
            if _plain(self.gate_proj, nn.Linear) and self.gate_proj.bias is None:
                with torch.autocast("cuda", enabled=False):
                    gate = ops.ProjectFn.apply(n.to(io), None, 0, None, 0, self.gate_proj.weight)
            else:
                gate = self.gate_proj(n)
        post = self.post_norm
        if post is not None and not _plain(post, RMSNorm):
            h, post = post(h), None
        dt = torch.promote_types(x.dtype, h.dtype)          # as in x + h: under autocast a float32 stream stays float32
        # two norms of unlike eps are not one kernel's: the next norm then runs by itself
        fused = next_norm if next_norm is not None and _plain(next_norm, RMSNorm) and (post is None or next_norm.eps == post.eps) else None
        eps = fused.eps if fused is not None else 0.0 if post is None else post.eps
        r, out = block_norm(x.to(dt), h.to(dt), gate=None if gate is None else gate.to(dt), scale=self.scale,
                            post_weight=None if post is None else post.weight, pre_weight=None if fused is None else fused.weight, eps=eps)
        if next_norm is not None and fused is None:
            out = next_norm(r)
        return r, out

    def advance(self, x, n=None, state=None, return_state=False, next_norm=None):
        """A joining block inside a stack: the residual stream `x` with ``n = norm(x)`` (None: not formed yet) -> (stream,
        ``next_norm(stream)`` or None without `next_norm`, State or None)."""
        n = self.norm(x) if n is None else n
        new = None
        if state is None and not return_state:
            h = self.mixer(n)
        else:
            h, new = self.mixer(n, state=state, return_state=True)
        r, out = self.join(x, n, h, next_norm)
        return r, out, new

    def forward(self, x, state=None, return_state=False):
        if self.joins:
            y, _, state = self.advance(x, None, state, return_state)
            return (y, state) if return_state else y
        fused = getattr(self.mixer, "fused_residual", False)      # this package's mixers add the residual in their output GEMM
        if state is None and not return_state:
            return self.mixer(self.norm(x), _residual=x) if fused else x + self.mixer(self.norm(x))
        if fused:
            y, state = self.mixer(self.norm(x), state=state, return_state=True, _residual=x)
        else:
            y, state = self.mixer(self.norm(x), state=state, return_state=True)
            y = x + y
        return (y, state) if return_state else y

    def step(self, x_t, state=None):
        """One token through the block: ``x_t [B, d_model]`` -> ``(x_t + mixer.step(norm(x_t)), State)`` (reference:
        src/orbit_ssm/model.py:110-115).  A missing `state` starts from zero carries."""
        if state is None:
            state = self.init_state(x_t.shape[0], device=x_t.device)
        n_t = self.norm(x_t)
        y_t, state = self.mixer.step(n_t, state)
        return (self.join(x_t, n_t, y_t)[0] if self.joins else x_t + y_t), state

    def init_state(self, batch_size, **kw):
        return self.mixer.init_state(batch_size, **kw)

    def validate_state(self, state, **kw):
        return self.mixer.validate_state(state, **kw)


def _joins(block):
    """Does the stack join the block's output to the stream itself?  (A block of its own forward or step, and one that somebody listens
    to, is called as a module.)"""
    return getattr(block, "joins", False) and type(block).forward is ResidualBlock.forward and type(block).step is ResidualBlock.step \
        and not {"forward", "step"} & block.__dict__.keys() and not _listened(block)


class BlockStack(nn.Module):
    checkpoint = None

    def __init__(self, blocks, d_model, *, residual_rescale=True):
        super().__init__()
        self.layers = nn.ModuleList(blocks)
        self.norm_f = RMSNorm(d_model)
        self.checkpoint = None
        self.residual_rescale = bool(residual_rescale)
        if self.residual_rescale and len(self.layers):
            n = sum(getattr(b, "n_residuals", 1) for b in self.layers)
            for p in self.parameters():                           # GPT-2 style depth rescale of tagged weights
                if getattr(p, "_normalize_w_num_layers", False):
                    nn.init.kaiming_uniform_(p, a=math.sqrt(5))
                    with torch.no_grad():
                        p.div_(math.sqrt(n))

    @classmethod
    def from_mixers(cls, mixers, d_model, d_mlp=0, *, residual_rescale=True, post_norm=False, gate=False, residual_scale=None):
        return cls([ResidualBlock(m, d_model, d_mlp, post_norm=post_norm, gate=gate, residual_scale=residual_scale) for m in mixers],
                   d_model, residual_rescale=residual_rescale)

    def set_checkpoint(self, mode):
        """``"int8"``: a training forward keeps of each block its input alone, in eight bits an element (`pack_activation`), and the
        backward pass runs the block again from it; None: every block keeps what its backward needs.  The gradients are then those of
        the blocks at the restored inputs (off by at most 1/127.5 of the largest of each 32 channels).  Blocks run one after another, each
        taking its norm from the stream as it is stored: outputs are those of the blocks called one by one, bit for bit.  That is also
        what a stack of plain blocks gives without the mode; in a stack of joining blocks the ordinary call forms each norm from the
        stream before its rounding, so that there outputs differ by that rounding (in bfloat16 2^-8 of each element before a norm).
        Calls with a state, or that return one, keep everything as without it.  A block that draws random numbers draws the same ones when
        it runs again; captured into a graph it is refused."""
        if mode not in (None, "int8"):
            raise ValueError(f"set_checkpoint: mode must be None or 'int8', got {mode!r}")
        if mode is not None:
            self._refuse_context_parallel()
        self.checkpoint = mode
        return self

    def _refuse_context_parallel(self):
        if any(getattr(m, "_cp", None) is not None for m in self.layers.modules()):
            raise ValueError("set_checkpoint: blocks that run context-parallel are not checkpointed (their exchanges would run twice)")

    def _next_norm(self, i):
        """The norm that follows joining block i, where that block may form it: the next joining block's or the final one."""
        return self.norm_f if i + 1 == len(self.layers) else self.layers[i + 1].norm if _joins(self.layers[i + 1]) else None

    @property
    def ssm_layers(self):
        return tuple(b.mixer for b in self.layers)

    def set_execution(self, execution):
        for m in self.ssm_layers:           # validate every target before changing any
            m._check_execution(as_execution(execution))
        for m in self.ssm_layers:
            m.set_execution(execution)
        return self

    def init_state(self, batch_size, **kw):
        return [b.init_state(batch_size, **kw) for b in self.layers]

    def step(self, x_t, state=None):
        """One token through every block and the final norm: ``x_t [B, d_model]`` -> ``(y_t, [State per layer])``."""
        states = list(state) if state is not None else [None] * len(self.layers)
        if len(states) != len(self.layers):
            raise ValueError(f"state must contain exactly {len(self.layers)} layer states")
        out = []
        n_t = None                       # the norm of x_t, where the block before formed it with its residual add
        for i, (b, s) in enumerate(zip(self.layers, states)):
            if not _joins(b):
                x_t, s = b.step(x_t, s)
                n_t = None
            else:
                s = b.init_state(x_t.shape[0], device=x_t.device) if s is None else s
                n_t = b.norm(x_t) if n_t is None else n_t
                y_t, s = b.mixer.step(n_t, s)
                x_t, n_t = b.join(x_t, n_t, y_t, self._next_norm(i))
            out.append(s)
        return (self.norm_f(x_t) if n_t is None else n_t), out

    def forward(self, x, state=None, return_state=False):
        if state is None and not return_state:
            if self.checkpoint is not None and torch.is_grad_enabled():
                self._refuse_context_parallel()             # (it may have been switched on since)
                for b in self.layers:
                    x = checkpoint_block(b, x)
                return self.norm_f(x)
            n = None
            for i, b in enumerate(self.layers):
                if _joins(b):
                    x, n, _ = b.advance(x, n, next_norm=self._next_norm(i))
                else:
                    x, n = b(x), None
            return self.norm_f(x) if n is None else n
        if state is not None:
            if not isinstance(state, (list, tuple)) or len(state) != len(self.layers):
                raise ValueError(f"state must contain exactly {len(self.layers)} layer states")
            for b, s in zip(self.layers, state):
                if s is not None:
                    b.validate_state(s, batch_size=x.shape[0], device=x.device)
        states = state if state is not None else [None] * len(self.layers)
        out = []
        n = None
        for i, (b, s) in enumerate(zip(self.layers, states)):
            if _joins(b):
                x, n, s = b.advance(x, n, s, True, self._next_norm(i))
            else:
                (x, s), n = b(x, state=s, return_state=True), None
            out.append(s)
        y = self.norm_f(x) if n is None else n
        return (y, out) if return_state else y
