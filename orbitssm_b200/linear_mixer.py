"""Linear attention with a constant decay for each head: the operators `linear_attention` (a sequence, differentiable,
with the state carried in and out) and `linear_attention_step` (one token), and the mixer layer `LinearAttention` on them.

    S_t = a S_{t-1} + v_t k_t^T,    y_t = scale S_t q_t,    a = exp(log_decay[head])

Where the SSD scan shares its maps over the heads and takes a decay for each token, here every head has keys and queries of
its own and one decay.  The state [B, H, Dv, Dk] is float32; its layout is that of the other layers' ``hidden_state``
[B, H, P, N] (channel, state row).
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from dataclasses import asdict, dataclass

import torch
import torch.nn as nn

from . import _lib, ops
from .block_ops import differentiated, io_code, launch, like, native, not_traced, same_device, wants_node
from .config import BACKENDS, PRECISIONS, _positive_int, _strict_from_dict, as_execution
from .state import State, StateLifecycle


# ----------------------------------------------------------------------------------------------------
#  the operators
# ----------------------------------------------------------------------------------------------------
def _operand(t):
    """`t` [B, L, H, D] as the kernels read it: a dense last axis; for bfloat16 heads of a multiple of 8 also 16-byte rows and no
    overlapping (expanded) axes, so that the tensor-core tiles can load it.  Copied only where it is not so already."""
    D = t.shape[3]
    tiles = t.dtype is torch.bfloat16 and D % 8 == 0
    if t.is_contiguous():
        return t if not tiles or t.data_ptr() % 16 == 0 else t.clone()
    sb, sl, sh, sd = t.stride()
    if sd != 1 and D > 1:
        return t.contiguous()
    if tiles:
        if t.data_ptr() % 16:
            return t.clone(memory_format=torch.contiguous_format)
        for n, s in zip(t.shape, (sb, sl, sh)):
            if n > 1 and (s % 8 or s <= 0):
                return t.contiguous()
    return t


def _strides(t):
    """(batch, token, head) strides; an axis of one element, whose stride is never used, gets an aligned one."""
    B, L, H, D = t.shape
    if t.is_contiguous():
        return (L * H * D, H * D, D)
    sb, sl, sh, _ = t.stride()
    return (sb if B > 1 else 8, sl if L > 1 else 8, sh if H > 1 else 8)


def _status(device):
    if (device.type, device.index) not in ops._STATUS and torch.cuda.is_current_stream_capturing():
        return 0                   # the word must not be born in a graph's memory pool
    word = ops._status_word(device).data_ptr()
    _lib.host().bind_status(device.index, word)
    return word


#: `orbit_la_args` in one call: filling the ctypes structure field by field costs the host 6 us more
_PACK = struct.Struct("@5if" + "P3q" * 3 + "PP" + "P3q" + "P" + "P3q" + "P" + "P3q" * 3 + "PPqP")
assert _PACK.size == C.sizeof(_lib.LaArgs)
_NONE = (0, 0, 0, 0)


def _run(name, fn, bwd, q, k, v, log_decay, state, scale, code, tail):
    """Pack the argument block (`tail`: its fields from `y` up to the workspace), ask for the workspace and launch."""
    dev = q.device
    B, L, H, Dk = q.shape
    Dv = v.shape[3]
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _run(name, fn, bwd, q, k, v, log_decay, state, scale, code, tail)
    fields = (B, L, H, Dk, Dv, scale, q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k), v.data_ptr(), *_strides(v),
              log_decay.data_ptr(), 0 if state is None else state.data_ptr(), *tail)
    status = _status(dev)
    lib = _lib.load()
    ws, nbytes = None, 0
    if L > 32:                     # a sequence of one tile is never split, whatever the kernels
        nbytes = lib.orbit_la_workspace_bytes(_PACK.pack(*fields, 0, 0, status), bwd, code)
        if nbytes:
            ws = torch.empty((nbytes,), device=dev, dtype=torch.uint8)
    launch(name, 1 if ws is None else 3, dev, fn, _PACK.pack(*fields, 0 if ws is None else ws.data_ptr(), nbytes, status), code)


def la_fwd(q, k, v, log_decay, state, scale, want_state):
    """Operands as `_operand` leaves them -> (y [B, L, H, Dv], state [B, H, Dv, Dk] | None)."""
    got = native("la_fwd", q, k, v, log_decay, state, scale, want_state)
    if got is not None:
        return got
    B, L, H, Dk = q.shape
    Dv = v.shape[3]
    y = like(v)
    new = None
    if want_state:
        new = torch.empty((B, H, Dv, Dk), device=q.device, dtype=torch.float32) if state is None else torch.empty_like(state)
    if B and (L or want_state):
        _run("linear_attention_fwd", _lib.load().orbit_la_fwd, 0, q, k, v, log_decay, state, scale, ops._DT[q.dtype],
             (y.data_ptr(), L * H * Dv, H * Dv, Dv, 0 if new is None else new.data_ptr(), *_NONE, 0, *_NONE, *_NONE, *_NONE, 0))
    return y, new


def la_bwd(q, k, v, log_decay, state, scale, dy, dstate, want_dstate0, outs=(None, None, None)):
    """Gradients (dq, dk, dv, dstate0 | None); `outs` may name tensors (any strides, dense last axis) that receive dq, dk, dv."""
    if outs[0] is None and outs[1] is None and outs[2] is None:
        got = native("la_bwd", q, k, v, log_decay, state, scale, dy, dstate, want_dstate0)
        if got is not None:
            return got
    dq, dk, dv = (like(t) if o is None else o for o, t in zip(outs, (q, k, v)))
    B, L, H, Dk = q.shape
    ds0 = torch.empty((B, H, v.shape[3], Dk), device=q.device, dtype=torch.float32) if want_dstate0 else None
    if B and (L or want_dstate0):
        _run("linear_attention_bwd", _lib.load().orbit_la_bwd, 1, q, k, v, log_decay, state, scale, ops._DT[q.dtype],
             (*_NONE, 0, dy.data_ptr(), *_strides(dy), 0 if dstate is None else dstate.data_ptr(), dq.data_ptr(), *_strides(dq),
              dk.data_ptr(), *_strides(dk), dv.data_ptr(), *_strides(dv), 0 if ds0 is None else ds0.data_ptr()))
    return dq, dk, dv, ds0


def _la(q, k, v, log_decay, state, scale, want_state):
    """(y, state | None) and what the backward pass reads."""
    q, k, v = _operand(q), _operand(k), _operand(v)
    if state is not None and not state.is_contiguous():
        state = state.contiguous()
    y, new = la_fwd(q, k, v, log_decay, state, scale, want_state)
    return y, new, (q, k, v, log_decay, state)


class LinearAttentionFn(torch.autograd.Function):
    """(y, state after the sequence | None).  `slots`: (GradArena, column-range index) of q, k and v, or None each."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, scale, want_state, slots):
        ctx.set_materialize_grads(False)
        got = native("la_fwd", q, k, v, log_decay, state, scale, want_state)     # (checks the call as well)
        if got is not None:
            y, new = got
            saved = (q, k, v, log_decay, state)
        else:
            scale, log_decay = _checked(q, k, v, log_decay, state, scale)
            y, new, saved = _la(q, k, v, log_decay, state, scale, want_state)
        ctx.save_for_backward(*saved)
        ctx.scale, ctx.slots = scale, slots
        return y, new

    @staticmethod
    @ops.first_order_only("linear attention")
    def backward(ctx, dy, dstate):
        if dy is None and dstate is None:
            return (None,) * 8
        q, k, v, log_decay, s0 = ctx.saved_tensors
        need = ctx.needs_input_grad
        dy = torch.zeros(v.shape, device=v.device, dtype=v.dtype) if dy is None else _operand(dy)
        dstate = None if dstate is None else dstate.contiguous()
        outs = [None] * 3
        if ctx.slots is not None:
            for i, (t, slot) in enumerate(zip((q, k, v), ctx.slots)):
                if slot is not None and need[i]:
                    B, L, H, D = t.shape
                    view = slot[0].view(slot[1], dy.new_empty((1,)).expand(B, L, H * D))     # a tensor of the range's shape
                    if view is not None and _operand(view.unflatten(2, (H, D))).data_ptr() == view.data_ptr():
                        outs[i] = view.unflatten(2, (H, D))
        scale = ctx.scale if ctx.scale is not None else q.shape[-1] ** -0.5
        dq, dk, dv, ds0 = la_bwd(q, k, v, log_decay, s0, scale, dy, dstate, need[4] and s0 is not None, outs)
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, ds0 if need[4] else None,
                None, None, None)


def _check_operands(who, q, k, v, log_decay, state, lead):
    """Shapes, dtypes and device of a call; `lead` names the axes before the heads."""
    qs, vs = q.shape, v.shape
    if len(qs) != len(lead) + 2 or k.shape != qs or len(vs) != len(qs) or vs[:-1] != qs[:-1]:
        axes = ", ".join(lead)
        raise ValueError(f"{who}: expected q, k [{axes}, H, Dk] and v [{axes}, H, Dv] (as many key heads as query heads: expand shared "
                         f"heads), got {tuple(qs)}, {tuple(k.shape)}, {tuple(vs)}")
    code = io_code(who, q)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{who}: q, k and v must have one dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    B, H, Dk, Dv = qs[0], qs[-2], qs[-1], vs[-1]
    if H < 1 or not 1 <= Dk <= 256 or not 1 <= Dv <= 256:
        raise NotImplementedError(f"{who}: at least one head, of widths 1..256, got H={H} Dk={Dk} Dv={Dv}")
    if log_decay.shape != (H,) or log_decay.dtype != torch.float32:
        raise ValueError(f"{who}: log_decay must be float32 [{H}], got {log_decay.dtype} {tuple(log_decay.shape)}")
    if differentiated(log_decay):
        raise ValueError(f"{who}: log_decay is a constant of the layer; its gradient is not served (detach it)")
    if state is not None and (state.shape != (B, H, Dv, Dk) or state.dtype != torch.float32):
        raise ValueError(f"{who}: state must be float32 {(B, H, Dv, Dk)}, got {state.dtype} {tuple(state.shape)}")
    same_device(who, q.get_device(), q, k, v, log_decay, state)
    return code


def _scale_of(who, scale, Dk):
    if scale is None:
        return Dk ** -0.5
    scale = float(scale)
    if not math.isfinite(scale) or scale == 0.0:
        raise ValueError(f"{who}: scale must be finite and not zero, got {scale!r}")
    return scale


def _checked(q, k, v, log_decay, state, scale):
    """Refuses what `linear_attention` does not serve -> the scale and the decays as the kernels take them."""
    _check_operands("linear_attention", q, k, v, log_decay, state, ("B", "L"))
    scale = _scale_of("linear_attention", scale, q.shape[-1])
    return scale, log_decay if log_decay.is_contiguous() and not log_decay.requires_grad else log_decay.detach().contiguous()


def linear_attention(q, k, v, log_decay, state=None, *, scale=None, return_state=False, _slots=None):
    """y_t = scale S_t q_t over a sequence, with S_t = exp(log_decay) S_{t-1} + v_t k_t^T for each head.

    q, k [B, L, H, Dk], v [B, L, H, Dv]: float32 or bfloat16, any strides (strided views with a dense last axis are read in
    place); log_decay [H] float32, at most 0, a constant; state [B, H, Dv, Dk] float32 before the sequence (None: zeros);
    scale: default Dk^-0.5.  Returns y [B, L, H, Dv] in the dtype of q, or (y, state after the sequence) with
    `return_state`.  L may be 0.  First-order differentiable in q, k, v and state, through y and the returned state.

    bfloat16 heads whose widths are multiples of 8 up to 128 run on tensor-core tiles (scales within 2^-40 to 2^40): products of the unrounded inputs with the
    scores or the state rounded once to bfloat16, float32 sums.  That makes the error of y and of the gradients of q, k and v about 1.4
    times that of their own rounding, at every length; scores are kept in two parts where a pass begins (for y and the gradient of q the
    first 32 tokens, for those of k and v the last 32 as far as they share the last chunk of 128), so that without a state these rows are
    rounded once.  The state itself is float32 throughout.  Other calls run on float32 kernels.  Values are expected to be finite: a NaN
    or infinity may reach every output of its head and sequence."""
    if differentiated(log_decay):
        _checked(q, k, v, log_decay, state, scale)               # refuses a gradient of it
    if wants_node(q, k, v, state):
        y, new = LinearAttentionFn.apply(q, k, v, log_decay, state, scale, bool(return_state), _slots)
        return (y, new) if return_state else y
    got = native("la_fwd", q, k, v, log_decay, state, scale, return_state)
    if got is None:
        scale, log_decay = _checked(q, k, v, log_decay, state, scale)
        got = _la(q, k, v, log_decay, state, scale, bool(return_state))
    return (got[0], got[1]) if return_state else got[0]


def linear_attention_step(q, k, v, log_decay, state, *, scale=None, out_state=None):
    """One token: q, k [B, H, Dk], v [B, H, Dv], state [B, H, Dv, Dk] float32 -> (y [B, H, Dv], state after the token).

    `out_state` (contiguous float32 of the state's shape) receives the new state; it may be `state` itself.  For inference: not
    differentiable (run `linear_attention` on a sequence of one token for gradients).  Everything else as there."""
    if out_state is None:
        got = native("la_step", q, k, v, log_decay, state, scale)
        if got is not None:
            return tuple(got)
    who = "linear_attention_step"
    not_traced(who)
    if state is None:
        raise ValueError(f"{who}: a state is required (zeros before the first token)")
    code = _check_operands(who, q, k, v, log_decay, state, ("B",))
    if differentiated(q, k, v, state):
        raise ValueError(f"{who}: gradients are not served; use linear_attention on a sequence of one token, or torch.no_grad()")
    if out_state is not None and (out_state.shape != state.shape or out_state.dtype != torch.float32 or not out_state.is_contiguous()
                                  or out_state.device != state.device):
        raise ValueError(f"{who}: out_state must be contiguous float32 {tuple(state.shape)} on {state.device}")
    scale = _scale_of(who, scale, q.shape[-1])
    B, H, Dk = q.shape
    Dv, dev = v.shape[2], q.device
    q, k, v = _dense_rows(q), _dense_rows(k), _dense_rows(v)
    if not state.is_contiguous():
        state = state.contiguous()
    if out_state is not None and out_state.data_ptr() != state.data_ptr() and _overlap(out_state, state):
        raise ValueError(f"{who}: out_state overlaps state without being it")
    if out_state is not None and any(_overlap(out_state, t) for t in (q, k, v, log_decay)):
        raise ValueError(f"{who}: out_state overlaps q, k, v or log_decay")
    new = torch.empty_like(state) if out_state is None else out_state
    if out_state is not None and not out_state.is_inference():
        torch.autograd.graph.increment_version(out_state)        # a graph that kept it must not read the new one
    y = like(v)
    if B:
        qb, qh, _ = q.stride()
        kb, kh, _ = k.stride()
        vb, vh, _ = v.stride()
        launch("linear_attention_step", 1, dev, _lib.load().orbit_la_step, q.data_ptr(), qb, qh, k.data_ptr(), kb, kh, v.data_ptr(), vb,
               vh, (log_decay if log_decay.is_contiguous() else log_decay.contiguous()).data_ptr(), state.data_ptr(), new.data_ptr(),
               y.data_ptr(), B, H, Dk, Dv, scale, code)
    return y, new


def _dense_rows(t):
    return t if t.shape[2] == 1 or t.stride(2) == 1 else t.contiguous()


def _extent(t):
    """The bytes from a tensor's first element to its last."""
    if t.numel() == 0:
        return 0, 0
    return t.data_ptr(), t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def _overlap(a, b):
    (a0, a1), (b0, b1) = _extent(a), _extent(b)
    return a0 < b1 and b0 < a1


# ----------------------------------------------------------------------------------------------------
#  the layer
# ----------------------------------------------------------------------------------------------------
@dataclass(frozen=True)
class LinearAttentionConfig:
    """`LinearAttention` layer.  Heads have keys of `d_key` and values of `d_value` channels (default d_model / n_heads
    each); head h forgets over a span that runs geometrically from `span_min` to `span_max` tokens: decay 1 - 1 / span.
    In bfloat16, widths that are multiples of 8 up to 128 run on tensor cores; others (up to 256) take the float32 kernels, which need
    about 30 times as long."""
    d_model: int
    n_heads: int
    d_key: int | None = None
    d_value: int | None = None
    span_min: float = 32.0
    span_max: float = 4096.0
    out_norm: bool = True
    norm_eps: float = 1e-5

    def __post_init__(self):
        _positive_int(self.d_model, "d_model")
        _positive_int(self.n_heads, "n_heads")
        for name in ("d_key", "d_value"):
            v = getattr(self, name)
            if v is None:
                if self.d_model % self.n_heads:
                    raise ValueError(f"{name}: n_heads={self.n_heads} does not divide d_model={self.d_model}; give the head width")
                object.__setattr__(self, name, self.d_model // self.n_heads)
            elif _positive_int(v, name) > 256:
                raise ValueError(f"{name} must be at most 256, got {v}")
            if getattr(self, name) > 256:
                raise ValueError(f"{name}={getattr(self, name)}: head widths go up to 256")
        if not 1.0 < self.span_min <= self.span_max:
            raise ValueError(f"spans must satisfy 1 < span_min <= span_max, got {self.span_min}, {self.span_max}")
        if not isinstance(self.out_norm, bool):
            raise TypeError("out_norm must be a bool")

    def to_dict(self):
        return asdict(self)

    @classmethod
    def from_dict(cls, d):
        return _strict_from_dict(cls, d)


class _OutNorm(nn.Module):
    """Parameter holder of the output RMSNorm; the arithmetic runs in the fused gate + norm kernel."""

    def __init__(self, d):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(d))


class LinearAttention(StateLifecycle, nn.Module):
    """Mixer: x -> [one GEMM: q | k | v | gate z] -> `linear_attention` -> y * silu(z) (+ RMSNorm) -> out_proj.

    ``LinearAttention(config, execution=None)``; same call, `State` and `step` contract as the package's other mixers, so it
    stands in `ResidualBlock`, `BlockStack`, `GraphedStep` and `GraphedDecode` beside them."""

    config_family = "linear_attention"
    fused_residual = True

    def __init__(self, config, execution=None):
        nn.Module.__init__(self)
        if isinstance(config, dict):
            config = LinearAttentionConfig.from_dict(config)
        if not isinstance(config, LinearAttentionConfig):
            raise TypeError(f"config must be a LinearAttentionConfig or its dict, got {type(config).__name__}")
        self.config = c = config
        self.d_model, self.H, self.Dk, self.Dv = c.d_model, c.n_heads, c.d_key, c.d_value
        dk, dv = self.H * self.Dk, self.H * self.Dv
        self.q_proj = nn.Linear(c.d_model, dk, bias=False)
        self.k_proj = nn.Linear(c.d_model, dk, bias=False)
        self.v_proj = nn.Linear(c.d_model, dv, bias=False)
        self.gate_proj = nn.Linear(c.d_model, dv, bias=False)
        spans = torch.logspace(math.log2(c.span_min), math.log2(c.span_max), self.H, base=2.0, dtype=torch.float64)
        self.register_buffer("log_decay", torch.log1p(-1.0 / spans).float(), persistent=True)
        self.norm = _OutNorm(dv) if c.out_norm else nn.Identity()
        self.out_proj = nn.Linear(dv, c.d_model, bias=False)
        # the columns of a bfloat16 slab stay 16-byte aligned for any head widths that the tensor-core tiles take
        self._pad = (-(2 * dk + 2 * dv)) % 8
        self.backend, self.precision, self.chunk_size, self.kernel_options = "cuda", "io", "auto", {}
        self._final_state = None
        self.set_execution(as_execution(execution))

    def _apply(self, fn, recurse=True):
        """Moves and casts the layer; the decays stay float32 (``.to(torch.bfloat16)`` would move a span of 4096 tokens by 8)."""
        kept = self.log_decay
        super()._apply(fn, recurse)
        if self.log_decay.dtype != torch.float32:
            self.log_decay = kept.to(self.log_decay.device)
        return self

    # -- execution ------------------------------------------------------------------------------------------
    def _check_execution(self, ex):
        f, out = ex.fields(), {}
        if "backend" in f:
            if f["backend"] not in BACKENDS:
                raise ValueError(f"LinearAttention: backend must be one of {BACKENDS}, got {f['backend']!r}")
            out["backend"] = f["backend"]
        if "precision" in f:
            if f["precision"] not in PRECISIONS:
                raise ValueError(f"LinearAttention: precision must be one of {PRECISIONS}, got {f['precision']!r}")
            if f["precision"] != "io":
                raise ValueError("LinearAttention: precision='ieee' is refused: the kernels go by the activations' dtype (float32 "
                                 "activations run in float32)")
        if "chunk_size" in f and f["chunk_size"] != "auto":
            raise ValueError(f"LinearAttention: chunk_size is the kernels' own ('auto'), got {f['chunk_size']!r}")
        if f.get("checkpoint"):
            raise ValueError("LinearAttention: checkpoint=True is refused (BlockStack.set_checkpoint keeps block inputs in 8 bits)")
        if f.get("kernel_options"):
            raise ValueError(f"LinearAttention: unknown kernel option(s) {sorted(f['kernel_options'])}; this layer has none")
        return out

    def set_execution(self, execution):
        for k, v in self._check_execution(as_execution(execution)).items():
            setattr(self, k, v)
        return self

    # -- state ----------------------------------------------------------------------------------------------
    def _init_state(self, batch_size, device=None, dtype=None):
        dev = device if device is not None else next(self.parameters()).device
        return State(hidden_state=torch.zeros(batch_size, self.H, self.Dv, self.Dk, device=dev,
                                              dtype=self._default_state_dtype() if dtype is None else dtype))

    def hidden_state_shape(self):
        return (self.H, self.Dv, self.Dk)

    # -- forward --------------------------------------------------------------------------------------------
    def forward(self, x, *, state=None, return_state=False, _residual=None):
        """x [B, L, d_model] -> y [B, L, d_model], or (y, State) with ``return_state=True``; `state` continues a previous call."""
        if x.dim() != 3 or x.shape[-1] != self.d_model:
            raise ValueError(f"LinearAttention: expected x of shape [B, L, {self.d_model}], got {tuple(x.shape)}")
        if not ops.on_device(x):
            raise ValueError("LinearAttention: got a CPU tensor; this layer runs on a CUDA device only")
        B, L, _ = x.shape
        H, Dk, Dv = self.H, self.Dk, self.Dv
        if state is not None:
            state = self.resolve_state(state, batch_size=B, device=x.device)
        io = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype
        if io not in (torch.float32, torch.bfloat16):
            raise NotImplementedError(f"LinearAttention: IO dtype must be float32 or bfloat16, got {io}")
        with torch.autocast("cuda", enabled=False):
            proj = ops.ProjectFn.apply(x.to(io), None, self._pad, None, 0, self.q_proj.weight, self.k_proj.weight, self.v_proj.weight,
                                       self.gate_proj.weight)
            arena = ops.GradArena()                  # the operators' backward passes write d(proj) in place
            q, k, v, z = ops.SplitColumnsFn.apply(proj, arena, H * Dk, H * Dk, H * Dv, H * Dv)
            q, k, v = q.unflatten(2, (H, Dk)), k.unflatten(2, (H, Dk)), v.unflatten(2, (H, Dv))
            s0 = None if state is None else state["hidden_state"].to(torch.float32)
            if L == 1 and s0 is not None and not torch.is_grad_enabled():
                y, new = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], self.log_decay, s0)
                y = y.unsqueeze(1)
            else:
                y = linear_attention(q, k, v, self.log_decay, s0, return_state=return_state,
                                     _slots=((arena, 0), (arena, 1), (arena, 2)))
                y, new = y if return_state else (y, None)
            y = y.flatten(2)
            if L > 0:
                y = ops.GateNormFn.apply(y, z, self.norm.weight if self.config.out_norm else None, self.config.norm_eps, (arena, 3))
            fuse = _residual is not None and _residual.dtype == io and _residual.shape == x.shape
            out = ops.ProjectFn.apply(y, _residual if fuse else None, 0, None, 0, self.out_proj.weight)
            if _residual is not None and not fuse:
                out = _residual + out
        if not return_state:
            return out
        ordered = self._conform_carries(State(hidden_state=new), state)
        self._final_state = ordered
        return out, ordered

    def step(self, x_t, state=None):
        """One token: ``x_t [B, d_model]``, `state` from `init_state` or a previous call -> ``(y_t [B, d_model], State)``.  Under
        ``torch.no_grad()`` the token runs in the one-launch step kernel; with gradients it is a sequence of one token."""
        if x_t.dim() != 2 or x_t.shape[-1] != self.d_model:
            raise ValueError(f"LinearAttention.step: expected x_t of shape [B, {self.d_model}], got {tuple(x_t.shape)}")
        if state is None:
            state = self.init_state(x_t.shape[0], device=x_t.device)
        y, new = self.forward(x_t.unsqueeze(1), state=state, return_state=True)
        return y.squeeze(1), new
