"""Operators around a block: the norms before and after it fused with gate, residual scale and residual add
(`block_norm`), and the 8-bit form in which a block's input waits for the backward pass (`pack_activation`,
`unpack_activation`).  `ResidualBlock` and `BlockStack` call them; they run `orbit_block_norm_*` and `orbit_act_*` of the
C-ABI library on the current stream of the tensors' device.
"""
from __future__ import annotations

import weakref
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib, ops

PACK_GROUP = 32      # elements of a row that share one exponent

_DT = ops._DT


def device_of(who, *tensors):
    """The one CUDA device the tensors live on; a CPU tensor or a second device is refused by name."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        d = t.device
        if d.type != "cuda":
            ops._require_cuda(who, t)
            raise ValueError(f"{who}: got a tensor on {d}; the kernels run on CUDA devices")
        if dev is None:
            dev = d
        elif d != dev:
            raise ValueError(f"{who}: tensors on {dev} and {d}; all of them have to be on one device")
    return dev


def launch(name, launches, device, fn, *args):
    """Call the C-ABI function `fn` with `args` and the current stream of `device`, with `device` current, counted as `launches`
    kernels under `name`; a nonzero status raises."""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return launch(name, launches, device, fn, *args)
    if ops._TIMING is None:
        ops.LAUNCHES += launches
        status = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with ops._timed(name, launches):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if status:
        _lib.check(status, fn.__name__)


def native(name, *args):
    """The outputs of host call `name` (`_lib.host`), or None where it leaves the call to the Python way."""
    if ops._TIMING is not None:
        return None                    # a timed region needs the events around the launch
    got = getattr(_lib._host or _lib.host(), name)(*args)
    if got is None:
        return None
    *outs, status, launches = got
    if status:
        _lib.check(status, name)
    ops.LAUNCHES += launches
    return outs


def tracing():
    """Is `torch.jit.trace` recording?  A call that is no autograd node would be recorded as its empty outputs."""
    return torch._C._get_tracing_state() is not None


def not_traced(who):
    if tracing():
        raise RuntimeError(f"{who}: cannot be recorded by torch.jit.trace (it is not an autograd node)")


def differentiated(*tensors):
    """Is a gradient of any of them recorded, or does one carry a forward-mode tangent?"""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                return True
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def wants_node(*tensors):
    """Does a call on them go through its autograd node?  Where it is differentiated (the node refuses forward mode) and under
    `torch.jit.trace`.  Elsewhere a call skips the node (about 10 us of host time)."""
    return tracing() or differentiated(*tensors)


def same_device(who, dev, *tensors):
    """Refuse (by name) unless every tensor is on CUDA device number `dev`."""
    for t in tensors:
        if t is not None and t.get_device() != dev or dev < 0:
            device_of(who, *tensors)


def like(t):
    """A new dense tensor of the shape and type of `t`."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, device=t.device, dtype=t.dtype)


def io_code(who, t):
    code = _DT.get(t.dtype)
    if code is None:
        raise NotImplementedError(f"{who}: activations must be float32 or bfloat16, got {t.dtype}")
    return code


def _ptr(t):
    return None if t is None else t.data_ptr()


def _weight(t):
    """A weight vector as the kernels read it: dense float32."""
    if t is None or (t.dtype is torch.float32 and t.is_contiguous()):
        return t
    return ops._f32(t)


# ----------------------------------------------------------------------------------------------------
#  norms around a block
# ----------------------------------------------------------------------------------------------------
def _rows_of(t, D):
    """[..., D] as [M, D] rows of one stride with a dense last axis; copied only where no view is one."""
    if t.dim() == 2 and t.stride(1) == 1:
        return t
    if t.is_contiguous():
        return t.view(-1, D)
    if t.stride(-1) != 1:
        return t.contiguous().view(-1, D)
    t = ops._as_rows(t, D)
    return t if t.stride(1) == 1 else t.contiguous()


def _stride(t):
    return t.shape[1] if t.shape[0] <= 1 else t.stride(0)      # the stride of a single row is never used


def block_norm_fwd(x, h, gate, scale, w_post, w_pre, eps, keep):
    """x, h, gate [M, D] (gate may be None), weights fp32 [D] or None -> (r, n | None, rstd_h | None, rstd_r | None);
    the rstd are kept where `keep`."""
    dev = x.device
    M, D = x.shape
    r = like(x)
    n = like(x) if w_pre is not None else None
    rh = torch.empty((M,), device=dev, dtype=torch.float32) if keep and w_post is not None else None
    rr = torch.empty((M,), device=dev, dtype=torch.float32) if keep and w_pre is not None else None
    if M:
        launch("block_norm_fwd", 1, dev, _lib.load().orbit_block_norm_fwd, x.data_ptr(), _stride(x), h.data_ptr(), _stride(h),
               _ptr(gate), 0 if gate is None else _stride(gate), _ptr(scale), _ptr(w_post), _ptr(w_pre), r.data_ptr(), _ptr(n),
               _ptr(rh), _ptr(rr), M, D, eps, _DT[x.dtype])
    return r, n, rh, rr


def block_norm_bwd(x, h, gate, scale, w_post, w_pre, rstd_h, rstd_r, dr, dn, want_sums=True):
    """Gradients of `block_norm_fwd`: (dx, dh, dgate | None, dscale | None, dw_post | None, dw_pre | None); dr or dn may
    be None (zeros).  Without `want_sums` the three column sums are left out."""
    dev = device_of("block_norm", x, dr, dn)
    M, D = x.shape
    f32 = torch.float32
    dx = like(x)
    dh = torch.empty_like(dx)
    dg = torch.empty_like(dx) if gate is not None else None
    sums = [torch.empty((D,), device=dev, dtype=f32) if (want_sums and w is not None) else None for w in (scale, w_post, w_pre)]
    lib = _lib.load()
    nbytes, ws = 0, None
    if any(s is not None for s in sums):
        nbytes = lib.orbit_block_norm_bwd_workspace_bytes(M, D)
        ws = torch.empty((nbytes,), device=dev, dtype=torch.uint8)
    launch("block_norm_bwd", (2 if ws is not None else 1) if M else 0, dev, lib.orbit_block_norm_bwd, x.data_ptr(), _stride(x),
           h.data_ptr(), _stride(h), _ptr(gate), 0 if gate is None else _stride(gate), _ptr(scale), _ptr(w_post), _ptr(w_pre),
           _ptr(rstd_h), _ptr(rstd_r), _ptr(dr), _ptr(dn), dx.data_ptr(), dh.data_ptr(), _ptr(dg), _ptr(sums[0]), _ptr(sums[1]),
           _ptr(sums[2]), _ptr(ws), nbytes, M, D, _DT[x.dtype])
    return (dx, dh, dg, *sums)


def _block_norm(x, h, gate, scale, w_post, w_pre, eps, keep):
    """(r, n | None) in the shape of x, and what the backward pass reads."""
    D = x.shape[-1]
    x2, h2 = _rows_of(x, D), _rows_of(h, D)
    g2 = None if gate is None else _rows_of(gate, D)
    s32, wo, wi = _weight(scale), _weight(w_post), _weight(w_pre)
    r, n, rh, rr = block_norm_fwd(x2, h2, g2, s32, wo, wi, eps, keep)
    if x.dim() != 2:
        r, n = r.view(x.shape), None if n is None else n.view(x.shape)
        # kept in the shape that the native call keeps: a run again on the other host way saves the like
        x2, h2, g2 = (None if t is None else t.view(x.shape) for t in (x2, h2, g2))
    return r, n, (x2, h2, g2, s32, wo, wi, rh, rr)


class BlockNormFn(torch.autograd.Function):
    """(r, n) of `block_norm`; n is None without a pre-norm weight."""

    @staticmethod
    def forward(ctx, x, h, gate, scale, w_post, w_pre, eps):
        ctx.set_materialize_grads(False)
        got = native("block_norm", x, h, gate, scale, w_post, w_pre, eps, True)
        if got is not None:
            r, n, rh, rr = got
            ctx.save_for_backward(x, h, gate, scale, w_post, w_pre, rh, rr)
        else:
            r, n, saved = _block_norm(x, h, gate, scale, w_post, w_pre, eps, True)
            ctx.save_for_backward(*saved)
        ctx.meta = (x.shape, [None if t is None else t.dtype for t in (scale, w_post, w_pre)])
        return r, n

    @staticmethod
    @ops.first_order_only("block norm")
    def backward(ctx, dr, dn):
        if dr is None and dn is None:
            return (None,) * 7
        x, h, gate, s32, wo, wi, rh, rr = ctx.saved_tensors
        shape, dts = ctx.meta
        need = ctx.needs_input_grad
        want_sums = need[3] or need[4] or need[5]
        got = native("block_norm_bwd", x, h, gate, s32, wo, wi, rh, rr, dr, dn, want_sums)
        if got is None:
            D = shape[-1]
            x2, h2, g2, dr2, dn2 = (None if t is None else _rows_of(t, D) for t in (x, h, gate, dr, dn))
            dr2, dn2 = (None if t is None else t.contiguous() for t in (dr2, dn2))
            got = block_norm_bwd(x2, h2, g2, s32, wo, wi, rh, rr, dr2, dn2, want_sums=want_sums)
        dx, dh, dg, *sums = got
        out = [dx.view(shape) if need[0] else None, dh.view(shape) if need[1] else None,
               dg.view(shape) if need[2] else None]
        out += [s.to(dt) if (need[3 + i] and s is not None) else None for i, (s, dt) in enumerate(zip(sums, dts))]
        return (*out, None)


def block_norm(x, h, *, gate=None, scale=None, post_weight=None, pre_weight=None, eps=1e-5):
    """Joins a block's output `h` to the residual stream `x` and normalises the sum for what follows, in one kernel:

        u = rms_norm(h) * post_weight        (u = h without `post_weight`)
        r = x + scale * u * sigmoid(gate)    (no gate factor without `gate`, scale 1 without `scale`)
        n = rms_norm(r) * pre_weight         (None without `pre_weight`)

    x, h, gate: [..., D] of one shape and dtype (float32 or bfloat16; a column slice of a wider buffer is read in place);
    scale, post_weight, pre_weight: [D].  Returns (r, n) in the dtype of x; arithmetic, norms and the weights' gradients are
    float32, and n is formed from the unrounded r.  First-order differentiable in every tensor argument."""
    got = native("block_norm", x, h, gate, scale, post_weight, pre_weight, eps, False)
    if got is not None:
        return tuple(got)
    who = "block_norm"
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"{who}: expected x [..., D] with D > 0, got {tuple(x.shape)}")
    io_code(who, x)
    for name, t in (("h", h), ("gate", gate)):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise ValueError(f"{who}: {name} must have the shape and dtype of x ({tuple(x.shape)}, {x.dtype}), got "
                             f"{tuple(t.shape)}, {t.dtype}")
    for name, t in (("scale", scale), ("post_weight", post_weight), ("pre_weight", pre_weight)):
        if t is not None and (t.dim() != 1 or t.shape[0] != x.shape[-1] or not t.is_floating_point()):
            raise ValueError(f"{who}: {name} must be a floating [{x.shape[-1]}] vector, got {tuple(t.shape)}, {t.dtype}")
    if not eps >= 0:
        raise ValueError(f"{who}: eps must be at least 0, got {eps!r}")
    same_device(who, x.get_device(), x, h, gate, scale, post_weight, pre_weight)
    if not wants_node(x, h, gate, scale, post_weight, pre_weight):
        return _block_norm(x, h, gate, scale, post_weight, pre_weight, float(eps), False)[:2]
    return BlockNormFn.apply(x, h, gate, scale, post_weight, pre_weight, float(eps))


# ----------------------------------------------------------------------------------------------------
#  activations in eight bits
# ----------------------------------------------------------------------------------------------------
class PackedActivation(NamedTuple):
    """An activation in eight bits: x ~ q * 2^(exponent - 127), one exponent for each 32 consecutive elements of a row."""
    q: torch.Tensor           # int8, the activation's shape
    exponent: torch.Tensor    # uint8 [..., ceil(D / 32)]
    dtype: torch.dtype        # what the activation was

    @property
    def nbytes(self):
        return self.q.numel() + self.exponent.numel()


def pack_activation(x):
    """x [..., D] (float32 or bfloat16, a dense last axis) -> `PackedActivation`: a signed byte an element and one power of
    two for each 32 elements of a row, the least under which the group's largest element rounds to at most 127 (never below
    2^-126).  Rounding is to nearest, ties to even: off by at most half a step, that is 1/127.5 of the group's largest element
    (2^-127 where that is more: a step is never below 2^-126; values within 2^122 of the type's largest are off by up to a step, so as
    to stay finite).  A non-finite element is restored as NaN and leaves its group's scale alone.  Not differentiable."""
    got = native("pack", x)
    if got is not None:
        return PackedActivation(*got, x.dtype)
    who = "pack_activation"
    not_traced(who)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"{who}: expected x [..., D] with D > 0, got {tuple(x.shape)}")
    code = io_code(who, x)
    if x.requires_grad:
        x = x.detach()
    dev = device_of(who, x)
    D = x.shape[-1]
    x2 = _rows_of(x, D)
    M = x2.shape[0]
    q = torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format)
    e = q.new_empty((*x.shape[:-1], -(-D // PACK_GROUP)), dtype=torch.uint8)
    if M:
        launch("act_pack", 1, dev, _lib.load().orbit_act_pack, x2.data_ptr(), _stride(x2), q.data_ptr(), e.data_ptr(), M, D, code)
    return PackedActivation(q, e, x.dtype)


def unpack_activation(packed, dtype=None):
    """The activation a `PackedActivation` stands for, in `dtype` (default: its own; exact in float32 and in bfloat16)."""
    who = "unpack_activation"
    not_traced(who)
    q, e, own_dtype = packed
    dtype = own_dtype if dtype is None else dtype
    if dtype not in _DT:
        raise NotImplementedError(f"{who}: activations must be float32 or bfloat16, got {dtype}")
    got = native("unpack", q, e, dtype is torch.bfloat16)
    if got is not None:
        return got[0]
    if q.dtype != torch.int8 or e.dtype != torch.uint8 or q.dim() < 1 or q.shape[-1] == 0 \
            or tuple(e.shape) != (*q.shape[:-1], -(-q.shape[-1] // PACK_GROUP)):
        raise ValueError(f"{who}: expected int8 q [..., D] with uint8 exponents [..., ceil(D / {PACK_GROUP})], got {q.dtype} "
                         f"{tuple(q.shape)} with {e.dtype} {tuple(e.shape)}")
    dev = device_of(who, q, e)
    q, e = q.contiguous(), e.contiguous()
    x = torch.empty_like(q, dtype=dtype)
    D = q.shape[-1]
    if q.numel():
        launch("act_unpack", 1, dev, _lib.load().orbit_act_unpack, q.data_ptr(), e.data_ptr(), x.data_ptr(), q.numel() // D, D, _DT[dtype])
    return x


#: block -> {the training flags of its modules: does it draw from the GPU's generator?}, as uncaptured runs have shown
_DRAWS = weakref.WeakKeyDictionary()


def _flags(block):
    return tuple(m.training for m in block.modules())


class _Drawn:
    """What a block's first run drew: the second one draws the same, and leaves the generators (the CPU's and the one of the block's
    device) as it found them."""

    def __init__(self, block, device):
        self.generators = [torch.default_generator]
        if device.type == "cuda":
            gpu = torch.cuda.default_generators[device.index]
            if not torch.cuda.is_current_stream_capturing():
                self.generators.append(gpu)
            else:
                # inside a capture a generator cannot be set back
                draws = _DRAWS.get(block, {}).get(_flags(block))
                if draws is None:
                    raise RuntimeError("8-bit activation checkpoint: run the block forward once, in the mode it is to be captured in, before "
                                       "the capture: only such a run shows whether it draws random numbers")
                if draws:
                    raise RuntimeError("8-bit activation checkpoint: a block that draws random numbers on the GPU cannot be captured into a "
                                       "graph: its second run would draw others than its first")
        self.states = [g.get_state() for g in self.generators]

    def note(self, block):
        drew = [not torch.equal(g.get_state(), s) for g, s in zip(self.generators, self.states)]
        if len(drew) == 2:
            _DRAWS.setdefault(block, {})[_flags(block)] = drew[1]
        self.generators, self.states = ([x for x, d in zip(xs, drew) if d] for xs in (self.generators, self.states))

    def __enter__(self):
        self.found = [g.get_state() for g in self.generators]
        for g, s in zip(self.generators, self.states):
            g.set_state(s)

    def __exit__(self, *exc):
        for g, s in zip(self.generators, self.found):
            g.set_state(s)


class _Checkpoint:
    """A block's run whose saved tensors are dropped (`drop` gives autograd a number for each) and formed again by a second run when
    the backward pass asks for the first of them (`fetch`)."""

    def __init__(self, block, x):
        params = list(block.parameters())
        self.block, self.packed, self.wanted = block, pack_activation(x), x.requires_grad
        self.versions = [(p, p._version) for p in params if not p.is_inference()]
        self.autocast = dict(dtype=torch.get_autocast_dtype("cuda"), enabled=torch.is_autocast_enabled("cuda"), cache_enabled=False)
        self.saved = []                  # shape, dtype and device of each
        self.again = {}                  # number -> tensor of the second run, until it is fetched
        self.drawn = _Drawn(block, x.device)

    def first(self, x):
        with torch.autograd.graph.saved_tensors_hooks(self.drop, self.fetch):
            y = self.block(x)
        self.drawn.note(self.block)
        return y

    def drop(self, t):
        self.saved.append((t.shape, t.dtype, t.device))
        return len(self.saved) - 1

    def fetch(self, i):
        if i not in self.again:          # (also where a kept graph is walked once more)
            self.again = self.second()
        return self.again.pop(i)

    def second(self):
        for p, version in self.versions:
            if p._version != version:
                raise RuntimeError(f"8-bit activation checkpoint: a parameter {tuple(p.shape)} that the block's backward pass needs was "
                                   f"modified by an inplace operation (version {p._version}, expected {version})")
        kept = []
        keep = torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.detach()), _never)
        with torch.enable_grad(), torch.autocast("cuda", **self.autocast), self.drawn, keep:
            self.block(unpack_activation(self.packed).requires_grad_(self.wanted))
        if [(t.shape, t.dtype, t.device) for t in kept] != self.saved:
            raise RuntimeError("8-bit activation checkpoint: the block's second run saved other tensors for its backward pass than its first "
                               f"({len(kept)} and {len(self.saved)} of them): its course has to depend on its input's shape alone")
        return dict(enumerate(kept))


def _never(t):
    raise RuntimeError("8-bit activation checkpoint: the graph of a block's second run is not differentiated")


def checkpoint_block(block, x):
    """``block(x)`` without keeping what the block's backward needs: its input waits in eight bits, and the backward pass restores
    it, runs the block again from it and differentiates the block's own graph with what that run saves (so that hooks of parameters
    and modules see one backward pass).  The second run draws the random numbers of the first (from torch's default generators, the
    CPU's and the input's device's).  Refused: a block that saves other tensors when it runs again, a parameter changed in place in between, and a block that draws on the GPU inside a graph capture.  An ordinary call where no gradient is wanted."""
    if not torch.is_grad_enabled() or not (x.requires_grad or any(p.requires_grad for p in block.parameters())):
        return block(x)
    return _Checkpoint(block, x).first(x)
