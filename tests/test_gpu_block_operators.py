"""-m gpu: linear attention, block norms and 8-bit activations against plain float64 restatements.

Tolerances are elementwise majorants, derived before the first run.  With u the half step of a type relative to the value
(2^-8 bfloat16, 2^-24 float32) and |.|-sums M taken over absolute values, a result that is a float32 sum of n terms is off by
at most n u32 M; an operand rounded to bfloat16 adds u16 M of its own sum, and the rounding of the result u |result|."""
import itertools

import pytest
import torch

import orbitssm_b200 as ob
from orbitssm_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U16, U32 = 2.0 ** -8, 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32
U = {BF: U16, F32: U32}


def _randn(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(DEV)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---------------------------------------------------------------------------------------------------------------------
#  linear attention
# ---------------------------------------------------------------------------------------------------------------------
def ref_attention(q, k, v, ld, s0, scale, dy=None, ds1=None):
    """Everything in float64, token by token from the definition: (y, S_L, dq, dk, dv, dS_0)."""
    q, k, v = (t.double() for t in (q, k, v))
    B, L, H, Dk = q.shape
    Dv = v.shape[-1]
    a = torch.exp(ld.double())[:, None, None]
    S = q.new_zeros(B, H, Dv, Dk) if s0 is None else s0.double()
    states, ys = [], []
    for t in range(L):
        S = a * S + v[:, t, :, :, None] * k[:, t, :, None, :]
        states.append(S)
        ys.append(scale * torch.einsum("bhvk,bhk->bhv", S, q[:, t]))
    y = torch.stack(ys, 1) if L else q.new_zeros(B, 0, H, Dv)
    if dy is None and ds1 is None:
        return y, S
    dy = torch.zeros_like(y) if dy is None else dy.double()
    R = torch.zeros_like(S) if ds1 is None else ds1.double()
    dq, dk, dv = [None] * L, [None] * L, [None] * L
    for t in reversed(range(L)):
        R = R + scale * dy[:, t, :, :, None] * q[:, t, :, None, :]
        dq[t] = scale * torch.einsum("bhvk,bhv->bhk", states[t], dy[:, t])
        dk[t] = torch.einsum("bhvk,bhv->bhk", R, v[:, t])
        dv[t] = torch.einsum("bhvk,bhk->bhv", R, k[:, t])
        R = a * R
    st = (lambda x, w: torch.stack(x, 1) if L else q.new_zeros(B, 0, H, w))
    return y, S, st(dq, Dk), st(dk, Dk), st(dv, Dv), R


def majorant(q, k, v, ld, s0, scale, dy=None, ds1=None):
    ab = lambda t: None if t is None else t.abs()  # noqa: E731
    return ref_attention(q.abs(), k.abs(), v.abs(), ld, ab(s0), abs(scale), ab(dy), ab(ds1))


def close(got, want, big, dtype, n, operand):
    """|got - want| <= u |want| + (operand rounding + n float32 additions) of the absolute sum."""
    err = (got.double() - want).abs()
    lim = U[dtype] * want.abs() + (operand + n * U32) * big + 1e-30
    bad = err > lim
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / lim).max()):.3g} of the bound"


CASES = [
    # B, L, H, Dk, Dv
    (1, 1, 1, 128, 128), (2, 2, 3, 64, 64), (1, 127, 2, 128, 128), (1, 128, 2, 128, 64), (2, 129, 1, 64, 128),
    (1, 257, 3, 80, 96), (2, 300, 2, 8, 16), (1, 1000, 2, 128, 128), (1, 640, 1, 40, 128), (3, 77, 2, 33, 20), (1, 70, 1, 200, 256),
    (1, 1700, 1, 72, 24),
]


def _inputs(B, L, H, Dk, Dv, dtype, seed, decay="span"):
    g = _gen(seed)
    q, k = _randn(g, B, L, H, Dk, dtype=dtype), _randn(g, B, L, H, Dk, dtype=dtype)
    v, dy = _randn(g, B, L, H, Dv, dtype=dtype), _randn(g, B, L, H, Dv, dtype=dtype)
    s0, ds1 = _randn(g, B, H, Dv, Dk, std=2.0), _randn(g, B, H, Dv, Dk, std=0.3)
    ld = {"span": torch.log1p(-torch.exp2(-(2.0 + 6.0 * torch.arange(H) / max(H - 1, 1)))),
          "none": torch.zeros(H), "strong": torch.full((H,), -40.0), "all": torch.full((H,), float("-inf"))}[decay].float().to(DEV)
    return q, k, v, ld, s0, dy, ds1


def _check_all(q, k, v, ld, s0, dy, ds1, dtype, scale=None, tensor=None):
    """Forward with state in and out, and every gradient through y and the state."""
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (q, k, v, s0)]
    y, s1 = ob.linear_attention(*leaves[:3], ld, leaves[3], scale=scale, return_state=True)
    keep = [t for t in leaves if t is not None]
    got = torch.autograd.grad((y, s1), keep, (dy, ds1))
    want, big = ref_attention(q, k, v, ld, s0, sc, dy, ds1), majorant(q, k, v, ld, s0, sc, dy, ds1)
    # a state entry or output is a sum over at most L + 2 Dk terms, in chunks; one operand of each product is rounded once
    n = 8 + 2 * max(q.shape[-1], v.shape[-1]) + 128 + 4 * (-(-q.shape[1] // 32))
    op = U16 if dtype == BF else 0.0
    close(y, want[0], big[0], dtype, n, op)
    close(s1, want[1], big[1], F32, n, 0.0)
    for i in range(3):
        close(got[i], want[2 + i], big[2 + i], dtype, n, op)
    if s0 is not None:
        close(got[3], want[5], big[5], F32, n, 0.0)
    ops.check_device_status()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("case", CASES)
def test_attention_and_gradients(case, dtype):
    q, k, v, ld, s0, dy, ds1 = _inputs(*case, dtype, 1)
    _check_all(q, k, v, ld, s0, dy, ds1, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("decay", ["none", "strong", "all"])
def test_attention_at_the_ends_of_the_decay_range(decay, dtype):
    q, k, v, ld, s0, dy, ds1 = _inputs(2, 300, 2, 64, 64, dtype, 2, decay)
    _check_all(q, k, v, ld, s0, dy, ds1, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_without_a_state_and_with_a_scale(dtype):
    q, k, v, ld, _, dy, ds1 = _inputs(1, 200, 2, 64, 80, dtype, 3)
    _check_all(q, k, v, ld, None, dy, ds1, dtype, scale=-1.7)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_reads_strided_and_expanded_operands(dtype):
    B, L, H, D = 2, 150, 4, 64
    g = _gen(4)
    wide = _randn(g, B, L, 3 * H * D + 8, dtype=dtype)
    q, k, v = (wide[..., 8 + i * H * D:8 + (i + 1) * H * D].unflatten(2, (H, D)) for i in range(3))
    _, _, _, ld, s0, dy, ds1 = _inputs(B, L, H, D, D, dtype, 5)
    _check_all(q, k, v, ld, s0, dy, ds1, dtype)
    odd = _randn(g, B, L, 3 * H * D + 5, dtype=dtype)[..., 5:]              # not 16-byte aligned
    q, k, v = (odd[..., i * H * D:(i + 1) * H * D].unflatten(2, (H, D)) for i in range(3))
    _check_all(q, k, v, ld, s0, dy, ds1, dtype)
    head_major = _randn(g, B, H, L, D, dtype=dtype).transpose(1, 2)
    one = _randn(g, B, L, 1, D, dtype=dtype)
    _check_all(head_major, one.expand(B, L, H, D), head_major.flip(1), ld, s0, dy, ds1, dtype)
    across = _randn(g, B, L, D, H, dtype=dtype).transpose(2, 3)            # the head axis is the dense one
    _check_all(across, across, across, ld, s0, dy, ds1, dtype)


def test_shared_key_heads_sum_their_gradients():
    B, L, H, D = 1, 140, 4, 64
    q, k, v, ld, s0, dy, ds1 = _inputs(B, L, H, D, D, F32, 6)
    k1 = k[:, :, :1].clone().requires_grad_(True)
    y = ob.linear_attention(q, k1.expand(B, L, H, D), v, ld, s0)
    got, = torch.autograd.grad(y, k1, dy)
    kk = k1.detach().expand(B, L, H, D)
    want, big = (f(q, kk, v, ld, s0, D ** -0.5, dy) for f in (ref_attention, majorant))
    close(got, want[3].sum(2, keepdim=True), big[3].sum(2, keepdim=True), F32, 400, 0.0)


def test_attention_gradients_agree_with_differences():
    B, L, H, D = 1, 33, 2, 8
    q, k, v, ld, s0, dy, ds1 = _inputs(B, L, H, D, D, F32, 7)
    leaves = [t.requires_grad_(True) for t in (q, k, v, s0)]

    def loss(a):
        y, s = ob.linear_attention(*a[:3], ld, a[3], return_state=True)
        return (y.double() * dy).sum() + (s.double() * ds1).sum()

    grads = torch.autograd.grad(loss(leaves), leaves)
    g = _gen(8)
    for i, t in enumerate(leaves):
        d = _randn(g, *t.shape)
        d = d / d.norm()
        h = 2.0 ** -3                                   # the loss is a polynomial of degree 3 in q, k, v at most: linear in each
        with torch.no_grad():
            up, dn = (loss([x + s * h * d if j == i else x for j, x in enumerate(leaves)]) for s in (1, -1))
        want = float((up - dn) / (2 * h))
        # the two losses are off by about 1e-6 of their absolute sums each, over a step of 2 h
        assert abs(float((grads[i] * d).sum()) - want) <= 2e-3 * max(1.0, abs(want))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_only_one_of_the_two_outputs_is_differentiated(dtype):
    q, k, v, ld, s0, dy, ds1 = _inputs(1, 140, 2, 64, 64, dtype, 9)
    n, op, sc = 8 + 128 + 128 + 20, U16 if dtype == BF else 0.0, 64 ** -0.5
    for through_y in (True, False):
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, s0)]
        y, s1 = ob.linear_attention(*leaves[:3], ld, leaves[3], return_state=True)
        got = torch.autograd.grad(y if through_y else s1, leaves, dy if through_y else ds1, allow_unused=True)
        args = (q, k, v, ld, s0, sc, dy if through_y else None, None if through_y else ds1)
        want, big = ref_attention(*args), majorant(*args)
        for i in range(3):
            close(got[i], want[2 + i], big[2 + i], dtype, n, op)
        close(got[3], want[5], big[5], F32, n, 0.0)


def test_empty_sequences_and_batches():
    for dtype in (BF, F32):
        q, k, v, ld, s0, _, ds1 = _inputs(2, 0, 2, 64, 64, dtype, 10)
        s = s0.clone().requires_grad_(True)
        qq = q.clone().requires_grad_(True)
        y, s1 = ob.linear_attention(qq, k, v, ld, s, return_state=True)
        assert y.shape == (2, 0, 2, 64) and torch.equal(s1, s0)
        gq, gs = torch.autograd.grad((y, s1), (qq, s), (torch.empty_like(y), ds1))
        assert gq.shape == q.shape and torch.equal(gs, ds1)
        _, z = ob.linear_attention(q, k, v, ld, return_state=True)
        assert z.shape == s0.shape and not bool(z.any())
        e = [t[:0] for t in (q, k, v)]
        y, s1 = ob.linear_attention(*e, ld, s0[:0], return_state=True)
        assert y.shape == (0, 0, 2, 64) and s1.shape == (0, 2, 64, 64)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_split_sequence_equals_the_whole(dtype):
    q, k, v, ld, s0, _, _ = _inputs(1, 700, 2, 128, 128, dtype, 11)
    y, s1 = ob.linear_attention(q, k, v, ld, s0, return_state=True)
    a, s = ob.linear_attention(q[:, :333], k[:, :333], v[:, :333], ld, s0, return_state=True)
    b, s = ob.linear_attention(q[:, 333:], k[:, 333:], v[:, 333:], ld, s, return_state=True)
    big = majorant(q, k, v, ld, s0, 128 ** -0.5)
    close(torch.cat([a, b], 1), y.double(), 2 * big[0], dtype, 600, U16 if dtype == BF else 0.0)
    close(s, s1.double(), 2 * big[1], F32, 600, 0.0)


# many heads (a CTA walks a whole head), few heads and long sequences (segments, joined), both; odd lengths, narrow and wide heads
SPREADS = [(5, 300, 40, 128, 96), (4, 130, 37, 64, 128), (1, 2001, 2, 128, 128), (2, 1300, 9, 40, 128), (1, 4099, 1, 128, 64),
           (2, 1025, 37, 128, 128)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("case", SPREADS)
def test_attention_spread_over_the_gpu_in_other_ways(case, dtype):
    q, k, v, ld, s0, dy, ds1 = _inputs(*case, dtype, 51)
    _check_all(q, k, v, ld, s0, dy, ds1, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("decay", ["none", "strong", "all"])
def test_joined_segments_at_the_ends_of_the_decay_range(decay, dtype):
    q, k, v, ld, s0, dy, ds1 = _inputs(1, 1999, 2, 128, 72, dtype, 52, decay)
    before = ops.LAUNCHES
    ob.linear_attention(q, k, v, ld, s0)
    assert ops.LAUNCHES - before == 3                                              # it is split: shares, join, walk
    _check_all(q, k, v, ld, s0, dy, ds1, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_decays_on_either_side_of_one_half(dtype):
    q, k, v, _, s0, dy, ds1 = _inputs(1, 700, 6, 96, 128, dtype, 54)
    ld = torch.tensor([-0.1, -0.69314, -0.69316, -0.8, -2.0, -5.0], device=DEV)
    _check_all(q, k, v, ld, s0, dy, ds1, dtype)


@pytest.mark.parametrize("case", [(3, 1, 2, 96, 32), (2, 2, 1, 72, 128), (1, 17, 3, 64, 64), (2, 32, 2, 128, 128)])
def test_short_sequences_are_rounded_once(case):
    """Without a state, up to 32 tokens: scores in two bfloat16 parts, off by 2^-16, and their decays by 2^-17 at most."""
    q, k, v, ld, _, dy, _ = _inputs(*case, BF, 55)
    sc = case[3] ** -0.5
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    y = ob.linear_attention(*leaves, ld)
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    zero = torch.zeros(case[0], case[2], case[4], case[3], device=DEV)
    want, big = ref_attention(q, k, v, ld, None, sc, dy, zero), majorant(q, k, v, ld, None, sc, dy, zero)
    for i, j in enumerate((0, 2, 3, 4)):
        close(got[i], want[j], big[j], BF, 8 + 2 * 128 + 128, 2.0 ** -16 + 2.0 ** -17)


def test_one_token_is_the_step():
    for dtype in (BF, F32):
        q, k, v, ld, s0, _, _ = _inputs(3, 1, 4, 72, 128, dtype, 53)
        y, s1 = ob.linear_attention(q, k, v, ld, s0, return_state=True)
        z, s2 = ob.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0)
        big = majorant(q, k, v, ld, s0, 72 ** -0.5)
        close(y[:, 0], z.double(), 2 * big[0][:, 0], dtype, 300, U16 if dtype == BF else 0.0)
        close(s1, s2.double(), 2 * big[1], F32, 300, 0.0)
        wide = torch.cat([v, v], 3)[..., :128]                                     # strided rows of one token
        a, b = ob.linear_attention(q, k, wide, ld, s0, return_state=True)
        assert torch.equal(a, y) and torch.equal(b, s1)


def test_rows_of_other_sequences_do_not_matter_and_repeats_are_bitwise():
    q, k, v, ld, s0, dy, ds1 = _inputs(3, 400, 2, 128, 128, BF, 12)

    def run(rows):
        leaves = [t[rows].detach().clone().requires_grad_(True) for t in (q, k, v, s0)]
        y, s1 = ob.linear_attention(*leaves[:3], ld, leaves[3], return_state=True)
        return [y, s1, *torch.autograd.grad((y, s1), leaves, (dy[rows], ds1[rows]))]

    whole, again = run(slice(0, 3)), run(slice(0, 3))
    assert all(torch.equal(a, b) for a, b in zip(whole, again))


STEP_CASES = [(1, 1, 128, 128), (3, 5, 64, 128), (2, 3, 32, 40), (2, 2, 72, 33), (1, 2, 7, 5), (2, 1, 256, 256), (129, 2, 128, 128)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("case", STEP_CASES)
def test_step(case, dtype):
    B, H, Dk, Dv = case
    q, k, v, ld, s0, _, _ = _inputs(B, 1, H, Dk, Dv, dtype, 13)
    want, big = (f(q, k, v, ld, s0, Dk ** -0.5) for f in (ref_attention, majorant))
    y, s1 = ob.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0)
    close(y, want[0][:, 0], big[0][:, 0], dtype, Dk + 8, 0.0)
    close(s1, want[1], big[1], F32, 8, 0.0)
    inplace = s0.clone()
    y2, s2 = ob.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, inplace, out_state=inplace)
    assert s2 is inplace and torch.equal(s2, s1) and torch.equal(y2, y)
    wide = torch.cat([q[:, 0], k[:, 0], v[:, 0]], -1)                       # strided heads
    y3, s3 = ob.linear_attention_step(wide[..., :Dk], wide[..., Dk:2 * Dk], wide[..., 2 * Dk:], ld, s0)
    assert torch.equal(y3, y) and torch.equal(s3, s1)


def test_steps_follow_the_sequence():
    q, k, v, ld, s0, _, _ = _inputs(2, 40, 2, 64, 64, F32, 14)
    y, s1 = ob.linear_attention(q, k, v, ld, s0, return_state=True)
    s, ys = s0, []
    for t in range(40):
        yt, s = ob.linear_attention_step(q[:, t], k[:, t], v[:, t], ld, s)
        ys.append(yt)
    big = majorant(q, k, v, ld, s0, 64 ** -0.5)
    close(torch.stack(ys, 1), y.double(), 2 * big[0], F32, 400, 0.0)
    close(s, s1.double(), 2 * big[1], F32, 400, 0.0)


# ---------------------------------------------------------------------------------------------------------------------
#  block norm
# ---------------------------------------------------------------------------------------------------------------------
def ref_block(x, h, gate, scale, post, pre, eps):
    rms = lambda t: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps)  # noqa: E731
    u = h if post is None else rms(h) * post
    m = u if gate is None else u * torch.sigmoid(gate)
    r = x + (m if scale is None else scale * m)
    return r, None if pre is None else rms(r) * pre


BLOCK_SHAPES = [(1, 8), (3, 64), (5, 100), (2, 7), (33, 256), (700, 512), (64, 1000), (130, 2048), (7, 4096), (3, 8192), (2, 9000), (1, 1)]
BLOCK_FLAGS = [(True, True, True, True), (False, True, True, True), (True, False, True, True), (False, False, True, True),
               (True, True, False, True), (True, True, True, False), (False, False, False, True), (False, False, False, False)]


def _block_inputs(M, D, dtype, flags, seed):
    g = _gen(seed)
    gate, scale, post, pre = flags
    x, h = _randn(g, M, D, dtype=dtype, std=2.0), _randn(g, M, D, dtype=dtype)
    vec = lambda on: (0.5 + 0.3 * torch.randn(D, generator=g)).to(DEV) if on else None  # noqa: E731
    return x, h, _randn(g, M, D, dtype=dtype) if gate else None, vec(scale), vec(post), vec(pre), \
        _randn(g, M, D, dtype=dtype), _randn(g, M, D, dtype=dtype) if pre else None


def _check_block(ins, dr, dn, dtype, eps=1e-5, lay=lambda t: t):
    leaves = [None if t is None else lay(t.detach().clone()).requires_grad_(True) for t in ins]
    r, n = ob.block_norm(leaves[0], leaves[1], gate=leaves[2], scale=leaves[3], post_weight=leaves[4], pre_weight=leaves[5], eps=eps)
    outs, douts = ((r, n), (dr, dn)) if n is not None else ((r,), (dr,))
    got = torch.autograd.grad(outs, [t for t in leaves if t is not None], douts)
    ref = [None if t is None else t.detach().double().requires_grad_(True) for t in ins]
    rr, rn = ref_block(*ref, eps)
    want = torch.autograd.grad((rr, rn) if n is not None else (rr,), [t for t in ref if t is not None], [d.double() for d in douts])
    # absolute sums of the terms that meet in each result (float64): a result is off by at most n u32 of them, n the roundings
    # on the longest path: row sums of D terms (twice), column sums of M terms, and fewer than 64 products, roots and sigmoids
    M, D = ins[0].shape
    x, h, gate, scale, post, pre = (None if t is None else t.detach().double() for t in ins)
    one = torch.ones(D, device=DEV, dtype=torch.float64)
    rms = lambda t: torch.rsqrt(t.square().mean(-1, keepdim=True) + eps)  # noqa: E731
    rs_h = rms(h) if post is not None else 1.0
    sig = 1.0 if gate is None else torch.sigmoid(gate)
    s, wo = one if scale is None else scale.abs(), one if post is None else post.abs()
    hh = (h * rs_h).abs()
    Ar = x.abs() + s * wo * hh * sig
    A = dr.double().abs()
    if pre is not None:
        rs_r = rms(rr.detach())
        rh, w = Ar * rs_r, dn.double().abs() * pre.abs()
        A = A + rs_r * (w + rh * (w * rh).mean(-1, keepdim=True))
    t = A * s * wo * sig
    n = (4 * D + 64) * U32
    assert bool(((r.double() - rr).abs() <= U[dtype] * rr.abs() + n * Ar).all())
    if pre is not None:
        assert bool((((ob_n := outs[1]).double() - rn).abs() <= U[dtype] * rn.abs() + n * rh * pre.abs()).all()), ob_n.shape
    big = [A, t if post is None else rs_h * (t + hh * (t * hh).mean(-1, keepdim=True)), t * hh,
           (A * wo * hh * sig).sum(0), (A * s * hh * sig).sum(0), None if pre is None else (dn.double().abs() * rh).sum(0)]
    left, want = list(got), list(want)
    for i, leaf in enumerate(ins):
        if leaf is None:
            continue
        a, b = left.pop(0), want.pop(0)
        assert a.dtype == leaf.dtype and a.shape == leaf.shape
        err, lim = (a.double() - b).abs(), (U[leaf.dtype] * b.abs() + (n + (M * U32 if i > 2 else 0)) * big[i] + 1e-30)
        assert bool((err <= lim).all()), (i, float((err / lim).max()))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", BLOCK_SHAPES)
def test_block_norm(shape, dtype):
    *ins, dr, dn = _block_inputs(*shape, dtype, BLOCK_FLAGS[0], 20)
    _check_block(ins, dr, dn, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("flags", BLOCK_FLAGS)
@pytest.mark.parametrize("shape", [(37, 256), (9, 100)])
def test_block_norm_without_some_factors(shape, flags, dtype):
    *ins, dr, dn = _block_inputs(*shape, dtype, flags, 21)
    _check_block(ins, dr, dn, dtype)


def test_block_norm_reads_column_slices():
    g = _gen(22)
    for off in (8, 3):                                    # aligned rows, and rows that only the scalar kernels can read
        wide = _randn(g, 40, 3 * 128 + 16, dtype=BF)
        x, h, gate = (wide[:, off + i * 128:off + (i + 1) * 128] for i in range(3))
        scale, post, pre = (_randn(g, 128) for _ in range(3))
        want = ob.block_norm(x.contiguous(), h.contiguous(), gate=gate.contiguous(), scale=scale, post_weight=post, pre_weight=pre)
        got = ob.block_norm(x, h, gate=gate, scale=scale, post_weight=post, pre_weight=pre)
        for a, b in zip(got, want):
            assert float((a.double() - b.double()).abs().max()) <= 2 * U16 * float(b.abs().max())
        t3 = wide.view(4, 10, -1)[..., off:off + 128]
        assert ob.block_norm(t3, t3, pre_weight=pre)[1].shape == t3.shape


def test_block_norm_of_nothing_and_of_zeros():
    z = torch.zeros(0, 64, device=DEV, dtype=BF, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    r, n = ob.block_norm(z, z, scale=w, post_weight=w, pre_weight=w)
    gz, gw = torch.autograd.grad((r, n), (z, w), (torch.zeros_like(r), torch.zeros_like(n)))
    assert r.shape == n.shape == (0, 64) and not bool(gw.any())
    x = torch.zeros(3, 64, device=DEV, requires_grad=True)
    r, n = ob.block_norm(x, x, gate=x, post_weight=w, pre_weight=w)         # rows of zeros: rsqrt(eps), finite gradients
    g = torch.autograd.grad((r, n), (x, w), (torch.ones_like(r), torch.ones_like(n)))
    assert not bool(r.any()) and all(bool(torch.isfinite(t).all()) for t in g)


def test_block_norm_gradient_of_one_output_alone():
    *ins, dr, dn = _block_inputs(11, 256, F32, BLOCK_FLAGS[0], 23)
    for pick in (0, 1):
        leaves = [t.detach().clone().requires_grad_(True) for t in ins]
        out = ob.block_norm(leaves[0], leaves[1], gate=leaves[2], scale=leaves[3], post_weight=leaves[4], pre_weight=leaves[5])[pick]
        got = torch.autograd.grad(out, leaves, (dr, dn)[pick], allow_unused=True)
        ref = [t.detach().double().requires_grad_(True) for t in ins]
        want = torch.autograd.grad(ref_block(*ref, 1e-5)[pick], ref, (dr, dn)[pick].double(), allow_unused=True)
        for a, b in zip(got, want):
            b = torch.zeros_like(a, dtype=torch.float64) if b is None else b
            a = torch.zeros_like(b) if a is None else a
            assert float((a.double() - b).abs().max()) <= 1e-4 * max(1.0, float(b.abs().max()))


# ---------------------------------------------------------------------------------------------------------------------
#  activations in eight bits
# ---------------------------------------------------------------------------------------------------------------------
def ref_pack(x):
    """Restored values in float64: the least step 2^e >= 2^-126 under which the group's largest rounds to 127 or less."""
    D = x.shape[-1]
    xd = x.double().cpu().reshape(-1, D)
    out = torch.empty_like(xd)
    for c in range(0, D, 32):
        g = xd[:, c:c + 32]
        fin = torch.where(torch.isfinite(g), g, 0.0)
        top = fin.abs().amax(-1, keepdim=True)
        e = torch.full_like(top, -126.0)
        for _ in range(300):
            e = torch.where(torch.round(top * torch.exp2(-e)) > 127, e + 1, e)
        top = torch.where(e == 122, 63.0, 127.0)                                    # 64 steps of 2^122 would be infinite
        q = torch.minimum(torch.maximum(torch.round(g * torch.exp2(-e)), -top), top)
        out[:, c:c + 32] = torch.where(torch.isfinite(g), q * torch.exp2(e), float("nan"))
    return out.reshape(x.shape)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 96), (4, 3, 100), (2, 2, 2048), (129, 512), (1, 4099), (64,)])
def test_pack_is_the_definition(shape, dtype):
    g = _gen(30)
    x = _randn(g, *shape) * torch.exp2(torch.randint(-30, 30, shape, generator=g).float()).to(DEV)
    x = x.to(dtype)
    p = ob.pack_activation(x)
    y = ob.unpack_activation(p)
    assert p.q.dtype == torch.int8 and p.q.shape == x.shape and y.dtype == dtype
    assert torch.equal(y.double().cpu(), ref_pack(x))
    assert torch.equal(ob.unpack_activation(p, F32).double(), y.double())           # exact in either type
    again = ob.pack_activation(y)
    assert torch.equal(ob.unpack_activation(again), y)                              # nothing is lost twice


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 50])
def test_pack_at_the_ends_of_the_range(D, dtype):
    big = torch.finfo(dtype).max
    rows = [torch.zeros(D), torch.full((D,), big), torch.full((D,), -big), torch.full((D,), 2.0 ** -140), torch.full((D,), 2.0 ** -127),
            torch.linspace(-1, 1, D) * 2.0 ** -120, torch.linspace(-127.5, 127.5, D), torch.full((D,), 127.5)]
    x = torch.stack(rows).to(dtype).to(DEV)
    assert torch.equal(ob.unpack_activation(ob.pack_activation(x)).double().cpu(), ref_pack(x))
    x[1, 3], x[2, 5], x[5, 7] = float("nan"), float("inf"), float("-inf")
    got, want = ob.unpack_activation(ob.pack_activation(x)).double().cpu(), ref_pack(x)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def test_pack_reads_strided_rows():
    x = _randn(_gen(31), 6, 300, dtype=BF)
    for view in (x[:, 8:200], x[:, 3:99], x[::2], x.t(), x.view(2, 3, 300)[:, :, 32:96]):
        got = ob.unpack_activation(ob.pack_activation(view))
        assert got.shape == view.shape and torch.equal(got, ob.unpack_activation(ob.pack_activation(view.contiguous())))
    assert ob.unpack_activation(ob.pack_activation(x[:0])).shape == (0, 300)


# ---------------------------------------------------------------------------------------------------------------------
#  the two ways to a launch
# ---------------------------------------------------------------------------------------------------------------------
def test_native_host_calls_and_the_python_way_give_the_same_bits():
    g = _gen(40)
    for dtype in (BF, F32):
        q, k, v, ld, s0, dy, ds1 = _inputs(2, 300, 2, 64, 72, dtype, 41)
        x, w = _randn(g, 5, 7, 96, dtype=dtype), _randn(g, 96)

        def run():
            leaves = [t.clone().requires_grad_(True) for t in (q, k, v, s0)]
            y, s = ob.linear_attention(*leaves[:3], ld, leaves[3], return_state=True)
            out = [y, s, *torch.autograd.grad((y, s), leaves, (dy, ds1))]
            with torch.no_grad():
                out += ob.linear_attention(q, k, v, ld, s0, scale=0.3, return_state=True)
                out += ob.linear_attention_step(q[:, 0].contiguous(), k[:, 0].contiguous(), v[:, 0].contiguous(), ld, s0)
                out += ob.block_norm(x, x, gate=x, scale=w, post_weight=w, pre_weight=w)
                out.append(ob.block_norm(x, x)[0])
                p = ob.pack_activation(x)
                out += [p.q, p.exponent, ob.unpack_activation(p), ob.unpack_activation(p, F32)]
            return out

        native = run()
        launches = ops.LAUNCHES
        run()
        launches = ops.LAUNCHES - launches
        timed = []
        ops.set_timing(timed)                             # a timed region takes the Python way
        try:
            before = ops.LAUNCHES
            python = run()
            assert ops.LAUNCHES - before == launches and timed
        finally:
            ops.set_timing(None)
        assert len(native) == len(python) and all(torch.equal(a, b) for a, b in zip(native, python))


@pytest.mark.parametrize("dtype", (BF, F32))
def test_block_norm_gradients_on_either_host_way_are_the_same_bits(dtype):
    g = _gen(43)
    x, h, z, dr, dn = (_randn(g, 3, 11, 72, dtype=dtype) for _ in range(5))
    s, wo, wi = (_randn(g, 72) for _ in range(3))

    def run(gate, post, scale, need):
        ins = [t.clone().requires_grad_(i in need) for i, t in enumerate((x, h, z, s, wo, wi))]
        a = [ins[0], ins[1], ins[2] if gate else None, ins[3] if scale else None, ins[4] if post else None, ins[5]]
        r, n = ob.block_norm(a[0], a[1], gate=a[2], scale=a[3], post_weight=a[4], pre_weight=a[5])
        leaves = [t for t in a if t is not None and t.requires_grad]
        out = [r, n, *torch.autograd.grad((r, n), leaves, (dr, dn), retain_graph=True)]
        out += torch.autograd.grad(n, leaves, dn, retain_graph=True, allow_unused=True)
        return out + list(torch.autograd.grad(r, leaves, dr[:, :1].expand_as(r), allow_unused=True))

    for gate, post, scale in itertools.product((True, False), repeat=3):
        for need in ((0, 1, 2, 3, 4, 5), (0, 1, 2), (3, 4, 5), (1,)):
            before = ops.LAUNCHES
            native = run(gate, post, scale, need)
            launches = ops.LAUNCHES - before
            ops.set_timing([])                            # a timed region takes the Python way
            try:
                before = ops.LAUNCHES
                python = run(gate, post, scale, need)
                assert ops.LAUNCHES - before == launches
            finally:
                ops.set_timing(None)
            for a, b in zip(native, python, strict=True):
                assert (a is None) == (b is None) and (a is None or torch.equal(a, b))


def test_a_state_written_in_place_is_seen_by_a_graph_that_kept_it():
    q, k, v, ld, s0, _, _ = _inputs(1, 70, 2, 64, 64, F32, 44)
    y = ob.linear_attention(q.requires_grad_(True), k, v, ld, s0)
    with torch.no_grad():
        ob.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0, out_state=s0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        s = s0.clone()
        z, new = ob.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s, out_state=s)
        want, _ = ob.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0)
        assert new is s and torch.equal(z, want)


def test_running_out_of_memory_keeps_its_type():
    x = torch.zeros(1 << 22, 32, device=DEV, dtype=BF)                     # its codes would take 128 MB
    torch.cuda.empty_cache()
    free = torch.cuda.memory_reserved() + (64 << 20)
    torch.cuda.set_per_process_memory_fraction(free / torch.cuda.get_device_properties(0).total_memory)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            ob.pack_activation(x)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert ob.pack_activation(x).q.shape == x.shape


def test_calls_on_tensors_of_another_type_or_place_are_refused_on_the_gpu_too():
    q, k, v, ld, s0, _, _ = _inputs(1, 4, 2, 8, 8, F32, 42)
    with pytest.raises(ValueError, match="one dtype"):
        ob.linear_attention(q, k.to(BF), v, ld)
    with pytest.raises(ValueError, match="CPU tensor|one device"):
        ob.linear_attention(q, k.cpu(), v, ld)
    with pytest.raises(ValueError, match="CPU tensor|one device"):
        ob.block_norm(q, q, pre_weight=torch.ones(8))
    with pytest.raises(ValueError, match="scale must be finite"):
        ob.linear_attention(q, k, v, ld, scale=float("inf"))
    with pytest.raises(ValueError, match="gradients are not served"):
        ob.linear_attention_step(q[:, 0].clone().requires_grad_(True), k[:, 0], v[:, 0], ld, s0)
    with pytest.raises(ValueError, match="out_state"):
        ob.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0, out_state=s0[:, :1])
    both = torch.zeros(3, 2, 8, 8, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        ob.linear_attention_step(*(t[:, 0].expand(2, 2, 8) for t in (q, k, v)), ld, both[:2], out_state=both[1:])
    with pytest.raises(RuntimeError, match="second-order"):
        qq = q.clone().requires_grad_(True)
        g, = torch.autograd.grad(ob.linear_attention(qq, k, v, ld).sum(), qq, create_graph=True)
        g.sum().backward()
