"""-m gpu: linear attention and block norms on operands that really lie as their case says: the leaves are the views themselves, and
each test asserts their strides and alignment before the call.  Bounds are those of the plain float64 restatements of
test_gpu_block_operators.py."""
import pytest
import torch

import orbitssm_b200 as ob
from orbitssm_b200 import ops
from test_gpu_block_operators import BF, BLOCK_FLAGS, DEV, F32, U, U16, U32, _block_inputs, _check_block, _gen, _inputs, _randn, close, \
    majorant, ref_attention

pytestmark = pytest.mark.gpu


def _attention(q, k, v, ld, s0, dy, ds1, dtype):
    """Forward, state and gradients of the views as they are; their neighbours in memory stay as they were."""
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (q, k, v, s0)]
    for a, b in zip(leaves, (q, k, v, s0)):
        assert a is None or (a.data_ptr() == b.data_ptr() and a.stride() == b.stride())
    y, s1 = ob.linear_attention(*leaves[:3], ld, leaves[3], return_state=True)
    got = torch.autograd.grad((y, s1), [t for t in leaves if t is not None], (dy, ds1))
    sc = q.shape[-1] ** -0.5
    want, big = ref_attention(q, k, v, ld, s0, sc, dy, ds1), majorant(q, k, v, ld, s0, sc, dy, ds1)
    n = 8 + 2 * max(q.shape[-1], v.shape[-1]) + 128 + 4 * (-(-q.shape[1] // 32))
    op = U16 if dtype == BF else 0.0
    close(y, want[0], big[0], dtype, n, op)
    close(s1, want[1], big[1], F32, n, 0.0)
    for i in range(3):
        assert got[i].shape == (q, k, v)[i].shape
        close(got[i], want[2 + i], big[2 + i], dtype, n, op)
    if s0 is not None:
        close(got[3], want[5], big[5], F32, n, 0.0)
    with torch.no_grad():                                # the way without a node takes the same operands
        y2, s2 = ob.linear_attention(q, k, v, ld, s0, return_state=True)
    assert torch.equal(y2, y) and torch.equal(s2, s1)
    ops.check_device_status()


def _columns(g, B, L, H, D, dtype, first, width):
    """q, k, v as column ranges of one buffer whose rows are `width` elements."""
    wide = _randn(g, B, L, width, dtype=dtype)
    return wide, [wide[..., first + i * H * D:first + (i + 1) * H * D].unflatten(2, (H, D)) for i in range(3)]


B, L, H, D = 2, 150, 4, 64


def _rest(dtype, seed):
    _, _, _, ld, s0, dy, ds1 = _inputs(B, L, H, D, D, dtype, seed)
    return ld, s0, dy, ds1


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("first,extra", [(8, 8), (5, 5), (0, 1), (4, 4)])
def test_attention_of_column_ranges(first, extra, dtype):
    wide, (q, k, v) = _columns(_gen(4), B, L, H, D, dtype, first, 3 * H * D + extra)
    es = q.element_size()
    assert q.stride() == (L * wide.shape[2], wide.shape[2], D, 1) and not q.is_contiguous()
    assert (q.data_ptr() % 16 == 0 and wide.shape[2] * es % 16 == 0) == (first * es % 16 == 0 and extra * es % 16 == 0)
    before = wide.clone()
    _attention(q, k, v, *_rest(dtype, 5), dtype)
    assert torch.equal(wide, before)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_of_other_orders_of_the_axes(dtype):
    g = _gen(6)
    head_major = _randn(g, B, H, L, D, dtype=dtype).transpose(1, 2)
    time_major = _randn(g, L, B, H, D, dtype=dtype).transpose(0, 1)
    across = _randn(g, B, L, D, H, dtype=dtype).transpose(2, 3)              # the head axis is the dense one
    assert head_major.stride(2) == L * D and time_major.stride(0) == H * D and across.stride(3) == H
    _attention(head_major, time_major, across, *_rest(dtype, 7), dtype)
    _attention(across, head_major, time_major, *_rest(dtype, 8), dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_of_expanded_and_overlapping_operands(dtype):
    g = _gen(9)
    one_head = _randn(g, B, L, 1, D, dtype=dtype).expand(B, L, H, D)
    one_row = _randn(g, 1, L, H, D, dtype=dtype).expand(B, L, H, D)
    one_token = _randn(g, B, 1, H, D, dtype=dtype).expand(B, L, H, D)
    assert one_head.stride(2) == 0 and one_row.stride(0) == 0 and one_token.stride(1) == 0
    _attention(one_head, one_row, one_token, *_rest(dtype, 10), dtype)
    line = _randn(g, 8 * (B * L * H + 32), dtype=dtype)
    for step in (8, 4):                                                      # windows that share most of their elements
        w = line.as_strided((B, L, H, D), (L * H * step, H * step, step, 1))
        _attention(w, w, w, *_rest(dtype, 11), dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_of_strided_states_decays_and_output_gradients(dtype):
    q, k, v, ld, s0, dy, ds1 = _inputs(B, L, H, D, D, dtype, 12)
    s0, ds1 = s0.transpose(2, 3), ds1.transpose(0, 1).contiguous().transpose(0, 1)
    ld = torch.stack([ld, ld], 1)[:, 0]
    assert not s0.is_contiguous() and not ds1.is_contiguous() and ld.stride(0) == 2
    for g in (dy[:, :1].expand_as(dy), dy.transpose(1, 2).contiguous().transpose(1, 2), torch.cat([dy, dy], 3)[..., 3:3 + D]):
        assert not g.is_contiguous()
        _attention(q, k, v, ld, s0, g, ds1, dtype)


def test_sequences_of_a_batch_do_not_see_each_other():
    q, k, v, ld, s0, dy, ds1 = _inputs(3, 400, 2, 128, 128, BF, 12)

    def run(rows):
        leaves = [t[rows].detach().requires_grad_(True) for t in (q, k, v, s0)]
        y, s1 = ob.linear_attention(*leaves[:3], ld, leaves[3], return_state=True)
        return [y, s1, *torch.autograd.grad((y, s1), leaves, (dy[rows], ds1[rows]))]

    whole, parts = run(slice(0, 3)), zip(run(slice(0, 1)), run(slice(1, 3)), strict=True)
    m = majorant(q, k, v, ld, s0, 128 ** -0.5, dy, ds1)
    for i, (got, (a, b)) in enumerate(zip(whole, parts, strict=True)):
        state = i in (1, 5)                              # either may be spread over the GPU in its own way: twice the bound of one
        close(torch.cat([a, b]), got.double(), 2 * m[i], F32 if state else BF, 600, 0.0 if state else U16)
    # a row of another sequence that is not finite stays there
    bad = [t.clone() for t in (q, k, v)]
    for t in bad:
        t[1, 7] = float("nan")
    y, s1 = ob.linear_attention(*bad, ld, s0, return_state=True)
    assert torch.equal(y[::2], whole[0][::2]) and torch.equal(s1[::2], whole[1][::2]) and bool(torch.isnan(y[1]).any())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(40, 128), (33, 100), (9, 2048)])
@pytest.mark.parametrize("offset,gap", [(8, 8), (3, 5), (0, 1)])
def test_block_norm_gradients_of_column_slices(shape, offset, gap, dtype):
    *ins, dr, dn = _block_inputs(*shape, dtype, BLOCK_FLAGS[0], 60)
    M, D2 = shape
    seen = []

    def lay(t):
        if t.dim() == 1:
            return t
        wide = torch.full((M, offset + D2 + gap), 7.0, device=DEV, dtype=dtype)
        view = wide[:, offset:offset + D2]
        view.copy_(t)
        assert view.stride() == (wide.shape[1], 1) and view.data_ptr() == wide.data_ptr() + offset * t.element_size()
        seen.append(view)
        return view

    _check_block(ins, dr, dn, dtype, lay=lay)
    assert len(seen) == 3
    # gradients that lie the same way, or repeat one row
    for give in (lay, lambda t: t[:1].expand_as(t)):
        leaves = [t.detach().clone().requires_grad_(True) for t in ins]
        r, n = ob.block_norm(leaves[0], leaves[1], gate=leaves[2], scale=leaves[3], post_weight=leaves[4], pre_weight=leaves[5])
        a, b = give(dr), give(dn)
        assert not a.is_contiguous()
        got = torch.autograd.grad((r, n), leaves, (a, b), retain_graph=True)
        want = torch.autograd.grad((r, n), leaves, (a.contiguous(), b.contiguous()))
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_block_norm_of_other_views(dtype):
    g = _gen(61)
    pre = _randn(g, 96)
    wide = _randn(g, 4, 10, 200, dtype=dtype)
    views = [wide[..., 8:104], wide[..., 3:99], wide[::2, 1::3, 8:104], wide.transpose(0, 1)[..., 8:104], wide[:, :1, 8:104].expand(4, 10, 96),
             wide[..., :192:2], wide[0, 0, 8:104]]
    for v in views:
        assert v.shape[-1] == 96
        c = v.contiguous()
        for a, b in zip(ob.block_norm(v, v, gate=v, pre_weight=pre), ob.block_norm(c, c, gate=c, pre_weight=pre)):
            # (rows may go to the kernel of aligned vectors or to the scalar one: sums of 96 terms in another order)
            assert a.shape == v.shape and bool(((a.double() - b.double()).abs() <= (2 * U[dtype] + 400 * U32) * b.double().abs() + 1e-6).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(300, 5120), (301, 8192), (299, 9001), (400, 4104)])
def test_block_norm_of_many_wide_rows(shape, dtype):
    """More rows than CTAs: the column sums of a CTA run over several rows."""
    *ins, dr, dn = _block_inputs(*shape, dtype, BLOCK_FLAGS[0], 62)
    _check_block(ins, dr, dn, dtype)
