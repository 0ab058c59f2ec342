"""-m gpu: where bfloat16 linear attention rounds.  A row's error is a matter of where the row stands, not of how many tokens the call
holds: what a pass begins with (the first 32 tokens for y and dq, for dk and dv the last 32 as far as they lie in the last chunk of
128) is rounded once, as a call of up to 32 tokens is and as the single-token step is."""
import pytest
import torch

import orbitssm_b200 as ob
from orbitssm_b200 import ops
from test_gpu_block_operators import BF, DEV, _inputs, close, majorant, ref_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("decay", [None, "strong", "fast"])
@pytest.mark.parametrize("case", [(2, 33, 2, 128, 128), (1, 40, 3, 64, 96), (2, 64, 1, 72, 128), (1, 97, 2, 128, 64), (1, 128, 2, 128, 128),
                                  (1, 129, 2, 96, 32), (1, 166, 2, 64, 64), (1, 300, 40, 128, 96), (1, 1999, 2, 128, 72), (3, 400, 2, 128, 128)])
def test_the_rows_that_a_pass_begins_with_are_rounded_once(case, decay):
    B, L, H, Dk, Dv = case
    q, k, v, ld, _, dy, _ = _inputs(*case, BF, 55, "span" if decay is None else "strong")
    if decay == "fast":                                  # a little below and above one half, where the tiles change their way
        ld = torch.tensor([-0.6, -0.8], device=DEV).repeat(H)[:H]
    sc = Dk ** -0.5
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    y = ob.linear_attention(*leaves, ld)
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    zero = torch.zeros(B, H, Dv, Dk, device=DEV)
    want, big = ref_attention(q, k, v, ld, None, sc, dy, zero), majorant(q, k, v, ld, None, sc, dy, zero)
    head, tail = slice(0, 32), slice(-min(32, (L - 1) % 128 + 1), None)
    for i, (j, rows) in enumerate(((0, head), (2, head), (3, tail), (4, tail))):
        # scores in two bfloat16 parts: off by 2^-16, their decays (at most 64 products) by 2^-17
        close(got[i][:, rows], want[j][:, rows], big[j][:, rows], BF, 8 + 2 * 128 + 128, 2.0 ** -16 + 2.0 ** -17)
    ops.check_device_status()


def test_tokens_after_a_row_do_not_change_it():
    q, k, v, ld, _, _, _ = _inputs(1, 64, 2, 128, 128, BF, 56)
    whole = ob.linear_attention(q, k, v, ld)
    for n in (1, 2, 31, 32, 33):
        assert torch.equal(ob.linear_attention(q[:, :n], k[:, :n], v[:, :n], ld)[:, :32], whole[:, :min(n, 32)])


@pytest.mark.parametrize("scale", [1e-30, 2.0 ** -41, 2.0 ** -40, -2.0 ** -39, 2.0 ** 40, -2.0 ** 41, 1e20, 1e30])
@pytest.mark.parametrize("L", [20, 200])
def test_any_scale_that_float32_holds(L, scale):
    q, k, v, _, s0, dy, ds1 = _inputs(1, L, 3, 64, 72, BF, 57)
    ld = torch.tensor([-0.69, -0.8, -0.01], device=DEV)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, s0)]
    y, s1 = ob.linear_attention(*leaves[:3], ld, leaves[3], scale=scale, return_state=True)
    got = [y, s1, *torch.autograd.grad((y, s1), leaves, (dy, ds1))]
    want, big = ref_attention(q, k, v, ld, s0, scale, dy, ds1), majorant(q, k, v, ld, s0, scale, dy, ds1)
    for i, (a, b, m) in enumerate(zip(got, want, big, strict=True)):
        u, op = (2.0 ** -24, 0.0) if i in (1, 5) else (2.0 ** -8, 2.0 ** -8)
        # the bound of the other tests, in the units of the largest sum: at 1e-30 their absolute slack would hide a result of zeros
        unit = float(m.max())
        err = (a.double() - b).abs() / unit
        assert bool((err <= (u * b.abs() + (op + 600 * 2.0 ** -24) * m) / unit).all()), i
    ops.check_device_status()


@pytest.mark.parametrize("powers", [(0, 0, -60, 0), (0, 0, 0, -60), (0, 0, 80, 0), (0, 0, 0, 80), (20, 20, 20, 20), (-20, -20, -20, -20)])
def test_values_far_from_one(powers):
    """Every head takes its decays without leaving the range of float32 where the operator's own terms are in it."""
    L, H, D = 200, 6, 64
    q, k, v, _, s0, dy, ds1 = _inputs(1, L, H, D, D, BF, 58)
    ld = torch.tensor([-0.01, -0.2, -0.3465, -0.3467, -0.5, -0.69], device=DEV)
    q, k, v, dy = (t * 2.0 ** e for t, e in zip((q, k, v, dy), powers))
    s0, ds1 = s0 * 2.0 ** (powers[1] + powers[2]), ds1 * 2.0 ** (powers[0] + powers[3])
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, s0)]
    y, s1 = ob.linear_attention(*leaves[:3], ld, leaves[3], return_state=True)
    got = [y, s1, *torch.autograd.grad((y, s1), leaves, (dy, ds1))]
    want, big = ref_attention(q, k, v, ld, s0, D ** -0.5, dy, ds1), majorant(q, k, v, ld, s0, D ** -0.5, dy, ds1)
    for i, (a, b, m) in enumerate(zip(got, want, big, strict=True)):
        u, op = (2.0 ** -24, 0.0) if i in (1, 5) else (2.0 ** -8, 2.0 ** -8)
        unit = float(m.max())
        assert bool(((a.detach().double() - b).abs() / unit <= (u * b.abs() + (op + 600 * 2.0 ** -24) * m) / unit).all()), i
    ops.check_device_status()
