"""The gated layer's gradients round [dg | du] to bf16 once, as operands of
the two products behind it, and lose nothing else.

The 64-bit formulas with that rounding put in. An element of dg or du that is
within its fp32 error (K 2^-23 sum|x w| through the activation, as in the other
tests of the layer) of the border between two bf16 values may round to
either: a step of 2^-7 of it. All others are the same value in both. Then dX
and dW are off by those steps times the other operand, by the accumulation (n
terms of 2^-23 of the magnitudes) and by their own rounding, 2^-8. That is well
below a quarter of what the rounding of [dg | du] itself adds to them.
"""

import pytest
import torch

from layer_reference import act64, assert_within

pytestmark = pytest.mark.gpu

H = 2.0 ** -8


def _border(v, err):
    """v in bf16 (as 64 bits), and a step where it might round either way."""
    r = v.bfloat16().double()
    lo, hi = (v - err).bfloat16().double(), (v + err).bfloat16().double()
    return r, hi - lo


@pytest.mark.parametrize("m,k1,k2,n", [(2000, 64, 0, 64), (3001, 40, 24, 136), (40000, 32, 32, 128)])
def test_one_rounding(cuda, m, k1, k2, n):
    from distributed_graph_flow_b200 import aggregation

    g = torch.Generator(device="cuda").manual_seed(m)

    def rnd(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    k = k1 + k2
    x1, x2 = rnd(m, k1).bfloat16(), rnd(m, k2).bfloat16() if k2 else None
    wg, wu = (0.2 * rnd(n, k)).bfloat16(), (0.2 * rnd(n, k)).bfloat16()
    bg, bu, dh = 0.1 * rnd(n), 0.1 * rnd(n), rnd(m, n).bfloat16()
    dx1, dx2, dwg, dwu, _, _ = aggregation.gated_dense_concat_backward(dh, x1, x2, wg, wu, bg, bu, activation="silu")
    aggregation.dense_check()
    x = (x1 if x2 is None else torch.cat([x1, x2], 1)).double()
    a, b = wg.double(), wu.double()
    gd, ud = x @ a.t() + bg.double(), x @ b.t() + bu.double()
    eg = (k + 4) * 2.0 ** -23 * (x.abs() @ a.abs().t() + bg.double().abs())
    eu = (k + 4) * 2.0 ** -23 * (x.abs() @ b.abs().t() + bu.double().abs())
    fast = 24 * 2.0 ** -24  # intrinsics and roundings of the epilogue, |g| below 12
    assert float(gd.abs().max()) < 12
    s = 1 / (1 + torch.exp(-gd))
    act, slope = gd * s, s * (1 + gd * (1 - s))
    assert torch.allclose(act, act64(gd, "silu"))
    d = dh.double()
    ea, es = 1.1 * eg + 2 * fast * act.abs(), 0.5 * eg + 2 * fast * (s + act.abs())
    du, eu_ = _border(d * act, d.abs() * (ea + 2.0 ** -23 * act.abs()))
    dg, eg_ = _border(d * ud * slope, d.abs() * (ud.abs() * es + eu * (slope.abs() + es) + 2.0 ** -22 * (ud * slope).abs()))
    dx = dg @ a + du @ b
    bx = eg_ @ a.abs() + eu_ @ b.abs() + 2 * n * 2.0 ** -23 * (dg.abs() @ a.abs() + du.abs() @ b.abs())
    got = dx1 if dx2 is None else torch.cat([dx1, dx2], 1)
    assert_within(got, dx.cpu(), (bx + H * (dx.abs() + bx)).cpu(), "dx")
    for name, p, q, e in (("dw_gate", dwg, dg, eg_), ("dw_up", dwu, du, eu_)):
        exp = q.t() @ x
        bw = e.t() @ x.abs() + (m + 64) * 2.0 ** -23 * q.abs().t() @ x.abs()
        assert_within(p, exp.cpu(), (bw + H * (exp.abs() + bw)).cpu(), name)
    # What the bound is worth: under a quarter of the rounding that it leaves out.
    assert float(eg_.sum() + eu_.sum()) < 0.25 * float((H * (dg.abs() + du.abs())).sum())
