"""Activations of the layer operators and their slopes, value by value.

A group norm whose weight is zero gives act(bias) exactly as the kernel computes
it, and with a gradient of one its bias gradient is act'(bias).

Bounds, u = 2^-24. Documented errors: ex2 4 u, rcp 2 u; every rounding u.
* sigmoid = 1 / (1 + e^-z): the exponent z log2(e) is rounded and its constant
  is off by 0.3 u, so e is off by (1.3 |z| + 4) u, of which 1 - s reaches the
  sum; the sum's rounding and rcp add 3 u: es = (1 - s) (1.3 |z| + 4) u + 3 u.
* silu one product more. Slopes: s (1 - s) and s (1 + z (1 - s)) with s off by
  es s and three roundings of terms of at most 1 + |z|.
* Phi(z) for gelu: the tail's fit 1.1e-8 (1 + z^2) + 2.3e-8 (coefficients in
  fp32) < (0.6 + 0.2 z^2) u; t = 1 / (1 + p |z|) is off by 4 u and enters with
  a logarithmic slope below 2.7: 11 u; eight steps of the polynomial, whose
  partial sums stay below twice its value: 6 u; two products, ex2: 6 u; the
  exponent z^2 / 2 log2(e), two roundings and a constant: 1.2 z^2 u. In all
  (24 + 1.4 z^2) u of the tail, and as much at most of one minus it; gelu one
  product more, its slope cdf + z e^(-z^2 / 2) / sqrt(2 pi).
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _values(reach):
    z = torch.linspace(-reach, reach, 1023).float()
    return torch.cat([z, torch.zeros(1)])


def _kernel(z, act):
    from distributed_graph_flow_b200 import aggregation

    off = torch.tensor([0, 1], device="cuda")
    x = torch.randn((1, z.numel()), device="cuda")
    w, b = torch.zeros(z.numel(), device="cuda"), z.cuda()
    y, mean, rstd = aggregation.segment_group_norm(x, off, 1, w, b, activation=act)
    _, _, db = aggregation.segment_group_norm_backward(torch.ones_like(x), x, off, mean, rstd, w, b, activation=act)
    return y[0].double().cpu(), db.double().cpu()


@pytest.mark.parametrize("reach", [1.0, 4.0, 12.0, 60.0])
@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
def test_values_and_slopes(cuda, act, reach):
    z = _values(reach)
    y, slope = _kernel(z, act)
    z = z.double()
    a = z.abs()
    s = 1 / (1 + torch.exp(-z))
    keep = 1 / (1 + torch.exp(z))
    es = keep * (1.3 * a + 4) * U + 3 * U
    if act == "sigmoid":
        exp, by = s, s * (es + U)
        dexp, dby = s * keep, s * (2 * es + 3 * U)
    elif act == "silu":
        exp, by = z * s, a * s * (es + 2 * U)
        dexp, dby = s * (1 + z * keep), s * ((1 + a) * 2 * es + 4 * (1 + a) * U)
    else:
        tail = 0.5 * torch.special.erfc(a / math.sqrt(2.0))
        cdf = torch.where(z < 0, tail, 1 - tail)
        ec = (24 + 1.4 * a * a) * U
        exp, by = z * cdf, a * (tail * ec + cdf * 2 * U)
        bell = a * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        dexp = cdf + torch.sign(z) * bell
        dby = tail * ec + bell * (8 + 1.4 * a * a) * U + (cdf + dexp.abs()) * 2 * U
    tiny = 2.0 ** -126 * (1 + a)  # flushed
    for what, got, e, bound in (("value", y, exp, by), ("slope", slope, dexp, dby)):
        bad = ~((got - e).abs() <= bound + tiny)
        i = int(((got - e).abs() / (bound + tiny)).argmax())
        assert not bool(bad.any()), (what, int(bad.sum()), float(z[i]), float(got[i]), float(e[i]), float(bound[i]))


@pytest.mark.parametrize("act", ["none", "relu"])
def test_exact_ones(cuda, act):
    z = _values(4.0)
    y, slope = _kernel(z, act)
    z = z.double()
    one = torch.ones_like(z)
    assert torch.equal(y, z if act == "none" else z.clamp_min(0))
    assert torch.equal(slope, one if act == "none" else (z > 0).double())


def test_strided_parameters_through_the_torch_operators(cuda):
    """Biases, weights and affine parameters strided or expanded: the values
    and gradients of their packed copies."""
    from distributed_graph_flow_b200 import torch_ops

    g = torch.Generator(device="cuda").manual_seed(3)
    off = torch.tensor([0, 30, 64], device="cuda")
    x = torch.randn((64, 32), generator=g, device="cuda")
    xb, w = x.bfloat16(), torch.randn((40, 32), generator=g, device="cuda").bfloat16()
    long = torch.randn(80, generator=g, device="cuda")

    def run(pack):
        base = long.clone().requires_grad_(True)
        one = torch.full((1,), 0.5, device="cuda", requires_grad=True)
        strided, expanded, affine = base[::2], one.expand(40), base[1:64:2]
        if pack:
            strided, expanded, affine = strided.contiguous(), expanded.contiguous(), affine.contiguous()
        h = torch.ops.dgfx.gated_dense_concat(xb, None, w, w, strided, expanded, "silu")
        y = torch_ops.segment_group_norm(x, off, 4, affine, one.expand(32) if not pack else one.expand(32).contiguous(),
                                         activation="silu")
        (h.float().square().sum() + y.square().sum()).backward()
        return h, y, base.grad, one.grad

    assert all(torch.equal(p, q) for p, q in zip(run(False), run(True)))
