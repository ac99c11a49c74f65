"""Gated dense layer over a concat (tensor cores) against the 64-bit formulas,
forward and backward.

Bounds. g and u are sums of K products of bf16 values, accumulated in fp32:
off by at most K 2^-23 sum|x w| each (the tensor core's adds may truncate: a
whole step, not half of one). The activation and its slope are Lipschitz (1.2, slopes of
the slope below 1); the intrinsics add 2^-19 relative. h is then rounded to
bf16: 2^-8 |h|. D = [dg | du] is rounded to bf16 (2^-8 relative) and enters
dX and dW as an operand, so those are off by 2^-8 sum|D||W| (sum|D||X|) plus
the accumulation, before their own rounding; the bias gradients are
fp32 sums of the unrounded values. All per element, with the sums of
magnitudes computed in 64 bits.
"""

import pytest
import torch

from layer_reference import act64, assert_within

pytestmark = pytest.mark.gpu

FAST = 2.0 ** -19
H = 2.0 ** -8


def _inputs(m, k1, k2, n, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    x1 = torch.randn((m, k1), generator=g).bfloat16()
    x2 = torch.randn((m, k2), generator=g).bfloat16() if k2 else None
    lim = (6.0 / (k1 + k2 + n)) ** 0.5
    wg, wu = (((torch.rand((n, k1 + k2), generator=g) * 2 - 1) * lim).bfloat16() for _ in range(2))
    bg, bu = (0.1 * torch.randn(n, generator=g) if bias else None for _ in range(2))
    dh = torch.randn((m, n), generator=g).bfloat16()
    return x1, x2, wg, wu, bg, bu, dh


def _slope64(z, act):
    z = z.clone().requires_grad_(True)
    act64(z, act).sum().backward()
    return z.grad


def _check(m, k1, k2, n, act="silu", bias=True, seed=0, inputs=None):
    from distributed_graph_flow_b200 import aggregation

    x1, x2, wg, wu, bg, bu, dh = inputs or _inputs(m, k1, k2, n, seed, bias)
    t = [None if v is None else v.cuda() for v in (x1, x2, wg, wu, bg, bu, dh)]
    h = aggregation.gated_dense_concat(*t[:6], activation=act)
    grads = aggregation.gated_dense_concat_backward(t[6], *t[:6], activation=act)
    aggregation.dense_check()
    # 64-bit values and magnitudes, on the device for speed.
    x = (t[0] if k2 == 0 else torch.cat([t[0], t[1]], 1)).double()
    wgd, wud = t[2].double(), t[3].double()
    zero = torch.zeros(n, dtype=torch.float64, device="cuda")
    bgd, bud = (zero if b is None else b.double() for b in t[4:6])
    g, u = x @ wgd.t() + bgd, x @ wud.t() + bud
    kk = k1 + k2
    eg = (kk + 4) * 2.0 ** -23 * (x.abs() @ wgd.abs().t() + bgd.abs())
    eu = (kk + 4) * 2.0 ** -23 * (x.abs() @ wud.abs().t() + bud.abs())
    a, s = act64(g, act), _slope64(g, act)
    eh = a * u
    ea = 1.2 * eg + FAST * (a.abs() + 1)
    bh = ea * u.abs() + a.abs() * eu + ea * eu
    assert_within(h, eh.cpu(), (bh + H * (eh.abs() + bh)).cpu() + 1e-30, "h")
    d = t[6].double()
    du, dg = d * a, d * u * s
    es = 1.0 * eg + FAST * (s.abs() + g.abs() + 1)
    if act == "relu":
        es = es + (g.abs() <= eg).double()  # either side of the jump
    edu, edg = d.abs() * ea, d.abs() * (u.abs() * es + eu * (s.abs() + es))
    names = ("dx1", "dx2", "dw_gate", "dw_up", "db_gate", "db_up")
    dx = dg @ wgd + du @ wud
    mag = (dg.abs() + edg) @ wgd.abs() + (du.abs() + edu) @ wud.abs()
    bx = edg @ wgd.abs() + edu @ wud.abs() + (H + 2 * n * 2.0 ** -23) * mag
    exp = {"dx1": (dx[:, :k1], bx[:, :k1]), "dx2": (dx[:, k1:], bx[:, k1:])}
    acc = H + (m + 64) * 2.0 ** -23
    for which, dd, ed in (("gate", dg, edg), ("up", du, edu)):
        exp["dw_" + which] = (dd.t() @ x, ed.t() @ x.abs() + acc * (dd.abs() + ed).t() @ x.abs())
        exp["db_" + which] = (dd.sum(0), ed.sum(0) + (m + 64) * 2.0 ** -24 * dd.abs().sum(0))
    for name, got in zip(names, grads):
        if got is None:
            assert (name == "dx2" and k2 == 0) or (name[:2] == "db" and not bias)
            continue
        e, bnd = exp[name]
        if got.dtype == torch.bfloat16:
            bnd = bnd + H * (e.abs() + bnd)
        assert_within(got, e.cpu(), bnd.cpu() + 1e-30, name)
    return h, grads


@pytest.mark.parametrize("m,k1,k2,n", [
    (128, 64, 0, 64),
    (1, 8, 0, 8),
    (1, 256, 256, 512),
    (2, 64, 64, 40),
    (127, 72, 8, 24),
    (129, 128, 64, 128),
    (300, 8, 200, 136),
    (515, 104, 0, 200),
    (1000, 320, 24, 264),
    (4097, 256, 256, 256),
    (20011, 40, 88, 72),
])
def test_shapes(cuda, m, k1, k2, n):
    _check(m, k1, k2, n, seed=m)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_activations(cuda, act, bias):
    _check(700, 64, 128, 192, act=act, bias=bias, seed=7)


@pytest.mark.parametrize("m,n", [(148 * 128, 256), (148 * 128 + 1, 512), (40000, 64), (6000, 1032)])
def test_tile_widths(cuda, m, n):
    """Every accumulator width, several tiles per CTA."""
    _check(m, 64, 0, n, seed=n)


def test_extreme_projections(cuda):
    """Projections far beyond where the exponential overflows."""
    x1, x2, wg, wu, bg, bu, dh = _inputs(200, 64, 0, 64, 11)
    bg = torch.linspace(-300, 300, 64)
    for act in ("silu", "gelu", "sigmoid", "relu"):
        _check(200, 64, 0, 64, act=act, inputs=(x1, x2, wg, wu, bg, bu, dh))


def test_nan_and_inf_rows(cuda):
    """A row with NaN or infinity leaves the other rows' outputs and input
    gradients as they were."""
    from distributed_graph_flow_b200 import aggregation

    x1, x2, wg, wu, bg, bu, dh = (t.cuda() for t in _inputs(300, 64, 64, 64, 12))
    ref = aggregation.gated_dense_concat(x1, x2, wg, wu, bg, bu)
    rdx = aggregation.gated_dense_concat_backward(dh, x1, x2, wg, wu, bg, bu)[:2]
    x1[7, 3], x2[250, 60] = float("nan"), float("inf")
    h = aggregation.gated_dense_concat(x1, x2, wg, wu, bg, bu)
    dx = aggregation.gated_dense_concat_backward(dh, x1, x2, wg, wu, bg, bu)[:2]
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[7] = keep[250] = False
    assert torch.equal(h[keep], ref[keep]) and bool(torch.isnan(h[7]).all())
    assert all(torch.equal(p[keep], q[keep]) for p, q in zip(dx, rdx))


def test_partial_gradients(cuda):
    from distributed_graph_flow_b200 import aggregation

    t = [v.cuda() for v in _inputs(1000, 64, 32, 96, 13)]
    full = aggregation.gated_dense_concat_backward(t[6], *t[:6])
    no_x = aggregation.gated_dense_concat_backward(t[6], *t[:6], need_input=False)
    no_w = aggregation.gated_dense_concat_backward(t[6], *t[:6], need_weight=False)
    assert no_x[:2] == (None, None) and no_w[2:4] == (None, None)
    assert all(torch.equal(p, q) for p, q in zip(full[2:], no_x[2:]))
    assert all(torch.equal(p, q) for p, q in zip(full[:2] + full[4:], no_w[:2] + no_w[4:]))


def test_rows_past_32_bits(cuda):
    """More than 2^31 values of h and 2^32 of the projections' gradients: the
    last rows (all others are zero). Operands and results are rounded to bf16
    once each, 2^-8 of the sum of magnitudes per rounding: four of them."""
    from distributed_graph_flow_b200 import aggregation

    rows, tail, n = (1 << 22) + 77, 300, 512
    x, dh = (torch.zeros((rows, w), dtype=torch.bfloat16, device="cuda") for w in (8, n))
    x1, _, wg, wu, _, _, d = _inputs(tail, 8, 0, n, 17, bias=False)
    x[-tail:], dh[-tail:] = x1.cuda(), d.cuda()
    wg, wu = wg.cuda(), wu.cuda()
    h = aggregation.gated_dense_concat(x, None, wg, wu)
    dx, _, dwg, dwu, _, _ = aggregation.gated_dense_concat_backward(dh, x, None, wg, wu)
    aggregation.dense_check()
    assert torch.count_nonzero(h[:-tail]) == 0 and torch.count_nonzero(dx[:-tail]) == 0
    xd, wgd, wud, dd = x1.double().cuda(), wg.double(), wu.double(), d.double().cuda()
    g, u = xd @ wgd.t(), xd @ wud.t()
    a, s = act64(g, "silu"), _slope64(g, "silu")
    dg, du = dd * u * s, dd * a

    def near(got, exp, magnitude, what):
        assert_within(got, exp.cpu(), (4 * H * magnitude + 1e-6).cpu(), what)

    near(h[-tail:], a * u, (a * u).abs(), "h")
    near(dx[-tail:], dg @ wgd + du @ wud, dg.abs() @ wgd.abs() + du.abs() @ wud.abs(), "dx")
    near(dwg, dg.t() @ xd, dg.abs().t() @ xd.abs(), "dw_gate")
    near(dwu, du.t() @ xd, du.abs().t() @ xd.abs(), "dw_up")


def test_no_rows(cuda):
    from distributed_graph_flow_b200 import aggregation

    t = [v.cuda() for v in _inputs(0, 64, 32, 96, 14)]
    assert aggregation.gated_dense_concat(*t[:6]).shape == (0, 96)
    grads = aggregation.gated_dense_concat_backward(t[6], *t[:6])
    assert grads[0].shape == (0, 64) and not any(bool(torch.count_nonzero(g)) for g in grads[2:])


def test_difference_quotient(cuda):
    """The weight gradient along a random direction against a central
    difference of the 64-bit layer: checks the formulas themselves."""
    from distributed_graph_flow_b200 import aggregation

    x1, x2, wg, wu, bg, bu, dh = _inputs(256, 64, 0, 64, 15)
    g = aggregation.gated_dense_concat_backward(dh.cuda(), x1.cuda(), None, wg.cuda(), wu.cuda(), bg.cuda(), bu.cuda(),
                                                activation="gelu")
    x = x1.double()
    gen = torch.Generator().manual_seed(1)

    def loss(a, b):
        return (act64(x @ a.t() + bg.double(), "gelu") * (x @ b.t() + bu.double()) * dh.double()).sum()

    for which, got in ((0, g[2]), (1, g[3])):
        v = torch.randn(wg.shape, generator=gen).double()
        step = [torch.zeros_like(v), torch.zeros_like(v)]
        step[which] = 1e-5 * v
        diff = (loss(wg.double() + step[0], wu.double() + step[1])
                - loss(wg.double() - step[0], wu.double() - step[1])) / 2e-5
        along = (got.double().cpu() * v).sum()
        # Rounding of D (2^-8 per term) and of dw (2^-8 per entry), all with one sign.
        bound = 2 * H * float((got.double().cpu().abs() * v.abs()).sum()) + 1e-3
        assert abs(float(along - diff)) <= bound


def test_results_repeat(cuda):
    from distributed_graph_flow_b200 import aggregation

    t = [v.cuda() for v in _inputs(50000, 128, 64, 256, 16)]
    first = None
    for _ in range(3):
        out = (aggregation.gated_dense_concat(*t[:6]), *aggregation.gated_dense_concat_backward(t[6], *t[:6]))
        first = first or out
        assert all(torch.equal(p, q) for p, q in zip(first, out))
    aggregation.dense_check()


def test_streams_and_graphs(cuda):
    from distributed_graph_flow_b200 import aggregation

    x1, x2, wg, wu, bg, bu, dh = (t.cuda() for t in _inputs(3000, 64, 64, 128, 17))

    def step(x):
        return (aggregation.gated_dense_concat(x, x2, wg, wu, bg, bu),
                *aggregation.gated_dense_concat_backward(dh, x, x2, wg, wu, bg, bu))

    other = (x1.float() * 2 + 1).bfloat16()
    eager, eager2 = step(x1), step(other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    h = aggregation.gated_dense_concat(x1, x2, wg, wu, bg, bu, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(h, eager[0])
    graphs = []
    for _ in range(2):
        xx = x1.clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(xx)
        graphs.append((g, xx, out))
    for k in range(2):
        for (g, xx, out), scale in zip(graphs, (k, 1 - k)):
            xx.copy_(other if scale else x1)
            g.replay()
        torch.cuda.synchronize()
        for (g, xx, out), scale in zip(graphs, (k, 1 - k)):
            assert all(torch.equal(p, q) for p, q in zip(out, eager2 if scale else eager))
    aggregation.dense_check()
