"""64-bit restatements of the layer operators, written from their formulas
with loops over segments and rows, and the bounds their tests share."""

import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # half a step, relative


def act64(z, kind):
    if kind == "none":
        return z
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))


def bounds_of(offsets, rows):
    """[(begin, end)] of the segments, as Python ints."""
    off = [int(v) for v in offsets]
    return list(zip(off[:-1], off[1:]))


def norm64(x, offsets, groups, weight, bias, eps, act, grad=None):
    """(y, dx, dweight, dbias) in 64 bits; zeros outside of the segments."""
    rows, c = x.shape
    w = torch.ones(c, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(c, dtype=torch.float64) if bias is None else bias.double()
    w, b = w.requires_grad_(True), b.requires_grad_(True)
    y = torch.zeros((rows, c), dtype=torch.float64)
    dx = torch.zeros((rows, c), dtype=torch.float64)
    for lo, hi in bounds_of(offsets, rows):
        if hi <= lo:
            continue
        xs = x[lo:hi].double().requires_grad_(True)
        v = xs.view(hi - lo, groups, c // groups)
        mean = v.mean(dim=(0, 2), keepdim=True)
        var = ((v - mean) ** 2).mean(dim=(0, 2), keepdim=True)
        z = ((v - mean) / torch.sqrt(var + eps)).reshape(hi - lo, c) * w + b
        ys = act64(z, act)
        y[lo:hi] = ys.detach()
        if grad is not None:
            ys.backward(grad[lo:hi].double())
            dx[lo:hi] = xs.grad
    zero = torch.zeros(c, dtype=torch.float64)
    return y, dx, zero if w.grad is None else w.grad, zero if b.grad is None else b.grad


def scan64(x, gate, offsets, initial, grad=None, grad_final=None):
    """(h, final, dx, dgate, dinitial) in 64 bits, row by row."""
    rows, c = x.shape
    segs = bounds_of(offsets, rows)
    h = torch.zeros((rows, c), dtype=torch.float64)
    dx, dgate = torch.zeros_like(h), torch.zeros_like(h)
    h0 = torch.zeros((len(segs), c), dtype=torch.float64) if initial is None else initial.double()
    final = h0.clone()
    dinit = torch.zeros_like(h0) if grad_final is None else grad_final.double().clone()
    for s, (lo, hi) in enumerate(segs):
        if hi <= lo:
            continue
        xs, gs = x[lo:hi].double(), gate[lo:hi].double()
        a, keep = 1 / (1 + torch.exp(-gs)), 1 / (1 + torch.exp(gs))
        st = h0[s]
        prev = []
        for t in range(hi - lo):
            prev.append(st)
            st = a[t] * st + keep[t] * xs[t]
            h[lo + t] = st
        final[s] = st
        e = torch.zeros(c, dtype=torch.float64) if grad_final is None else grad_final[s].double()
        for t in range(hi - lo - 1, -1, -1):
            d = e if grad is None else grad[lo + t].double() + e
            dx[lo + t] = keep[t] * d
            dgate[lo + t] = d * (prev[t] - xs[t]) * a[t] * keep[t]
            e = a[t] * d
        dinit[s] = e
    return h, final, dx, dgate, dinit


def assert_within(got, exp, bound, what=""):
    """|got - exp| <= bound elementwise; bound in 64 bits."""
    got = got.detach().double().cpu()
    assert got.shape == exp.shape, f"{what}: {tuple(got.shape)} vs {tuple(exp.shape)}"
    err = (got - exp).abs()
    bad = ~(err <= bound)
    if bool(bad.any()):
        i = int((err / bound).nan_to_num(nan=math.inf).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off; worst {float(err.flatten()[i]):.3e} "
                             f"against a bound of {float(torch.as_tensor(bound).expand_as(err).flatten()[i]):.3e}")
