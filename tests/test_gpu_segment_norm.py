"""Group norm with activation over ragged segments against the 64-bit
formulas, forward and backward.

Bounds, derived from the arithmetic: u = 2^-24 is fp32's half step and n a
bound on the additions behind one sum (a thread's rows, then the block's
row lanes, then the group's channels: at most rows + C). The mean is off by
n u mean|x| at most, so the normalised value xhat by about
m = rstd (|x| + mean|x|) times (n + 16) u (the variance's error counts once
more through rstd, hence twice n); the activation and its slope are
Lipschitz (at most 1.2) and the exponential intrinsic adds under 2^-19
relative. Outputs add half a step of their type. Gradients: every term of dx
is at most rstd |w dz| (or the group's mean of it, times |xhat|) with the same
relative error, amplified by how far xhat is off.
"""

import pytest
import torch

from layer_reference import HALF, assert_within, norm64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FAST = 2.0 ** -19  # exponential and reciprocal intrinsics


def _offsets(lengths, first=0):
    off = [first]
    for n in lengths:
        off.append(off[-1] + n)
    return torch.tensor(off, dtype=torch.int64)


def _inputs(rows, c, dtype, seed, dev="cpu"):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, c), generator=g) * 1.3 + torch.randn(c, generator=g)).to(dtype)
    w = 1 + 0.3 * torch.randn(c, generator=g)
    b = 0.3 * torch.randn(c, generator=g)
    dy = torch.randn((rows, c), generator=g).to(dtype)
    return x, w, b, dy


def _check(x, off, groups, w, b, dy, act, eps=1e-5, what=""):
    from distributed_graph_flow_b200 import aggregation

    rows, c = x.shape
    dtype = x.dtype
    dev = "cuda"
    t = [None if v is None else v.to(dev) for v in (x, off, w, b, dy)]
    y, mean, rstd = aggregation.segment_group_norm(t[0], t[1], groups, t[2], t[3], eps=eps, activation=act)
    dx, dw, db = aggregation.segment_group_norm_backward(t[4], t[0], t[1], mean, rstd, t[2], t[3], activation=act)
    ey, edx, edw, edb = norm64(x, off, groups, w, b, eps, act, dy)
    assert y.dtype == dtype and dx.dtype == dtype
    # Per-row magnitudes of the bounds: the segment's rstd and mean |x|.
    rel = torch.zeros((rows, 1), dtype=torch.float64)
    mag = torch.zeros((rows, c), dtype=torch.float64)   # rstd (|x| + mean |x|)
    rst = torch.zeros((rows, c), dtype=torch.float64)
    gmag = torch.zeros((rows, c), dtype=torch.float64)  # the group's largest |w dz|
    for s in range(off.numel() - 1):
        lo, hi = int(off[s]), int(off[s + 1])
        if hi <= lo:
            continue
        v = x[lo:hi].double().view(hi - lo, groups, -1)
        r = 1 / torch.sqrt(v.var(dim=(0, 2), unbiased=False) + eps)
        ma = v.abs().mean(dim=(0, 2))
        m = r[None, :, None] * (v.abs() + ma[None, :, None])
        mag[lo:hi] = m.reshape(hi - lo, c)
        rst[lo:hi] = r[None, :, None].expand_as(v).reshape(hi - lo, c)
        gm = (dy[lo:hi].double().abs().view(v.shape) * 1.2 * (1 if w is None else w.double().abs().view(1, groups, -1)))
        gmag[lo:hi] = gm.amax(dim=(0, 2))[None, :, None].expand_as(v).reshape(hi - lo, c)
        rel[lo:hi] = (2 * (hi - lo + c) + 16) * U
    wa = torch.ones(c, dtype=torch.float64) if w is None else w.double().abs()
    off_xhat = mag * rel
    by = 1.2 * (off_xhat * wa + 4 * U * (mag * wa + 1)) + FAST * (ey.abs() + mag * wa + 1)
    assert_within(y, ey, by + HALF[dtype] * (ey.abs() + by) + 1e-30, what + " y")
    xm = 1 + mag
    bdx = rst * gmag * (xm * xm * rel + off_xhat * (1 + wa) * xm + FAST * xm * xm)
    if act != "relu":  # relu's slope jumps: only where z is not within its own error of the jump
        assert_within(dx, edx, bdx + HALF[dtype] * (edx.abs() + bdx) + 1e-30, what + " dx")
        n = rows + 4 * 592
        bw = ((n * U + FAST) * dy.double().abs() * 1.2 * xm + dy.double().abs() * off_xhat * 2).nan_to_num().sum(0) + 1e-30
        if w is not None:
            assert_within(dw, edw, bw, what + " dweight")
        if b is not None:
            assert_within(db, edb, bw, what + " dbias")
    return y, dx


LENGTHS = {
    "one": [1],
    "ones": [1] * 40,
    "two": [2, 0, 3],
    "tree": [61, 1, 17, 44, 0, 0, 30, 8],
    "long": [700, 3, 1300],
    "all_empty": [0, 0, 0],
}


@pytest.mark.parametrize("lengths", sorted(LENGTHS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_segments(cuda, lengths, dtype):
    off = _offsets(LENGTHS[lengths])
    x, w, b, dy = _inputs(max(int(off[-1]), 1), 64, dtype, 1)
    _check(x[:int(off[-1])], off, 8, w, b, dy[:int(off[-1])], "silu", what=lengths)


@pytest.mark.parametrize("c,groups", [(8, 1), (8, 8), (24, 3), (200, 25), (200, 1), (256, 32), (256, 256), (1024, 4),
                                      (1000, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_channels(cuda, c, groups, dtype):
    off = _offsets([5, 33, 0, 70])
    x, w, b, dy = _inputs(108, c, dtype, 2)
    _check(x, off, groups, w, b, dy, "gelu", what=f"{c}/{groups}")


@pytest.mark.parametrize("c,groups", [(80, 40), (80, 80), (8, 1), (264, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_segments_with_many_groups(cuda, c, groups, dtype):
    """Row tiles joined per 32 groups and up to 32 lanes, short and empty segments
    between the long ones, spare rows on both ends (zeros)."""
    lengths = [2600, 3, 0, 9000, 1, 0, 3100]
    off = _offsets(lengths, first=7)
    used = int(off[-1])
    x, w, b, dy = _inputs(used + 500, c, dtype, 6)
    y, dx = _check(x[:used], off, groups, w, b, dy[:used], "silu", what=f"{c}/{groups}")
    for t in (y, dx):
        assert torch.count_nonzero(t[:7]) == 0
    from distributed_graph_flow_b200 import aggregation

    wide = [t.cuda() for t in (x, off, w, b, dy)]
    y2, mean, rstd = aggregation.segment_group_norm(wide[0], wide[1], groups, wide[2], wide[3], activation="silu")
    dx2 = aggregation.segment_group_norm_backward(wide[4], wide[0], wide[1], mean, rstd, wide[2], wide[3],
                                                  activation="silu")[0]
    assert torch.count_nonzero(y2[used:]) == 0 and torch.count_nonzero(dx2[used:]) == 0


def test_single_values_have_no_gradient(cuda):
    """A segment and group of one value: its normalised value is zero and its
    gradient exactly zero, however large rstd = 1 / sqrt(eps) is."""
    from distributed_graph_flow_b200 import aggregation

    x, w, b, dy = (t.cuda() for t in _inputs(200, 40, torch.float32, 5))
    off = _offsets([1] * 200).cuda()
    y, mean, rstd = aggregation.segment_group_norm(x, off, 40, w, b)
    assert torch.equal(mean, x) and torch.equal(y, b.expand(200, 40))
    dx, dw, _ = aggregation.segment_group_norm_backward(dy, x, off, mean, rstd, w, b)
    assert torch.count_nonzero(dx) == 0 and torch.count_nonzero(dw) == 0


def test_widest_rows(cuda):
    off = _offsets([3, 20])
    x, w, b, dy = _inputs(23, 2048, torch.bfloat16, 3)
    _check(x, off, 2048, w, b, dy, "silu")
    _check(x, off, 1, w, b, dy, "none")


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("affine", [(True, True), (False, True), (True, False), (False, False)])
def test_activations(cuda, act, affine):
    off = _offsets([20, 50, 3])
    x, w, b, dy = _inputs(73, 32, torch.float32, 4)
    _check(x, off, 4, w if affine[0] else None, b if affine[1] else None, dy, act)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_outside_are_zero_and_unused(cuda, dtype):
    """Spare rows before and behind the segments hold NaN and infinities."""
    off = _offsets([9, 0, 30], first=5)
    rows = 5 + 39 + 11
    x, w, b, dy = _inputs(rows, 40, dtype, 5)
    clean = _check(x, off, 5, w, b, dy, "silu")
    for bad in (float("nan"), float("inf"), -float("inf")):
        xb, dyb = x.clone(), dy.clone()
        for t in (xb, dyb):
            t[:5] = bad
            t[44:] = bad
        from distributed_graph_flow_b200 import aggregation

        y, mean, rstd = aggregation.segment_group_norm(xb.cuda(), off.cuda(), 5, w.cuda(), b.cuda(), activation="silu")
        dx, dw, db = aggregation.segment_group_norm_backward(dyb.cuda(), xb.cuda(), off.cuda(), mean, rstd, w.cuda(),
                                                             b.cuda(), activation="silu")
        assert torch.equal(y, clean[0]) and torch.equal(dx, clean[1])
        assert torch.count_nonzero(y[:5]) == 0 and torch.count_nonzero(y[44:]) == 0
        assert bool(torch.isfinite(dw).all()) and bool(torch.isfinite(db).all())


def test_nan_stays_in_its_segment(cuda):
    from distributed_graph_flow_b200 import aggregation

    off = _offsets([8, 12, 7])
    x, w, b, _ = _inputs(27, 16, torch.float32, 6)
    ref = aggregation.segment_group_norm(x.cuda(), off.cuda(), 2, w.cuda(), b.cuda(), activation="relu")[0]
    x[10, 3] = float("nan")
    y = aggregation.segment_group_norm(x.cuda(), off.cuda(), 2, w.cuda(), b.cuda(), activation="relu")[0]
    assert torch.equal(y[:8], ref[:8]) and torch.equal(y[20:], ref[20:])
    assert bool(torch.isnan(y[8:20, :8]).all()) and torch.equal(y[8:20, 8:], ref[8:20, 8:])


def test_large_mean_keeps_its_variance(cuda):
    """mean / spread = 2000: squares are summed around the mean."""
    off = _offsets([500])
    g = torch.Generator().manual_seed(7)
    x = torch.randn((500, 16), generator=g) + 2000.0
    _check(x, off, 4, None, None, torch.randn((500, 16), generator=g), "none")


@pytest.mark.parametrize("rows", [3, 700])
def test_values_whose_square_overflows(cuda, rows):
    """A mean of 1e20 with a spread of 1e17: squares of the distances stay
    finite, and threads without rows add nothing (not 0 times infinity)."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn((rows, 16), generator=g) * 1e17 + 1e20
    _check(x, _offsets([rows]), 4, None, None, torch.randn((rows, 16), generator=g), "none")


def test_bad_offsets_stay_in_bounds(cuda):
    """Offsets past the rows (or descending) are clamped, never followed."""
    from distributed_graph_flow_b200 import aggregation

    x = torch.randn((50, 16), device="cuda")
    for off in ([0, 10, 1 << 40], [-5, 20, 50], [0, 40, 10, 50], [60, 70, 80]):
        o = torch.tensor(off, dtype=torch.int64, device="cuda")
        y, mean, rstd = aggregation.segment_group_norm(x, o, 4)
        aggregation.segment_group_norm_backward(x, x, o, mean, rstd)
    torch.cuda.synchronize()


def test_results_repeat(cuda):
    from distributed_graph_flow_b200 import aggregation

    off = _offsets([3000, 41, 0, 900, 5000]).cuda()
    x, w, b, dy = (t.cuda() for t in _inputs(8941, 96, torch.bfloat16, 8))
    first = None
    for _ in range(3):
        y, mean, rstd = aggregation.segment_group_norm(x, off, 12, w, b, activation="silu")
        out = (y, *aggregation.segment_group_norm_backward(dy, x, off, mean, rstd, w, b, activation="silu"))
        first = first or out
        assert all(torch.equal(p, q) for p, q in zip(first, out))


def test_long_buffers_past_32_bits(cuda):
    """More than 2^32 bytes and 2^31 values: the last segment's rows."""
    from distributed_graph_flow_b200 import aggregation

    rows, c = (1 << 23) + 77, 264
    x = torch.zeros((rows, c), dtype=torch.bfloat16, device="cuda")
    tail = torch.randn((500, c), device="cuda").to(torch.bfloat16)
    x[-500:] = tail
    off = torch.tensor([0, 10, rows - 500, rows], device="cuda")
    y, mean, rstd = aggregation.segment_group_norm(x, off, 33, activation="silu")
    ey, edx, _, _ = norm64(tail.cpu(), torch.tensor([0, 500]), 33, None, None, 1e-5, "silu", tail.cpu())
    assert_within(y[-500:], ey, 2.0 ** -7 * (1 + ey.abs()), "y")
    dx, _, _ = aggregation.segment_group_norm_backward(x, x, off, mean, rstd, activation="silu")
    assert_within(dx[-500:], edx, 2.0 ** -6 * (1 + edx.abs()), "dx")


def test_streams_and_graphs(cuda):
    """Another stream than the current one, and two captured graphs replayed
    in turn on changed inputs, give the eager values bit for bit."""
    from distributed_graph_flow_b200 import aggregation

    off = _offsets([300, 41, 0, 90]).cuda()
    x, w, b, dy = (t.cuda() for t in _inputs(431, 64, torch.float32, 9))

    def step(xx):
        y, mean, rstd = aggregation.segment_group_norm(xx, off, 8, w, b, activation="gelu")
        return (y, *aggregation.segment_group_norm_backward(dy, xx, off, mean, rstd, w, b, activation="gelu"))

    eager, eager2 = step(x), step(2 * x + 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y, mean, rstd = aggregation.segment_group_norm(x, off, 8, w, b, activation="gelu", stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, eager[0])
    graphs = []
    for _ in range(2):
        xx = x.clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(xx)
        graphs.append((g, xx, out))
    for k in range(2):
        for (g, xx, out), scale in zip(graphs, (k, 1 - k)):
            xx.copy_(2 * x + 1 if scale else x)
            g.replay()
        torch.cuda.synchronize()
        for (g, xx, out), scale in zip(graphs, (k, 1 - k)):
            assert all(torch.equal(p, q) for p, q in zip(out, eager2 if scale else eager))
