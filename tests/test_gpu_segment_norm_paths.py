"""Group norm: gradients of relu, bf16 forms of every activation, and the
kernels for long segments (list, row tiles, join, apply) against the 64-bit formulas.

A call takes the long segments' kernels where its rows exceed 24 steps of the
largest team, and of its segments those of more than three to eight steps: 24
x 2048 rows of 8 bf16 channels, 24 x 512 rows of 16 fp32 ones, fewer of wider rows.

Bounds, u = 2^-24. Whatever the segment's length, a sum is a chain of at most
256 rows of one thread, 69 values of its group and 69 row tiles: N = 400
additions (or rows + C, if that is less), each off by u of what was summed. The
squares are taken around values of the segment, so the variance and with it
rstd are off by 2 N u. The mean is a sum of at most 75 means of threads, 80 u
mean|x| with their own roundings, taken as N u mean|x| unless said; the sums
inside of a thread (32 rows here) and over the tiles (37 + 32) run around one of the values or
tile means, which may lie as far out as the largest value does: 80 u max|x|
more. The rest as in the arithmetic of one
value: the activation and its slope are Lipschitz (at most 1.2), their
intrinsics add 2^-19, outputs half a step of their type; a term of dx is at
most rstd |w dz| times 1 + |xhat|^2. The sums for weight and bias are chains of at most 256 rows of a thread,
256 threads of a block, and 344 of the blocks' sums.

relu's slope jumps: where |z| is below MARGIN, far above what z can be off by, the
gradient that arrives is zero, so that the slope there does not matter, and all others
are compared as those of any activation.
"""

import pytest
import torch

from layer_reference import HALF, act64, assert_within, norm64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FAST = 2.0 ** -19
CHAIN = 400
MARGIN = 2.0 ** -8


def _offsets(lengths, first=0):
    off = [first]
    for n in lengths:
        off.append(off[-1] + n)
    return torch.tensor(off, dtype=torch.int64)


def _inputs(rows, c, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, c), generator=g) * 1.3 + torch.randn(c, generator=g)).to(dtype)
    w = 1 + 0.3 * torch.randn(c, generator=g)
    b = 0.3 * torch.randn(c, generator=g)
    dy = torch.randn((rows, c), generator=g).to(dtype)
    return x, w, b, dy


def _away_from_the_jump(x, off, groups, w, b, dy):
    """dy with zeros where |z| < MARGIN."""
    z = norm64(x, off, groups, w, b, 1e-5, "none")[0]
    assert float((z.abs() < MARGIN).double().mean()) < 0.05
    return torch.where(z.abs() < MARGIN, torch.zeros((), dtype=dy.dtype), dy)


def _run(x, off, groups, w, b, dy, act):
    from distributed_graph_flow_b200 import aggregation

    t = [None if v is None else v.cuda() for v in (x, off, w, b, dy)]
    y, mean, rstd = aggregation.segment_group_norm(t[0], t[1], groups, t[2], t[3], activation=act)
    return (y, *aggregation.segment_group_norm_backward(t[4], t[0], t[1], mean, rstd, t[2], t[3], activation=act))


def _check(x, off, groups, w, b, dy, act, mean_units=None, what=""):
    rows, c = x.shape
    dtype = x.dtype
    y, dx, dw, db = _run(x, off, groups, w, b, dy, act)
    ey, edx, edw, edb = norm64(x, off, groups, w, b, 1e-5, act, dy)
    off_xhat, xhat, rst, gmag = (torch.zeros((rows, c), dtype=torch.float64) for _ in range(4))
    rel = torch.zeros((rows, 1), dtype=torch.float64)
    wa = torch.ones(c, dtype=torch.float64) if w is None else w.double().abs()
    for lo, hi in zip(off[:-1].tolist(), off[1:].tolist()):
        if hi <= lo:
            continue
        v = x[lo:hi].double().view(hi - lo, groups, -1)
        mu = v.mean(dim=(0, 2), keepdim=True)
        r = 1 / torch.sqrt(v.var(dim=(0, 2), unbiased=False, keepdim=True) + 1e-5)
        n = min(hi - lo + c, CHAIN)
        n_mean = n if mean_units is None else mean_units
        rel[lo:hi] = (2 * n + 16) * U
        ma, most = v.abs().mean(dim=(0, 2), keepdim=True), v.abs().amax(dim=(0, 2), keepdim=True)
        xh = r * (v - mu).abs()
        # The mean's error, the subtraction's and rstd's.
        off_xhat[lo:hi] = (r * (n_mean * U * ma + 80 * U * most + U * (v.abs() + ma)) + xh * (2 * n + 16) * U).reshape(hi - lo, c)
        xhat[lo:hi] = xh.reshape(hi - lo, c)
        rst[lo:hi] = r.expand_as(v).reshape(hi - lo, c)
        gm = dy[lo:hi].double().abs().view(v.shape) * 1.2 * wa.view(1, groups, -1)
        gmag[lo:hi] = gm.amax(dim=(0, 2), keepdim=True).expand_as(v).reshape(hi - lo, c)
    by = 1.2 * (off_xhat * wa + 4 * U * (xhat * wa + 1)) + FAST * (ey.abs() + xhat * wa + 1)
    if act == "relu":
        assert float(by[xhat * wa < 2].max()) < MARGIN  # z near the jump is known to be on its side
    assert_within(y, ey, by + HALF[dtype] * (ey.abs() + by) + 1e-30, what + " y")
    xm = 1 + xhat
    bdx = rst * gmag * (xm * xm * rel + off_xhat * (1 + wa) * xm + FAST * xm * xm)
    assert_within(dx, edx, bdx + HALF[dtype] * (edx.abs() + bdx) + 1e-30, what + " dx")
    da = dy.double().abs()
    bw = ((min(rows, 256) + 600) * U * 1.2 * da * xm + FAST * da * 1.2 * xm + da * off_xhat * (2 + wa * xm)).sum(0) + 1e-30
    for got, exp, name in ((dw, edw, " dweight"), (db, edb, " dbias")):
        if got is not None:
            assert_within(got, exp, bw, what + name)
    return y, dx


LENGTHS = {
    "ones": [1] * 40,
    "tree": [61, 1, 17, 44, 0, 0, 30, 8],
    "long": [2600, 3, 0, 9000, 1, 0, 3100],
}


@pytest.mark.parametrize("lengths", sorted(LENGTHS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("affine", [(True, True), (False, False)])
def test_relu_gradients(cuda, lengths, dtype, affine):
    off = _offsets(LENGTHS[lengths])
    x, w, b, dy = _inputs(int(off[-1]), 64, dtype, 21)
    w, b = w if affine[0] else None, b if affine[1] else None
    dy = _away_from_the_jump(x, off, 8, w, b, dy)
    _check(x, off, 8, w, b, dy, "relu", what=lengths)


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("lengths", ["tree", "long"])
def test_bf16_activations(cuda, act, lengths):
    off = _offsets(LENGTHS[lengths])
    x, w, b, dy = _inputs(int(off[-1]), 40, torch.bfloat16, 22)
    _check(x, off, 5, w, b, dy, act, what=lengths)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["relu", "gelu"])
def test_narrow_rows_in_tiles(cuda, dtype, act):
    """8 channels: 64,004 rows are more than 24 steps of the largest team."""
    off = _offsets([30000, 3, 0, 25000, 1, 9000])
    x, w, b, dy = _inputs(int(off[-1]), 8, dtype, 23)
    if act == "relu":
        dy = _away_from_the_jump(x, off, 1, w, b, dy)
    _check(x, off, 1, w, b, dy, act)


def test_tiles_far_from_zero(cuda):
    """mean / spread = 2000 over 30,000 rows: squares are summed around values
    of the segment, and tiles joined around the first one's mean."""
    off = _offsets([30000, 5, 20000])
    g = torch.Generator().manual_seed(24)
    x = torch.randn((50005, 16), generator=g) + 2000.0
    _check(x, off, 4, None, None, torch.randn(x.shape, generator=g), "none", mean_units=80)


@pytest.mark.parametrize("shift", [1000.0, -3e4])
def test_first_tile_apart_from_the_rest(cuda, shift):
    """The join runs around the first tile's mean: one far from all others."""
    off = _offsets([40000, 20000])
    g = torch.Generator().manual_seed(25)
    x = torch.randn((60000, 16), generator=g)
    x[:1500] += shift
    x[40000:40200] -= shift
    _check(x, off, 4, None, None, torch.randn(x.shape, generator=g), "silu")


def test_nan_stays_in_its_long_segment(cuda):
    off = _offsets([20000, 15000, 4, 18000])
    x, w, b, dy = _inputs(int(off[-1]), 16, torch.float32, 26)
    ref = _run(x, off, 2, w, b, dy, "silu")
    x[25000, 3] = float("nan")
    y, dx, dw, db = _run(x, off, 2, w, b, dy, "silu")
    hit = torch.zeros(x.shape, dtype=torch.bool, device="cuda")
    hit[20000:35000, :8] = True
    for got, exp in ((y, ref[0]), (dx, ref[1])):
        assert bool(torch.isnan(got[hit]).all()) and torch.equal(got[~hit], exp[~hit])
    for got, exp in ((dw, ref[2]), (db, ref[3])):
        assert bool(torch.isnan(got[:8]).all()) and torch.equal(got[8:], exp[8:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_long_segments(cuda, dtype):
    """Forward and backward with the long segments' kernels in two captured
    graphs, replayed in turn on changed inputs and offsets: the eager bits."""
    from distributed_graph_flow_b200 import aggregation

    lengths = ([2600, 3, 0, 9000, 1, 0, 3100], [9000, 0, 2600, 0, 3100, 3, 1])
    offs = [_offsets(n, first=7).cuda() for n in lengths]
    rows = int(offs[0][-1]) + 290
    x, w, b, dy = (t.cuda() for t in _inputs(rows, 264, dtype, 27))
    xs = [x, (2 * x.float() + 1).to(dtype)]

    def step(xx, off):
        y, mean, rstd = aggregation.segment_group_norm(xx, off, 33, w, b, activation="gelu")
        return (y, *aggregation.segment_group_norm_backward(dy, xx, off, mean, rstd, w, b, activation="gelu"))

    eager = [step(p, q) for p, q in zip(xs, offs)]
    graphs = []
    for _ in range(2):
        xx, oo = xs[0].clone(), offs[0].clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(xx, oo)
        graphs.append((g, xx, oo, out))
    for turn in range(4):
        for k, (g, xx, oo, out) in enumerate(graphs):
            xx.copy_(xs[(turn + k) % 2])
            oo.copy_(offs[(turn + k) % 2])
            g.replay()
        torch.cuda.synchronize()
        for k, (g, xx, oo, out) in enumerate(graphs):
            assert all(torch.equal(p, q) for p, q in zip(out, eager[(turn + k) % 2]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["none", "relu"])
def test_hundreds_of_thousands_of_segments(cuda, dtype, act):
    """Segments of one row, or none, with one group: a layer norm of each row."""
    g = torch.Generator(device="cuda").manual_seed(28)
    c, nseg = 64, 400_000
    lengths = (torch.rand(nseg, generator=g, device="cuda") < 0.75).long()
    off = torch.cat([lengths.new_zeros(1), torch.cumsum(lengths, 0)])
    rows = int(off[-1])
    x = (torch.randn((rows, c), generator=g, device="cuda") * 1.3 + 0.4).to(dtype)
    w = 1 + 0.3 * torch.randn(c, generator=g, device="cuda")
    b = 0.3 * torch.randn(c, generator=g, device="cuda")
    xd = x.double().requires_grad_(True)
    v = xd - xd.mean(1, keepdim=True)
    wd, bd = w.double().requires_grad_(True), b.double().requires_grad_(True)
    rstd = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5)
    z = v * rstd * wd + bd
    dy = torch.randn((rows, c), generator=g, device="cuda").to(dtype)
    dy = torch.where(z.detach().abs() < MARGIN, torch.zeros((), dtype=dtype, device="cuda"), dy)
    exp = act64(z, act)
    exp.backward(dy.double())
    from distributed_graph_flow_b200 import aggregation

    y, mean, rs = aggregation.segment_group_norm(x, off, 1, w, b, activation=act)
    dx, dw, db = aggregation.segment_group_norm_backward(dy, x, off, mean, rs, w, b, activation=act)
    n = c + 1
    xm = (v * rstd).detach().abs()
    r, wa = rstd.detach(), w.double().abs()
    off_xhat = r * ((n + 1) * U * x.double().abs().mean(1, keepdim=True) + U * x.double().abs()) + xm * (2 * n + 16) * U
    by = off_xhat * wa + 4 * U * (xm * wa + 1)
    assert_within(y, exp.detach().cpu(), (by + HALF[dtype] * (exp.detach().abs() + by)).cpu(), "y")
    gmag = (dy.double().abs() * wa).amax(1, keepdim=True)
    bdx = r * gmag * ((1 + xm) ** 2 * (2 * n + 16) * U + off_xhat * (1 + wa) * (1 + xm))
    assert_within(dx, xd.grad.cpu(), (bdx + HALF[dtype] * (xd.grad.abs() + bdx)).cpu(), "dx")
    # A slot of the parameters' sums adds at most 400,000 / 592 rows, then the slots are added: 3000 in all.
    bw = ((3000 * U * (1 + xm) + off_xhat * 2) * dy.double().abs()).sum(0)
    assert_within(dw, wd.grad.cpu(), bw.cpu(), "dweight")
    assert_within(db, bd.grad.cpu(), bw.cpu(), "dbias")
    empty = lengths == 0
    assert torch.count_nonzero(mean[empty]) == 0
