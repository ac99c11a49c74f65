"""Gated recurrence over ragged windows against the 64-bit formulas, row by
row, forward, backward and single step.

Bounds, with u = 2^-24, M the largest magnitude among states and inputs and n
the window's length. Rounding: a row adds at most 8 u M to the state's error,
and a_t < 1 only shrinks what was there: 8 n u M. The gate: FAST = 2^-19 bounds
the relative error of the exponential for |gate| < 8 (and of the reciprocal);
it moves a_t by at most a_t (1 - a_t) FAST, hence row t's state by 2 M (1 -
a_t) FAST, and the sum over rows of (1 - a_t) times the product of the later
gates telescopes to at most 1: 2 FAST M in all, taken twice. The same for the
gradients, with M the largest accumulated gradient (times twice the largest
state or input for dgate). Outputs add half a step of their type.
"""

import pytest
import torch

from layer_reference import HALF, assert_within, scan64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FAST = 2.0 ** -19


def _offsets(lengths, first=0):
    off = [first]
    for n in lengths:
        off.append(off[-1] + n)
    return torch.tensor(off, dtype=torch.int64)


def _inputs(rows, c, nseg, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, c), generator=g).to(dtype)
    gate = (1.5 * torch.randn((rows, c), generator=g) + 2.0).to(dtype)
    dh = torch.randn((rows, c), generator=g).to(dtype)
    h0 = 0.7 * torch.randn((nseg, c), generator=g)
    df = torch.randn((nseg, c), generator=g)
    return x, gate, dh, h0, df


def _check(x, gate, off, h0, dh, df, what=""):
    from distributed_graph_flow_b200 import aggregation

    dev = "cuda"
    dt = x.dtype
    t = [None if v is None else v.to(dev) for v in (x, gate, off, h0, dh, df)]
    h, final, saved = aggregation.gated_scan(t[0], t[1], t[2], initial=t[3], return_saved=True)
    dx, dgate, dinit = aggregation.gated_scan_backward(t[4], t[0], t[1], t[2], saved, initial=t[3], grad_final=t[5])
    only = aggregation.gated_scan(t[0], t[1], t[2], initial=t[3], return_sequence=False)
    assert only[0] is None and torch.equal(only[1], final)
    eh, ef, edx, edg, edi = scan64(x, gate, off, h0, dh, df)
    inside = torch.zeros((x.shape[0], 1), dtype=torch.bool)
    inside[int(off[0]):int(off[-1])] = True
    n = max([int(v) for v in off[1:] - off[:-1]] + [1])
    r = 8 * n * U + 4 * FAST
    xm = torch.where(inside, x.double(), torch.zeros((), dtype=torch.float64)).abs()
    m = max(float(xm.max()) if xm.numel() else 0.0, 0.0 if h0 is None or not h0.numel() else float(h0.abs().max()), 1.0)
    bh = torch.full_like(eh, r * m)
    assert h.dtype == dt and final.dtype == torch.float32
    assert_within(h, eh, bh + HALF[dt] * (eh.abs() + bh), what + " h")
    assert_within(final, ef, torch.full_like(ef, r * m), what + " final")
    gm = 1.0
    if dh is not None or df is not None:
        gs = torch.where(inside, torch.zeros_like(eh) if dh is None else dh.double(), torch.zeros_like(eh))
        # Accumulated gradient: |delta| <= the largest |dx / (1 - a)|.
        keep = 1 / (1 + torch.exp(gate.double()))
        acc = torch.where(inside, edx / keep, torch.zeros_like(edx)).abs()
        gm = max(float(acc.max()) if acc.numel() else 0.0, float(gs.abs().max()) if gs.numel() else 0.0,
                 0.0 if df is None or not df.numel() else float(df.abs().max()), 1.0)
    bd = torch.full_like(edx, r * gm)
    assert_within(dx, edx, bd + HALF[dt] * (edx.abs() + bd), what + " dx")
    bg = torch.full_like(edx, r * gm * 2 * m)
    assert_within(dgate, edg, bg + HALF[dt] * (edg.abs() + bg), what + " dgate")
    if h0 is not None:
        assert_within(dinit, edi, torch.full_like(edi, r * gm), what + " dinitial")
    else:
        assert dinit is None
    return h, final, dx, dgate


LENGTHS = {
    "one": [1],
    "ones": [1] * 300,
    "empties": [0, 0, 3, 0, 0, 5, 0],
    "windows": [30, 1, 200, 7, 0, 64, 129, 128, 127],
    "long": [2500],
    "two_long": [1300, 0, 1100],
    "runs_of_empties": [0] * 700 + [3] + [0] * 300 + [1, 0, 2] + [0] * 1000 + [40] + [0] * 513,
    "empty_but_the_first": [20] + [0] * 900,
    "empty_but_the_last": [0] * 900 + [20],
}


@pytest.mark.parametrize("lengths", sorted(LENGTHS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("initial", [True, False])
def test_windows(cuda, lengths, dtype, initial):
    off = _offsets(LENGTHS[lengths])
    x, gate, dh, h0, df = _inputs(int(off[-1]), 64, off.numel() - 1, dtype, 1)
    _check(x, gate, off, h0 if initial else None, dh, df, lengths)


@pytest.mark.parametrize("c", [4, 8, 12, 20, 64, 68, 96, 128, 260])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_channels(cuda, c, dtype):
    off = _offsets([300, 5, 0, 1000, 33])
    x, gate, dh, h0, df = _inputs(1338, c, 5, dtype, 2)
    _check(x, gate, off, h0, dh, df, str(c))


def test_one_window_over_many_tiles(cuda):
    """A window that crosses chunks of 16 rows, groups of 32 chunks and supergroups
    of 1024, short ones on either side."""
    off = _offsets([100, 70000, 50, 0, 3])
    x, gate, dh, h0, df = _inputs(70153, 64, 5, torch.float32, 12)
    _check(x, gate, off, h0, dh, df)


@pytest.mark.parametrize("initial", [True, False])
def test_windows_end_at_chunk_edges(cuda, initial):
    """Windows that begin and end at the edges of chunks (16 rows), groups (512)
    and supergroups (16384), and one row to either side of them."""
    lengths = [16384, 512, 16, 16368 - 512, 512 * 31, 512, 1, 16383, 15, 0, 17, 511, 513, 16 * 900, 0, 5000]
    off = _offsets(lengths, first=16)
    rows = int(off[-1]) + 40
    x, gate, dh, h0, df = _inputs(rows, 64, len(lengths), torch.float32, 13)
    _check(x, gate, off, h0 if initial else None, dh, df)


@pytest.mark.parametrize("have", [(True, False), (False, True), (False, False)])
def test_missing_gradients(cuda, have):
    off = _offsets([40, 0, 200])
    x, gate, dh, h0, df = _inputs(240, 32, 3, torch.float32, 3)
    _check(x, gate, off, h0, dh if have[0] else None, df if have[1] else None)


@pytest.mark.parametrize("rows", [0, 1, 127, 128, 129, 256, 257])
def test_row_counts(cuda, rows):
    off = _offsets([rows])
    x, gate, dh, h0, df = _inputs(rows, 64, 1, torch.float32, 4)
    _check(x, gate, off, h0, dh, df)


def test_no_segments(cuda):
    off = torch.zeros(1, dtype=torch.int64)
    x, gate, dh, h0, df = _inputs(70, 64, 0, torch.bfloat16, 4)
    h, _, dx, dgate = _check(x, gate, off, h0, dh, df)
    assert not any(bool(torch.count_nonzero(t)) for t in (h, dx, dgate))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_outside_are_zero_and_unused(cuda, dtype):
    off = _offsets([9, 0, 200], first=5)
    rows = 5 + 209 + 300
    x, gate, dh, h0, df = _inputs(rows, 64, 3, dtype, 5)
    clean = _check(x, gate, off, h0, dh, df)
    for bad in (float("nan"), float("inf"), -float("inf")):
        t = [v.clone() for v in (x, gate, dh)]
        for v in t:
            v[:5] = bad
            v[214:] = bad
        got = _check(t[0], t[1], off, h0, t[2], df)
        assert all(torch.equal(p, q) for p, q in zip(clean, got))
        assert torch.count_nonzero(got[0][:5]) == 0 and torch.count_nonzero(got[2][214:]) == 0


def test_nan_stays_in_its_window(cuda):
    """A NaN reaches the rows after it in its window (before it, going
    backward) and no other window."""
    from distributed_graph_flow_b200 import aggregation

    off = _offsets([400, 300, 500])
    x, gate, dh, h0, df = _inputs(1200, 32, 3, torch.float32, 6)
    ref = _check(x, gate, off, h0, dh, df)
    x[550, 3] = float("nan")
    dh[560, 4] = float("nan")
    t = [v.cuda() for v in (x, gate, off, h0, dh, df)]
    h, final, saved = aggregation.gated_scan(*t[:3], initial=t[3], return_saved=True)
    dx, dgate, dinit = aggregation.gated_scan_backward(t[4], *t[:3], saved, initial=t[3], grad_final=t[5])
    mask = torch.zeros_like(h, dtype=torch.bool)
    mask[550:700, 3] = True
    assert torch.equal(torch.isnan(h), mask) and torch.equal(h[~mask], ref[0][~mask])
    up = torch.zeros_like(mask)
    up[400:561, 4] = True
    assert torch.equal(torch.isnan(dx), up) and torch.equal(dx[~up], ref[2][~up])
    assert bool(torch.isnan(dinit[1, 4])) and int(torch.isnan(dinit).sum()) == 1
    assert int(torch.isnan(final).sum()) == 1


def test_extreme_gates(cuda):
    """Gates that close or open fully: |gate| far beyond where exp overflows."""
    off = _offsets([260])
    x, gate, dh, h0, df = _inputs(260, 16, 1, torch.float32, 7)
    gate[::3] = 200.0
    gate[1::3] = -200.0
    _check(x, gate, off, h0, dh, df)
    gate[:] = 300.0  # a = 1: the state passes unchanged
    _check(x, gate, off, h0, dh, df)
    gate[:] = float("inf")
    from distributed_graph_flow_b200 import aggregation

    h, final = aggregation.gated_scan(x.cuda(), gate.cuda(), off.cuda(), initial=h0.cuda())
    assert torch.equal(final.cpu(), h0) and torch.equal(h.cpu(), h0.expand(260, 16))


def test_bad_offsets_stay_in_bounds(cuda):
    from distributed_graph_flow_b200 import aggregation

    x = torch.randn((500, 16), device="cuda")
    for off in ([0, 10, 1 << 40], [-5, 20, 50], [0, 400, 10, 500], [600, 700, 800]):
        o = torch.tensor(off, dtype=torch.int64, device="cuda")
        h, final, saved = aggregation.gated_scan(x, x, o, return_saved=True)
        aggregation.gated_scan_backward(x, x, x, o, saved)
    torch.cuda.synchronize()


def test_results_repeat(cuda):
    from distributed_graph_flow_b200 import aggregation

    off = _offsets([60000, 41, 0, 900, 50000]).cuda()
    x, gate, dh, h0, df = (t.cuda() for t in _inputs(110941, 64, 5, torch.bfloat16, 8))
    first = None
    for _ in range(4):
        h, final, saved = aggregation.gated_scan(x, gate, off, initial=h0, return_saved=True)
        out = (h, final, *aggregation.gated_scan_backward(dh, x, gate, off, saved, initial=h0, grad_final=df))
        first = first or out
        assert all(torch.equal(p, q) for p, q in zip(first, out))


def test_long_buffers_past_32_bits(cuda):
    from distributed_graph_flow_b200 import aggregation

    rows, c = (1 << 23) + 77, 264
    x = torch.zeros((rows, c), dtype=torch.bfloat16, device="cuda")
    tail = torch.randn((300, c), device="cuda").to(torch.bfloat16)
    x[-300:] = tail
    off = torch.tensor([0, 10, rows - 300, rows], device="cuda")
    h, final, saved = aggregation.gated_scan(x, x, off, return_saved=True)
    eh, ef, edx, edg, _ = scan64(tail.cpu(), tail.cpu(), torch.tensor([0, 300]), None, tail.cpu(), None)
    assert_within(h[-300:], eh, 2.0 ** -7 * (0.5 + eh.abs()), "h")
    assert_within(final[2:], ef, 1e-3 * (1 + ef.abs()), "final")
    dx, dgate, _ = aggregation.gated_scan_backward(x, x, x, off, saved)
    assert_within(dx[-300:], edx, 2.0 ** -7 * (0.5 + edx.abs()), "dx")
    assert_within(dgate[-300:], edg, 2.0 ** -7 * (0.5 + edg.abs()), "dgate")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [0, 1, 33, 5000])
def test_step(cuda, dtype, n):
    """The single step equals the scan over windows of one row, in place too."""
    from distributed_graph_flow_b200 import aggregation

    x, gate, _, h0, _ = (t.cuda() for t in _inputs(n, 24, n, dtype, 9))
    h, state = aggregation.gated_scan_step(x, gate, h0)
    off = torch.arange(n + 1, device="cuda")
    eh, ef = aggregation.gated_scan(x, gate, off, initial=h0)
    assert torch.equal(h, eh) and torch.equal(state, ef)
    e = scan64(x.cpu(), gate.cpu(), off.cpu(), h0.cpu())
    assert_within(state, e[1], (8 * U + 4 * FAST) * 5, "state")
    own = h0.clone()
    h2, s2 = aggregation.gated_scan_step(x, gate, own, out_state=own)
    assert s2 is own and torch.equal(own, state) and torch.equal(h2, h)


def test_streams_and_graphs(cuda):
    from distributed_graph_flow_b200 import aggregation

    off = _offsets([3000, 41, 0, 900]).cuda()
    x, gate, dh, h0, df = (t.cuda() for t in _inputs(3941, 64, 4, torch.float32, 10))

    def step(xx):
        h, final, saved = aggregation.gated_scan(xx, gate, off, initial=h0, return_saved=True)
        return (h, final, *aggregation.gated_scan_backward(dh, xx, gate, off, saved, initial=h0, grad_final=df))

    eager, eager2 = step(x), step(2 * x + 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    h, final = aggregation.gated_scan(x, gate, off, initial=h0, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(h, eager[0]) and torch.equal(final, eager[1])
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
