"""The layer operators as torch operators, and a run of them together: a
trained layer over a sampled batch.

Causal windows of every sampled node -> gated scan (the window's last state is
the node's feature) -> mean over the sampled neighbours and gated update ->
group norm per sampled graph -> dense head. Outputs and all gradients against
the same formulas in 64 bits (autograd over the formulas, on the rounded
values where an operator rounds).

Tolerance: every stage rounds its output and its operands' gradients to bf16
(2^-8 relative each at most) and passes earlier roundings on; over S stages in
a row that is at most about S 2^-8 of the magnitude that is rounded, and relative
to the norm of a whole tensor, where the signs are random, well below the
sum of all of them: 5 roundings on the way forward, 5 back, 10 x 2^-8 = 4e-2.
"""

import pytest
import torch

from layer_reference import act64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(cuda):
    from distributed_graph_flow_b200 import torch_ops

    return torch_ops


def _near(got, exp, rel, what):
    got, exp = got.detach().double().cpu(), exp.detach().double().cpu()
    assert got.shape == exp.shape
    err = float((got - exp).norm() / exp.norm().clamp_min(1e-12))
    assert err <= rel, f"{what}: relative error {err:.2e}"


def test_opcheck(ops):
    g = torch.Generator(device="cuda").manual_seed(0)

    def rnd(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda").to(dtype).requires_grad_(True)

    bf = torch.bfloat16
    off = torch.tensor([0, 9, 9, 40], device="cuda")
    torch.library.opcheck(torch.ops.dgfx.gated_dense_concat.default,
                          (rnd(40, 16, dtype=bf), rnd(40, 8, dtype=bf), rnd(32, 24, dtype=bf), rnd(32, 24, dtype=bf),
                           rnd(32), rnd(32), "gelu"))
    torch.library.opcheck(torch.ops.dgfx.gated_dense_concat.default,
                          (rnd(40, 16, dtype=bf), None, rnd(32, 16, dtype=bf), rnd(32, 16, dtype=bf), None, None,
                           "silu"))
    torch.library.opcheck(torch.ops.dgfx.segment_group_norm.default,
                          (rnd(40, 16), off, 4, rnd(16), rnd(16), 1e-5, "silu"))
    torch.library.opcheck(torch.ops.dgfx.segment_group_norm.default,
                          (rnd(40, 16, dtype=bf), off, 4, None, None, 1e-5, "none"))
    torch.library.opcheck(torch.ops.dgfx.gated_scan.default, (rnd(40, 16), rnd(40, 16), off, rnd(3, 16), True))
    torch.library.opcheck(torch.ops.dgfx.gated_scan.default,
                          (rnd(40, 16, dtype=bf), rnd(40, 16, dtype=bf), off, None, True))


def test_gradients_by_differences(ops):
    """float32 operators against central differences of themselves along
    random directions, with a step h = 2^-7. The quotient is off by the
    values' rounding, 2^-24 |y| / h, and by h^2 / 6 times the third derivative along
    the direction, below 10 for these scales: 1e-3 in all, relative to the
    magnitude of the terms."""
    g = torch.Generator(device="cuda").manual_seed(1)
    off = torch.tensor([0, 9, 9, 40], device="cuda")

    def rnd(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def check(fn, *inputs):
        leaves = [t.clone().requires_grad_(True) for t in inputs]
        w = [rnd(*o.shape) / o.numel() ** 0.5 for o in fn(*inputs)]

        def loss(*a):
            return sum((o.double() * v.double()).sum() for o, v in zip(fn(*a), w))

        loss(*leaves).backward()
        for i, t in enumerate(inputs):
            d = rnd(*t.shape) / t.numel() ** 0.5
            h = 2.0 ** -7
            up, down = list(inputs), list(inputs)
            up[i], down[i] = t + h * d, t - h * d
            diff = float(loss(*up) - loss(*down)) / (2 * h)
            along = float((leaves[i].grad.double() * d.double()).sum())
            assert abs(along - diff) <= 1e-3 * (1 + abs(diff)), (i, along, diff)

    check(lambda x, w, b: (ops.segment_group_norm(x, off, 4, w, b, activation="gelu"),), rnd(40, 16), rnd(16), rnd(16))
    check(lambda x, gate, h0: ops.gated_scan(x, gate, off, h0), rnd(40, 16), rnd(40, 16), rnd(3, 16))


def test_expanded_and_strided_gradients(ops):
    """Gradients that arrive expanded (from a sum) or strided (from a slice)."""
    off = torch.tensor([0, 30, 64], device="cuda")
    x = torch.randn((64, 32), device="cuda", requires_grad=True)
    gate = torch.randn((64, 32), device="cuda", requires_grad=True)
    ops.segment_group_norm(x, off, 4, activation="silu").sum().backward()
    first = x.grad.clone()
    x.grad = None
    (ops.segment_group_norm(x, off, 4, activation="silu") * 1.0).sum().backward()
    assert torch.allclose(first, x.grad, rtol=0, atol=1e-6)
    x.grad = None
    h, final = ops.gated_scan(x, gate, off)
    h[:, ::2].sum().backward()
    assert bool(torch.isfinite(x.grad).all()) and bool((x.grad[:, 1::2] == 0).all())
    x.grad = gate.grad = None
    final2 = ops.gated_scan(x, gate, off)[1]
    final2.sum().backward()
    assert bool((x.grad != 0).any())
    xb = torch.randn((64, 32), device="cuda").bfloat16().requires_grad_(True)
    w = torch.randn((32, 32), device="cuda").bfloat16().requires_grad_(True)
    torch.ops.dgfx.gated_dense_concat(xb, None, w, w, None, None, "relu").sum().backward()
    assert bool(torch.isfinite(xb.grad).all()) and bool((w.grad != 0).any())


def test_scan_without_gradient_keeps_nothing(ops):
    x = torch.randn((64, 32), device="cuda", requires_grad=True)
    off = torch.tensor([0, 64], device="cuda")
    with torch.no_grad():
        h, final = ops.gated_scan(x, x, off)
    assert not h.requires_grad
    with pytest.raises(RuntimeError, match="keep_states"):
        torch.ops.dgfx.gated_scan(x, x, off, None, False)


def _batch():
    """A sampled merged batch (one node set) and its CSR."""
    from distributed_graph_flow_b200 import _native, aggregation, synth
    from distributed_graph_flow_b200.sampling import _in_memory_sampler_ext as ext
    from distributed_graph_flow_b200.sampling import config as cfg

    dev = torch.device("cuda", 0)
    spec = synth.GraphSpec(3000, 30_000, 2.1, 500, seed=1, ts_range=(0, 50))
    index, _, _ = synth.build_graph(spec, dev)
    plan = cfg.explicit_plan("v", "e", [6, 4])
    s = ext.create_device_sampler(plan, ["v"], [spec.num_nodes], ["e"], [index], [None], _native.MODE_FIRST, seed=3,
                                  has_temporal=True)
    seeds = synth.uniform_int(64, 0, spec.num_nodes, 21, 9, dev)
    sts = synth.uniform_int(64, 10, 55, 22, 9, dev)
    batch = s.sample_merged(seeds, sts)
    rowptr, col = aggregation.batch_csr(batch)
    return batch, rowptr, col[: int(rowptr[-1])]  # the matrix's gradient takes the entries without spare capacity


def test_layer_over_a_sampled_batch(ops):
    from distributed_graph_flow_b200 import aggregation

    batch, rowptr, col = _batch()
    nodes = int(batch.node_offsets[-1])
    rows_cap = int(batch.node_ids.numel())
    assert rows_cap > nodes  # spare capacity behind the last graph
    g = torch.Generator(device="cuda").manual_seed(2)
    f, n_out = 32, 64

    def rnd(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype).requires_grad_(True)

    bf = torch.bfloat16
    lengths = torch.randint(0, 30, (rows_cap,), generator=g, device="cuda")
    windows = torch.cat([lengths.new_zeros(1), torch.cumsum(lengths, 0)])
    obs = int(windows[-1])
    x, gate = rnd(obs, f, dtype=bf), rnd(obs, f, dtype=bf, scale=1.5)
    h0 = rnd(rows_cap, f, scale=0.5)
    wg, wu = rnd(n_out, 2 * f, dtype=bf, scale=0.15), rnd(n_out, 2 * f, dtype=bf, scale=0.15)
    bg, bu = rnd(n_out, scale=0.1), rnd(n_out, scale=0.1)
    nw, nb = rnd(n_out), rnd(n_out)
    head = (torch.randn((64, n_out), generator=g, device="cuda") * 0.1).to(bf)
    leaves = (x, gate, h0, wg, wu, bg, bu, nw, nb)

    _, final = ops.gated_scan(x, gate, windows, h0)
    feats = final.to(bf)
    upd = ops.sage_mean_gated(rowptr, col, feats, wg, wu, bg, bu, "silu")
    normed = ops.segment_group_norm(upd, batch.node_offsets, 8, nw, nb, activation="gelu")
    weights = torch.randn(normed.shape, generator=g, device="cuda") / nodes ** 0.5
    (normed.float() * weights).sum().backward()
    out = aggregation.dense_concat(normed.detach(), None, head, None, relu=False)
    aggregation.dense_check()
    assert torch.count_nonzero(normed[nodes:]) == 0 and torch.count_nonzero(out[nodes:]) == 0

    # The same in 64 bits.
    d = [t.detach().double().requires_grad_(True) for t in leaves]
    dx, dgate, dh0, dwg, dwu, dbg, dbu, dnw, dnb = d
    a = torch.sigmoid(dgate)
    state = dh0
    step = torch.arange(int(lengths.max()), device="cuda")
    for t in step.tolist():
        live = lengths > t
        r = (windows[:-1] + t).clamp_max(obs - 1)
        state = torch.where(live[:, None], a[r] * state + (1 - a[r]) * dx[r], state)
    deg = (rowptr[1:] - rowptr[:-1])
    row = torch.repeat_interleave(torch.arange(rows_cap, device="cuda"), deg)
    agg = torch.zeros((rows_cap, f), dtype=torch.float64, device="cuda").index_add(0, row, state[col.long()])
    cat = torch.cat([state, agg / deg.clamp_min(1)[:, None]], 1)
    u = act64(cat @ dwg.t() + dbg, "silu") * (cat @ dwu.t() + dbu)
    seg = torch.repeat_interleave(torch.arange(64, device="cuda"), batch.node_offsets[1:] - batch.node_offsets[:-1])
    v = u[:nodes].view(nodes, 8, -1)
    cnt = torch.bincount(seg, minlength=64).double()[:, None].clamp_min(1)

    def seg_mean(t):
        return (torch.zeros((64, 8), dtype=torch.float64, device="cuda").index_add(0, seg, t.mean(2)) / cnt)[seg][:, :, None]

    c = v - seg_mean(v)
    z = (c / torch.sqrt(seg_mean(c * c) + 1e-5)).reshape(nodes, n_out) * dnw + dnb
    y = act64(z, "gelu")
    (y * weights[:nodes].double()).sum().backward()
    _near(normed[:nodes], y, 4e-2, "output")
    _near(out[:nodes], y @ head.double().t(), 4e-2, "head")
    names = ("x", "gate", "initial", "w_gate", "w_up", "b_gate", "b_up", "norm weight", "norm bias")
    for name, got, exp in zip(names, leaves, d):
        assert got.grad.dtype == got.dtype
        _near(got.grad, exp.grad, 4e-2, "gradient of " + name)


def test_captured_layer_matches_eager(ops):
    """Forward and backward of the layer operators captured in one CUDA graph:
    replays on new inputs give the eager values and gradients bit for bit."""
    off = torch.tensor([0, 300, 300, 777, 900], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)

    def rnd(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    bf = torch.bfloat16
    gate, w = rnd(1000, 64, dtype=bf), rnd(64, 64, dtype=bf, scale=0.2)
    nw = rnd(64)

    def step(x, gt, wt, nwt):
        h, final = ops.gated_scan(x, gt, off)
        y = ops.segment_group_norm(torch.ops.dgfx.gated_dense_concat(h, None, wt, wt, None, None, "silu"), off, 8, nwt,
                                   None, activation="relu")
        loss = y.float().square().sum() + final.sum()
        return (y, final, *torch.autograd.grad(loss, (x, gt, wt, nwt)))

    def leaves(x):
        return [t.clone().requires_grad_(True) for t in (x, gate, w, nw)]

    xs = [rnd(1000, 64, dtype=bf) for _ in range(3)]
    eager = [[t.detach().clone() for t in step(*leaves(x))] for x in xs]
    static = leaves(xs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)  # warm-up outside of the capture
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for x, exp in zip(xs, eager):
        with torch.no_grad():
            static[0].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, exp))


def test_tensor_form_of_the_gated_layer(ops):
    """aggregation.sage_mean_gated (into given buffers, on another stream)
    against the torch operator, bit for bit."""
    from distributed_graph_flow_b200 import aggregation

    batch, rowptr, col = _batch()
    rows = int(rowptr.numel()) - 1
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((rows, 32), generator=g, device="cuda").to(torch.bfloat16)
    wg, wu = (0.2 * torch.randn((2, 40, 64), generator=g, device="cuda")).to(torch.bfloat16)
    bg = torch.randn(40, generator=g, device="cuda")
    ref = ops.sage_mean_gated(rowptr, col, x, wg.contiguous(), wu.contiguous(), bg, None, "gelu")
    agg = torch.empty((rows, 32), dtype=torch.bfloat16, device="cuda")
    out = torch.empty((rows, 40), dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = aggregation.sage_mean_gated(rowptr, col, x, wg.contiguous(), wu.contiguous(), bg, None, "gelu", agg=agg, out=out,
                                      stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, ref)
    aggregation.dense_check()
