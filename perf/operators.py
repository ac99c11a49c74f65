"""Cases and plain forms of the layer operators around the neighbour aggregation.

Three operators, each with its backward pass:

* gated dense layer over a concat: h = act(g) * u with g = [x1 | x2] Wg^T + bg and u = [x1 | x2] Wu^T + bu;
* group norm with an activation over the ragged segments of a merged batch, channels last;
* gated linear recurrence h_t = a_t h_{t-1} + (1 - a_t) x_t, a_t = sigmoid(gate_t), over ragged windows, and its
  single step.

``own`` selects the framework's kernels; otherwise ``run`` computes the plain form in elementary torch operations.
"""

import math

import numpy as np
import torch

own = False

_EPS = 1e-5
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _gated(name, rows, k1, k2, n, act, train):
    return {"name": name, "op": "gated", "rows": rows, "k1": k1, "k2": k2, "n": n, "act": act, "train": train}


def _norm(name, segments, rows, spare, channels, groups, dtype, act, lengths, train):
    return {"name": name, "op": "norm", "segments": segments, "rows": rows, "spare": spare, "channels": channels,
            "groups": groups, "dtype": dtype, "act": act, "lengths": lengths, "train": train}


def _scan(name, segments, rows, spare, channels, dtype, initial, lengths, train):
    return {"name": name, "op": "scan", "segments": segments, "rows": rows, "spare": spare, "channels": channels,
            "dtype": dtype, "initial": initial, "lengths": lengths, "train": train}


def listed():
    return [
        # One node scored online: the update of a single row, all weights read for it.
        _gated("gated one row", 1, 256, 256, 512, "silu", False),
        # A mid-sized batch with feature widths that are no multiple of a tile.
        _gated("gated odd widths", 10007, 104, 0, 200, "relu", False),
        # The update of a full GraphSAGE layer (256 own + 256 aggregated features), inference.
        _gated("gated layer", 500000, 256, 256, 512, "silu", False),
        # The same layer in training: output and all six gradients.
        _gated("gated layer train", 500000, 256, 256, 512, "silu", True),
        # A handful of small sampled graphs: latency of one small call.
        _norm("norm few small graphs", 8, 200, 0, 64, 8, "bf16", "silu", "tree", False),
        # A merged batch of 1024 seeds, [10, 5] trees, in buffers with room for more rows.
        _norm("norm merged batch", 1024, 41003, 9000, 256, 32, "bf16", "relu", "tree", False),
        # One whole graph as one segment, training.
        _norm("norm whole graph train", 1, 1000000, 0, 256, 16, "bf16", "silu", "tree", True),
        # A batch of whole graphs of very different sizes (empty ones among them), fp32, training.
        _norm("norm ragged graphs train", 300, 250001, 1000, 200, 25, "f32", "gelu", "zipf", True),
        # Online update of one new observation per tracked node.
        {"name": "scan step", "op": "step", "segments": 512, "channels": 256, "dtype": "bf16"},
        # Causal windows of the sampled nodes of a batch, encoded for inference.
        _scan("scan windows", 20000, 600011, 5000, 64, "bf16", False, "zipf", False),
        # Windows of a training batch, with states carried over from earlier windows.
        _scan("scan windows train", 30000, 1200007, 0, 128, "bf16", True, "tree", True),
        # A few long series (sensor histories), fp32, training.
        _scan("scan long series train", 3, 393209, 0, 96, "f32", True, "tree", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gated", "norm", "scan", "gated", "norm", "scan", "step"])
    if op == "gated":
        case = {"op": op, "k1": 8 * _log(rng, 1, 64), "k2": rng.choice([0, 1]) * 8 * _log(rng, 1, 64),
                "n": 8 * _log(rng, 1, 128), "act": rng.choice(["silu", "gelu", "sigmoid"]),
                "train": rng.random() < 0.5}
        most = min(500000, 500000 * 512 * 512 // ((case["k1"] + case["k2"]) * case["n"]))
        return {**case, "rows": _log(rng, 1, max(2, most))}
    if op == "step":
        return {"op": op, "segments": _log(rng, 1, 60000), "channels": 8 * _log(rng, 1, 64),
                "dtype": rng.choice(["bf16", "f32"])}
    dtype = rng.choice(["bf16", "f32"])
    segments = _log(rng, 1, 30000)
    channels = 8 * _log(rng, 1, 64 if op == "norm" else 32)
    rows = _log(rng, 10, min(1000000, 100_000_000 // channels))
    case = {"op": op, "segments": segments, "rows": rows, "spare": rng.choice([0, rows // 5]), "channels": channels,
            "dtype": dtype, "lengths": rng.choice(["tree", "zipf"]), "train": rng.random() < 0.5}
    if op == "norm":
        return {**case, "groups": rng.choice([g for g in range(1, channels + 1) if channels % g == 0]),
                "act": rng.choice(["none", "silu", "gelu"])}
    return {**case, "initial": rng.random() < 0.5}


def work(case):
    if case["op"] == "gated":
        m, k, n = case["rows"], case["k1"] + case["k2"], case["n"]
        moved, flops = 2 * (m * k + 2 * n * k + m * n) + 8 * n, 4 * m * n * k
        if case["train"]:
            moved += 2 * (m * n + m * k + 2 * n * k) + 8 * n
            flops *= 3
        return {"bytes": moved, "flops": flops}
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "step":
        elems = case["segments"] * case["channels"]
        return {"bytes": elems * (3 * e + 8), "flops": 8 * elems}
    used, held = case["rows"] * case["channels"], (case["rows"] + case["spare"]) * case["channels"]
    if case["op"] == "norm":
        moved = e * (used + held) + 8 * case["segments"] + 8 * case["channels"]
        if case["train"]:
            moved += e * (used + held) + 8 * case["channels"]
        return {"bytes": moved, "flops": (30 if case["train"] else 10) * used}
    states = 4 * case["segments"] * case["channels"]
    moved = e * (2 * used + held) + 8 * case["segments"] + states * (2 if case["initial"] else 1)
    if case["train"]:
        moved += e * (used + 2 * held) + states * (2 if case["initial"] else 1)
    return {"bytes": moved, "flops": (24 if case["train"] else 8) * used}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _lengths(case, seed):
    """Lengths of the segments, in sum case["rows"]."""
    rng = np.random.default_rng(seed)
    s, rows = case["segments"], case["rows"]
    if case["lengths"] == "zipf":  # many short ones, a few very long ones, empty ones
        share = rng.pareto(1.1, s) + 1e-3
    else:  # sampled trees: sizes within a factor of a few of each other
        share = rng.gamma(3.0, 1.0, s) + 0.1
    lengths = np.floor(share / share.sum() * rows).astype(np.int64)
    lengths[int(np.argmax(lengths))] += rows - lengths.sum()
    return lengths


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)

    def normal(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=gen, device=dev) * scale + shift).to(dtype)

    state = {"case": case}
    if case["op"] == "gated":
        m, k1, k2, n = case["rows"], case["k1"], case["k2"], case["n"]
        lim = math.sqrt(6.0 / (k1 + k2 + n))
        for name in ("w_gate", "w_up"):
            w = (torch.rand((n, k1 + k2), generator=gen, device=dev) * 2 - 1) * lim
            state[name] = w.to(torch.bfloat16)
        state["b_gate"], state["b_up"] = normal(n, scale=0.1), normal(n, scale=0.1)
        state["x1"] = normal(m, k1, dtype=torch.bfloat16)
        state["x2"] = normal(m, k2, dtype=torch.bfloat16) if k2 else None
        state["grad"] = normal(m, n, dtype=torch.bfloat16) if case["train"] else None
        return state
    dtype = _TYPES[case["dtype"]]
    c = case["channels"]
    if case["op"] == "step":
        s = case["segments"]
        state["x"], state["gate"] = normal(s, c, dtype=dtype), normal(s, c, dtype=dtype, scale=1.5, shift=1.0)
        state["state"] = normal(s, c, scale=0.7)
        return state
    lengths = _lengths(case, seed)
    state["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)).to(dev)
    state["longest"] = int(lengths.max())
    held = case["rows"] + case["spare"]
    if case["op"] == "norm":
        # Features are not centred: a channel's mean is as large as its spread.
        state["x"] = (torch.randn((held, c), generator=gen, device=dev) * 1.3
                      + torch.randn(c, generator=gen, device=dev)).to(dtype)
        state["weight"], state["bias"] = normal(c, scale=0.3, shift=1.0), normal(c, scale=0.3)
        state["grad"] = normal(held, c, dtype=dtype) if case["train"] else None
        return state
    state["x"] = normal(held, c, dtype=dtype)
    state["gate"] = normal(held, c, dtype=dtype, scale=1.5, shift=2.0)  # mostly long memories
    state["initial"] = normal(case["segments"], c, scale=0.7) if case["initial"] else None
    if case["train"]:
        state["grad"] = normal(held, c, dtype=dtype)
        state["grad_final"] = normal(case["segments"], c)
    return state


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _act(z, kind):
    if kind == "none":
        return z
    if kind == "relu":
        return z.clamp_min(0)
    if kind == "sigmoid":
        return torch.sigmoid(z)
    if kind == "silu":
        return z * torch.sigmoid(z)
    return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))  # gelu


def _act_grad(z, kind):
    if kind == "none":
        return torch.ones_like(z)
    if kind == "relu":
        return (z > 0).to(z.dtype)
    s = torch.sigmoid(z)
    if kind == "sigmoid":
        return s * (1.0 - s)
    if kind == "silu":
        return s * (1.0 + z * (1.0 - s))
    return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_gated(st):
    case = st["case"]
    x = st["x1"].float() if st["x2"] is None else torch.cat([st["x1"], st["x2"]], 1).float()
    wg, wu = st["w_gate"].float(), st["w_up"].float()
    g = x @ wg.t() + st["b_gate"]
    u = x @ wu.t() + st["b_up"]
    a = _act(g, case["act"])
    out = {"h": (a * u).to(torch.bfloat16)}
    if case["train"]:
        dh = st["grad"].float()
        du = dh * a
        dg = dh * u * _act_grad(g, case["act"])
        dx = (dg @ wg + du @ wu).to(torch.bfloat16)
        out["dx1"] = dx[:, :case["k1"]]
        if case["k2"]:
            out["dx2"] = dx[:, case["k1"]:]
        out["dw_gate"], out["dw_up"] = (dg.t() @ x).to(torch.bfloat16), (du.t() @ x).to(torch.bfloat16)
        out["db_gate"], out["db_up"] = dg.double().sum(0).float(), du.double().sum(0).float()
    return out


def _row_segments(offsets, rows):
    """Segment of each row; rows outside of every segment get the number of segments."""
    r = torch.arange(rows, device=offsets.device)
    s = torch.searchsorted(offsets[1:].contiguous(), r, right=True)
    return torch.where(r < offsets[0], torch.full_like(s, offsets.numel() - 1), s)


def _plain_norm(st):
    case, x = st["case"], st["x"]
    s, g = case["segments"], case["groups"]
    rows, c = x.shape
    seg = _row_segments(st["offsets"], rows)
    inside = (seg < s)[:, None, None]
    xf = x.float().view(rows, g, c // g)
    count = ((st["offsets"][1:] - st["offsets"][:-1]).clamp_min(1) * (c // g)).double()
    count = torch.cat([count, count.new_ones(1)])[:, None]

    def mean_of(v):  # mean over each segment's rows and each group's channels, back at the rows
        sums = torch.zeros((s + 1, g), dtype=torch.float64, device=x.device)
        sums.index_add_(0, seg, v.sum(2).double())
        return (sums / count).float()[seg][:, :, None]

    centred = xf - mean_of(xf)
    rstd = torch.rsqrt(mean_of(centred * centred) + _EPS)
    xhat = centred * rstd
    w, b = st["weight"].view(1, g, -1), st["bias"].view(1, g, -1)
    z = xhat * w + b
    zero = torch.zeros((), device=x.device)
    out = {"y": torch.where(inside, _act(z, case["act"]), zero).view(rows, c).to(x.dtype)}
    if case["train"]:
        dz = torch.where(inside, st["grad"].float().view(rows, g, -1) * _act_grad(z, case["act"]), zero)
        dxhat = dz * w
        dx = rstd * (dxhat - mean_of(dxhat) - xhat * mean_of(dxhat * xhat))
        out["dx"] = torch.where(inside, dx, zero).view(rows, c).to(x.dtype)
        out["dweight"] = torch.where(inside, dz * xhat, zero).view(rows, c).double().sum(0).float()
        out["dbias"] = dz.view(rows, c).double().sum(0).float()
    return out


def _doubling(a, u, longest):
    """h_t = a_t h_{t-1} + u_t down the rows (a_t = 0 at the first row of a segment), spans doubled step by step."""
    span = 1
    while span < longest:
        u = torch.cat([u[:span], u[span:] + a[span:] * u[:-span]])
        a = torch.cat([a[:span], a[span:] * a[:-span]])
        span *= 2
    return u


def _plain_scan(st):
    case, off = st["case"], st["offsets"]
    rows, c = st["x"].shape
    s = case["segments"]
    seg = _row_segments(off, rows)
    inside = (seg < s)[:, None]
    r = torch.arange(rows, device=off.device)
    ends = torch.cat([off, off[-1:]])
    begins = torch.cat([off[:-1], off[-1:]])
    first = (r == begins[seg])[:, None]
    last = (r == ends[seg + 1] - 1)[:, None]
    x, gate = st["x"].float(), st["gate"].float()
    a, keep = torch.sigmoid(gate), torch.sigmoid(-gate)
    h0 = torch.zeros((s, c), device=x.device) if st["initial"] is None else st["initial"]
    before = torch.cat([h0, h0.new_zeros(1, c)])[seg]
    zero = torch.zeros((), device=x.device)
    u = keep * x + torch.where(first, a * before, zero)
    h = _doubling(torch.where(first | ~inside, zero, a), torch.where(inside, u, zero), st["longest"])
    filled = (off[1:] > off[:-1])[:, None]
    final = torch.where(filled, h[(off[1:] - 1).clamp_min(0)], h0)
    out = {"h": h.to(st["x"].dtype), "final": final}
    if case["train"]:
        tail = torch.cat([st["grad_final"], h0.new_zeros(1, c)])[seg]
        d = torch.where(inside, st["grad"].float() + torch.where(last, tail, zero), zero)
        nxt = torch.where(last | ~inside, zero, torch.cat([a[1:], a[:1]]))
        delta = _doubling(nxt.flip(0), d.flip(0), st["longest"]).flip(0)
        prev = torch.where(first, before, torch.cat([h[:1], h[:-1]]))
        out["dx"] = torch.where(inside, keep * delta, zero).to(st["x"].dtype)
        out["dgate"] = torch.where(inside, delta * (prev - x) * a * keep, zero).to(st["x"].dtype)
        if case["initial"]:
            at = off[:-1].clamp_max(rows - 1)
            out["dinitial"] = torch.where(filled, (a * delta)[at], st["grad_final"])
    return out


def _plain_step(st):
    gate = st["gate"].float()
    h = torch.sigmoid(gate) * st["state"] + torch.sigmoid(-gate) * st["x"].float()
    return {"h": h.to(st["x"].dtype), "state": h}


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------
def _own_gated(st):
    from distributed_graph_flow_b200 import aggregation

    act = st["case"]["act"]
    args = (st["x1"], st["x2"], st["w_gate"], st["w_up"], st["b_gate"], st["b_up"])
    out = {"h": aggregation.gated_dense_concat(*args, activation=act)}
    if st["case"]["train"]:
        names = ("dx1", "dx2", "dw_gate", "dw_up", "db_gate", "db_up")
        grads = aggregation.gated_dense_concat_backward(st["grad"], *args, activation=act)
        out.update({n: g for n, g in zip(names, grads) if g is not None})
    return out


def _own_norm(st):
    from distributed_graph_flow_b200 import aggregation

    case = st["case"]
    y, mean, rstd = aggregation.segment_group_norm(st["x"], st["offsets"], case["groups"], st["weight"], st["bias"],
                                                   eps=_EPS, activation=case["act"])
    out = {"y": y}
    if case["train"]:
        out["dx"], out["dweight"], out["dbias"] = aggregation.segment_group_norm_backward(
            st["grad"], st["x"], st["offsets"], mean, rstd, st["weight"], st["bias"], activation=case["act"])
    return out


def _own_scan(st):
    from distributed_graph_flow_b200 import aggregation

    case = st["case"]
    if not case["train"]:
        h, final = aggregation.gated_scan(st["x"], st["gate"], st["offsets"], initial=st["initial"])
        return {"h": h, "final": final}
    h, final, saved = aggregation.gated_scan(st["x"], st["gate"], st["offsets"], initial=st["initial"],
                                             return_saved=True)
    dx, dgate, dinitial = aggregation.gated_scan_backward(st["grad"], st["x"], st["gate"], st["offsets"], saved,
                                                          initial=st["initial"], grad_final=st["grad_final"])
    out = {"h": h, "final": final, "dx": dx, "dgate": dgate}
    if case["initial"]:
        out["dinitial"] = dinitial
    return out


def _own_step(st):
    from distributed_graph_flow_b200 import aggregation

    h, state = aggregation.gated_scan_step(st["x"], st["gate"], st["state"])
    return {"h": h, "state": state}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"gated": _own_gated, "norm": _own_norm, "scan": _own_scan, "step": _own_step}[op](state)
    return {"gated": _plain_gated, "norm": _plain_norm, "scan": _plain_scan, "step": _plain_step}[op](state)


# ---------------------------------------------------------------------------
# 64-bit values, from the definitions
# ---------------------------------------------------------------------------
def _act64(z, kind):
    fn = {"none": lambda t: t, "relu": torch.relu, "sigmoid": torch.sigmoid, "silu": lambda t: t / (1 + torch.exp(-t)),
          "gelu": lambda t: t * (0.5 * torch.erfc(-t / math.sqrt(2.0)))}[kind]
    return fn(z)


def _exact_gated(st):
    case = st["case"]
    leaf = {k: st[k].double().requires_grad_(case["train"])
            for k in ("x1", "x2", "w_gate", "w_up", "b_gate", "b_up") if st[k] is not None}
    k1 = case["k1"]

    def project(w, b):
        p = torch.addmm(b, leaf["x1"], w[:, :k1].t())
        return p if st["x2"] is None else torch.addmm(p, leaf["x2"], w[:, k1:].t())

    h = _act64(project(leaf["w_gate"], leaf["b_gate"]), case["act"]) * project(leaf["w_up"], leaf["b_up"])
    out = {"h": h.detach()}
    if case["train"]:
        h.backward(st["grad"].double())
        out.update({"d" + k: v.grad for k, v in leaf.items()})
    return out


def _exact_norm(st):
    case, off = st["case"], st["offsets"]
    lo, hi = int(off[0]), int(off[-1])
    lengths = off[1:] - off[:-1]
    g = case["groups"]
    x = st["x"][lo:hi].double().requires_grad_(case["train"])
    w, b = (st[k].double().requires_grad_(case["train"]) for k in ("weight", "bias"))
    full = lengths[lengths > 0]
    marks = torch.cumsum(full, 0)

    def averages(v):  # [rows, channels] -> [filled segments, groups], by differences of running sums
        v = v.reshape(v.shape[0], g, -1).mean(2)
        run_ = torch.cat([v.new_zeros(1, g), torch.cumsum(v, 0)])
        return (run_[marks] - run_[marks - full]) / full[:, None]

    def spread(v):
        return torch.repeat_interleave(v, full, dim=0).repeat_interleave(case["channels"] // g, dim=1)

    dev = x - spread(averages(x))
    y = _act64(dev / torch.sqrt(spread(averages(dev ** 2)) + _EPS) * w + b, case["act"])

    def placed(v):
        p = torch.zeros(st["x"].shape, dtype=torch.float64, device=v.device)
        p[lo:hi] = v
        return p

    out = {"y": placed(y.detach())}
    if case["train"]:
        y.backward(st["grad"][lo:hi].double())
        out.update({"dx": placed(x.grad), "dweight": w.grad, "dbias": b.grad})
    return out


def _recur64(a, u):
    """h_t = a_t h_{t-1} + u_t from h = 0: step by step within blocks of rows, then over the blocks' ends."""
    t, c = u.shape
    size = max(1, int(math.sqrt(t)))
    blocks = -(-t // size)
    pad = (0, 0, 0, blocks * size - t)
    a, u = (torch.nn.functional.pad(v, pad).view(blocks, size, c).clone() for v in (a, u))
    for i in range(1, size):
        u[:, i] += a[:, i] * u[:, i - 1]
        a[:, i] *= a[:, i - 1]
    carry = torch.zeros((blocks, c), dtype=u.dtype, device=u.device)
    for j in range(1, blocks):
        carry[j] = u[j - 1, -1] + a[j - 1, -1] * carry[j - 1]
    return (u + a * carry[:, None]).view(blocks * size, c)[:t]


def _exact_scan(st):
    case = st["case"]
    off = st["offsets"].cpu().numpy()
    lo, hi = int(off[0]), int(off[-1])
    lengths = np.diff(off)
    filled = torch.from_numpy(np.flatnonzero(lengths > 0)).to(st["x"].device)
    start = torch.from_numpy(off[:-1][lengths > 0] - lo).to(st["x"].device)
    end = torch.from_numpy(off[1:][lengths > 0] - lo - 1).to(st["x"].device)
    x, gate = st["x"][lo:hi].double(), st["gate"][lo:hi].double()
    h0 = torch.zeros((case["segments"], case["channels"]), dtype=torch.float64, device=x.device)
    if st["initial"] is not None:
        h0 = st["initial"].double()
    a = 1 / (1 + torch.exp(-gate))
    u = x / (1 + torch.exp(gate))
    u[start] += a[start] * h0[filled]
    linked = a.clone()
    linked[start] = 0
    h = _recur64(linked, u)
    final = h0.clone()
    final[filled] = h[end]

    def placed(v):
        p = torch.zeros(st["x"].shape, dtype=torch.float64, device=v.device)
        p[lo:hi] = v
        return p

    out = {"h": placed(h), "final": final}
    if case["train"]:
        d = st["grad"][lo:hi].double()
        gf = st["grad_final"].double()
        d[end] += gf[filled]
        later = torch.cat([linked[1:], linked.new_zeros(1, linked.shape[1])])
        delta = torch.flip(_recur64(torch.flip(later, [0]), torch.flip(d, [0])), [0])
        prev = torch.cat([h.new_zeros(1, h.shape[1]), h[:-1]])
        prev[start] = h0[filled]
        out["dx"] = placed(delta / (1 + torch.exp(gate)))
        out["dgate"] = placed(delta * (prev - x) * a / (1 + torch.exp(gate)))
        if case["initial"]:
            out["dinitial"] = gf.clone()
            out["dinitial"][filled] = a[start] * delta[start]
    return out


def _exact_step(st):
    e = torch.exp(-st["gate"].double())
    h = (st["state"].double() + e * st["x"].double()) / (1 + e)
    return {"h": h, "state": h.clone()}


def exact(case, seed):
    st = prepare(case, seed)
    return {"gated": _exact_gated, "norm": _exact_norm, "scan": _exact_scan, "step": _exact_step}[case["op"]](st)
