"""Sparse neighbour aggregation on B200 (torch tensors in and out).

The two forms the reference's GNN layers use:
  * ``segment_sum(data, segment_ids, num_segments, mean=...)`` —
    jax.ops.segment_sum as called in hetero_gnn.py:283-295 (mean divides by
    max(count, 1)); out-of-range ids are dropped.
  * ``csr_spmm(rowptr, col, x, val=None, normalize=...)`` — the
    ``SparseMatrix @ dense`` of homo_gnn_sparse_deferred.py:138-161 with rows
    = message targets and columns = message sources (message_passing.py:
    24-38); normalize=True is the row-normalised (mean) aggregation.
Both run in hand-written sm_100a kernels (csrc/aggregate.cu) and accumulate
in fp32; inputs/outputs are fp32 or bf16.

Around the aggregation, the operators of the layers, with their gradients:
``dense_concat`` and ``gated_dense_concat`` (the update, csrc/dense.cu and
csrc/gated.cu), ``segment_group_norm`` (per-graph norm of a merged batch,
csrc/segment_norm.cu) and ``gated_scan`` (recurrence over ragged windows,
csrc/gated_scan.cu).
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch

from distributed_graph_flow_b200 import _native


def _dtype_code(t) -> int:
    torch = _native.require_cuda()
    if t == torch.float32:
        return _native.F32
    if t == torch.bfloat16:
        return _native.BF16
    raise ValueError(f"unsupported dtype {t}; expected float32 or bfloat16")


def _temporary(shape, dtype, device, stream):
    """Memory that only the kernels of a call on ``stream`` (None: the current
    one) use: from that stream's pool, so that it is not handed out again
    before they are done, however soon the call drops it."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def csr_spmm(rowptr, col, x, val=None, normalize: bool = False, out=None, out_dtype=None, num_rows: Optional[int] = None,
             workspace=None, stream=None):
    """Y[r] = scale_r * sum_j val_j * X[col_j] over CSR row r.

    rowptr int64 [R+1], col int32 [nnz], val float32 [nnz] or None (ones),
    x [N, F] float32/bfloat16 (row-major, F a multiple of 8). normalize gives
    scale_r = 1 / max(deg_r, 1).
    """
    torch = _native.require_cuda()
    if x.get_device() not in (-1, _native.current_device()):  # launches go to x's device
        with torch.cuda.device(x.get_device()):
            return csr_spmm(rowptr, col, x, val, normalize, out, out_dtype, num_rows, workspace, stream)
    R = int(rowptr.numel()) - 1 if num_rows is None else int(num_rows)
    nnz = int(col.numel())
    F = int(x.shape[1])
    if out is None:
        out = torch.empty((R, F), dtype=out_dtype or x.dtype, device=x.device)
    if col.dtype != torch.int32 or rowptr.dtype != torch.int64:
        raise ValueError("rowptr must be int64 and col int32")
    if not x.is_contiguous() or not out.is_contiguous():
        raise ValueError("x and out must be contiguous")
    need = ctypes.c_size_t()
    _native.check(_native.lib().dgfx_spmm_workspace_size(R, nnz, F, ctypes.byref(need)))
    if workspace is None or workspace.numel() < need.value:
        workspace = _temporary((need.value,), torch.uint8, x.device, stream)
    _native.check(
        _native.lib().dgfx_spmm_csr(
            _native.ptr(rowptr), _native.ptr(col), _native.ptr(val), R, int(x.shape[0]), nnz, _native.ptr(x),
            _dtype_code(x.dtype), _native.ptr(out), _dtype_code(out.dtype), F, int(bool(normalize)),
            _native.ptr(workspace), need.value, _native.stream_handle(stream),
        )
    )
    return out


def spmm_workspace(num_rows: int, nnz: int, feat: int, device):
    torch = _native.require_cuda()
    need = ctypes.c_size_t()
    _native.check(_native.lib().dgfx_spmm_workspace_size(num_rows, nnz, feat, ctypes.byref(need)))
    return torch.empty(need.value, dtype=torch.uint8, device=device)


def segment_sum(data, segment_ids, num_segments: int, mean: bool = False, indices_are_sorted: bool = False,
                out_dtype=None, stream=None):
    """jax.ops.segment_sum(data, segment_ids, num_segments) [/ max(count, 1)]."""
    torch = _native.require_cuda()
    n, F = int(data.shape[0]), int(data.shape[1])
    out = torch.empty((num_segments, F), dtype=out_dtype or data.dtype, device=data.device)
    ids = segment_ids.to(torch.int64).contiguous()
    need = ctypes.c_size_t()
    _native.check(_native.lib().dgfx_segment_sum_workspace_size(n, F, num_segments, ctypes.byref(need)))
    ws = torch.empty(max(1, need.value), dtype=torch.uint8, device=data.device)
    _native.check(
        _native.lib().dgfx_segment_sum(
            _native.ptr(data.contiguous()), _dtype_code(data.dtype), _native.ptr(ids), n, F, int(num_segments),
            int(bool(mean)), int(bool(indices_are_sorted)), _native.ptr(out), _dtype_code(out.dtype),
            _native.ptr(ws), need.value, _native.stream_handle(stream),
        )
    )
    return out


def segment_softmax(logits, messages, segment_ids, num_segments: int, indices_are_sorted: bool = False,
                    out_dtype=None, stream=None):
    """Attention-weighted segment sum (hetero_graph_attention_network.py:
    242-263): softmax of ``logits`` [E, H] over the items of each segment
    (per head, max-subtracted, + 1e-9 in the denominator) weighting
    ``messages`` [E, H, D]; returns [num_segments, H, D]. One pass over the
    items (online softmax), fp32 accumulation."""
    torch = _native.require_cuda()
    if logits.dtype != torch.float32:
        raise ValueError("segment_softmax: logits must be float32")
    E, H = int(logits.shape[0]), int(logits.shape[1])
    if messages.dim() != 3 or int(messages.shape[0]) != E or int(messages.shape[1]) != H:
        raise ValueError("segment_softmax: messages must be [E, H, D] matching logits [E, H]")
    D = int(messages.shape[2])
    out = torch.empty((num_segments, H, D), dtype=out_dtype or messages.dtype, device=messages.device)
    ids = segment_ids.to(torch.int64).contiguous()
    need = ctypes.c_size_t()
    _native.check(_native.lib().dgfx_segment_softmax_workspace_size(
        E, num_segments, H, D, _dtype_code(messages.dtype), int(bool(indices_are_sorted)), ctypes.byref(need)))
    ws = torch.empty(max(1, need.value), dtype=torch.uint8, device=messages.device)
    _native.check(_native.lib().dgfx_segment_softmax(
        _native.ptr(logits.contiguous()), H, _native.ptr(messages.contiguous()), _dtype_code(messages.dtype), D,
        _native.ptr(ids), E, int(num_segments), int(bool(indices_are_sorted)), _native.ptr(out),
        _dtype_code(out.dtype), _native.ptr(ws), need.value, _native.stream_handle(stream)))
    return out


def gather_rows(table, ids, stream=None):
    """out[i] = table[ids[i]] (rows of any dtype whose byte width is a
    multiple of 16; ids outside the table give zero rows)."""
    torch = _native.require_cuda()
    n = int(ids.numel())
    row_bytes = table.element_size() * (table.numel() // max(1, table.shape[0]))
    out = torch.empty((n,) + tuple(table.shape[1:]), dtype=table.dtype, device=table.device)
    _native.check(
        _native.lib().dgfx_gather_rows(
            _native.ptr(table), int(table.shape[0]), row_bytes, _native.ptr(ids.to(torch.int64).contiguous()), n,
            _native.ptr(out), _native.stream_handle(stream),
        )
    )
    return out


def dense_concat(x1, x2, weight, bias=None, relu: bool = True, out=None, stream=None):
    """act(concat[x1, x2] @ weight.T + bias) in bf16 on the tensor cores
    (tcgen05, fp32 accumulation): the Dense(+ReLU) update after aggregation
    (hetero_gnn.py:302-312). x1 [M, K1], x2 [M, K2] or None, weight [N, K1+K2]
    (torch Linear layout), bias fp32 [N] or None; K1, K2 and N multiples of 64.
    The concat is read from the two inputs, never materialised."""
    torch = _native.require_cuda()
    if x1.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16 or (x2 is not None and x2.dtype != torch.bfloat16):
        raise ValueError("dense_concat: x1, x2 and weight must be bfloat16")
    m, k1 = int(x1.shape[0]), int(x1.shape[1])
    k2 = 0 if x2 is None else int(x2.shape[1])
    if x2 is not None and int(x2.shape[0]) != m:
        raise ValueError("dense_concat: x1 and x2 must have the same number of rows")
    n = int(weight.shape[0])
    if int(weight.shape[1]) != k1 + k2:
        raise ValueError(f"dense_concat: weight is [{n}, {int(weight.shape[1])}], expected [N, {k1 + k2}]")
    for t in (x1, x2, weight):
        if t is not None and not t.is_contiguous():
            raise ValueError("dense_concat: inputs must be contiguous")
    if bias is not None and (bias.dtype != torch.float32 or int(bias.numel()) != n):
        raise ValueError("dense_concat: bias must be float32 [N]")
    if out is None:
        out = x1.new_empty((m, n))
    _native.check(_native.lib().dgfx_dense_concat_bf16(
        _native.ptr(x1), k1, _native.ptr(x2), k2, m, _native.ptr(weight), _native.ptr(bias), n, int(bool(relu)),
        _native.ptr(out), _native.stream_handle(stream)))
    return out


def dense_check(stream=None):
    """Raises if a dense_concat launch hit a pipeline timeout since the last
    check (synchronises the stream)."""
    _native.check(_native.lib().dgfx_dense_check(_native.stream_handle(stream)))


def sage_mean_linear_relu(rowptr, col, x, weight, bias=None, agg=None, workspace=None, out=None, stream=None):
    """GraphSAGE-mean layer: agg = mean over in-neighbours (CSR rows = target
    nodes, col = source nodes) of x, then relu(concat[x, agg] @ weight.T +
    bias). x bf16 [N, F]; weight bf16 [N_out, 2F]. Two launches: the SpMM
    (HBM-bound gather, bf16 out) and the tensor-core dense layer."""
    _native.require_cuda()
    n_rows = int(rowptr.numel()) - 1
    if agg is None:
        agg = _temporary((n_rows, int(x.shape[1])), torch.bfloat16, x.device, stream)
    csr_spmm(rowptr, col, x, normalize=True, out=agg, workspace=workspace, stream=stream)
    return dense_concat(x[:n_rows], agg, weight, bias, relu=True, out=out, stream=stream)


def sage_mean_gated(rowptr, col, x, w_gate, w_up, b_gate=None, b_up=None, activation: str = "silu", agg=None,
                    workspace=None, out=None, stream=None):
    """GraphSAGE-mean layer with a gated update: agg = mean over in-neighbours
    of x (as ``sage_mean_linear_relu``), then act(concat[x, agg] @ w_gate.T +
    b_gate) * (concat[x, agg] @ w_up.T + b_up) (``gated_dense_concat``). x bf16
    [N, F], w_gate and w_up bf16 [N_out, 2F]; agg, if given, must not overlap x."""
    who = "sage_mean_gated"
    n_rows = rowptr.numel() - 1
    nodes, feat = _layer_matrix(who, "x", x, torch.bfloat16)
    if not 0 <= n_rows <= nodes:
        raise ValueError(f"{who}: rowptr has {n_rows} rows, x {nodes}")
    if agg is not None:
        _layer_operand(who, "agg", agg, (n_rows, feat), torch.bfloat16)
        _layer_apart(who, "agg", agg, x=x)
    _gated_operands(who, x[:n_rows], x[:n_rows], w_gate, w_up, b_gate, b_up)  # agg is as large as x[:n_rows]
    _activation_code(who, activation)
    if out is not None:
        _layer_operand(who, "out", out, (n_rows, w_gate.shape[0]), torch.bfloat16)
    # Both steps under one guard: agg, the SpMM's workspace and the launches
    # share one device and stream, so that memory freed here is not handed out
    # while another stream's kernels still use it.
    guard = _layer_guard(who, stream, x, rowptr, col, w_gate, w_up, b_gate, b_up, agg, workspace, out)
    if guard is not None:
        with guard:
            return sage_mean_gated(rowptr, col, x, w_gate, w_up, b_gate, b_up, activation, agg, workspace, out)
    if agg is None:
        agg = x.new_empty((n_rows, feat))
    csr_spmm(rowptr, col, x, normalize=True, out=agg, workspace=workspace)
    return gated_dense_concat(x[:n_rows], agg, w_gate, w_up, b_gate, b_up, activation, out=out)


# ---------------------------------------------------------------------------
# Propagation matrices of the reference's sparse GNN layers, CSR transpose,
# segment-sum gradient, mean aggregation over a sampled batch.
# ---------------------------------------------------------------------------
def _symmetric_structure(src, dst, num_nodes: int, stream=None):
    """CSR (rowptr int64, col int32) of A + A^T for an edge list on one node
    set: every edge contributes (dst, src) and (src, dst); duplicates and
    self loops are kept (the sum of COO matrices keeps them too). Rows are
    sorted by column."""
    torch = _native.require_cuda()
    from distributed_graph_flow_b200.sampling import _in_memory_sampler_ext as ext

    s = src.to(torch.int64).contiguous()
    d = dst.to(torch.int64).contiguous()
    rows = torch.cat([d, s])
    cols = torch.cat([s, d])
    idx = ext.build_adjacency_index_device(rows, cols, None, num_nodes, num_nodes, False, False, stream=stream)
    return idx.rowptr, idx.col


def _add_diagonal(rowptr, col, num_nodes: int, diag: float, normalize: bool, stream=None):
    torch = _native.require_cuda()
    nnz = int(col.numel()) + num_nodes
    out_rowptr = torch.empty(num_nodes + 1, dtype=torch.int64, device=rowptr.device)
    out_col = torch.empty(max(nnz, 1), dtype=torch.int32, device=rowptr.device)[:nnz]
    out_val = torch.empty(max(nnz, 1), dtype=torch.float32, device=rowptr.device)[:nnz]
    _native.check(_native.lib().dgfx_csr_add_diagonal(
        _native.ptr(rowptr), _native.ptr(col), num_nodes, float(diag), int(bool(normalize)), _native.ptr(out_rowptr),
        _native.ptr(out_col), _native.ptr(out_val), _native.stream_handle(stream)))
    return out_rowptr, out_col, out_val


def gcn_matrix(src, dst, num_nodes: int, stream=None):
    """D^-1/2 (A + A^T + I) D^-1/2 as CSR (rowptr int64, col int32, val
    float32), D = row sums: the reference's GCN propagation matrix
    ``(adj + adj.transpose()).add_eye().normalize_symmetric()``
    (homo_gnn_sparse_deferred.py:293). Symmetric, so it is its own
    transpose."""
    rowptr, col = _symmetric_structure(src, dst, num_nodes, stream)
    return _add_diagonal(rowptr, col, num_nodes, 1.0, True, stream)


def gin_matrix(src, dst, num_nodes: int, epsilon: float = 0.0, stream=None):
    """A + A^T + (1 + epsilon) I as CSR (rowptr, col, val): the reference's
    GIN propagation matrix ``(adj + adj.transpose()).add_eye(1 +
    epsilon)`` (homo_gnn_sparse_deferred.py:526)."""
    rowptr, col = _symmetric_structure(src, dst, num_nodes, stream)
    return _add_diagonal(rowptr, col, num_nodes, 1.0 + float(epsilon), False, stream)


def csr_row_ids(rowptr, stream=None):
    """int64 row of every CSR entry."""
    torch = _native.require_cuda()
    R = int(rowptr.numel()) - 1
    nnz = int(rowptr[-1].item()) if R >= 0 else 0
    rows = torch.empty(max(nnz, 1), dtype=torch.int64, device=rowptr.device)[:nnz]
    _native.check(_native.lib().dgfx_csr_row_ids(_native.ptr(rowptr), R, _native.ptr(rows),
                                                 _native.stream_handle(stream)))
    return rows


def csr_transpose(rowptr, col, val, num_cols: int, stream=None):
    """Transpose of a CSR matrix [R, num_cols] -> [num_cols, R] (rowptr,
    col int32, val float32 or None); entries of a transposed row are in
    original row order."""
    torch = _native.require_cuda()
    from distributed_graph_flow_b200.sampling import _in_memory_sampler_ext as ext

    R = int(rowptr.numel()) - 1
    nnz = int(col.numel())
    rows = torch.empty(max(nnz, 1), dtype=torch.int64, device=rowptr.device)[:nnz]
    _native.check(_native.lib().dgfx_csr_row_ids(_native.ptr(rowptr), R, _native.ptr(rows),
                                                 _native.stream_handle(stream)))
    idx = ext.build_adjacency_index_device(rows, col.to(torch.int64), None, R, int(num_cols), True, val is not None,
                                           stream=stream)
    val_t = None
    if val is not None:
        val_t = torch.empty_like(val)
        val_t[idx.edge_pos] = val
    return idx.rowptr, idx.col, val_t


def segment_counts(segment_ids, num_segments: int, stream=None):
    torch = _native.require_cuda()
    ids = segment_ids.to(torch.int64).contiguous()
    cnt = torch.empty(max(1, num_segments), dtype=torch.int32, device=ids.device)[:num_segments]
    _native.check(_native.lib().dgfx_segment_counts(_native.ptr(ids), int(ids.numel()), int(num_segments),
                                                    _native.ptr(cnt), _native.stream_handle(stream)))
    return cnt


def gather_rows_scaled(src, segment_ids, num_segments: int, counts=None, stream=None):
    """out[i] = src[ids[i]] / max(counts[ids[i]], 1) (no division if counts is
    None); zero rows for ids outside [0, num_segments)."""
    torch = _native.require_cuda()
    ids = segment_ids.to(torch.int64).contiguous()
    src = src.contiguous()
    F = int(src.numel() // max(1, src.shape[0])) if src.dim() > 1 else 1
    out = torch.empty((int(ids.numel()),) + tuple(src.shape[1:]), dtype=src.dtype, device=src.device)
    _native.check(_native.lib().dgfx_gather_rows_scaled(
        _native.ptr(src), _dtype_code(src.dtype), _native.ptr(ids), int(ids.numel()), int(num_segments), F,
        _native.ptr(counts), _native.ptr(out), _native.stream_handle(stream)))
    return out


def batch_csr(batch, stream=None):
    """CSR over the batch nodes of a merged sampled batch (one node set, one
    edge set): rowptr int64 [capacity + 1] (rows past the batch's node count
    empty), col int32 [edge capacity], col = batch index of the sampled
    neighbour. No host synchronisation."""
    torch = _native.require_cuda()
    cap = int(batch.node_ids.numel())
    ecap = int(batch.edge_src.numel())
    rowptr = torch.empty(cap + 1, dtype=torch.int64, device=batch.node_ids.device)
    col = torch.empty(max(ecap, 1), dtype=torch.int32, device=batch.node_ids.device)[:ecap]
    _native.check(_native.lib().dgfx_batch_csr(
        _native.ptr(batch.node_offsets), _native.ptr(batch.edge_offsets), _native.ptr(batch.edge_src),
        _native.ptr(batch.edge_dst), int(batch.B), cap, _native.ptr(rowptr), _native.ptr(col),
        _native.stream_handle(stream)))
    return rowptr, col


def batch_mean_aggregate(batch, features, out=None, stream=None):
    """Mean aggregation over a merged sampled batch (jax.ops.segment_sum
    mean pooling of hetero_gnn.py:282-294, messages = the features of the
    sampled neighbours flowing to the node that sampled them): out[v] =
    mean of features[u] over the batch edges v -> u, zero rows for nodes
    without sampled neighbours; rows past the batch's node count are left
    as they are. features [capacity, F] in batch order (the rows gathered
    for batch.node_ids). One kernel (dgfx_batch_mean); the same values as
    csr_spmm(*batch_csr(batch), features, normalize=True)."""
    torch = _native.require_cuda()
    cap = int(batch.node_ids.numel())
    F = int(features.numel() // max(1, features.shape[0]))
    if out is None:
        out = torch.empty_like(features)
    _native.check(_native.lib().dgfx_batch_mean(
        _native.ptr(batch.node_offsets), _native.ptr(batch.edge_offsets), _native.ptr(batch.edge_src),
        _native.ptr(batch.edge_dst), int(batch.B), cap, _native.ptr(features), _dtype_code(features.dtype), F,
        _native.ptr(out), _native.stream_handle(stream)))
    return out


# ---------------------------------------------------------------------------
# Layer operators around the aggregation: gated dense layer, group norm over
# the segments of a merged batch, gated recurrence over ragged windows.
# ---------------------------------------------------------------------------
def _activation_code(who: str, activation: str) -> int:
    code = _native.ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"{who}: unknown activation {activation!r}; expected one of {sorted(_native.ACTIVATIONS)}")
    return code


def _short(dtype) -> str:
    return str(dtype).replace("torch.", "")


def _layer_operand(who: str, name: str, t, shape, dtype) -> None:
    """Checks one operand: type, shape, contiguity."""
    if t.dtype is not dtype:
        raise ValueError(f"{who}: {name} must be {_short(dtype)}")
    if t.shape != shape:
        raise ValueError(f"{who}: {name} is {list(t.shape)}, expected {list(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{who}: {name} must be contiguous")


def _layer_matrix(who: str, name: str, t, dtype):
    """Checks a matrix whose extents are free and returns them."""
    shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"{who}: {name} is {list(shape)}, expected a matrix")
    _layer_operand(who, name, t, shape, dtype)
    return shape


def _layer_input(who: str, x):
    """Checks the main input [rows, channels] (float32 or bfloat16); (rows, channels, dtype code)."""
    code = _native.BF16 if x.dtype is torch.bfloat16 else _native.F32
    if code == _native.F32 and x.dtype is not torch.float32:
        raise ValueError(f"{who}: x must be float32 or bfloat16")
    rows, channels = _layer_matrix(who, "x", x, x.dtype)
    return rows, channels, code


def _layer_offsets(who: str, offsets) -> int:
    """Checks segment offsets (int64 [segments + 1]) and returns the number of segments."""
    if offsets.dtype is not torch.int64 or offsets.dim() != 1 or offsets.numel() < 1 or not offsets.is_contiguous():
        raise ValueError(f"{who}: offsets must be a contiguous int64 vector of segments + 1 values")
    return offsets.numel() - 1


def _layer_apart(who: str, name: str, out, **inputs) -> None:
    """Refuses an output that shares memory with an input: other blocks of the
    kernel may still read what one has overwritten."""
    begin, end = out.data_ptr(), out.data_ptr() + out.numel() * out.element_size()
    for other, t in inputs.items():
        if t is not None and t.data_ptr() < end and begin < t.data_ptr() + t.numel() * t.element_size():
            raise ValueError(f"{who}: {name} must not overlap {other}")


class _LayerGuard:
    """Device and stream of a call that does not run where the caller stands:
    the operands' device becomes the current one and ``stream`` the current
    stream, so that allocations inside belong to it; the operands are recorded on it, so
    that their memory is not handed out while the call still runs."""

    def __init__(self, who: str, stream, device: int, operands):
        if stream is not None and stream.device_index != device:
            raise ValueError(f"{who}: the stream belongs to cuda:{stream.device_index}, the tensors to cuda:{device}")
        self._guards = [torch.cuda.device(device)]
        if stream is not None:
            self._guards.append(torch.cuda.stream(stream))
            for t in operands:
                if t is not None:
                    t.record_stream(stream)

    def __enter__(self):
        for g in self._guards:
            g.__enter__()

    def __exit__(self, *exc):
        for g in reversed(self._guards):
            g.__exit__(*exc)
        return False


def _layer_guard(who: str, stream, *operands):
    """None when the call runs on the current device and stream as it is, else
    the guard to run it under. Refuses operands that are not on one CUDA
    device."""
    device = operands[0].get_device()
    for t in operands:
        if t is not None and (t.get_device() != device or device < 0):
            _native.require_cuda()
            raise ValueError(f"{who}: all tensors must be on one CUDA device, got "
                             + ", ".join(sorted({str(o.device) for o in operands if o is not None})))
    if device == _native.current_device() and (stream is None or stream.cuda_stream == _native.raw_stream(device)):
        return None
    return _LayerGuard(who, stream, device, operands)


def _layer_workspace(device, nbytes: int):
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(function: str, *sizes) -> int:
    """A *_workspace_size query (a function of the sizes alone)."""
    need = ctypes.c_size_t()
    _native.check(getattr(_native.lib(), function)(*sizes, ctypes.byref(need)))
    return need.value


@functools.lru_cache(maxsize=1024)
def _scan_sizes(rows: int, channels: int, code: int):
    need, saved = ctypes.c_size_t(), ctypes.c_size_t()
    _native.check(_native.lib().dgfx_gated_scan_workspace_size(rows, channels, code, ctypes.byref(need),
                                                               ctypes.byref(saved)))
    return need.value, saved.value // 4


def _gated_operands(who: str, x1, x2, w_gate, w_up, b_gate, b_up):
    """Checks the operands of the gated dense layer; (m, k1, k2, n)."""
    m, k1 = _layer_matrix(who, "x1", x1, torch.bfloat16)
    k2 = 0
    if x2 is not None:
        m2, k2 = _layer_matrix(who, "x2", x2, torch.bfloat16)
        if m2 != m:
            raise ValueError(f"{who}: x2 is {list(x2.shape)}, expected {m} rows")
    n, k = _layer_matrix(who, "w_gate", w_gate, torch.bfloat16)
    if k != k1 + k2:
        raise ValueError(f"{who}: w_gate is {list(w_gate.shape)}, expected {k1 + k2} columns")
    _layer_operand(who, "w_up", w_up, (n, k), torch.bfloat16)
    if b_gate is not None:
        _layer_operand(who, "b_gate", b_gate, (n,), torch.float32)
    if b_up is not None:
        _layer_operand(who, "b_up", b_up, (n,), torch.float32)
    return m, k1, k2, n


def gated_dense_concat(x1, x2, w_gate, w_up, b_gate=None, b_up=None, activation: str = "silu", out=None, stream=None):
    """act(X @ w_gate.T + b_gate) * (X @ w_up.T + b_up) with X = concat[x1,
    x2] on the tensor cores: the gated form of the dense update after the
    aggregation (``dense_concat``). Both projections, the activation and the product run in one
    kernel; neither the concat nor the projections are written to memory.

    x1 [M, K1], x2 [M, K2] or None, w_gate and w_up [N, K1 + K2] (torch Linear
    layout) bfloat16, biases float32 [N] or None; K1, K2 and N multiples of 8;
    contiguous; out must not overlap them. activation: silu, gelu (erf form),
    relu, sigmoid or none. fp32 accumulation, one rounding to bfloat16. ``dense_check`` reports pipeline
    timeouts of this call too."""
    who = "gated_dense_concat"
    m, k1, k2, n = _gated_operands(who, x1, x2, w_gate, w_up, b_gate, b_up)
    act = _activation_code(who, activation)
    if out is not None:
        _layer_operand(who, "out", out, (m, n), torch.bfloat16)
        _layer_apart(who, "out", out, x1=x1, x2=x2, w_gate=w_gate, w_up=w_up, b_gate=b_gate, b_up=b_up)
    _workspace_bytes("dgfx_gated_dense_concat_backward_workspace_size", k1, k2, m, n)  # refuses sizes before devices
    guard = _layer_guard(who, stream, x1, x2, w_gate, w_up, b_gate, b_up, out)
    if guard is not None:
        with guard:
            return gated_dense_concat(x1, x2, w_gate, w_up, b_gate, b_up, activation, out)
    if out is None:
        out = x1.new_empty((m, n))
    ptr = _native.ptr
    _native.check(_native.lib().dgfx_gated_dense_concat_bf16(
        ptr(x1), k1, ptr(x2), k2, m, ptr(w_gate), ptr(w_up), ptr(b_gate), ptr(b_up), n, act, ptr(out),
        _native.raw_stream(x1.get_device())))
    return out


def gated_dense_concat_backward(grad, x1, x2, w_gate, w_up, b_gate=None, b_up=None, activation: str = "silu",
                                need_input: bool = True, need_weight: bool = True, stream=None):
    """Gradients of ``gated_dense_concat``: (dx1, dx2, dw_gate, dw_up, db_gate,
    db_up) from the gradient of its output (bfloat16 [M, N]) and its inputs;
    None where the input is None. The projections are computed again instead
    of being kept, and the gradients of the two projections (2 M N values of
    workspace) are rounded to bfloat16 once, as operands of the products that
    follow, so that dx and dw are off by 2.3e-3 (2-norm, relative) where their
    own rounding is 1.7e-3; the bias gradients (float32) are summed before that rounding.
    need_input=False skips dx1 and dx2, need_weight=False dw_gate and dw_up
    (returned as None). Sums run in a fixed order."""
    who = "gated_dense_concat_backward"
    m, k1, k2, n = _gated_operands(who, x1, x2, w_gate, w_up, b_gate, b_up)
    _layer_operand(who, "grad", grad, (m, n), torch.bfloat16)
    act = _activation_code(who, activation)
    need = _workspace_bytes("dgfx_gated_dense_concat_backward_workspace_size", k1, k2, m, n)
    guard = _layer_guard(who, stream, x1, x2, w_gate, w_up, b_gate, b_up, grad)
    if guard is not None:
        with guard:
            return gated_dense_concat_backward(grad, x1, x2, w_gate, w_up, b_gate, b_up, activation, need_input,
                                               need_weight)
    dx1 = torch.empty_like(x1) if need_input else None
    dx2 = torch.empty_like(x2) if need_input and x2 is not None else None
    dwg = torch.empty_like(w_gate) if need_weight else None
    dwu = torch.empty_like(w_up) if need_weight else None
    dbg = None if b_gate is None else torch.empty_like(b_gate)
    dbu = None if b_up is None else torch.empty_like(b_up)
    ws = _layer_workspace(x1.device, need)
    ptr = _native.ptr
    _native.check(_native.lib().dgfx_gated_dense_concat_backward_bf16(
        ptr(grad), ptr(x1), k1, ptr(x2), k2, m, ptr(w_gate), ptr(w_up), ptr(b_gate), ptr(b_up), n, act, ptr(dx1),
        ptr(dx2), ptr(dwg), ptr(dwu), ptr(dbg), ptr(dbu), ptr(ws), need, _native.raw_stream(x1.get_device())))
    return dx1, dx2, dwg, dwu, dbg, dbu


def segment_group_norm(x, offsets, groups: int, weight=None, bias=None, eps: float = 1e-5, activation: str = "none",
                       stream=None):
    """Group norm with an activation over ragged segments, channels last:
    every segment (rows offsets[s] .. offsets[s+1] of x, e.g. the graphs of a
    merged batch with offsets = its node_offsets) and every group of C /
    ``groups`` adjacent channels is normalised by its own mean and biased
    variance, y = act((x - mean) * rstd * weight + bias). With one segment per
    graph this is the per-graph norm of a GNN layer; with groups = C an
    instance norm. With groups = 1 and one row per segment it computes a layer
    norm, but it is not made for that: a segment costs a fixed amount of work,
    and rows of 64 bfloat16 values run at 0.2 TB/s.

    x [rows, C] float32 / bfloat16 (rows a multiple of 16 bytes, at most
    4096), offsets int64 [segments + 1] ascending, on the device (no host
    synchronisation), weight and bias float32 [C] or None, activation one of
    none, relu, silu, gelu (erf form), sigmoid. Rows outside of every segment
    (a merged batch's spare capacity) give zeros and are never used, whatever they
    hold. Returns (y, mean, rstd); mean and rstd, float32 [segments, groups],
    are what ``segment_group_norm_backward`` takes."""
    who = "segment_group_norm"
    rows, channels, code = _layer_input(who, x)
    nseg = _layer_offsets(who, offsets)
    act = _activation_code(who, activation)
    if weight is not None:
        _layer_operand(who, "weight", weight, (channels,), torch.float32)
    if bias is not None:
        _layer_operand(who, "bias", bias, (channels,), torch.float32)
    groups = int(groups)
    need = _workspace_bytes("dgfx_segment_group_norm_workspace_size", rows, channels, groups, nseg, code, 0)
    if not eps > 0:
        raise ValueError(f"{who}: eps must be positive")
    guard = _layer_guard(who, stream, x, offsets, weight, bias)
    if guard is not None:
        with guard:
            return segment_group_norm(x, offsets, groups, weight, bias, eps, activation)
    y = torch.empty_like(x)
    mean = x.new_empty((nseg, groups), dtype=torch.float32)
    rstd = torch.empty_like(mean)
    ws = _layer_workspace(x.device, need) if need else None
    ptr = _native.ptr
    _native.check(_native.lib().dgfx_segment_group_norm(
        ptr(x), code, rows, channels, groups, ptr(offsets), nseg, ptr(weight), ptr(bias), eps, act, ptr(y), ptr(mean),
        ptr(rstd), ptr(ws), need, _native.raw_stream(x.get_device())))
    return y, mean, rstd


def segment_group_norm_backward(grad, x, offsets, mean, rstd, weight=None, bias=None, activation: str = "none",
                                stream=None):
    """Gradients of ``segment_group_norm``: (dx, dweight, dbias) from the
    gradient of y, the forward inputs and the returned mean and rstd. dx has
    x's type, dweight and dbias are float32 sums over all segments (None for
    a weight or bias that is None), in a fixed order. Rows outside of every
    segment get zeros, and what grad holds there is not used."""
    who = "segment_group_norm_backward"
    rows, channels, code = _layer_input(who, x)
    _layer_operand(who, "grad", grad, x.shape, x.dtype)
    nseg = _layer_offsets(who, offsets)
    act = _activation_code(who, activation)
    segments, groups = _layer_matrix(who, "mean", mean, torch.float32)
    if segments != nseg:
        raise ValueError(f"{who}: mean is {list(mean.shape)}, expected {nseg} rows")
    _layer_operand(who, "rstd", rstd, (nseg, groups), torch.float32)
    if weight is not None:
        _layer_operand(who, "weight", weight, (channels,), torch.float32)
    if bias is not None:
        _layer_operand(who, "bias", bias, (channels,), torch.float32)
    need = _workspace_bytes("dgfx_segment_group_norm_workspace_size", rows, channels, groups, nseg, code, 1)
    guard = _layer_guard(who, stream, grad, x, offsets, mean, rstd, weight, bias)
    if guard is not None:
        with guard:
            return segment_group_norm_backward(grad, x, offsets, mean, rstd, weight, bias, activation)
    dx = torch.empty_like(x)
    dw = None if weight is None else torch.empty_like(weight)
    db = None if bias is None else torch.empty_like(bias)
    ws = _layer_workspace(x.device, need)
    ptr = _native.ptr
    _native.check(_native.lib().dgfx_segment_group_norm_backward(
        ptr(grad), ptr(x), code, rows, channels, groups, ptr(offsets), nseg, ptr(mean), ptr(rstd), ptr(weight),
        ptr(bias), act, ptr(dx), ptr(dw), ptr(db), ptr(ws), need, _native.raw_stream(x.get_device())))
    return dx, dw, db


def gated_scan(x, gate, offsets, initial=None, return_sequence: bool = True, return_saved: bool = False, stream=None):
    """Gated linear recurrence over ragged windows (e.g. the causal windows
    of sampled nodes' time series): per channel and segment,

        a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t.

    x and gate [rows, C] float32 / bfloat16 (C a multiple of 4), offsets int64
    [segments + 1] ascending, on the device; initial float32 [segments, C] is
    the state before each segment's first row (None: zeros). Returns (h,
    final): h [rows, C] in x's type, zeros in rows outside of every segment
    (whose inputs are never used), and final float32 [segments, C], the state
    after each segment's last row (its initial state if it has no rows).
    States are float32 throughout. return_sequence=False skips h (returned as
    None); return_saved=True appends what ``gated_scan_backward`` takes."""
    who = "gated_scan"
    rows, channels, code = _layer_input(who, x)
    _layer_operand(who, "gate", gate, x.shape, x.dtype)
    nseg = _layer_offsets(who, offsets)
    if initial is not None:
        _layer_operand(who, "initial", initial, (nseg, channels), torch.float32)
    need, saved_n = _scan_sizes(rows, channels, code)
    guard = _layer_guard(who, stream, x, gate, offsets, initial)
    if guard is not None:
        with guard:
            return gated_scan(x, gate, offsets, initial, return_sequence, return_saved)
    h = torch.empty_like(x) if return_sequence else None
    final = x.new_empty((nseg, channels), dtype=torch.float32)
    saved = torch.empty(saved_n, dtype=torch.float32, device=x.device) if return_saved else None
    ws = _layer_workspace(x.device, need)
    ptr = _native.ptr
    _native.check(_native.lib().dgfx_gated_scan(
        ptr(x), ptr(gate), code, rows, channels, ptr(offsets), nseg, ptr(initial), ptr(h), ptr(final), ptr(saved),
        ptr(ws), need, _native.raw_stream(x.get_device())))
    return (h, final, saved) if return_saved else (h, final)


def gated_scan_backward(grad, x, gate, offsets, saved, initial=None, grad_final=None, stream=None):
    """Gradients of ``gated_scan``: (dx, dgate, dinitial) from the gradients
    of h (None: zeros) and of final (None: zeros), the forward inputs and
    ``saved``. dinitial is None where initial is. Rows outside of every
    segment get zeros."""
    who = "gated_scan_backward"
    rows, channels, code = _layer_input(who, x)
    _layer_operand(who, "gate", gate, x.shape, x.dtype)
    if grad is not None:
        _layer_operand(who, "grad", grad, x.shape, x.dtype)
    nseg = _layer_offsets(who, offsets)
    if initial is not None:
        _layer_operand(who, "initial", initial, (nseg, channels), torch.float32)
    if grad_final is not None:
        _layer_operand(who, "grad_final", grad_final, (nseg, channels), torch.float32)
    need, saved_n = _scan_sizes(rows, channels, code)
    _layer_operand(who, "saved", saved, (saved_n,), torch.float32)
    guard = _layer_guard(who, stream, x, grad, gate, offsets, saved, initial, grad_final)
    if guard is not None:
        with guard:
            return gated_scan_backward(grad, x, gate, offsets, saved, initial, grad_final)
    dx, dgate = torch.empty_like(x), torch.empty_like(gate)
    dinitial = None if initial is None else torch.empty_like(initial)
    ws = _layer_workspace(x.device, need)
    ptr = _native.ptr
    _native.check(_native.lib().dgfx_gated_scan_backward(
        ptr(x), ptr(gate), code, rows, channels, ptr(offsets), nseg, ptr(initial), ptr(saved), ptr(grad),
        ptr(grad_final), ptr(dx), ptr(dgate), ptr(dinitial), ptr(ws), need, _native.raw_stream(x.get_device())))
    return dx, dgate, dinitial


def gated_scan_step(x, gate, state, out_state=None, stream=None):
    """One step of ``gated_scan`` for n independent sequences (online use):
    state' = a state + (1 - a) x with a = sigmoid(gate). x and gate [n, C],
    state float32 [n, C]; returns (h, state'), h in x's type. out_state may be
    ``state`` itself, which is then updated in place."""
    who = "gated_scan_step"
    n, channels, code = _layer_input(who, x)
    _layer_operand(who, "gate", gate, x.shape, x.dtype)
    _layer_operand(who, "state", state, (n, channels), torch.float32)
    if out_state is not None:
        _layer_operand(who, "out_state", out_state, (n, channels), torch.float32)
        in_place = out_state.data_ptr() == state.data_ptr()
        _layer_apart(who, "out_state", out_state, x=x, gate=gate, state=None if in_place else state)
    guard = _layer_guard(who, stream, x, gate, state, out_state)
    if guard is not None:
        with guard:
            return gated_scan_step(x, gate, state, out_state)
    h = torch.empty_like(x)
    new_state = torch.empty_like(state) if out_state is None else out_state
    ptr = _native.ptr
    _native.check(_native.lib().dgfx_gated_scan_step(
        ptr(x), ptr(gate), code, n, channels, ptr(state), ptr(h), ptr(new_state), _native.raw_stream(x.get_device())))
    return h, new_state
