"""The aggregation boundary as torch custom operators (``torch.library``).

The reference's GNN layers call their aggregation inside trained models:
``jax.ops.segment_sum`` over an edge list
(dgf/src/learning/jax/layers/hetero_gnn.py:282-294) and ``SparseMatrix @
dense`` (homo_gnn_sparse_deferred.py:138-161, 292-297, 525-530). Here the
same operations are torch operators in the ``dgfx`` namespace, with fake
(meta) implementations for tracing and export, and autograd where the
reference's layers need gradients:

* ``dgfx::csr_spmm(rowptr, col, val, x, normalize, num_rows)`` —
  Y = S A X with A the CSR matrix (rows = message targets, columns =
  sources), S = diag(1 / max(deg, 1)) when normalize. Gradient with
  respect to x: A^T S dY, one SpMM over the transposed CSR (built on the
  device). The matrix values are constants (the reference's propagation
  matrices are built from the graph): a val that requires grad is rejected.
* ``dgfx::segment_sum(data, segment_ids, num_segments, mean)`` — gradient:
  d data[i] = dY[ids[i]] (/ max(count, 1) for the mean), a row gather.
  The two gradients are operators of their own (``dgfx::csr_spmm_grad_x``,
  ``dgfx::segment_sum_grad``), so backward graphs trace with fake tensors.
* ``dgfx::gated_dense_concat(x1, x2, w_gate, w_up, b_gate, b_up, activation)``,
  ``dgfx::segment_group_norm(x, offsets, groups, weight, bias, eps,
  activation)`` and ``dgfx::gated_scan(x, gate, offsets, initial,
  keep_states)`` — the layer operators around the aggregation, with their
  gradients (operators too: ``*_grad``). ``gated_scan``, ``segment_group_norm``
  and ``sage_mean_gated`` below are the calls a model makes.
* ``dgfx::segment_softmax(logits, messages, segment_ids, num_segments)`` and
  ``dgfx::sage_mean_linear_relu(rowptr, col, x, weight, bias)`` — forward
  (inference) operators with fake implementations.

Every operator runs the library's sm_100a kernels (no fallback): the inputs
must be CUDA tensors.
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from distributed_graph_flow_b200 import aggregation

_LIB = "dgfx"


# ---------------------------------------------------------------------------
# csr_spmm
# ---------------------------------------------------------------------------
@torch.library.custom_op(f"{_LIB}::csr_spmm", mutates_args=())
def csr_spmm(rowptr: torch.Tensor, col: torch.Tensor, val: Optional[torch.Tensor], x: torch.Tensor,
             normalize: bool = False, num_rows: int = -1) -> torch.Tensor:
    rows = int(rowptr.numel()) - 1 if num_rows < 0 else int(num_rows)
    return aggregation.csr_spmm(rowptr, col, x.contiguous(), val=val, normalize=normalize, num_rows=rows)


@csr_spmm.register_fake
def _csr_spmm_fake(rowptr, col, val, x, normalize=False, num_rows=-1):
    rows = rowptr.shape[0] - 1 if num_rows < 0 else num_rows
    return x.new_empty((rows, x.shape[1]))


def _csr_spmm_setup(ctx, inputs, output):
    rowptr, col, val, x, normalize, num_rows = inputs
    if val is not None and val.requires_grad:
        raise RuntimeError("dgfx::csr_spmm: gradients with respect to the matrix values are not supported")
    ctx.save_for_backward(rowptr, col, val)
    ctx.normalize = normalize
    ctx.num_x_rows = x.shape[0]
    ctx.x_dtype = x.dtype


@torch.library.custom_op(f"{_LIB}::csr_spmm_grad_x", mutates_args=())
def csr_spmm_grad_x(rowptr: torch.Tensor, col: torch.Tensor, val: Optional[torch.Tensor], grad: torch.Tensor,
                    normalize: bool, num_x_rows: int) -> torch.Tensor:
    """A^T S dY: the transposed CSR (device build) times dY."""
    v = val
    if normalize:
        # Entry (r, c) of S A is val_rc / max(deg_r, 1).
        deg = (rowptr[1:] - rowptr[:-1]).clamp_min(1).to(torch.float32)
        scale = (1.0 / deg)[aggregation.csr_row_ids(rowptr)]
        v = scale if val is None else val * scale
    rp_t, col_t, val_t = aggregation.csr_transpose(rowptr, col, v, int(num_x_rows))
    return aggregation.csr_spmm(rp_t, col_t, grad.contiguous(), val=val_t, normalize=False, num_rows=int(num_x_rows))


@csr_spmm_grad_x.register_fake
def _csr_spmm_grad_x_fake(rowptr, col, val, grad, normalize, num_x_rows):
    return grad.new_empty((num_x_rows, grad.shape[1]))


def _csr_spmm_backward(ctx, grad):
    rowptr, col, val = ctx.saved_tensors
    dx = None
    if ctx.needs_input_grad[3]:
        dx = torch.ops.dgfx.csr_spmm_grad_x(rowptr, col, val, grad.to(ctx.x_dtype), ctx.normalize, ctx.num_x_rows)
    return None, None, None, dx, None, None


csr_spmm.register_autograd(_csr_spmm_backward, setup_context=_csr_spmm_setup)


# ---------------------------------------------------------------------------
# segment_sum
# ---------------------------------------------------------------------------
@torch.library.custom_op(f"{_LIB}::segment_sum", mutates_args=())
def segment_sum(data: torch.Tensor, segment_ids: torch.Tensor, num_segments: int, mean: bool = False) -> torch.Tensor:
    return aggregation.segment_sum(data.contiguous(), segment_ids, int(num_segments), mean=mean)


@segment_sum.register_fake
def _segment_sum_fake(data, segment_ids, num_segments, mean=False):
    return data.new_empty((num_segments, data.shape[1]))


def _segment_sum_setup(ctx, inputs, output):
    data, segment_ids, num_segments, mean = inputs
    ctx.save_for_backward(segment_ids)
    ctx.num_segments = int(num_segments)
    ctx.mean = bool(mean)
    ctx.data_dtype = data.dtype


@torch.library.custom_op(f"{_LIB}::segment_sum_grad", mutates_args=())
def segment_sum_grad(grad: torch.Tensor, segment_ids: torch.Tensor, num_segments: int, mean: bool) -> torch.Tensor:
    """d data[i] = dY[ids[i]] (/ max(count, 1) for the mean)."""
    counts = aggregation.segment_counts(segment_ids, int(num_segments)) if mean else None
    return aggregation.gather_rows_scaled(grad.contiguous(), segment_ids, int(num_segments), counts)


@segment_sum_grad.register_fake
def _segment_sum_grad_fake(grad, segment_ids, num_segments, mean):
    return grad.new_empty((segment_ids.shape[0], grad.shape[1]))


def _segment_sum_backward(ctx, grad):
    (ids,) = ctx.saved_tensors
    d = None
    if ctx.needs_input_grad[0]:
        d = torch.ops.dgfx.segment_sum_grad(grad.to(ctx.data_dtype), ids, ctx.num_segments, ctx.mean)
    return d, None, None, None


segment_sum.register_autograd(_segment_sum_backward, setup_context=_segment_sum_setup)


# ---------------------------------------------------------------------------
# Forward-only operators
# ---------------------------------------------------------------------------
@torch.library.custom_op(f"{_LIB}::segment_softmax", mutates_args=())
def segment_softmax(logits: torch.Tensor, messages: torch.Tensor, segment_ids: torch.Tensor,
                    num_segments: int) -> torch.Tensor:
    return aggregation.segment_softmax(logits.contiguous(), messages.contiguous(), segment_ids, int(num_segments))


@segment_softmax.register_fake
def _segment_softmax_fake(logits, messages, segment_ids, num_segments):
    return messages.new_empty((num_segments, messages.shape[1], messages.shape[2]))


@torch.library.custom_op(f"{_LIB}::sage_mean_linear_relu", mutates_args=())
def sage_mean_linear_relu(rowptr: torch.Tensor, col: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                          bias: Optional[torch.Tensor]) -> torch.Tensor:
    return aggregation.sage_mean_linear_relu(rowptr, col, x.contiguous(), weight.contiguous(), bias)


@sage_mean_linear_relu.register_fake
def _sage_fake(rowptr, col, x, weight, bias):
    return x.new_empty((rowptr.shape[0] - 1, weight.shape[0]))


def gcn_propagate(x: torch.Tensor, matrix) -> torch.Tensor:
    """adj_symnorm @ x of the reference's GCN layer, matrix = (rowptr, col,
    val) from aggregation.gcn_matrix (differentiable in x)."""
    rowptr, col, val = matrix
    return torch.ops.dgfx.csr_spmm(rowptr, col, val, x, False, -1)


def gin_propagate(x: torch.Tensor, matrix) -> torch.Tensor:
    """(adj + adj^T + (1 + eps) I) @ x of the reference's GIN layer, matrix
    from aggregation.gin_matrix (differentiable in x)."""
    rowptr, col, val = matrix
    return torch.ops.dgfx.csr_spmm(rowptr, col, val, x, False, -1)


# ---------------------------------------------------------------------------
# gated_dense_concat
# ---------------------------------------------------------------------------
def _like_or_none(t: Optional[torch.Tensor], like: torch.Tensor) -> torch.Tensor:
    """An operator's outputs are tensors: an empty one stands for None."""
    return like.new_empty(0) if t is None else t


def _packed(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """A strided or expanded operand as the kernels read it."""
    return None if t is None else t.contiguous()


@torch.library.custom_op(f"{_LIB}::gated_dense_concat", mutates_args=())
def gated_dense_concat(x1: torch.Tensor, x2: Optional[torch.Tensor], w_gate: torch.Tensor, w_up: torch.Tensor,
                       b_gate: Optional[torch.Tensor], b_up: Optional[torch.Tensor],
                       activation: str = "silu") -> torch.Tensor:
    return aggregation.gated_dense_concat(x1.contiguous(), _packed(x2), w_gate.contiguous(), w_up.contiguous(),
                                          _packed(b_gate), _packed(b_up), activation)


@gated_dense_concat.register_fake
def _gated_dense_concat_fake(x1, x2, w_gate, w_up, b_gate, b_up, activation="silu"):
    return x1.new_empty((x1.shape[0], w_gate.shape[0]))


@torch.library.custom_op(f"{_LIB}::gated_dense_concat_grad", mutates_args=())
def gated_dense_concat_grad(grad: torch.Tensor, x1: torch.Tensor, x2: Optional[torch.Tensor], w_gate: torch.Tensor,
                            w_up: torch.Tensor, b_gate: Optional[torch.Tensor], b_up: Optional[torch.Tensor],
                            activation: str, need_input: bool, need_weight: bool) -> List[torch.Tensor]:
    """[dx1, dx2, dw_gate, dw_up, db_gate, db_up], empty where there is none."""
    grads = aggregation.gated_dense_concat_backward(
        grad.contiguous(), x1.contiguous(), _packed(x2), w_gate.contiguous(), w_up.contiguous(), _packed(b_gate),
        _packed(b_up), activation, need_input, need_weight)
    return [_like_or_none(g, grad) for g in grads]


@gated_dense_concat_grad.register_fake
def _gated_dense_concat_grad_fake(grad, x1, x2, w_gate, w_up, b_gate, b_up, activation, need_input, need_weight):
    def like(t, wanted=True):
        return torch.empty(t.shape, dtype=t.dtype, device=t.device) if t is not None and wanted else grad.new_empty(0)

    return [like(x1, need_input), like(x2, need_input), like(w_gate, need_weight), like(w_up, need_weight),
            like(b_gate), like(b_up)]


def _gated_dense_concat_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:6])
    ctx.activation = inputs[6]


def _gated_dense_concat_backward(ctx, grad):
    x1, x2, w_gate, w_up, b_gate, b_up = ctx.saved_tensors
    need = ctx.needs_input_grad
    grads = torch.ops.dgfx.gated_dense_concat_grad(grad, x1, x2, w_gate, w_up, b_gate, b_up, ctx.activation,
                                                   need[0] or need[1], need[2] or need[3])
    return (*(g if n else None for g, n in zip(grads, need)), None)


gated_dense_concat.register_autograd(_gated_dense_concat_backward, setup_context=_gated_dense_concat_setup)


def sage_mean_gated(rowptr, col, x, w_gate, w_up, b_gate=None, b_up=None, activation: str = "silu") -> torch.Tensor:
    """GraphSAGE-mean layer with a gated update (aggregation.sage_mean_gated),
    differentiable in x, the weights and the biases."""
    agg = torch.ops.dgfx.csr_spmm(rowptr, col, None, x, True, -1)
    return torch.ops.dgfx.gated_dense_concat(x[: rowptr.shape[0] - 1], agg, w_gate, w_up, b_gate, b_up, activation)


# ---------------------------------------------------------------------------
# segment_group_norm
# ---------------------------------------------------------------------------
@torch.library.custom_op(f"{_LIB}::segment_group_norm", mutates_args=())
def _segment_group_norm(x: torch.Tensor, offsets: torch.Tensor, groups: int, weight: Optional[torch.Tensor],
                        bias: Optional[torch.Tensor], eps: float,
                        activation: str) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return aggregation.segment_group_norm(x.contiguous(), offsets.contiguous(), groups, _packed(weight), _packed(bias), eps,
                                          activation)


@_segment_group_norm.register_fake
def _segment_group_norm_fake(x, offsets, groups, weight, bias, eps, activation):
    stats = (offsets.shape[0] - 1, groups)
    return (x.new_empty(x.shape), x.new_empty(stats, dtype=torch.float32), x.new_empty(stats, dtype=torch.float32))


@torch.library.custom_op(f"{_LIB}::segment_group_norm_grad", mutates_args=())
def _segment_group_norm_grad(grad: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor, mean: torch.Tensor,
                             rstd: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
                             activation: str) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias), empty where there is no weight or bias."""
    dx, dw, db = aggregation.segment_group_norm_backward(grad.contiguous(), x.contiguous(), offsets.contiguous(), mean,
                                                         rstd, _packed(weight), _packed(bias), activation)
    return dx, _like_or_none(dw, mean), _like_or_none(db, mean)


@_segment_group_norm_grad.register_fake
def _segment_group_norm_grad_fake(grad, x, offsets, mean, rstd, weight, bias, activation):
    return (x.new_empty(x.shape), mean.new_empty(0) if weight is None else weight.new_empty(weight.shape),
            mean.new_empty(0) if bias is None else bias.new_empty(bias.shape))


def _segment_group_norm_setup(ctx, inputs, output):
    x, offsets, groups, weight, bias, eps, activation = inputs
    _, mean, rstd = output
    ctx.mark_non_differentiable(mean, rstd)
    ctx.save_for_backward(x, offsets, mean, rstd, weight, bias)
    ctx.activation = activation


def _segment_group_norm_backward(ctx, grad, grad_mean, grad_rstd):
    x, offsets, mean, rstd, weight, bias = ctx.saved_tensors
    dx, dw, db = torch.ops.dgfx.segment_group_norm_grad(grad.to(x.dtype), x, offsets, mean, rstd, weight, bias,
                                                        ctx.activation)
    need = ctx.needs_input_grad
    return dx if need[0] else None, None, None, dw if need[3] else None, db if need[4] else None, None, None


_segment_group_norm.register_autograd(_segment_group_norm_backward, setup_context=_segment_group_norm_setup)


def segment_group_norm(x, offsets, groups: int, weight=None, bias=None, eps: float = 1e-5,
                       activation: str = "none") -> torch.Tensor:
    """Group norm with an activation over the segments of a merged batch
    (aggregation.segment_group_norm), differentiable in x, weight and bias."""
    return torch.ops.dgfx.segment_group_norm(x, offsets, groups, weight, bias, eps, activation)[0]


# ---------------------------------------------------------------------------
# gated_scan
# ---------------------------------------------------------------------------
def _scan_states(x):
    """Values that the backward pass of a scan over x keeps: one state per
    channel before every 8th row, every 4th in float32."""
    block = 4 if x.dtype == torch.float32 else 8
    return (x.shape[0] + block - 1) // block * x.shape[1]


@torch.library.custom_op(f"{_LIB}::gated_scan", mutates_args=())
def _gated_scan(x: torch.Tensor, gate: torch.Tensor, offsets: torch.Tensor, initial: Optional[torch.Tensor],
                keep_states: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(h, final, states for the backward pass: empty unless keep_states)."""
    out = aggregation.gated_scan(x.contiguous(), gate.contiguous(), offsets.contiguous(),
                                 _packed(initial), return_saved=keep_states)
    return out if keep_states else (*out, out[1].new_empty(0))


@_gated_scan.register_fake
def _gated_scan_fake(x, gate, offsets, initial, keep_states):
    return (x.new_empty(x.shape), x.new_empty((offsets.shape[0] - 1, x.shape[1]), dtype=torch.float32),
            x.new_empty(_scan_states(x) if keep_states else 0, dtype=torch.float32))


@torch.library.custom_op(f"{_LIB}::gated_scan_grad", mutates_args=())
def _gated_scan_grad(grad: Optional[torch.Tensor], grad_final: Optional[torch.Tensor], x: torch.Tensor,
                     gate: torch.Tensor, offsets: torch.Tensor, saved: torch.Tensor,
                     initial: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dgate, dinitial), the last empty without initial."""
    dx, dgate, dinitial = aggregation.gated_scan_backward(
        _packed(grad), x.contiguous(), gate.contiguous(), offsets.contiguous(), saved, _packed(initial),
        _packed(grad_final))
    return dx, dgate, _like_or_none(dinitial, saved)


@_gated_scan_grad.register_fake
def _gated_scan_grad_fake(grad, grad_final, x, gate, offsets, saved, initial):
    return (x.new_empty(x.shape), gate.new_empty(gate.shape),
            saved.new_empty(0) if initial is None else initial.new_empty(initial.shape))


def _gated_scan_setup(ctx, inputs, output):
    x, gate, offsets, initial, keep_states = inputs
    if not keep_states:
        raise RuntimeError("dgfx::gated_scan: gradients need keep_states=True")
    ctx.mark_non_differentiable(output[2])
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x, gate, offsets, output[2], initial)


def _gated_scan_backward(ctx, grad, grad_final, grad_saved):
    x, gate, offsets, saved, initial = ctx.saved_tensors
    need = ctx.needs_input_grad
    if grad is None and grad_final is None:
        return None, None, None, None, None
    dx, dgate, dinitial = torch.ops.dgfx.gated_scan_grad(grad, grad_final, x, gate, offsets, saved, initial)
    return dx if need[0] else None, dgate if need[1] else None, None, dinitial if need[3] else None, None


_gated_scan.register_autograd(_gated_scan_backward, setup_context=_gated_scan_setup)


def gated_scan(x, gate, offsets, initial=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gated linear recurrence over ragged windows (aggregation.gated_scan):
    (h, final), differentiable in x, gate and initial. The states that the
    backward pass needs are only kept where a gradient can be asked for."""
    keep = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, gate, initial))
    return torch.ops.dgfx.gated_scan(x, gate, offsets, initial, keep)[:2]
