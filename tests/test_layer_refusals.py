"""Calls of the layer operators that are refused before anything runs on a
device (no GPU needed)."""

import pytest
import torch

from distributed_graph_flow_b200 import _native, aggregation

OFF = torch.tensor([0, 3, 8])


def _x(rows=8, c=16, dtype=torch.float32):
    return torch.zeros((rows, c), dtype=dtype)


BF = torch.bfloat16


def _gated(x1=None, x2=None, w_gate=None, w_up=None, **kw):
    x1 = _x(8, 16, BF) if x1 is None else x1
    x2 = _x(8, 16, BF) if x2 is None else x2
    k = x1.shape[1] + x2.shape[1]
    w_gate = _x(16, k, BF) if w_gate is None else w_gate
    w_up = _x(16, k, BF) if w_up is None else w_up
    return aggregation.gated_dense_concat(x1, x2, w_gate, w_up, **kw)


@pytest.mark.parametrize("call,match", [
    (lambda: aggregation.segment_group_norm(_x(dtype=torch.float16), OFF, 4), "x must be float32 or bfloat16"),
    (lambda: aggregation.segment_group_norm(_x()[:, ::2], OFF, 4), "contiguous"),
    (lambda: aggregation.segment_group_norm(_x(), OFF.int(), 4), "offsets"),
    (lambda: aggregation.segment_group_norm(_x(), OFF[:0], 4), "offsets"),
    (lambda: aggregation.segment_group_norm(_x(), OFF, 3), "divide the channels"),
    (lambda: aggregation.segment_group_norm(_x(), OFF, 0), "divide the channels"),
    (lambda: aggregation.segment_group_norm(_x(c=6), OFF, 3), "multiple of 16 bytes"),
    (lambda: aggregation.segment_group_norm(_x(c=4, dtype=torch.bfloat16), OFF, 1), "multiple of 16 bytes"),
    (lambda: aggregation.segment_group_norm(_x(), OFF, 4, activation="tanh"), "unknown activation"),
    (lambda: aggregation.segment_group_norm(_x(), OFF, 4, eps=0.0), "eps"),
    (lambda: aggregation.segment_group_norm(_x(), OFF, 4, eps=float("nan")), "eps"),
    (lambda: aggregation.segment_group_norm(_x(), OFF, 4, weight=torch.ones(8)), "weight is"),
    (lambda: aggregation.segment_group_norm(_x(), OFF, 4, bias=torch.ones(16, dtype=torch.bfloat16)), "bias must be"),
    (lambda: aggregation.segment_group_norm_backward(_x(7), _x(), OFF, torch.zeros(2, 4), torch.zeros(2, 4)), "grad is"),
    (lambda: aggregation.segment_group_norm_backward(_x(), _x(), OFF, torch.zeros(3, 4), torch.zeros(2, 4)), "mean is"),
    (lambda: aggregation.segment_group_norm_backward(_x(), _x(), OFF, torch.zeros(2, 4), torch.zeros(2, 2)), "rstd is"),
    (lambda: aggregation.gated_scan(_x(c=6), _x(c=6), OFF), "multiple of 4"),
    (lambda: aggregation.gated_scan(_x(), _x(7), OFF), "gate is"),
    (lambda: aggregation.gated_scan(_x(), _x(dtype=torch.bfloat16), OFF), "gate must be float32"),
    (lambda: aggregation.gated_scan(_x(), _x(), OFF, initial=torch.zeros(3, 16)), "initial is"),
    (lambda: aggregation.gated_scan(_x(), _x(), OFF.float()), "offsets"),
    (lambda: aggregation.gated_scan_backward(_x(), _x(), _x(), OFF, torch.zeros(3)), "saved is"),
    (lambda: _gated(x1=_x(8, 12, BF)), "multiples of 8"),
    (lambda: _gated(x1=_x(8, 16)), "x1 must be bfloat16"),
    (lambda: _gated(x2=_x(7, 16, BF)), "x2 is"),
    (lambda: _gated(w_gate=_x(24, 32, BF)), "w_up is"),
    (lambda: _gated(w_up=_x(16, 24, BF)), "w_up is"),
    (lambda: _gated(w_gate=_x(12, 32, BF), w_up=_x(12, 32, BF)), "multiples of 8"),
    (lambda: _gated(w_gate=_x(32, 16, BF).t()), "w_gate must be contiguous"),
    (lambda: _gated(b_gate=torch.zeros(16, dtype=BF)), "b_gate must be float32"),
    (lambda: _gated(b_up=torch.zeros(8)), "b_up is"),
    (lambda: _gated(activation="swish"), "unknown activation"),
    (lambda: _gated(out=_x(8, 16)), "out must be bfloat16"),
    (lambda: aggregation.gated_dense_concat_backward(_x(8, 24, BF), _x(8, 16, BF), None, _x(16, 16, BF),
                                                     _x(16, 16, BF)), "grad is"),
    (lambda: aggregation.gated_scan_step(_x(), _x(), torch.zeros(8, 8)), "state is"),
    (lambda: aggregation.gated_scan_step(_x(), _x(), torch.zeros(16, 8).t()), "state must be contiguous"),
])
def test_refused(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def test_overlapping_outputs():
    """An output over an input would be read by other blocks after it is
    written; the step's state in place is each thread's own."""
    buf = torch.zeros((12, 16), dtype=BF)
    for name, kw in (("x1", {"x1": buf[:8]}), ("x2", {"x2": buf[4:]}), ("w_gate", {"w_gate": _x(24, 32, BF)[:16]})):
        out = buf[2:10] if name != "w_gate" else kw["w_gate"].view(-1)[128:256].view(8, 16)
        with pytest.raises(ValueError, match=f"out must not overlap {name}"):
            _gated(out=out, **kw)
    state = torch.zeros(9, 16)
    with pytest.raises(ValueError, match="out_state must not overlap state"):
        aggregation.gated_scan_step(_x(), _x(), state[:8], out_state=state[1:])
    x = _x()
    with pytest.raises(ValueError, match="out_state must not overlap x"):
        aggregation.gated_scan_step(x, _x(), state[:8], out_state=x)


def test_rows_too_wide():
    with pytest.raises(RuntimeError, match="at most 4096 bytes"):
        aggregation.segment_group_norm(_x(c=1028), OFF, 4)


def test_host_tensors_are_refused():
    """Without a device the call says so; with one, host tensors are refused."""
    with pytest.raises((RuntimeError, ValueError), match="CUDA device"):
        aggregation.segment_group_norm(_x(), OFF, 4)
    with pytest.raises((RuntimeError, ValueError), match="CUDA device"):
        aggregation.gated_scan(_x(), _x(), OFF)


def test_native_checks_need_no_gpu():
    lib = _native.lib()
    bad = _native.ERR_INVALID_ARGUMENT
    assert lib.dgfx_segment_group_norm(None, 0, 4, 16, 4, None, 1, None, None, 1e-5, 0, None, None, None, None, 0,
                                       None) == bad
    assert lib.dgfx_segment_group_norm(None, 0, 4, 16, 4, None, 1, None, None, 1e-5, 9, None, None, None, None, 0,
                                       None) == bad
    assert lib.dgfx_segment_group_norm(256, 0, 4, 16, 4, 256, 1, None, None, 1e-5, 0, 264, 256, 256, None, 0, None) == bad
    assert "aligned" in _native.last_error()
    assert lib.dgfx_segment_group_norm_backward(256, 256, 0, 4, 16, 4, 256, 1, 256, 256, None, None, 0, 256, None, None,
                                                None, 0, None) == _native.ERR_WORKSPACE
    assert lib.dgfx_gated_scan(256, 256, 0, 4, 16, None, 1, None, None, None, None, None, 0, None) == bad
    assert lib.dgfx_gated_scan(264, 256, 0, 4, 16, 256, 1, None, None, None, None, None, 0, None) == bad
    assert lib.dgfx_gated_scan(256, 256, 0, 4, 16, 256, 1, None, None, None, None, 256, 8, None) == _native.ERR_WORKSPACE
    assert lib.dgfx_gated_scan(256, 256, 0, 1 << 50, 1 << 20, 256, 1, None, None, None, None, 256, 8,
                               None) == _native.ERR_UNSUPPORTED
    assert lib.dgfx_gated_scan_step(None, None, 1, 4, 16, None, None, None, None) == bad
