"""Where the layer operators allocate and launch when a stream is given: no
GPU needed, the guard and the kernels are stand-ins that write down the order."""

import contextlib

import pytest
import torch

from distributed_graph_flow_b200 import _native, aggregation

BF = torch.bfloat16


class _Stream:
    cuda_stream = 7
    device_index = 0


@pytest.fixture
def log(monkeypatch):
    events = []

    @contextlib.contextmanager
    def entered():
        events.append("enter")
        yield
        events.append("leave")

    def guard(who, stream, *operands):
        events.append(("guard", sum(t is not None for t in operands)))
        return None if stream is None else entered()

    def spmm(rowptr, col, x, normalize, out, workspace=None, stream=None):
        events.append(("spmm", stream))
        return out

    def gated(x1, x2, *args, out=None, stream=None):
        events.append(("gated", stream))
        return x1.new_empty((x1.shape[0], args[0].shape[0])) if out is None else out

    monkeypatch.setattr(_native, "require_cuda", lambda: torch)
    monkeypatch.setattr(aggregation, "_layer_guard", guard)
    monkeypatch.setattr(aggregation, "csr_spmm", spmm)
    monkeypatch.setattr(aggregation, "gated_dense_concat", gated)
    return events


def _operands():
    return (torch.tensor([0, 1, 3]), torch.zeros(3, dtype=torch.int32), torch.zeros((4, 16), dtype=BF),
            torch.zeros((24, 32), dtype=BF), torch.zeros((24, 32), dtype=BF))


def test_both_steps_of_the_gated_sage_layer_run_under_one_guard(log):
    """agg and the workspace of the mean come from the pool of the stream that
    uses them: nothing is allocated or launched outside of the guard."""
    out = aggregation.sage_mean_gated(*_operands(), stream=_Stream())
    assert out.shape == (2, 24)
    calls = [e for e in log if e in ("enter", "leave") or e[0] in ("spmm", "gated")]
    assert calls == ["enter", ("spmm", None), ("gated", None), "leave"]
    # Everything that the launches read or write is recorded on the stream.
    log.clear()
    rowptr, col, x, wg, wu = _operands()
    agg, work = torch.zeros((2, 16), dtype=BF), torch.zeros(64, dtype=torch.uint8)
    aggregation.sage_mean_gated(rowptr, col, x, wg, wu, torch.zeros(24), torch.zeros(24), agg=agg, workspace=work,
                                out=torch.zeros((2, 24), dtype=BF), stream=_Stream())
    assert log[0] == ("guard", 10)


@pytest.mark.parametrize("change,match", [
    (dict(x=torch.zeros((4, 16))), "x must be bfloat16"),
    (dict(rowptr=torch.zeros(6, dtype=torch.int64)), "rowptr has 5 rows"),
    (dict(w_gate=torch.zeros((24, 16), dtype=BF)), "w_gate is"),
    (dict(agg=torch.zeros((3, 16), dtype=BF)), "agg is"),
    (dict(out=torch.zeros((2, 16), dtype=BF)), "out is"),
    (dict(activation="swish"), "unknown activation"),
])
def test_the_gated_sage_layer_refuses_before_it_runs(log, change, match):
    call = dict(zip(("rowptr", "col", "x", "w_gate", "w_up"), _operands())) | change
    with pytest.raises(ValueError, match=match):
        aggregation.sage_mean_gated(**call)
    assert not log


def test_the_gated_sage_layer_refuses_a_mean_over_its_input(log):
    rowptr, col, x, wg, wu = _operands()
    with pytest.raises(ValueError, match="agg must not overlap x"):
        aggregation.sage_mean_gated(rowptr, col, x, wg, wu, agg=x[1:3])


def test_temporaries_of_the_mean_come_from_the_streams_pool(monkeypatch):
    """csr_spmm drops its workspace, and sage_mean_linear_relu its mean, while
    the kernels may still run: both belong to the stream that runs them."""
    current, made = [None], []

    @contextlib.contextmanager
    def stream_context(stream):
        current.append(stream)
        yield
        current.pop()

    class _Lib:
        def dgfx_spmm_workspace_size(self, rows, nnz, feat, need):
            need._obj.value = 4096
            return 0

        def dgfx_spmm_csr(self, *args):
            return 0

    empty = torch.empty

    def recorded(shape, *args, **kw):
        made.append((tuple(shape) if not isinstance(shape, int) else (shape,), current[-1]))
        return empty(shape, *args, **kw)

    monkeypatch.setattr(_native, "require_cuda", lambda: torch)
    monkeypatch.setattr(_native, "lib", _Lib)
    monkeypatch.setattr(torch.cuda, "stream", stream_context)
    monkeypatch.setattr(torch, "empty", recorded)
    monkeypatch.setattr(aggregation, "dense_concat", lambda x1, x2, *args, **kw: x2)
    rowptr, col, x, weight, _ = _operands()
    stream = _Stream()
    aggregation.csr_spmm(rowptr, col, x, stream=stream)
    assert made == [((2, 16), None), ((4096,), stream)]  # the result is the caller's
    made.clear()
    aggregation.sage_mean_linear_relu(rowptr, col, x, weight, stream=stream)
    assert made == [((2, 16), stream), ((4096,), stream)]


def test_the_mean_runs_on_the_device_of_its_operands(monkeypatch):
    """Whatever device is the current one: its streams do not take the launches."""
    device, launched = [0], []

    class _Elsewhere(torch.Tensor):
        def get_device(self):
            return 1

    @contextlib.contextmanager
    def device_context(index):
        device.append(index)
        yield
        device.pop()

    class _Lib:
        def dgfx_spmm_workspace_size(self, rows, nnz, feat, need):
            need._obj.value = 64
            return 0

        def dgfx_spmm_csr(self, *args):
            launched.append((device[-1], args[-1]))
            return 0

    monkeypatch.setattr(_native, "require_cuda", lambda: torch)
    monkeypatch.setattr(_native, "lib", _Lib)
    monkeypatch.setattr(_native, "current_device", lambda: device[-1])
    monkeypatch.setattr(_native, "stream_handle", lambda stream=None: 100 + device[-1] if stream is None else stream.cuda_stream)
    monkeypatch.setattr(torch.cuda, "device", device_context)
    rowptr, col, x, _, _ = _operands()
    aggregation.csr_spmm(rowptr, col, x)
    there = torch.Tensor._make_subclass(_Elsewhere, x)
    out = aggregation.csr_spmm(rowptr, col, there, None, True, None, torch.float32)
    assert launched == [(0, 100), (1, 101)] and device == [0]
    assert out.shape == (2, 16) and out.dtype == torch.float32
