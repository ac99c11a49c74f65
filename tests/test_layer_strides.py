"""The torch operators take every operand strided or expanded: what they hand
to the kernels is packed. No GPU needed, the kernels are stand-ins."""

import torch

from distributed_graph_flow_b200 import aggregation, torch_ops  # noqa: F401 (registers the operators)

BF = torch.bfloat16


def _strided(rows, cols=None, dtype=torch.float32):
    return torch.zeros((2 * rows,) if cols is None else (2 * rows, cols), dtype=dtype)[::2]


def _packed_only(seen, result):
    def call(*args, **kw):
        seen.append([t for t in (*args, *kw.values()) if isinstance(t, torch.Tensor)])
        return tuple(t.clone() for t in result) if isinstance(result, tuple) else result.clone()

    return call


def test_operands_are_packed(monkeypatch):
    seen = []
    x, w, b = _strided(8, 16, BF), _strided(24, 32, BF), _strided(24)
    monkeypatch.setattr(aggregation, "gated_dense_concat", _packed_only(seen, torch.zeros((8, 24), dtype=BF)))
    torch.ops.dgfx.gated_dense_concat(x, x, w, w, b, torch.zeros(1).expand(24), "silu")
    monkeypatch.setattr(aggregation, "gated_dense_concat_backward", _packed_only(seen, (torch.zeros(1),) * 6))
    torch.ops.dgfx.gated_dense_concat_grad(_strided(8, 24, BF), x, x, w, w, b, torch.zeros(1).expand(24), "silu", True,
                                           True)
    xf, off, s = _strided(8, 16), _strided(3).long(), torch.zeros(2, 4)
    off = torch.stack([off, off], 1)[:, 0]
    monkeypatch.setattr(aggregation, "segment_group_norm", _packed_only(seen, (torch.zeros(8, 16), s, s + 1)))
    torch.ops.dgfx.segment_group_norm(xf, off, 4, _strided(16), torch.zeros(1).expand(16), 1e-5, "none")
    monkeypatch.setattr(aggregation, "segment_group_norm_backward",
                        _packed_only(seen, (torch.zeros(8, 16), torch.zeros(16), torch.zeros(16))))
    torch.ops.dgfx.segment_group_norm_grad(xf, xf, off, s, s, _strided(16), torch.zeros(1).expand(16), "none")
    h0 = _strided(2, 16)
    monkeypatch.setattr(aggregation, "gated_scan", _packed_only(seen, (torch.zeros(8, 16), torch.zeros(2, 16),
                                                                      torch.zeros(32))))
    torch.ops.dgfx.gated_scan(xf, xf, off, h0, True)
    monkeypatch.setattr(aggregation, "gated_scan_backward",
                        _packed_only(seen, (torch.zeros(8, 16), torch.zeros(8, 16), torch.zeros(2, 16))))
    torch.ops.dgfx.gated_scan_grad(xf, h0, xf, xf, off, torch.zeros(32), h0)
    assert [len(call) for call in seen] == [6, 7, 4, 7, 4, 7]
    assert all(t.is_contiguous() for call in seen for t in call)
