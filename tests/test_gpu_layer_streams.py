"""Layer operators on another stream than the current one, while the current
stream allocates and fills memory of the sizes that the call uses inside."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _graph(rows, degree, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    col = torch.randint(0, rows, (rows * degree,), generator=g, device="cuda", dtype=torch.int32)
    rowptr = torch.arange(0, rows * degree + 1, degree, device="cuda")
    return g, rowptr, col


def test_gated_sage_layer_keeps_its_memory_on_its_stream(cuda):
    """The mean and its workspace are the side stream's: what the current
    stream allocates and fills right after the call never touches them."""
    from distributed_graph_flow_b200 import aggregation

    rows, feat = 60000, 128
    g, rowptr, col = _graph(rows, 32, 1)
    x = torch.randn((rows, feat), generator=g, device="cuda").bfloat16()
    wg, wu = (0.1 * torch.randn((64, 2 * feat), generator=g, device="cuda")).bfloat16(), torch.ones(
        (64, 2 * feat), dtype=torch.bfloat16, device="cuda")
    ref = aggregation.sage_mean_gated(rowptr, col, x, wg, wu)
    need = aggregation.spmm_workspace(rows, col.numel(), feat, "cuda").numel()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    side = torch.cuda.Stream()
    for _ in range(5):
        got = aggregation.sage_mean_gated(rowptr, col, x, wg, wu, stream=side)
        junk = [torch.full((need,), 255, dtype=torch.uint8, device="cuda"),
                torch.full((rows, feat), float("nan"), dtype=torch.bfloat16, device="cuda")]
        torch.cuda.synchronize()
        assert torch.equal(got, ref)
        del junk, got
    aggregation.dense_check()


def test_mean_and_dense_layer_keep_their_memory_on_their_stream(cuda):
    from distributed_graph_flow_b200 import aggregation

    rows, feat = 60000, 128
    g, rowptr, col = _graph(rows, 32, 2)
    x = torch.randn((rows, feat), generator=g, device="cuda").bfloat16()
    weight = (0.1 * torch.randn((64, 2 * feat), generator=g, device="cuda")).bfloat16()
    ref = aggregation.csr_spmm(rowptr, col, x, normalize=True)
    ref_layer = aggregation.sage_mean_linear_relu(rowptr, col, x, weight)
    need = aggregation.spmm_workspace(rows, col.numel(), feat, "cuda").numel()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    side = torch.cuda.Stream()
    for _ in range(3):
        got = aggregation.csr_spmm(rowptr, col, x, normalize=True, stream=side)
        layer = aggregation.sage_mean_linear_relu(rowptr, col, x, weight, stream=side)
        junk = [torch.full((need,), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
        junk.append(torch.full((rows, feat), float("nan"), dtype=torch.bfloat16, device="cuda"))
        torch.cuda.synchronize()
        assert torch.equal(got, ref) and torch.equal(layer, ref_layer)
        del junk, got, layer
    aggregation.dense_check()
