"""Workspaces of the layer operators that are refused before anything runs on
a device (no GPU needed; the pointers are never followed)."""

import ctypes

import pytest

from distributed_graph_flow_b200 import _native

BIG = 1 << 40


def _calls():
    lib = _native.lib()

    def scan(ws, size):
        return lib.dgfx_gated_scan(256, 256, 0, 64, 16, 256, 2, None, 256, 256, None, ws, size, None)

    def scan_backward(ws, size):
        return lib.dgfx_gated_scan_backward(256, 256, 0, 64, 16, 256, 2, None, 256, 256, None, 256, 256, None, ws, size,
                                            None)

    def norm(ws, size):  # long enough for the list and the row tiles
        return lib.dgfx_segment_group_norm(256, 0, 1 << 20, 16, 4, 256, 2, None, None, 1e-5, 0, 256, 256, 256, ws, size,
                                           None)

    def norm_backward(ws, size):
        return lib.dgfx_segment_group_norm_backward(256, 256, 0, 64, 16, 4, 256, 2, 256, 256, None, None, 0, 256, None,
                                                    None, ws, size, None)

    def gated_backward(ws, size):
        return lib.dgfx_gated_dense_concat_backward_bf16(256, 256, 16, None, 0, 64, 256, 256, None, None, 16, 2, 256, None,
                                                         256, 256, None, None, ws, size, None)

    return {f.__name__: f for f in (scan, scan_backward, norm, norm_backward, gated_backward)}


@pytest.mark.parametrize("name", ["scan", "scan_backward", "norm", "norm_backward", "gated_backward"])
def test_refused(name):
    call = _calls()[name]
    assert call(256, 8) == _native.ERR_WORKSPACE
    assert call(None, BIG) == _native.ERR_WORKSPACE
    for odd in (260, 264):
        assert call(odd, BIG) == _native.ERR_INVALID_ARGUMENT
        assert "16-byte aligned" in _native.last_error()


def test_sizes_are_multiples_of_the_alignment():
    """Workspaces carved one behind the other stay aligned."""
    lib, need = _native.lib(), ctypes.c_size_t()
    for rows in (1, 7, 1000, 65537):
        assert lib.dgfx_gated_scan_workspace_size(rows, 20, 1, ctypes.byref(need), None) == 0
        assert need.value % 16 == 0
        assert lib.dgfx_segment_group_norm_workspace_size(rows, 24, 3, 5, 0, 1, ctypes.byref(need)) == 0
        assert need.value % 16 == 0
        assert lib.dgfx_gated_dense_concat_backward_workspace_size(24, 8, rows, 40, ctypes.byref(need)) == 0
        assert need.value % 16 == 0
