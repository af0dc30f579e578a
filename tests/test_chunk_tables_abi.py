"""kv800_hip_decode_chunk_sized (CPU, no GPU calls): widths of the tables apart from their strides, bad ones rejected on the host."""
import ctypes

import pytest

import lfm3_kv800_amd.kv800_hip as kh
from test_chunk_abi import A, lib, paged, refused  # noqa: F401


def test_widths_are_checked(lib):
    ws = lib.kv800_hip_decode_chunk_workspace(2, 8, 4)

    def f(bcols=4, ecols=4, T=8, **P):
        return lib.kv800_hip_decode_chunk_sized(ctypes.byref(paged(**P)), bcols, ecols, A, A, 2, T, A, A, 512, A, 1 << 20, 1 << 20, 0, A, A,
                                                ws, None)
    assert f(T=0) == 0
    for k in (dict(ecols=0), dict(ecols=-1), dict(bcols=0), dict(bcols=-1), dict(eoff_stride=-1), dict(boff_stride=-1)):
        refused(lib, f(**k), b"decode_chunk")


@pytest.mark.parametrize("stride,shape,want", [((1, 1), (1, 9), 9), ((20, 1), (1, 9), 20), ((20, 1), (3, 9), 20), ((0, 1), (3, 9), 0)])
def test_row_stride(stride, shape, want):
    import torch
    assert kh._row_stride(torch.zeros(80, dtype=torch.int64).as_strided(shape, stride)) == want
