"""Which products round their tokens inside (no workspace) and which apart (CPU, sizes only)."""
import pytest

from test_int8_abi import lib


@pytest.mark.parametrize("R,N,K,gated,inside", [
    (1, 8192, 4096, 0, True), (4, 8192, 4096, 0, True), (5, 8192, 2048, 0, False), (1, 8192, 4104, 0, False),     # one tile of the weight a workgroup
    (1, 8256, 2048, 0, True), (4, 16384, 2048, 0, True), (1, 8256, 2056, 0, False), (1, 16448, 2048, 0, False),   # two
    (1, 64, 2048, 1, True), (4, 16384, 2048, 1, True), (1, 64, 2056, 1, False), (1, 8192, 4096, 1, False), (1, 16448, 2048, 1, False)])
def test_rounding_inside(lib, R, N, K, gated, inside):
    need = lib.lfm3_hip_linear8_workspace(R, N, K, gated)
    assert (need == 0) == inside
    if not inside:
        assert need == 32 * (-(-K // 128) * 128) + 32 * 4
