"""Where the parts of linear attention's workspace lie, told from its size."""
import pytest


@pytest.fixture(scope="module")
def lib():
    from csn_b200 import _build, _lib
    _build.build()
    return _lib.load()


@pytest.mark.parametrize("packed", [0, 1])
@pytest.mark.parametrize("rows,H,Dk,Dv", [(3, 3, 12, 8), (37, 2, 10, 64), (150, 2, 9, 64), (5, 3, 36, 104), (5, 3, 7, 8)])
def test_partial_gradients_begin_on_whole_sectors(lib, packed, rows, H, Dk, Dv):
    """Shared heads, sequences too short to be cut: the workspace is the float32 gradients of k and of v for every head of q, the
    second behind the first.  Their rows are written 32 bytes at a time."""
    nbytes = lib.csn_linear_attention_workspace_bytes(1, rows, H, 1, Dk, Dv, packed, 1, 0, 1)
    of_v = -(-rows * H * Dv * 4 // 32) * 32
    assert nbytes % 32 == 0 and nbytes - of_v >= rows * H * Dk * 4
    assert nbytes - of_v < rows * H * Dk * 4 + 32
