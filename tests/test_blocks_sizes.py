"""The gated block's workspaces over their sizes, without a GPU: what a layer asks for is enough for its own calls."""
import pytest


def _lib():
    from tcbnn_amd import _lib
    return _lib


ROWS = [1, 3, 5, 17, 130, 257, 1000, 4099, 12000, 33333, 47951, 60000, 123457, 400000]
INNER = [3, 24, 519, 615, 1023, 1024, 2501, 4095]
OUTER = [5, 100, 1000, 4001, 20000, 65537, 131072, 227888, 500000]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_room_for_copies_is_room_without(dtype):
    """Each call asks for as much as its size without copies, and a layer whose operands lie anywhere has the size with them."""
    lib, dt = _lib().lib, _lib().DTYPES[dtype]
    for f in (lib.tcbnn_linear_loss_workspace_bytes, lib.tcbnn_linear_loss_grad_workspace_bytes, lib.tcbnn_gated_grad_workspace_bytes):
        for m in ROWS:
            for k in INNER:
                for n in OUTER:
                    assert f(m, k, n, dt, 1) >= f(m, k, n, dt, 0), (f.__name__, m, k, n)
