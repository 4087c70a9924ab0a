"""What the softmax loss asks its caller for (no GPU needed)."""
import ctypes as C

import pytest

import apoe


@pytest.fixture(scope="module")
def L():
    import build as apoe_build
    apoe_build.build()
    return apoe.lib()


@pytest.mark.parametrize("rows", [1, 32, 1000, 1001, 8192, 8193, 32768, 65000, 131073, 300000, 1 << 20])
def test_the_losses_workspace_is_bounded(L, rows):
    """64 MB of partial results or 512 bytes of each row, and 8 more of it, rounded to 256: whatever the number of documents."""
    size = C.c_size_t(0)
    for docs in (1, 2, 255, 256, 257, 1000, 8191, 8192, 8193, 8461, 16384, 16385, 100000, 100003, 1 << 24, 1 << 30):
        assert L.ap_softmax_loss_workspace(0, rows, docs, 1024, 0, size) == 0
        assert 0 < size.value <= max(64 << 20, rows * 512) + rows * 8 + 512, (docs, size.value)
