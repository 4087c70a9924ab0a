"""Addresses the dense operators refuse on the host: a kernel that read or wrote there would fault (no GPU needed)."""
import pytest

import apoe

BF16 = 2
GOOD = 1 << 12       # an aligned address that is never read


@pytest.fixture(scope="module")
def L():
    import build as apoe_build
    apoe_build.build()
    return apoe.lib()


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("which", ["target", "loss", "lse", "grad"])
def test_vectors_off_4_byte_boundaries_are_refused(L, which, off):
    at = {name: GOOD + (off if name == which else 0) for name in ("target", "loss", "lse", "grad")}
    # workspaces too small to pass, so that no call goes on to the device
    calls = [L.ap_softmax_loss_backward_device(0, 8, 64, 64, BF16, GOOD, 64, GOOD, 64, at["target"], 1.0, at["loss"], at["lse"], at["grad"], GOOD, 64,
                                               GOOD, 64, GOOD, 0, None)]
    assert "4-byte" in L.ap_last_error().decode()
    if which != "grad":
        calls.append(L.ap_softmax_loss_forward_device(0, 8, 64, 64, BF16, GOOD, 64, GOOD, 64, at["target"], 1.0, at["loss"], at["lse"], GOOD, 0, None))
        assert "4-byte" in L.ap_last_error().decode()
    assert all(rc == 1 for rc in calls)
