"""The scan gradient's sums across a wave's lanes, on the CPU: the kernel's own
steps (csrc/scan_lanes.h) on 64 modelled lanes."""
import ctypes
import os
import subprocess

import numpy as np
import pytest


@pytest.fixture(scope="module")
def model():
    here = os.path.dirname(os.path.abspath(__file__))
    # by make's rule, so that the steps tested are the present ones
    subprocess.run(["make", "-s", "-C", here, "liblane_model.so"], check=True)
    f = ctypes.CDLL(os.path.join(here, "liblane_model.so")).lane_model

    def run(tpc, x):
        x = np.ascontiguousarray(x, np.float32)
        out = [np.zeros(64, t) for t in (np.float32, np.float32, np.int32, np.int32)]
        f(tpc, *[ctypes.c_void_p(a.ctypes.data) for a in (x, *out)])
        return out
    return run


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("tpc", [4, 8])
def test_sums_over_lanes(model, tpc, seed):
    """Whole numbers, whose sums have no rounding: each lane's value is the sum
    that its address stands for."""
    x = np.random.default_rng(seed).integers(-40, 41, (13, 64)).astype(np.float32)
    sums, bc, states, slot = model(tpc, x)
    n, lane = 4 * tpc, np.arange(64)
    channels = 64 // tpc
    for c in range(channels):  # every channel's lanes hold all its states
        assert sorted(states[c * tpc:(c + 1) * tpc]) == list(range(tpc))
    over = x[:3].reshape(3, channels, tpc).sum(2)  # y, I, M
    assert (sums == over[np.minimum(lane & 3, 2), lane // tpc]).all()

    want = np.zeros(2 * n)
    for i in range(64):
        for k in range(4):
            want[4 * states[i] + k] += x[5 + k, i] * x[3, i]      # dB: dh du
            want[n + 4 * states[i] + k] += x[9 + k, i] * x[4, i]  # dC: h dy
    assert set(slot) == set(range(2 * n))
    assert (bc == want[slot]).all(), f"lanes {np.nonzero(bc != want[slot])[0]} hold other sums"


@pytest.mark.parametrize("tpc", [4, 8])
def test_lanes_of_one_address_agree(model, tpc):
    """Any values: lanes that store to one address store the same bits."""
    x = np.random.default_rng(9).standard_normal((13, 64)).astype(np.float32)
    sums, bc, _, slot = model(tpc, x)
    for value, address in ((bc, slot), (sums, (np.arange(64) // tpc) * 3
                                        + np.minimum(np.arange(64) & 3, 2))):
        for a in set(address):
            assert len({v.tobytes() for v in value[address == a]}) == 1, a
