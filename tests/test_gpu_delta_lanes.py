"""The gated delta rule over more lanes than are put in order, and at the number
up to which they are: a lane's results are the same bits as in smaller batches."""
import pytest
import torch

import boa_hip
from test_gpu_delta import compare, inputs, run
from test_gpu_training import BF16, F32, codec, lens_of  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lanes,dtype", [(2048, F32), (2049, BF16), (5000, F32)])
def test_batches_do_not_matter(codec, lanes, dtype):  # noqa: F811
    T, dk, dv = 70, 16, 12
    s, g = inputs(lanes, T, 1, 1, dk, dv, dtype)
    lens = lens_of("ragged", lanes, T, g)
    got, live = run(codec, s, 1, lens, "dense")
    for at in range(0, lanes, 1000):
        part = slice(at, at + 1000)
        some = {n: v[part] for n, v in s.items()}
        want, _ = run(codec, some, 1, lens[part], "dense")
        for n in want:
            assert torch.equal(got[n][part], want[n]), (n, at)
    few = {n: v[:8] for n, v in s.items()}
    compare({n: v[:8] for n, v in got.items()}, few, 1, live[:8])


def test_many_lanes_are_linear_in_memory():
    """What the order takes does not grow beyond the lanes that are put in order."""
    need = [boa_hip.delta_rule_work_bytes(n, 100, 1, 1, 64, 64) / n for n in (1000, 2048, 60000)]
    assert need[0] >= need[1] >= need[2]
