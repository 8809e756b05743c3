"""The gated delta rule on the GPU, whole lanes against the 64-bit recurrence
within limits on norms (delta_limits.py): states that live on through many
segments, keys that repeat, no decay."""
import pytest
import torch

import boa_hip
import delta_limits as lim
import training_ref
from delta_limits import SHAPES
from test_gpu_delta import GRADS, run
from test_gpu_training import BF16, F32, codec, lens_of  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lanes,T,heads,hv,dk,dv,layout,kind,data", SHAPES)
def test_lanes(codec, lanes, T, heads, hv, dk, dv, layout, kind, data, dtype):  # noqa: F811
    s, g = lim.inputs(lanes, T, heads, hv, dk, dv, dtype, data)
    lens = lens_of(kind, lanes, T, g)
    got, live = run(codec, s, heads, lens, layout)
    want = lim.exact(s, heads, 0.3, live)
    limits = lim.limits(s, heads, 0.3, live, want)
    for n in ["out", "state_out", "dstate_in"] + GRADS:
        limit = limits[n] + (2.0 ** -8 if got[n].dtype == BF16 else 0)
        t = got[n].cpu() if n.endswith(("state_in", "state_out")) else torch.where(
            live[..., None], got[n].cpu(), torch.zeros((), dtype=got[n].dtype))
        seen = lim.off(t, want[n])
        print(n, "off by", f"{seen.max():.2g}, {(seen / limit).max():.2g} of the limit")
        assert (seen <= limit).all(), (n, seen, limit)
    # the forward pass alone, without what the gradient needs
    again, _ = run(codec, s, heads, lens, layout, train=False)
    assert (lim.off(again["state_out"].cpu(), want["state_out"]) <= limits["state_out"]).all()
