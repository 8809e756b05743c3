"""The limits of delta_limits.py: that they are tight enough to see a term or a
segment's move that is missing or mistaken."""
import pytest
import torch

import delta_limits as lim
import delta_ref as ref
import training_ref
from delta_limits import SHAPES


def lens_of(kind, lanes, T, g):
    n = torch.randint(0, T + 1, (lanes,), generator=g, dtype=torch.int32)
    n[0] = T
    return None if kind == "full" else n


@pytest.mark.parametrize("lanes,T,heads,hv,dk,dv,layout,kind,data", SHAPES)
def test_limits_are_tight(lanes, T, heads, hv, dk, dv, layout, kind, data):
    s, g = lim.inputs(lanes, T, heads, hv, dk, dv, torch.float32, data)
    live = training_ref.mask(lens_of(kind, lanes, T, g), lanes, T)
    want = lim.exact(s, heads, 0.3, live)
    limits = lim.limits(s, heads, 0.3, live, want)
    for n, limit in limits.items():  # under a thousandth, where zero is off by one
        assert (limit <= 1e-3).all(), (n, limit)
    # the chunks in 64 bits are the recurrence
    s64 = {n: t.double() for n, t in s.items()}
    same = lim.results(lambda x: lim.chunked(x, heads, 0.3, live, torch.float64), s64, True)
    assert all((lim.off(same[n], want[n]) <= 1e-9).all() for n in want)
    # no write, and no read of what was written before, is within them
    for missing in ("v", "k"):
        less = dict(s64, **{missing: s64[missing].clone()})
        less[missing][:, T // 2:T // 2 + 8] = 0  # (some of them have a beta of 0)
        got = lim.results(lambda x: lim.chunked(x, heads, 0.3, live, torch.float64), less, False)
        seen = lim.off(got["out"], want["out"])
        assert (seen[0] > limits["out"][0]).all(), (missing, seen[0], limits["out"][0])
    each = ref._segment(lanes, hv, T, dk, dv)
    if each == -(-T // 64):
        return
    for mode, name in (("right", "state_out"), ("drop", "out"), ("drop", "state_out"),
                       ("across", "out"), ("across", "state_out"), ("back drop", "dstate_in"),
                       ("back across", "dstate_in")):
        got = lim.results(lambda x: lim.chunked(x, heads, 0.3, live, torch.float64, each, mode),
                          s64, mode.startswith("back"))
        seen = lim.off(got[name], want[name])
        if mode == "right":
            assert (seen <= limits[name]).all()
        else:
            assert seen[0] > 3 * limits[name][0], (mode, name, seen[0].item(), limits[name][0].item())
