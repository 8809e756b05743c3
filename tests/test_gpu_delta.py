"""The gated delta rule on the GPU against its 64-bit form (delta_ref.py, whose
error bounds are the tolerances): one position to several chunks, odd widths,
shared heads, lanes of length 0, strided and unaligned rows, decays that forget
everything, keys that repeat, refusals, streams and graphs."""
import math

import pytest
import torch

import boa_hip
import delta_ref as ref
import training_ref
from test_gpu_training import (BF16, F32, SKIP, codec, dev, empty, lens_of, place,  # noqa: F401
                               untouched, work, zeroed)

pytestmark = pytest.mark.gpu

GRADS = ["dq", "dk", "dv", "dg", "dbeta"]


def inputs(lanes, T, heads, hv, dk, dv, dtype, kind="plain", seed=0):
    g = torch.Generator().manual_seed(seed + lanes * 1000 + T + dk + 3 * dv)
    r = lambda *n: torch.randn(n, generator=g)  # noqa: E731
    s = {"q": r(lanes, T, heads * dk), "k": r(lanes, T, heads * dk), "v": r(lanes, T, hv * dv),
         "g": -torch.exp(r(lanes, T, hv) - 2), "beta": torch.sigmoid(r(lanes, T, hv)),
         "state_in": r(lanes, hv, dk, dv) * 0.3, "dout": r(lanes, T, hv * dv),
         "dstate_out": r(lanes, hv, dk, dv) * 0.3}
    if kind == "same":     # one key again and again, taken whole
        s["k"] = s["k"][:, :1].expand(lanes, T, heads * dk) + 1e-3 * s["k"]
        s["beta"] = torch.ones_like(s["beta"])
        s["g"] = s["g"] * 1e-3
    elif kind == "reset":  # a sequence behind another: nothing of the state is left
        s["g"][torch.rand(s["g"].shape, generator=g) < 0.05] = -math.inf
        s["g"][torch.rand(s["g"].shape, generator=g) < 0.05] = -300.0
    elif kind == "none":   # no decay, no write
        s["g"] = torch.zeros_like(s["g"])
        s["beta"] = s["beta"] * (torch.rand(s["beta"].shape, generator=g) < 0.5)
    elif kind == "tiny":   # rows of zeros, and rows far below the epsilon
        s["k"][:, ::3] = 0
        s["q"][:, 1::3] *= 1e-6
    for n in ("q", "k", "v", "dout"):
        s[n] = s[n].to(dtype)
    return s, g


def run(codec, s, heads, lens, layout, scale=0.3, unit=True, train=True, in_place=False):  # noqa: F811
    lanes, T, hv = s["g"].shape
    dt, dk, dv = s["q"].dtype, s["q"].shape[2] // heads, s["v"].shape[2] // hv
    live = training_ref.mask(lens, lanes, T)
    held = {}
    for n in ("q", "k", "v", "g", "beta", "dout"):
        t = s[n].clone()
        t[~live] = math.nan  # never read
        held[n] = place(t, layout, math.nan)
    sizes = (lanes, T, heads, hv, dk, dv)
    out = empty(lanes, T, hv * dv, dt, layout)
    state = dev(s["state_in"])
    state_out = state if in_place else torch.full((lanes, hv, dk, dv), SKIP, device="cuda")
    saved = torch.full((boa_hip.delta_rule_saved_floats(*sizes),), math.nan, device="cuda")
    w = work(boa_hip.delta_rule_work_bytes(*sizes, grad=train))
    args = [held[n] for n in ("q", "k", "v", "g", "beta")]
    how = dict(heads=heads, scale=scale, unit_qk=unit, d_lens=dev(lens))
    first = None if s["state_in"] is None else state.clone()
    codec.delta_rule(*args, out, w, d_state_in=state, d_state_out=state_out,
                     d_saved=saved if train else None, **how)
    got = {"out": out, "state_out": state_out}
    untouched(out, live, "out")
    if train:
        g = {"dq": empty(lanes, T, heads * dk, dt, layout), "dk": empty(lanes, T, heads * dk, dt, layout),
             "dv": empty(lanes, T, hv * dv, dt, layout), "dg": empty(lanes, T, hv, F32, layout),
             "dbeta": empty(lanes, T, hv, F32, layout)}
        ds_out = dev(s["dstate_out"])
        ds_in = ds_out if in_place and ds_out is not None else torch.full((lanes, hv, dk, dv), SKIP,
                                                                         device="cuda")
        codec.delta_rule_grad(*args, saved, held["dout"], *[g[n] for n in GRADS], w,
                              d_state_in=first, d_dstate_out=ds_out, d_dstate_in=ds_in, **how)
        for n in GRADS:
            zeroed(g[n], live, n)
        got.update(g, dstate_in=ds_in)
    return got, live


def compare(got, s, heads, live, scale=0.3, unit=True, train=True):
    want, dwant = ref.recurrence(s, heads, scale, unit, live, train)
    err, derr = ref.bounds(s, heads, scale, unit, live, train)
    ref.check("out", got["out"].cpu()[live], want["out"][live], err["out"][live], s["q"].dtype)
    ref.check("state_out", got["state_out"], want["state_out"], err["state_out"])
    if train:
        for n in GRADS:
            ref.check(n, got[n].cpu()[live], dwant[n][live], derr[n][live], got[n].dtype)
        if "dstate_in" in dwant:
            ref.check("dstate_in", got["dstate_in"], dwant["dstate_in"], derr["dstate_in"])


SHAPES = [  # lanes, T, heads, v heads, d_k, d_v, layout, lens, kind
    (1, 1, 1, 1, 64, 64, "dense", "full", "plain"), (3, 1, 2, 2, 1, 1, "dense", "full", "plain"),
    (3, 1, 1, 3, 80, 80, "wide", "ragged", "plain"), (4, 3, 2, 4, 128, 128, "dense", "ragged", "reset"),
    (2, 4, 1, 1, 17, 33, "odd", "ragged", "tiny"), (5, 2, 1, 2, 64, 128, "time", "ragged", "none"),
    (2, 5, 1, 1, 64, 64, "dense", "full", "plain"), (2, 17, 2, 2, 16, 16, "wide", "ragged", "tiny"),
    (1, 63, 1, 1, 64, 64, "dense", "full", "same"), (1, 64, 1, 2, 64, 128, "dense", "full", "reset"),
    (1, 65, 2, 2, 128, 64, "time", "full", "plain"), (3, 130, 1, 2, 80, 80, "wide", "ragged", "plain"),
    (3, 129, 2, 4, 128, 128, "dense", "ragged", "same"), (2, 200, 1, 3, 33, 100, "odd", "ragged", "reset"),
    (5, 70, 2, 2, 64, 128, "dense", "ragged", "none"), (2, 300, 1, 1, 127, 7, "odd", "ragged", "plain"),
    (1, 513, 1, 1, 64, 64, "dense", "full", "plain"), (3, 12, 1, 2, 100, 36, "dense", "ragged", "same"),
    (2, 9, 2, 2, 64, 64, "odd", "ragged", "reset"), (4, 13, 1, 1, 128, 128, "time", "ragged", "tiny"),
    # more blocks than CUs: the longest lanes first
    (70, 150, 2, 4, 33, 20, "dense", "ragged", "plain"), (300, 70, 1, 1, 16, 100, "wide", "ragged", "reset"),
    # cut into segments
    (1, 1100, 1, 1, 64, 64, "dense", "full", "plain"), (2, 1029, 1, 2, 33, 80, "odd", "ragged", "reset"),
    (3, 1500, 1, 2, 80, 70, "wide", "ragged", "same"), (1, 2000, 2, 2, 128, 128, "dense", "full", "none")]


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lanes,T,heads,hv,dk,dv,layout,kind,data", SHAPES)
def test_delta(codec, lanes, T, heads, hv, dk, dv, layout, kind, data, dtype, train):  # noqa: F811
    s, g = inputs(lanes, T, heads, hv, dk, dv, dtype, data)
    got, live = run(codec, s, heads, lens_of(kind, lanes, T, g), layout, train=train)
    compare(got, s, heads, live, train=train)


@pytest.mark.parametrize("T", [1, 3, 90])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_raw_rows_and_no_states(codec, dtype, T):  # noqa: F811
    """q and k as they are, no first state and no gradient of the last one."""
    s, g = inputs(2, T, 1, 2, 64, 64, dtype)
    for n in ("q", "k"):
        s[n] = (s[n].float() * 0.1).to(dtype)
    s["state_in"] = s["dstate_out"] = None
    got, live = run(codec, s, 1, None, "dense", scale=1.7, unit=False)
    compare(got, s, 1, live, scale=1.7, unit=False)


@pytest.mark.parametrize("T", [1, 4, 150, 1200])
def test_states_in_place(codec, T):  # noqa: F811
    s, g = inputs(3, T, 1, 2, 64, 128, F32)
    lens = lens_of("ragged", 3, T, g)
    got, live = run(codec, s, 1, lens, "dense", in_place=True)
    compare(got, s, 1, live)


@pytest.mark.parametrize("T,at", [(200, 64), (200, 77), (130, 3), (1200, 1100)])
def test_pieces_make_the_whole(codec, T, at):  # noqa: F811
    """A sequence in two calls, the state handed on."""
    s, _ = inputs(2, T, 1, 2, 64, 64, F32)
    live = training_ref.mask(None, 2, T)
    outs, state = [], s["state_in"]
    for part in (slice(0, at), slice(at, T)):
        piece = {n: v[:, part] if n in ("q", "k", "v", "g", "beta", "dout") else v
                 for n, v in s.items()}
        piece["state_in"] = state
        got, _ = run(codec, piece, 1, None, "dense", train=False)
        outs.append(got["out"].cpu())
        state = got["state_out"].cpu()
    compare({"out": torch.cat(outs, 1), "state_out": state}, s, 1, live, train=False)


def test_gradient_against_differences(codec):  # noqa: F811
    """The call's own outputs, moved a little: a central difference is off by
    h^2 of a third derivative (about 1e-4 of the slope here) and by the fp32
    outputs' rounding over 2 h; both lie well under 1 %."""
    lanes, T, heads, hv, dk, dv = 1, 70, 1, 2, 8, 8
    s, g = inputs(lanes, T, heads, hv, dk, dv, F32)
    got, _ = run(codec, s, heads, None, "dense")

    def loss(t):
        o, _ = run(codec, t, heads, None, "dense", train=False)
        return (o["out"].double().cpu() * s["dout"].double()).sum() + (
            o["state_out"].double().cpu() * s["dstate_out"].double()).sum()

    for n in ("q", "k", "v", "g", "beta", "state_in"):
        way = torch.randn(s[n].shape, generator=g)
        h = 1e-2
        up, down = (loss(dict(s, **{n: s[n] + sign * h * way})) for sign in (1, -1))
        slope = (got["d" + n].double().cpu() * way.double()).sum()
        size = (got["d" + n].double().cpu() * way.double()).norm()
        assert abs((up - down) / (2 * h) - slope) < 0.01 * size + 0.01 * slope.abs(), n


def test_other_lanes_do_not_matter(codec):  # noqa: F811
    """A lane's results are the same bits alone and beside others, one of which
    is not finite."""
    for T in (1, 3, 100):
        s, _ = inputs(5, T, 1, 2, 64, 64, F32)
        got, _ = run(codec, s, 1, None, "dense")
        s["v"][3] = math.nan
        more, _ = run(codec, s, 1, None, "dense")
        one = {n: v[2:3] for n, v in s.items()}
        alone, _ = run(codec, one, 1, None, "dense")
        for n in got:
            assert torch.equal(got[n][2:3], alone[n]), n
            assert torch.equal(got[n][:3], more[n][:3]), n


def test_two_calls_are_the_same_bits(codec):  # noqa: F811
    s, g = inputs(4, 333, 2, 4, 64, 128, BF16)
    lens = lens_of("ragged", 4, 333, g)
    a, b = (run(codec, s, 2, lens, "wide")[0] for _ in range(2))
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_capture(codec):  # noqa: F811
    """Forward and gradient captured once, replayed on new inputs."""
    lanes, T, sizes = 3, 100, (3, 100, 1, 2, 64, 64)
    s, _ = inputs(lanes, T, 1, 2, 64, 64, F32)
    d = {n: dev(v) for n, v in s.items()}
    z = lambda *n: torch.zeros(n, device="cuda")  # noqa: E731
    out, state = z(lanes, T, 128), z(lanes, 2, 64, 64)
    saved, w = z(boa_hip.delta_rule_saved_floats(*sizes)), work(
        boa_hip.delta_rule_work_bytes(*sizes, grad=True))
    g = [z(lanes, T, 64), z(lanes, T, 64), z(lanes, T, 128), z(lanes, T, 2), z(lanes, T, 2)]
    args = [d[n] for n in ("q", "k", "v", "g", "beta")]

    def step():
        codec.delta_rule(*args, out, w, heads=1, d_state_in=d["state_in"], d_state_out=state,
                         d_saved=saved)
        codec.delta_rule_grad(*args, saved, d["dout"], *g, w, heads=1, d_state_in=d["state_in"],
                              d_dstate_out=d["dstate_out"])

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        codec.set_stream(torch.cuda.current_stream().cuda_stream)
        step()
    codec.set_stream(torch.cuda.current_stream().cuda_stream)
    for seed in (1, 2, 3):
        new, _ = inputs(lanes, T, 1, 2, 64, 64, F32, seed=seed)
        for n in d:
            d[n].copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in [out, state] + g]
        for t in [out, state] + g:
            t.zero_()
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, [out, state] + g))


def test_refusals(codec):  # noqa: F811
    z = lambda *n, dt=F32: torch.zeros(n, dtype=dt, device="cuda")  # noqa: E731
    ok = dict(q=z(2, 20, 64), k=z(2, 20, 64), v=z(2, 20, 128), g=z(2, 20, 2), beta=z(2, 20, 2),
              out=z(2, 20, 128), w=work(boa_hip.delta_rule_work_bytes(2, 20, 1, 2, 64, 64)), heads=1)

    def call(**new):
        a = dict(ok, **new)
        codec.delta_rule(a["q"], a["k"], a["v"], a["g"], a["beta"], a["out"], a["w"],
                         heads=a["heads"], d_state_in=a.get("state_in"),
                         d_state_out=a.get("state_out"), d_saved=a.get("saved"))

    call()
    # few positions need no workspace, unless what the gradient needs is to be kept
    few = dict(ok, **{n: ok[n][:, :12] for n in ("q", "k", "v", "g", "beta", "out")})
    assert boa_hip.delta_rule_work_bytes(2, 12, 1, 2, 64, 64) == 0
    call(**dict(few, w=None))
    with pytest.raises(boa_hip.BoaError, match="workspace"):
        call(**dict(few, w=None, saved=z(boa_hip.delta_rule_saved_floats(2, 12, 1, 2, 64, 64))))
    for bad, why in [(dict(w=None), "workspace"), (dict(w=ok["w"][:-16]), "workspace"),
                     (dict(out=ok["v"]), "input"), (dict(out=z(2, 20, 64).repeat(1, 1, 1)), "out"),
                     (dict(q=z(2, 20, 64, dt=BF16)), "k"), (dict(g=z(2, 20, 2, dt=BF16)), "g"),
                     (dict(q=z(2, 20, 192), k=z(2, 20, 192)), "128"),
                     (dict(q=z(2, 20, 192), k=z(2, 20, 192), heads=3), "multiple"),
                     (dict(heads=0), "heads"), (dict(heads=5), "heads"),
                     (dict(state_in=z(2, 2, 64, 32)), "state_in"),
                     (dict(q=z(2, 20, 64).cpu()), "cpu"),
                     (dict(out=z(1, 20, 128).expand(2, 20, 128)), "overlap")]:
        with pytest.raises((boa_hip.BoaError, ValueError), match=why):
            call(**bad)
