"""Outputs of a gated-delta-rule predictor's operators that begin where another
output or an input does are refused; what may be in place still is."""
import itertools

import pytest
import torch

import boa_hip
from test_gpu_training import BF16, F32, codec, work  # noqa: F401

pytestmark = pytest.mark.gpu

LANES, T, H, HV, DK, DV = 2, 20, 1, 1, 64, 64
SIZES = (LANES, T, H, HV, DK, DV)


def z(*n, dt=F32):
    return torch.zeros(n, dtype=dt, device="cuda")


def refused(call, tensors, outs, allowed=()):
    """Every output in place of another tensor of its shape and type."""
    call(**tensors)
    tried = 0
    for a, b in itertools.product(outs, tensors):
        x, y = tensors[a], tensors[b]
        if a == b or (a, b) in allowed or (b, a) in allowed:
            continue
        if x.dtype != y.dtype:
            y = y.view(x.dtype) if y.is_contiguous() else y
        if y.dtype != x.dtype or y.numel() < x.numel():
            continue
        y = y.flatten()[:x.numel()].view(x.shape)
        with pytest.raises((boa_hip.BoaError, ValueError), match="output is"):
            call(**dict(tensors, **{a: y}))
        tried += 1
    assert tried >= len(outs), tried


def test_norm(codec):  # noqa: F811
    # as wide as a lane is long, so that weight and scale8 could be each other
    w = LANES * T
    t = {"x": z(LANES, T, w), "residual": z(LANES, T, w), "weight": z(w), "sum": z(LANES, T, w),
         "out": z(LANES, T, w), "out8": z(LANES, T, w, dt=torch.int8), "scale8": z(LANES, T)}

    def call(**a):
        codec.rms_norm(a["x"], a["out"], d_weight=a["weight"], d_residual=a["residual"],
                       d_sum=a["sum"], d_out8=a["out8"], d_scale8=a["scale8"])

    refused(call, t, ["sum", "out", "out8", "scale8"], allowed=[("sum", "x"), ("sum", "residual")])
    codec.rms_norm(t["x"], t["out"], d_residual=t["residual"], d_sum=t["x"])
    codec.rms_norm(t["x"], t["out"], d_residual=t["residual"], d_sum=t["residual"])


def test_norm_grad(codec):  # noqa: F811
    w = 64
    t = {"h": z(LANES, T, w), "dout": z(LANES, T, w), "dsum": z(LANES, T, w), "weight": z(w),
         "dx": z(LANES, T, w), "dweight": z(w),
         "work": work(boa_hip.rms_norm_grad_work_bytes(LANES, T, w))}

    def call(**a):
        codec.rms_norm_grad(a["h"], a["dout"], a["dx"], a["work"], d_weight=a["weight"],
                            d_dsum=a["dsum"], d_dweight=a["dweight"])

    refused(call, t, ["dx", "dweight", "work"], allowed=[("dx", "dout"), ("dx", "dsum")])
    for n in ("dout", "dsum"):
        call(**dict(t, dx=t[n]))


def test_8_bits(codec):  # noqa: F811
    n, k = 64, LANES * T
    t = {"x": z(LANES, T, k), "out8": z(LANES, T, k, dt=torch.int8), "scale8": z(LANES, T)}
    refused(lambda **a: codec.int8_rows(a["x"], a["out8"], a["scale8"]), t, ["out8", "scale8"])
    t = {"x8": z(LANES, T, 4 * n, dt=torch.int8), "scale8": z(LANES, T), "wscale": z(n),
         "bias": z(n), "packed": z(boa_hip.int8_pack_bytes(n, 4 * n), dt=torch.uint8),
         "out": z(LANES, T, n)}

    def call(**a):
        codec.int8_matmul(a["x8"], a["scale8"], a["packed"], a["wscale"], a["out"],
                          d_bias=a["bias"])

    refused(call, t, ["out"])


def rule(codec, T=T):  # noqa: F811
    q = {n: z(LANES, T, 64) for n in ("q", "k", "v", "out")}
    q.update(g=z(LANES, T, 1), beta=z(LANES, T, 1), state_in=z(LANES, 1, 64, 64),
             state_out=z(LANES, 1, 64, 64),
             saved=z(boa_hip.delta_rule_saved_floats(LANES, T, *SIZES[2:])),
             work=work(boa_hip.delta_rule_work_bytes(LANES, T, *SIZES[2:], grad=True)))
    return q


def test_rule(codec):  # noqa: F811
    t = rule(codec)

    def call(**a):
        codec.delta_rule(a["q"], a["k"], a["v"], a["g"], a["beta"], a["out"], a["work"], heads=1,
                         d_state_in=a["state_in"], d_state_out=a["state_out"], d_saved=a["saved"])

    refused(call, t, ["out", "state_out", "saved", "work"], allowed=[("state_out", "state_in")])
    call(**dict(t, state_out=t["state_in"]))
    # few positions use no workspace, so it may be anything
    few = rule(codec, 4)
    codec.delta_rule(few["q"], few["k"], few["v"], few["g"], few["beta"], few["out"], few["q"],
                     heads=1)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rule_grad(codec, dtype):  # noqa: F811
    t = rule(codec)
    for n in ("q", "k", "v"):
        t[n] = t[n].to(dtype)
    del t["out"], t["state_out"]
    t.update({"d" + n: torch.zeros_like(t[n]) for n in ("q", "k", "v", "g", "beta", "state_in")})
    t.update(dout=torch.zeros_like(t["v"]), dstate_out=z(LANES, 1, 64, 64))

    def call(**a):
        codec.delta_rule_grad(a["q"], a["k"], a["v"], a["g"], a["beta"], a["saved"], a["dout"],
                              a["dq"], a["dk"], a["dv"], a["dg"], a["dbeta"], a["work"], heads=1,
                              d_state_in=a["state_in"], d_dstate_out=a["dstate_out"],
                              d_dstate_in=a["dstate_in"])

    call(**t)
    refused(call, t, ["dq", "dk", "dv", "dg", "dbeta", "work"])
    refused(call, t, ["dstate_in"], allowed=[("dstate_in", "dstate_out"), ("dstate_in", "state_in")])
    call(**dict(t, dstate_in=t["dstate_out"]))
    # side by side in one tensor, as their inputs may be
    d = torch.zeros((LANES, T, 192), dtype=dtype, device="cuda")
    call(**dict(t, dq=d[..., :64], dk=d[..., 64:128], dv=d[..., 128:]))


def test_sample(codec):  # noqa: F811
    t = {"logits": z(LANES, T, 256), "bias": z(256), "uniform": z(LANES, T), "params": z(LANES, 4),
         "bytes": z(LANES, T, dt=torch.uint8), "logp": z(LANES, T)}

    def call(**a):
        codec.sample_bytes(a["logits"], a["uniform"], a["bytes"], d_bias=a["bias"],
                           d_logp=a["logp"], d_params=a["params"])

    refused(call, t, ["bytes", "logp"])
