"""The 64-bit form of the gated delta rule against differences, and what can be
asked of its operators without a GPU: sizes and refusals."""
import ctypes

import pytest
import torch

import boa_hip
import delta_ref as ref


def test_recurrence_gradient_against_differences():
    g = torch.Generator().manual_seed(0)
    lanes, T, h, hv, dk, dv = 2, 7, 1, 2, 5, 3
    r = lambda *n: torch.randn(n, generator=g, dtype=torch.float64)  # noqa: E731
    s = {"q": r(lanes, T, h * dk), "k": r(lanes, T, h * dk), "v": r(lanes, T, hv * dv),
         "g": -r(lanes, T, hv).abs(), "beta": torch.sigmoid(r(lanes, T, hv)),
         "state_in": r(lanes, hv, dk, dv), "dout": r(lanes, T, hv * dv),
         "dstate_out": r(lanes, hv, dk, dv)}
    live = torch.ones((lanes, T), dtype=torch.bool)
    live[1, 4:] = False

    def total(x):
        got, _ = ref.recurrence(x, h, 0.3, True, live)
        return ((got["out"] * x["dout"]).sum() + (got["state_out"] * x["dstate_out"]).sum()).item()

    _, grads = ref.recurrence(s, h, 0.3, True, live, True)
    for n in ("q", "k", "v", "g", "beta", "state_in"):
        d = torch.randn(s[n].shape, generator=g, dtype=torch.float64)
        hi, lo = (total(dict(s, **{n: s[n] + e * d})) for e in (1e-5, -1e-5))
        want = (grads["d" + n] * d).sum().item()
        # a third derivative of the size of the sum, times 1e-10
        assert abs((hi - lo) / 2e-5 - want) <= 1e-6 * max(1.0, abs(want)), n


def test_sizes():
    lib = boa_hip.lib()
    assert boa_hip.delta_rule_work_bytes(1000, 1, 4, 4, 64, 128) == 0  # a decode step
    assert boa_hip.delta_rule_work_bytes(1000, 1, 4, 4, 64, 128, grad=True) > 0
    assert boa_hip.delta_rule_work_bytes(2, 100, 1, 2, 64, 64) > 0
    # S and N of every chunk, fp32
    assert boa_hip.delta_rule_saved_floats(3, 129, 1, 2, 60, 50) == 3 * 2 * 3 * 50 * (64 + 64)
    # few long sequences keep what their segments make of a state, too
    assert (boa_hip.delta_rule_saved_floats(1, 4096, 1, 1, 64, 64)
            > 64 * 64 * (64 + 64) * 1)
    assert boa_hip.int8_pack_bytes(1, 1) == 128 * 64
    assert boa_hip.int8_pack_bytes(129, 513) == 256 * 768
    assert boa_hip.rms_norm_grad_work_bytes(5, 7, 64) >= 0
    for bad in [(0, 1, 1, 1, 64, 64), (1, 0, 1, 1, 64, 64), (1, 1, 2, 3, 64, 64), (1, 1, 1, 0, 64, 64),
                (1, 1, 1, 1, 129, 64), (1, 1, 1, 1, 64, 129), (1, 1, 1, 1, 0, 64), (1, 1, 0, 1, 64, 64),
                (1, 1, 1, 1025, 64, 64), (65536, 1, 1, 1, 64, 64), (2, 1 << 30, 1, 1, 64, 64)]:
        assert lib.boa_delta_rule_work_bytes(*bad, 0) == -1, bad
        assert lib.boa_delta_rule_saved_floats(*bad) == -1, bad
        with pytest.raises(ValueError):
            boa_hip.delta_rule_work_bytes(*bad)
    for bad in [(0, 1), (1, 0), (65537, 1), (1, 16385)]:
        assert lib.boa_int8_pack_bytes(*bad) == -1


def test_sizes_beyond_32_bits_are_refused():
    """What ctypes would cut to 32 bits, to sizes that are in range."""
    for f, good in ((boa_hip.delta_rule_work_bytes, (1, 5, 1, 2, 64, 64)),
                    (boa_hip.delta_rule_saved_floats, (1, 5, 1, 2, 64, 64)),
                    (boa_hip.rms_norm_grad_work_bytes, (1, 5, 64)),
                    (boa_hip.int8_pack_bytes, (5, 64))):
        f(*good)
        for i in range(len(good)):
            bad = list(good)
            bad[i] += 2 ** 32
            with pytest.raises(ValueError, match="range"):
                f(*bad)


def test_null_context_is_refused():
    lib, r = boa_hip.lib(), boa_hip.Rows(None, 0, 0)
    p = ctypes.byref(r)
    d, how = boa_hip.Delta(), boa_hip.Sampling(1.0, 0, 1.0, 0.0)
    for rc in (lib.boa_rms_norm(None, p, None, None, None, 1, 1, 64, 0, 1e-6, None, p, None, None),
               lib.boa_rms_norm_grad(None, p, None, None, 1, 1, 64, 0, 1e-6, p, None, p, None, None, 0),
               lib.boa_int8_rows(None, p, None, 1, 1, 64, 0, p, None),
               lib.boa_int8_pack(None, None, 1, 1, None),
               lib.boa_int8_matmul(None, p, None, None, 1, 1, 64, None, None, 1, None, 0, p),
               lib.boa_delta_rule(None, ctypes.byref(d), p, None, None, None, 0),
               lib.boa_delta_rule_grad(None, ctypes.byref(d), None, p, None,
                                       ctypes.byref(boa_hip.DeltaGrads()), None, 0),
               lib.boa_sample_bytes(None, p, None, None, None, 1, 1, 0, ctypes.byref(how), None, None,
                                    0, None)):
        assert rc == boa_hip.BOA_E_ARG
