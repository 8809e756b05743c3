"""The 64-bit forms of the training operators that the GPU tests compare with:
their gradients against differences of their forwards, and the argument
checks of the binding that need no GPU."""
import ctypes
import math

import pytest
import torch

import boa_hip
import training_ref as ref


def _scan_inputs(lanes, T, ch, n, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    return {"u": r(lanes, T, ch), "delta": r(lanes, T, ch) * 0.5, "z": r(lanes, T, ch),
            "B": r(lanes, T, n), "C": r(lanes, T, n), "A": -torch.rand((ch, n), generator=g).double() * 4,
            "D": r(ch), "delta_bias": r(ch) - 1, "state_in": r(lanes, ch, n),
            "dout": r(lanes, T, ch), "dstate_out": r(lanes, ch, n)}


def test_scan_gradient_against_differences():
    s = _scan_inputs(3, 7, 5, 16, 0)
    live = ref.mask(torch.tensor([7, 4, 0]), 3, 7)

    def value(s):
        out, state, _ = ref.scan(s, live)
        return ((out.val * s["dout"])[live].sum() + (state.val * s["dstate_out"]).sum()).item()

    _, _, kept = ref.scan(s, live)
    grads = ref.scan_grad(s, live, kept)
    g = torch.Generator().manual_seed(1)
    for name, key in [("du", "u"), ("ddelta", "delta"), ("dz", "z"), ("dB", "B"), ("dC", "C"),
                      ("dA", "A"), ("dD", "D"), ("ddelta_bias", "delta_bias"),
                      ("dstate_in", "state_in")]:
        d = torch.randn(s[key].shape, generator=g, dtype=torch.float64)
        eps = 1e-5
        diff = (value(dict(s, **{key: s[key] + eps * d}))
                - value(dict(s, **{key: s[key] - eps * d}))) / (2 * eps)
        along = (grads[name].val * d).sum().item()
        # central differences: eps^2 times a third derivative, 1e-16 / eps of rounding
        assert abs(diff - along) <= 1e-6 * max(1.0, abs(along)), name


def test_loss_gradient_against_differences():
    g = torch.Generator().manual_seed(2)
    x = torch.randn((2, 5, 256), generator=g, dtype=torch.float64) * 3
    b = torch.randn(256, generator=g, dtype=torch.float64)
    tgt = torch.randint(0, 256, (2, 5), generator=g, dtype=torch.uint8)
    live = ref.mask(torch.tensor([5, 3]), 2, 5)
    f = lambda x, b: ref.loss(x, b, tgt, 1.0, live)[1].val.item()  # noqa: E731
    _, _, dx, db = ref.loss(x, b, tgt, 1.0, live)
    for grad, i in ((dx, 0), (db, 1)):
        d = torch.randn(grad.val.shape, generator=g, dtype=torch.float64)
        hi = f(*[v + 1e-5 * d if k == i else v for k, v in enumerate((x, b))])
        lo = f(*[v - 1e-5 * d if k == i else v for k, v in enumerate((x, b))])
        assert abs((hi - lo) / 2e-5 - (grad.val * d).sum().item()) <= 1e-6


def test_loss_matches_log_softmax():
    g = torch.Generator().manual_seed(3)
    x = torch.randn((1, 9, 256), generator=g, dtype=torch.float64) * 5
    x[0, :, 128:] = -math.inf
    tgt = torch.randint(0, 128, (1, 9), generator=g, dtype=torch.uint8)
    out, _, _, _ = ref.loss(x, None, tgt, 1.0, ref.mask(None, 1, 9))
    want = torch.nn.functional.cross_entropy(x[0], tgt[0].long(), reduction="none")
    assert torch.allclose(out.val[0], want, rtol=1e-12, atol=1e-12)


def test_work_sizes_refuse_bad_sizes():
    lib = boa_hip.lib()
    assert boa_hip.embed_grad_work_bytes(1, 1, 1) == 0  # one block does it all
    assert boa_hip.next_byte_loss_work_bytes(1, 128) == 0
    assert boa_hip.selective_scan_saved_floats(3, 17, 5, 16) == 3 * 2 * 5 * 16
    for bad in [(0, 1, 64), (1, 0, 64), (65536, 1, 64), (1, 1, 513), (1, 1, 0), (2, 1 << 30, 64)]:
        assert lib.boa_embed_grad_work_bytes(*bad) == -1
        with pytest.raises(ValueError):
            boa_hip.embed_grad_work_bytes(*bad)
    for bad in [(0, 1, 64, 16), (1, 0, 64, 16), (1, 1, 0, 16), (1, 1, 4097, 16), (1, 1, 64, 24)]:
        assert lib.boa_selective_scan_work_bytes(*bad, 1) == -1
        assert lib.boa_selective_scan_saved_floats(*bad) == -1
    assert lib.boa_next_byte_loss_work_bytes(1, (1 << 30) + 1) == -1


def test_null_context_is_refused():
    lib = boa_hip.lib()
    assert lib.boa_device(None) == boa_hip.BOA_E_ARG
    r = boa_hip.Rows(None, 0, 0)
    assert lib.boa_embed(None, None, 0, None, 1, 1, None, 64, 0, 1.0,
                         ctypes.byref(r)) == boa_hip.BOA_E_ARG
    assert lib.boa_next_byte_loss(None, ctypes.byref(r), None, None, 0, None, 1, 1, 0, 1.0, None,
                                  None, None, None, None, 0) == boa_hip.BOA_E_ARG


def test_binding_refuses_wrong_tensors():
    t = torch.zeros((2, 3, 8))
    with pytest.raises(ValueError, match="is on"):  # not on the context's device
        boa_hip._rows(t, "x", 2, 3, 8, torch.float32, 0)
    with pytest.raises(ValueError, match="want"):  # shape
        boa_hip._rows(t, "x", 2, 3, 9, torch.float32, 0)
    with pytest.raises(ValueError, match="want"):  # type
        boa_hip._rows(t.half(), "x", 2, 3, 8, torch.float32, 0)
    with pytest.raises(ValueError):
        boa_hip._precision(t.half(), "x")
    with pytest.raises(ValueError):
        boa_hip._bytes(torch.zeros((2, 3)), "tokens", 0)


def test_sizes_beyond_32_bits_are_refused():
    """What ctypes would cut to 32 bits, to sizes that are in range."""
    far = 2 ** 32
    for f, good in ((boa_hip.embed_grad_work_bytes, (1, 1, 64)),
                    (boa_hip.selective_scan_saved_floats, (1, 5, 64, 16)),
                    (boa_hip.selective_scan_work_bytes, (1, 5, 64, 16)),
                    (boa_hip.next_byte_loss_work_bytes, (1, 1))):
        f(*good)
        for i in range(len(good)):
            bad = list(good)
            bad[i] += far
            with pytest.raises(ValueError, match="range"):
                f(*bad)
    meta = lambda *s, **k: torch.empty(s, device="meta", **k)  # noqa: E731
    for s in ((1, far + 3), (far + 3, 1)):
        with pytest.raises(ValueError, match="range"):
            boa_hip._bytes(meta(*s, dtype=torch.uint8), "tokens", -1)
    codec = boa_hip.Codec.__new__(boa_hip.Codec)  # no context: the checks before the call
    codec.h, codec.device = None, -1
    for lanes, T, ch, n in ((1, far + 5, 64, 16), (1, 5, far + 64, 16), (1, 5, 64, far + 16)):
        rows, bc, a = meta(lanes, T, ch), meta(lanes, T, n), meta(ch, n)
        with pytest.raises(ValueError, match="range"):
            codec._scan_args(rows, rows, rows, bc, bc, a, meta(ch), meta(ch), None, None)
