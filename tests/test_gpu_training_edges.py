"""The training operators beside infinities and NaN, on the GPU: what a row, a
lane or a state that is not finite may reach, and what it may not."""
import math

import pytest
import torch

import boa_hip
import training_ref as ref
from test_gpu_training import BF16, F32, codec, dev, run_scan, scan_inputs, work  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradient_of_a_nan_among_ruled_out_bytes(codec, dtype):  # noqa: F811
    """A row of -inf and a NaN has a gradient of NaN like any row with a NaN; a
    row of nothing but -inf and one past its lane's length keep zero."""
    x = torch.full((2, 128, 256), -math.inf)
    x[0, torch.arange(128), 2 * torch.arange(128)] = math.nan
    x[1, 1] = 0.0
    x[1, 100:] = math.nan  # past the length
    tgt = torch.full((2, 128), 9, dtype=torch.uint8)
    lens = torch.tensor([128, 100], dtype=torch.int32)
    loss, dx = torch.zeros((2, 128), device="cuda"), torch.ones((2, 128, 256), dtype=dtype,
                                                                device="cuda")
    dbias = torch.zeros(256, device="cuda")
    w = work(boa_hip.next_byte_loss_work_bytes(2, 128))
    codec.next_byte_loss(x.to(dtype).cuda(), dev(tgt), loss, w, d_dlogits=dx, d_dbias=dbias,
                         d_lens=dev(lens))
    assert loss[0].isnan().all() and dx[0].isnan().all() and dbias.isnan().all()
    assert (dx[1, 0] == 0).all() and (dx[1, 2:] == 0).all()
    codec.next_byte_loss(x[1:].to(dtype).cuda(), dev(tgt[1:]), loss[1:], w, d_dlogits=dx[1:],
                         d_dbias=dbias, d_lens=dev(lens[1:]))
    assert dbias.isfinite().all()


def _lanes_alone(s, lens):
    """dA of the lanes one by one, each as long as it is, summed: no position
    past a lane's end takes part in the formula at all."""
    total = None
    for i, n in enumerate(lens.tolist()):
        one = {k: v if v.shape[0] != len(lens) else v[i:i + 1] for k, v in s.items()}
        one = {k: v[:, :n] if v.dim() == 3 and k in ("u", "delta", "z", "B", "C", "dout") else v
               for k, v in one.items()}
        live = ref.mask(None, 1, n)
        dA = ref.scan_grad(one, live, ref.scan(one, live)[2])["dA"]
        total = dA if total is None else total + dA
    return total


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [16, 32])
@pytest.mark.parametrize("ch", [64, 70])
def test_decay_gradient_beside_infinite_states(codec, ch, n, dtype):  # noqa: F811
    """dA is the sum over the lanes' positions: an infinite last state, or an
    infinite gradient of it, meets no position past the lane's end."""
    s, _ = scan_inputs(3, 45, ch, n, dtype, "full")
    lens = torch.tensor([21, 17, 35], dtype=torch.int32)
    s["u"][0, 20, 5] = math.inf   # the lane's last position: only its last state is infinite
    s["u"][2, 34, 60] = -math.inf
    # one channel in which every state and decay is positive, so that the
    # infinite gradient of lane 1 makes dA +inf, and not NaN
    s["u"][:, :, 9] = s["u"][:, :, 9].abs()
    s["B"][:] = s["B"].abs()
    s["state_in"][:] = s["state_in"].abs()
    s["dstate_out"][1, 9, 2] = math.inf
    got, _ = run_scan(codec, s, lens, "dense")
    want = _lanes_alone(s, lens)
    dA = got["dA"].cpu()
    assert dA[9, 2] == math.inf
    finite = torch.ones((ch, n), dtype=torch.bool)
    finite[9, 2] = False
    ref.check("dA", dA[finite], want[finite])


@pytest.mark.parametrize("T", [300, 700])
def test_growing_states_that_are_zero(codec, T):  # noqa: F811
    """A > 0 over segments whose decay overflows: a state (and a gradient) of
    zero stays zero until something enters it."""
    s, _ = scan_inputs(1, T, 64, 16, F32, "full", state=False)
    s["A"] = s["A"].abs().clamp(8, 12)
    s["delta"][:], s["delta_bias"][:] = 0.0, 0.0  # delta = log 2: e^(A delta 16) > 1e38
    s["u"][:, :-6] = 0.0     # the state is zero until six positions before the end
    s["dout"][:, 6:] = 0.0   # and its gradient down to the sixth position
    got, live = run_scan(codec, s, None, "dense")
    out, state, kept = ref.scan(s, live)
    ref.check("out", got["out"], out)
    ref.check("state_out", got["state_out"], state)
    for k, want in ref.scan_grad(s, live, kept).items():
        ref.check(k, got[k], want)


@pytest.mark.parametrize("T", [30, 600])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_segments_whose_decay_leaves_the_range(codec, sign, T):  # noqa: F811
    """A segment's decay may overflow (underflow) where the state that goes
    through it does not."""
    s, _ = scan_inputs(1, T, 64, 16, F32, "full")
    size = 2.0 ** 83                                # a segment of 16 positions: 2^(16 * 9) = 2^144
    s["A"] = torch.full((64, 16), sign * 9.0)
    s["delta"][:], s["delta_bias"][:] = -200.0, 0.0   # delta = 0
    s["delta"][:, :16] = 0.0                          # delta = log 2, in the first segment only
    s["u"][:] = 0.0
    s["state_in"] = s["state_in"].abs().clamp(0.5, 1.5) * size ** -sign
    s["dstate_out"] = s["dstate_out"].abs().clamp(0.5, 1.5) * size ** -sign
    got, live = run_scan(codec, s, None, "dense")
    out, state, kept = ref.scan(s, live)
    # the chain's own roundings: 16 deltas added up, the exponent's three, the
    # two factors' four -- relative to the state, whose exponent is 16 * 9 log 2
    more = ref.U * ((16 + 3) * 16 * 9 * math.log(2) + 4)
    state.err = state.err + more * state.val.abs()
    ref.check("state_out", got["state_out"], state)
    # dout's terms grow by 2^144 on their way to the first position, so where
    # A > 0 dstate_in is out of fp32's range
    want = ref.scan_grad(s, live, kept)["dstate_in"]
    if sign > 0:
        assert (want.val.abs() > torch.finfo(F32).max).all()
        assert torch.equal(got["dstate_in"].cpu().double(), want.val.sign() * math.inf)
    else:
        want.err = want.err + more * want.val.abs()
        ref.check("dstate_in", got["dstate_in"], want)
    # and without them it is dstate_out times the decay
    s["dout"][:] = 0.0
    got, _ = run_scan(codec, s, None, "dense")
    want = ref.scan_grad(s, live, kept | {"w": dict(kept["w"], dout=ref.V(s["dout"].double()))})
    want = want["dstate_in"]
    want.err = want.err + more * want.val.abs()
    ref.check("dstate_in", got["dstate_in"], want)
