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
