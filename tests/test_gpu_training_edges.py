"""The training operators beside infinities and NaN, on the GPU: what a row, a
lane or a state that is not finite may reach, and what it may not."""
import math

import pytest
import torch

import boa_hip
from test_gpu_training import BF16, F32, codec, dev, work  # noqa: F401

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
