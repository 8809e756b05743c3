"""Rows in 8 bits as wide as the product takes them."""
import pytest
import torch

import boa_hip
import training_ref as ref
from test_gpu_training import BF16, F32, SKIP, codec, dev, empty, lens_of, place, work  # noqa: F401
from training_ref import U, V

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width,layout", [(8193, "odd"), (8200, "dense"), (12000, "wide"),
                                          (16384, "dense"), (16383, "odd"), (16384, "time")])
def test_rows_and_their_product(codec, width, layout, dtype):  # noqa: F811
    lanes, T, n = 3, 7, 33
    g = torch.Generator().manual_seed(width)
    x = torch.randn((lanes, T, width), generator=g).to(dtype)
    x[0, 1] = 0
    lens = lens_of("ragged", lanes, T, g)
    live = ref.mask(lens, lanes, T)
    q = torch.full((lanes, T, width), 99, dtype=torch.int8, device="cuda")
    s8 = torch.full((lanes, T), SKIP, device="cuda")
    codec.int8_rows(place(x, layout), q, s8, d_lens=dev(lens))
    top = x.double().abs().amax(-1, keepdim=True)
    want = torch.round(x.double() * 127 / top.clamp_min(1e-300)).to(torch.int8)
    assert torch.equal(q.cpu()[live], want[live])
    off = (s8.cpu().double() - top[..., 0] / 127).abs()[live]
    assert (off <= U * top[..., 0][live] / 127).all()
    assert (q.cpu()[~live] == 99).all() and (s8.cpu()[~live] == SKIP).all()
    # weights come from rows, too: one lane, a row for each channel
    wf = torch.randn((1, n, width), generator=g).to(dtype)
    w8 = torch.zeros((1, n, width), dtype=torch.int8, device="cuda")
    ws, packed = torch.zeros((1, n), device="cuda"), work(boa_hip.int8_pack_bytes(n, width))
    codec.int8_rows(dev(wf), w8, ws)
    codec.int8_pack(w8[0], packed)
    out = empty(lanes, T, n, F32, "dense")
    codec.int8_matmul(q, s8, packed, ws[0], out, d_lens=dev(lens))
    acc = want.double() @ w8[0].cpu().double().t()
    y = V(acc, U * acc.abs()) * (V(s8.cpu().double()[..., None].expand_as(acc))
                                 * V(ws[0].cpu().double().expand_as(acc)))
    ref.check("out", out.cpu()[live], y[live])


def test_refusals(codec):  # noqa: F811
    x, q = torch.zeros((1, 1, 16385), device="cuda"), torch.zeros((1, 1, 16385), dtype=torch.int8,
                                                                 device="cuda")
    with pytest.raises(boa_hip.BoaError, match="16384"):
        codec.int8_rows(x, q, torch.zeros((1, 1), device="cuda"))
    with pytest.raises(boa_hip.BoaError, match="8192"):
        codec.rms_norm(x[..., :8193], d_out8=q[..., :8193], d_scale8=torch.zeros((1, 1), device="cuda"))
