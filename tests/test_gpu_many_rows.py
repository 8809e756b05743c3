"""Norm, its gradient and the 8-bit product at sizes at which blocks go on from
row to row and from tile to tile."""
import pytest
import torch

import boa_hip
from test_gpu_training import BF16, F32, codec, work  # noqa: F401
from training_ref import U

pytestmark = pytest.mark.gpu


# more tiles of 128 x 128 than the small kernel takes, and K of every count of
# 64s that has a kernel of its own, beyond 512, and in odd rows; from 4096 tiles on
# a block takes several of a row
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,n,k,pad", [
    (1300, 1024, 64, 0), (1300, 1030, 128, 0), (2000, 777, 192, 0), (1300, 1024, 320, 16),
    (1500, 1025, 384, 0), (1300, 1030, 448, 0), (1300, 1024, 1024, 0), (1290, 1030, 1008, 0),
    (1300, 1025, 528, 16), (1300, 1024, 513, 0), (2600, 600, 1000, 3), (1300, 1030, 63, 0),
    (1300, 1025, 300, 1), (1400, 1030, 400, 3), (1300, 1025, 509, 1), (1300, 1024, 1001, 0),
    (33000, 2050, 64, 0), (33000, 2064, 600, 8), (33001, 2050, 512, 0), (70001, 2050, 131, 0),
    (131100, 2050, 80, 0), (4500, 16390, 192, 0)])
def test_product(codec, rows, n, k, pad, dtype):  # noqa: F811
    g = torch.Generator("cuda").manual_seed(rows + n + k)
    r8 = lambda *s: torch.randint(-127, 128, s, generator=g, device="cuda", dtype=torch.int8)  # noqa: E731
    x = r8(1, rows, k + pad)[..., pad:]
    w, packed = r8(n, k), work(boa_hip.int8_pack_bytes(n, k))
    sx, sw = (torch.rand(s, generator=g, device="cuda") for s in ((1, rows), (n,)))
    bias = torch.randn((n,), generator=g, device="cuda") * 100
    out = torch.zeros((1, rows, n), dtype=dtype, device="cuda")
    codec.int8_pack(w, packed)
    codec.int8_matmul(x, sx, packed, sw, out, d_bias=bias)
    wt = w.float().t().contiguous()
    for at in range(0, rows, 16384):
        part = slice(at, at + 16384)
        # 1024 x 127 x 127 < 2^24: fp32 holds every sum
        acc = x[0, part].float() @ wt
        want = acc * (sx[0, part, None] * sw) + bias
        assert torch.equal(out[0, part], want.to(dtype)), at


ROWS = [(33000, 64), (70003, 50), (40000, 128), (9001, 256), (8500, 511), (4500, 1024), (5000, 700),
        (2500, 4096), (2100, 2000), (2300, 8190)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", ROWS)
def test_norm(codec, rows, width, dtype):  # noqa: F811
    g = torch.Generator("cuda").manual_seed(rows + width)
    x = torch.randn((1, rows, width), generator=g, device="cuda").to(dtype)
    w = 1 + 0.2 * torch.randn((width,), generator=g, device="cuda")
    out, q = torch.zeros_like(x), torch.zeros(x.shape, dtype=torch.int8, device="cuda")
    s8 = torch.zeros((1, rows), device="cuda")
    codec.rms_norm(x, out, d_weight=w, d_out8=q, d_scale8=s8, eps=1e-5)
    t = x.double() * w.double()
    r = 1 / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-5)
    # r: half the sum's relative error, root, quotient, eps; then two products
    limit = ((width + 1) / 2 + 8) * U + (2.0 ** -8 if dtype == BF16 else 0)
    assert ((out.double() - t * r).abs() <= (t * r).abs() * limit + 2.0 ** -126).all()
    top = t.abs().amax(-1, keepdim=True)
    assert torch.equal(q, torch.round(t * 127 / top).to(torch.int8))
    scale = (top * r / 127)[..., 0]
    assert ((s8.double() - scale).abs() <= scale * ((width + 1) / 2 + 8) * U).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", ROWS)
def test_norm_grad(codec, rows, width, dtype):  # noqa: F811
    g = torch.Generator("cuda").manual_seed(rows + width)
    h, dy = (torch.randn((1, rows, width), generator=g, device="cuda").to(dtype) for _ in range(2))
    w = 1 + 0.2 * torch.randn((width,), generator=g, device="cuda")
    dx, dw = torch.zeros_like(h), torch.zeros((width,), device="cuda")
    codec.rms_norm_grad(h, dy, dx, work(boa_hip.rms_norm_grad_work_bytes(1, rows, width)),
                        d_weight=w, d_dweight=dw, eps=1e-5)
    hd, wdy = h.double(), w.double() * dy.double()
    r = 1 / torch.sqrt((hd ** 2).mean(-1, keepdim=True) + 1e-5)
    n, rel = hd * r, ((width + 1) / 2 + 8) * U
    m = (n * wdy).mean(-1, keepdim=True)
    want = r * (wdy - n * m)
    size = r * (wdy.abs() + 2 * n.abs() * (n * wdy).abs().mean(-1, keepdim=True))
    limit = size * (rel * 2 + (width + 8) * U) + (2.0 ** -8 * want.abs() if dtype == BF16 else 0)
    assert ((dx.double() - want).abs() <= limit * 1.01 + 2.0 ** -126).all()
    # a term's n, its product; at most 20 rows one after the other, 16 groups of a
    # block; the blocks in 64 bits: less than a row's share in 70,003 of them
    terms = (dy.double() * n).abs().sum((0, 1))
    assert ((dw.double() - (dy.double() * n).sum((0, 1))).abs() <= terms * (rel + 40 * U)).all()
