"""Norm, its gradient and its rows in 8 bits over all that fp32 and bfloat16
hold: rows whose squares leave fp32's range, at either end, against the 64-bit
forms whose error bounds are the tolerances."""
import pytest
import torch

import boa_hip
import training_ref as ref
from test_gpu_norm_int8 import lift, root
from test_gpu_training import BF16, F32, codec, dev, place, work  # noqa: F401
from training_ref import U, V

pytestmark = pytest.mark.gpu

# powers of two that rows are multiplied with; neighbours share a wave
SIZES = [-120, 0, -90, 124, -58, 100, -55, 66, -50, 51, -64, 48, 0, -100]
WIDTHS = [(64, "dense"), (80, "odd"), (512, "wide"), (1000, "dense"), (4096, "dense"), (8191, "odd")]


def rows(width, dtype, seed, even=True):
    g = torch.Generator().manual_seed(seed)
    size = torch.tensor([2.0 ** e for e in SIZES], dtype=torch.float64)[None, :, None]
    x = torch.randn((1, len(SIZES), width), generator=g).double()
    if not even:  # a few elements far above the others
        x = torch.where(torch.rand(x.shape, generator=g) < 0.9, x * 2.0 ** -20, x)
    return (x * size).to(dtype), g


@pytest.mark.parametrize("even", [True, False])
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -20, 2.0 ** -116])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width,layout", WIDTHS)
def test_norm(codec, width, layout, dtype, eps, even):  # noqa: F811
    x, g = rows(width, dtype, width, even)
    w = 1 + 0.3 * torch.randn((width,), generator=g)
    out, q = place(torch.zeros_like(x), layout), torch.zeros(x.shape, dtype=torch.int8, device="cuda")
    s8 = torch.zeros(x.shape[:2], device="cuda")
    codec.rms_norm(place(x, layout), out, d_weight=dev(w), d_out8=q, d_scale8=s8, eps=eps)
    h = V(x.double())
    rn = lift(root(h, eps), h.val)
    ref.check("out", out, h * rn * V(w.double().expand_as(h.val)), dtype)
    t = h.val * w.double()
    top = t.abs().amax(-1, keepdim=True)
    assert torch.equal(q.cpu(), torch.round(t * 127 / top).to(torch.int8))
    scale = (top * rn.val[..., :1] / 127)[..., 0]
    # what is less than the least normal number has steps of 2^-149
    limit = scale * (rn.err / rn.val)[..., 0] + 3 * U * scale + 2.0 ** -149
    assert ((s8.cpu().double() - scale).abs() <= limit).all()


@pytest.mark.parametrize("size", [0, -60, -100])
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -20, 2.0 ** -116])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width,layout", WIDTHS)
def test_norm_grad(codec, width, layout, dtype, eps, size):  # noqa: F811
    x, g = rows(width, dtype, width)
    dy = (torch.randn(x.shape, generator=g) * 2.0 ** size).to(dtype)
    w = 1 + 0.3 * torch.randn((width,), generator=g)
    dx, dw = place(torch.zeros_like(x), layout), torch.zeros((width,), device="cuda")
    codec.rms_norm_grad(place(x, layout), place(dy, layout), dx,
                        work(boa_hip.rms_norm_grad_work_bytes(*x.shape)), d_weight=dev(w),
                        d_dweight=dw, eps=eps)
    hv = V(x.double())
    rn = lift(root(hv, eps), hv.val)
    n, wdy = hv * rn, V(w.double().expand_as(hv.val)) * V(dy.double())
    # the mean of n w dy, whichever of its factors comes first
    c = (n * wdy).sum(-1)
    m = lift(V(c.val / width, c.err / width + U * c.val.abs() / width)[..., None], hv.val)
    ref.check("dx", dx, rn * (wdy - n * m), dtype)
    ref.check("dweight", dw, (V(dy.double()) * n).sum((0, 1)))


@pytest.mark.parametrize("width", [64, 1000])
def test_a_residual_beside_large_rows(codec, width):  # noqa: F811
    """The sum as it is stored, and its norm."""
    x, g = rows(width, F32, 3)
    res = -x * 0.5
    out, total = torch.zeros_like(x).cuda(), torch.zeros_like(x).cuda()
    codec.rms_norm(dev(x), out, d_residual=dev(res), d_sum=total, eps=0.0)
    h = V(x.double()) + V(res.double())
    ref.check("sum", total, h, F32)
    ref.check("out", out, h * lift(root(h, 0.0), h.val), F32)


def test_rows_without_gradients(codec):  # noqa: F811
    """Nothing comes back where nothing came in, beside rows where it did."""
    g = torch.Generator().manual_seed(1)
    x, dy = (torch.randn((4, 9, 256), generator=g) for _ in range(2))
    dy[1] = 0
    dy[2, ::2] = 0
    dx = torch.ones_like(x).cuda()
    codec.rms_norm_grad(dev(x), dev(dy), dx, eps=1e-6)
    assert (dx[1] == 0).all() and (dx[2, ::2] == 0).all()
    one = torch.ones((1, 1, 256), device="cuda")
    codec.rms_norm_grad(dev(x[2:3, 1:2]), dev(dy[2:3, 1:2]), one, eps=1e-6)
    assert torch.equal(one[0, 0], dx[2, 1])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", [64, 256, 4096])
def test_rows_do_not_matter_to_each_other(codec, width, dtype):  # noqa: F811
    """A row's bits are the same alone as beside rows of any size."""
    x, g = rows(width, dtype, 7)
    x, dy = dev(x), dev(torch.randn(x.shape, generator=g).to(dtype))

    def run(x, dy):
        out, dx, q = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x, dtype=torch.int8)
        s8 = torch.zeros(x.shape[:2], device="cuda")
        codec.rms_norm(x, out, d_out8=q, d_scale8=s8, eps=2.0 ** -116)
        codec.rms_norm_grad(x, dy, dx, eps=2.0 ** -116)
        return out, dx, q, s8

    whole = run(x, dy)
    for i in range(len(SIZES)):
        for a, b in zip(run(x[:, i:i + 1].clone(), dy[:, i:i + 1].clone()), whole):
            assert torch.equal(a, b[:, i:i + 1])
