"""Norm, rows in 8 bits and their product on the GPU against 64-bit forms whose
error bounds are the tolerances."""
import math

import pytest
import torch

import boa_hip
import training_ref as ref
from training_ref import U, V
from test_gpu_training import (BF16, F32, SKIP, codec, dev, empty, lens_of, place,  # noqa: F401
                               untouched, work, zeroed)

pytestmark = pytest.mark.gpu

ROWS = [(1, 1, 1, "dense", "full"), (3, 1, 64, "dense", "full"), (2, 5, 80, "wide", "ragged"),
        (4, 33, 256, "dense", "ragged"), (3, 19, 7, "odd", "ragged"), (2, 65, 512, "time", "ragged"),
        (5, 9, 513, "odd", "ragged"), (3, 70, 1000, "wide", "ragged"), (2, 7, 4096, "dense", "full"),
        (2, 3, 8192, "dense", "ragged"), (2, 3, 8191, "odd", "full"), (40, 301, 64, "dense", "ragged")]


def root(h, eps):
    """1 / root of the mean square and its bound: the sum's roundings, then its
    root (half of its relative error), quotient and the addition of eps"""
    n = h.val.shape[-1]
    ss = V(h.val * h.val, 2 * h.val.abs() * h.err + U * h.val ** 2).sum(-1)
    m = ss.val / n + eps
    r = 1 / torch.sqrt(m)
    return V(r, r * (ss.err / (n * m) + 6 * U))[..., None]


def lift(v, like):
    return V(v.val.expand_as(like), v.err.expand_as(like))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lanes,T,width,layout,kind", ROWS)
def test_norm(codec, lanes, T, width, layout, kind, dtype):  # noqa: F811
    g = torch.Generator().manual_seed(lanes + T + width)
    r = lambda *n: torch.randn(n, generator=g)  # noqa: E731
    x, res, w = r(lanes, T, width).to(dtype), (2 * r(lanes, T, width)).to(dtype), 1 + 0.3 * r(width)
    lens = lens_of(kind, lanes, T, g)
    live = ref.mask(lens, lanes, T)
    for residual in (res, None):
        held = x.clone()
        held[~live] = math.nan
        out, total = empty(lanes, T, width, dtype, layout), empty(lanes, T, width, dtype, layout)
        q = torch.full((lanes, T, width + 8), 99, dtype=torch.int8, device="cuda")[..., 4:4 + width]
        s8 = torch.full((lanes, T), SKIP, device="cuda")
        codec.rms_norm(place(held, layout, math.nan), out, d_weight=dev(w),
                       d_residual=None if residual is None else place(residual, layout),
                       d_sum=total, d_out8=q, d_scale8=s8, eps=1e-5, d_lens=dev(lens))
        h = V(x.double()) + (V(res.double()) if residual is not None else V(torch.zeros_like(x).double()))
        rn = lift(root(h, 1e-5), h.val)
        y = h * rn * V(w.double().expand_as(h.val))
        ref.check("sum", total.cpu()[live], h[live], dtype)
        ref.check("out", out.cpu()[live], y[live], dtype)
        untouched(out, live, "out"), untouched(total, live, "sum")
        assert (q.cpu()[~live] == 99).all() and (s8.cpu()[~live] == SKIP).all()
        # in 8 bits: whole numbers, of values computed in 64 bits here and there
        t = h.val * w.double()
        top = t.abs().amax(-1, keepdim=True)
        want = torch.round(t * 127 / top)
        assert torch.equal(q.cpu()[live], want[live].to(torch.int8))
        scale = (top * rn.val[..., :1] / 127)[..., 0]
        off = (s8.cpu().double() - scale).abs()[live]
        assert (off <= scale[live] * (rn.err / rn.val)[..., 0][live] + 3 * U * scale[live]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lanes,T,width,layout,kind", ROWS)
def test_norm_grad(codec, lanes, T, width, layout, kind, dtype):  # noqa: F811
    g = torch.Generator().manual_seed(lanes + T + width)
    r = lambda *n: torch.randn(n, generator=g)  # noqa: E731
    h, dy, ds = (r(lanes, T, width).to(dtype) for _ in range(3))
    w = 1 + 0.3 * r(width)
    lens = lens_of(kind, lanes, T, g)
    live = ref.mask(lens, lanes, T)
    held = h.clone()
    held[~live] = math.nan
    dx, dw = empty(lanes, T, width, dtype, layout), torch.full((width,), SKIP, device="cuda")
    wk = work(boa_hip.rms_norm_grad_work_bytes(lanes, T, width))
    args = (place(held, layout, math.nan), place(dy, layout), dx, wk)
    codec.rms_norm_grad(*args, d_weight=dev(w), d_dsum=place(ds, layout), d_dweight=dw, eps=1e-5,
                        d_lens=dev(lens))
    hv, on = V(h.double()), live[..., None].double()
    rn = lift(root(hv, 1e-5), hv.val)
    n, wdy = hv * rn, V(w.double().expand_as(hv.val)) * V(dy.double())
    # c = sum of h w dy; its mean times r
    c = (hv * wdy).sum(-1)
    m = lift(V(c.val / width, c.err / width + U * c.val.abs() / width)[..., None], hv.val) * rn
    want = rn * (wdy - n * m) + V(ds.double())
    ref.check("dx", dx.cpu()[live], want[live], dtype)
    zeroed(dx, live, "dx")
    p = V(dy.double()) * n
    ref.check("dweight", dw, V(p.val * on, p.err * on).sum((0, 1)))
    # without a weight, the residual's gradient or the weight's; into dout itself
    into = place(dy, layout)
    codec.rms_norm_grad(place(h, layout), into, into, eps=1e-5, d_lens=dev(lens))
    c = (hv * V(dy.double())).sum(-1)
    m = lift(V(c.val / width, c.err / width + U * c.val.abs() / width)[..., None], hv.val) * rn
    want = rn * (V(dy.double()) - n * m)
    ref.check("dx", into.cpu()[live], want[live], dtype)
    zeroed(into, live, "dx")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sum_in_place(codec, dtype):  # noqa: F811
    g = torch.Generator().manual_seed(1)
    x, res = (torch.randn((3, 11, 256), generator=g).to(dtype).cuda() for _ in range(2))
    outs = []
    for into in ("new", "x", "res"):
        a, b = x.clone(), res.clone()
        total = {"new": torch.empty_like(a), "x": a, "res": b}[into]
        out = torch.empty_like(a)
        codec.rms_norm(a, out, d_residual=b, d_sum=total)
        outs.append((out, total))
    assert all(torch.equal(o, outs[0][0]) and torch.equal(t, outs[0][1]) for o, t in outs)


def test_rows_that_are_zero_or_not_finite(codec):  # noqa: F811
    x = torch.ones((1, 5, 64))
    x[0, 1] = 0
    x[0, 2, 7] = math.nan
    x[0, 3, 9] = math.inf
    q, s = torch.zeros((1, 5, 64), dtype=torch.int8, device="cuda"), torch.zeros((1, 5), device="cuda")
    for norm in (True, False):
        if norm:
            codec.rms_norm(dev(x), d_out8=q, d_scale8=s)
        else:
            codec.int8_rows(dev(x), q, s)
        values = q.float() * s[..., None]
        assert values[0, 0].isfinite().all() and values[0, 4].isfinite().all()
        assert (q[0, 1] == 0).all() and s[0, 1] == 0
        assert not values[0, 2].isfinite().any() and not values[0, 3].isfinite().any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lanes,T,width,layout,kind", ROWS)
def test_int8_rows(codec, lanes, T, width, layout, kind, dtype):  # noqa: F811
    g = torch.Generator().manual_seed(lanes + T + width)
    x = torch.randn((lanes, T, width), generator=g).to(dtype)
    lens = lens_of(kind, lanes, T, g)
    live = ref.mask(lens, lanes, T)
    q = torch.full((lanes, T, width), 99, dtype=torch.int8, device="cuda")
    s8 = torch.full((lanes, T), SKIP, device="cuda")
    codec.int8_rows(place(x, layout), q, s8, d_lens=dev(lens))
    top = x.double().abs().amax(-1, keepdim=True)
    assert torch.equal(q.cpu()[live], torch.round(x.double() * 127 / top)[live].to(torch.int8))
    off = (s8.cpu().double() - top[..., 0] / 127).abs()[live]
    assert (off <= U * top[..., 0][live] / 127).all()  # 127 / 127 of 64 bits, rounded once
    assert (q.cpu()[~live] == 99).all() and (s8.cpu()[~live] == SKIP).all()


PRODUCTS = [(1, 1, 1, 1, "dense", "full"), (64, 1, 256, 1032, "dense", "full"),
            (3, 1, 80, 324, "wide", "full"), (2, 33, 64, 260, "dense", "ragged"),
            (3, 19, 7, 33, "odd", "ragged"), (5, 130, 513, 100, "time", "ragged"),
            (2, 70, 1000, 129, "wide", "ragged"), (1, 5, 16384, 40, "dense", "full"),
            (70, 130, 512, 640, "dense", "ragged"), (64, 65, 130, 1000, "odd", "ragged"),
            (33, 257, 96, 1025, "dense", "ragged")]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lanes,T,k,n,layout,kind", PRODUCTS)
def test_int8_matmul(codec, lanes, T, k, n, layout, kind, dtype):  # noqa: F811
    g = torch.Generator().manual_seed(lanes + T + k + n)
    x = torch.randint(-128, 128, (lanes, T, k), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    sx, sw = torch.rand((lanes, T), generator=g), torch.rand((n,), generator=g)
    bias = torch.randn((n,), generator=g) * 100
    lens = lens_of(kind, lanes, T, g)
    live = ref.mask(lens, lanes, T)
    packed = torch.full((boa_hip.int8_pack_bytes(n, k),), 0xFF, dtype=torch.uint8, device="cuda")
    codec.int8_pack(dev(w), packed)
    acc = (x.view(-1, k).double() @ w.double().t()).view(lanes, T, n)  # exact
    for b in (bias, None):
        out = empty(lanes, T, n, dtype, layout)
        codec.int8_matmul(place(x, layout, 99), dev(sx), packed, dev(sw), out, d_bias=dev(b),
                          d_lens=dev(lens))
        # the sum may have more digits than fp32: one rounding of its own
        y = V(acc, U * acc.abs()) * (V(sx.double()[..., None].expand_as(acc))
                                     * V(sw.double().expand_as(acc)))
        if b is not None:
            y = y + V(b.double().expand_as(acc))
        ref.check("out", out.cpu()[live], y[live], dtype)
        untouched(out, live, "out")


def test_the_batch_does_not_matter(codec):  # noqa: F811
    """A lane's product is the same bits alone and among a thousand."""
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-127, 128, (1000, 40, 256), generator=g, dtype=torch.int8).cuda()
    w = torch.randint(-127, 128, (700, 256), generator=g, dtype=torch.int8).cuda()
    sx, sw = torch.rand((1000, 40), generator=g).cuda(), torch.rand((700,), generator=g).cuda()
    packed = torch.zeros((boa_hip.int8_pack_bytes(700, 256),), dtype=torch.uint8, device="cuda")
    codec.int8_pack(w, packed)
    many = torch.zeros((1000, 40, 700), device="cuda")
    codec.int8_matmul(x, sx, packed, sw, many)
    for lane in (0, 517, 999):
        one = torch.zeros((1, 40, 700), device="cuda")
        codec.int8_matmul(x[lane:lane + 1], sx[lane:lane + 1], packed, sw, one)
        assert torch.equal(one[0], many[lane])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_capture(codec, dtype):  # noqa: F811
    """Norm in both forms, its gradient in place and the product, replayed on new
    values between eager calls."""
    lanes, T, width, n = 5, 37, 256, 130
    new = lambda *s, dt=dtype: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731
    x, res, dy = new(lanes, T, width), new(lanes, T, width), new(lanes, T, width)
    total, out, dx, y = new(lanes, T, width), new(lanes, T, width), new(lanes, T, width), new(lanes, T, n)
    x8, s8 = new(lanes, T, width, dt=torch.int8), new(lanes, T, dt=F32)
    w, dw, ws = torch.ones((width,), device="cuda"), new(width, dt=F32), torch.ones((n,), device="cuda")
    packed = work(boa_hip.int8_pack_bytes(n, width))
    codec.int8_pack(torch.randint(-127, 128, (n, width), dtype=torch.int8, device="cuda"), packed)
    wk = work(boa_hip.rms_norm_grad_work_bytes(lanes, T, width))

    def step():
        codec.rms_norm(x, out, d_weight=w, d_residual=res, d_sum=total, d_out8=x8, d_scale8=s8)
        codec.int8_matmul(x8, s8, packed, ws, y)
        dx.copy_(dy)
        codec.rms_norm_grad(total, dx, dx, wk, d_weight=w, d_dweight=dw)

    results = [total, out, x8, s8, y, dx, dw]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        codec.set_stream(torch.cuda.current_stream().cuda_stream)
        step()
    codec.set_stream(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        for t in (x, res, dy, w):
            t.normal_()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in results]
        for t in results:
            t.zero_()
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, results))
        apart = torch.zeros_like(dx)  # not into dout itself
        dw.zero_()
        codec.rms_norm_grad(total, dy, apart, wk, d_weight=w, d_dweight=dw)
        torch.cuda.synchronize()
        assert torch.equal(apart, dx) and torch.equal(dw, replayed[-1])


def test_refusals(codec):  # noqa: F811
    z = lambda *n, dt=F32: torch.zeros(n, dtype=dt, device="cuda")  # noqa: E731
    x, i8 = z(2, 4, 64), z(2, 4, 64, dt=torch.int8)
    s8, packed = z(2, 4), z(boa_hip.int8_pack_bytes(32, 64), dt=torch.uint8)
    bad = [
        (lambda: codec.rms_norm(x), "no output"),
        (lambda: codec.rms_norm(x, x), "input"),
        (lambda: codec.rms_norm(x, z(2, 4, 64, dt=BF16)), "out"),
        (lambda: codec.rms_norm(x, d_out8=i8), "scale8"),
        (lambda: codec.rms_norm(x, z(2, 4, 64), eps=-1.0), "eps"),
        (lambda: codec.rms_norm(x, z(2, 4, 64), d_weight=z(63)), "weight"),
        (lambda: codec.rms_norm(z(1, 1, 8193), z(1, 1, 8193)), "8192"),
        (lambda: codec.rms_norm_grad(x, x.clone(), x), "input"),
        (lambda: codec.rms_norm_grad(x, x.clone(), z(2, 4, 64), d_dweight=z(64)), "workspace"),
        (lambda: codec.int8_rows(x, z(2, 4, 64), s8), "int8"),
        (lambda: codec.int8_matmul(i8, s8, packed, z(129), z(2, 4, 129)), "packed"),
        (lambda: codec.int8_matmul(i8, s8, packed[:100], z(32), z(2, 4, 32)), "packed"),
        (lambda: codec.int8_matmul(i8, s8, packed, z(32), z(1, 4, 32).expand(2, 4, 32)), "overlap"),
        (lambda: codec.int8_pack(z(32, 20000, dt=torch.int8), packed), "16384|packed"),
    ]
    for call, why in bad:
        with pytest.raises((boa_hip.BoaError, ValueError), match=why):
            call()
    for sizes in [(0, 1, 64), (1, 0, 64), (1, 1, 0), (1, 1, 8193), (70000, 1, 64)]:
        with pytest.raises(ValueError):
            boa_hip.rms_norm_grad_work_bytes(*sizes)
