"""The choice of a byte on the GPU against its 64-bit form: the same bytes."""
import math

import pytest
import torch

import boa_hip
from test_gpu_training import BF16, F32, codec, dev, lens_of, place, work  # noqa: F401
import training_ref as ref

pytestmark = pytest.mark.gpu


def choose(x, u, temp, k, p, m):
    """One row: (byte, log of its share), from the definition in 64 bits."""
    x = x.double()
    if not x.isfinite().any() or x.isnan().any() or (x == math.inf).any():
        return 0, math.nan
    order = sorted(range(256), key=lambda i: (-x[i].item(), i))
    w = torch.exp((x - x.max()) / (temp if temp > 0 else 1.0))
    ranked = [w[i].item() for i in order]
    n = 256 if k < 1 else min(256, math.ceil(k))
    if temp <= 0:
        n = 1
    kept = ranked[:n]
    if p < 1:
        total, run, cut = sum(kept), 0.0, len(kept)
        for i, v in enumerate(kept):
            if i and run >= p * total:
                cut = i
                break
            run += v
        kept = kept[:cut]
    kept = [v for i, v in enumerate(kept) if i == 0 or v >= m]
    chosen = sorted(order[:len(kept)])
    total, run = sum(kept), 0.0
    for b in chosen:
        run += w[b].item()
        if run > u * total and w[b] > 0:
            return b, math.log(w[b].item() / total)
    return chosen[-1], math.log(w[chosen[-1]].item() / total)


HOW = [(1.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.02), (0.0, 5, 0.5, 0.0), (2.5, 1, 1.0, 0.0),
       (1.3, 0, 0.3, 0.0), (1.0, 0, 0.0, 0.0), (0.9, 0, 1.0, 0.3), (0.1, 256, 0.99, 1.0),
       (5.0, 3.5, 2.0, -1.0), (1.0, 1000, 1.5, 0.0), (1.0, 0, 1.0, 1.5), (3.0, 200, 0.999, 1e-3)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lanes,T,layout,kind,data", [
    (1, 1, "dense", "full", "plain"), (7, 1, "wide", "ragged", "masked"),
    (5, 13, "odd", "ragged", "plain"), (3, 9, "time", "ragged", "ties"),
    (10, 6, "dense", "full", "masked"), (4, 5, "dense", "full", "one")])
def test_sample(codec, lanes, T, layout, kind, data, dtype):  # noqa: F811
    g = torch.Generator().manual_seed(lanes + T)
    x = torch.randn((lanes, T, 256), generator=g) * 3
    if data == "ties":
        x = torch.round(x)
    elif data == "masked":
        x[..., torch.randperm(256, generator=g)[:100]] = -math.inf
    elif data == "one":  # all but one byte ruled out
        keep = torch.randint(0, 256, (lanes, T, 1), generator=g)
        x = torch.full_like(x, -math.inf).scatter(-1, keep, 1.0)
    x = x.to(dtype)
    bias = torch.randn((256,), generator=g) if data != "ties" else None
    u = torch.rand((lanes, T), generator=g)
    u[0, 0] = 0.0
    u[-1, -1] = 1 - 2.0 ** -24
    lens = lens_of(kind, lanes, T, g)
    live = ref.mask(lens, lanes, T)
    y = x.double() + (bias.double() if bias is not None else 0)
    each = torch.tensor([HOW[i % len(HOW)] for i in range(lanes)])
    for how in [each] + HOW[:4]:
        out = torch.full((lanes, T + 3), 99, dtype=torch.uint8, device="cuda")[:, :T]
        logp = torch.full((lanes, T), 7.5, device="cuda")
        args = dict(d_params=dev(each)) if how is each else dict(
            zip(("temperature", "top_k", "top_p", "min_p"), how))
        codec.sample_bytes(place(x, layout), dev(u), out, d_bias=dev(bias), d_logp=logp,
                           d_lens=dev(lens), **args)
        for l in range(lanes):
            h = each[l].tolist() if how is each else how
            h = [float(torch.tensor(v, dtype=F32)) for v in h]
            for t in range(T):
                if not live[l, t]:
                    assert out[l, t] == 99 and logp[l, t] == 7.5
                    continue
                b, lp = choose(y[l, t], u[l, t].item(), *h)
                assert out[l, t].item() == b, (l, t, h)
                # one rounding to fp32, and 64-bit arithmetic far below it
                assert abs(logp[l, t].item() - lp) <= 2.0 ** -23 * abs(lp) + 1e-12


def test_rows_without_a_choice(codec):  # noqa: F811
    x = torch.zeros((4, 1, 256))
    x[0] = -math.inf
    x[1, 0, 3] = math.nan
    x[2, 0, 200] = math.inf
    x[3, 0, 77] = 80.0
    out, logp = torch.full((4, 1), 9, dtype=torch.uint8, device="cuda"), torch.zeros((4, 1), device="cuda")
    codec.sample_bytes(dev(x), torch.full((4, 1), 0.5, device="cuda"), out, d_logp=logp)
    assert out[:, 0].tolist() == [0, 0, 0, 77]
    assert logp[:3].isnan().all() and logp[3] == 0


def test_numbers_outside_the_unit(codec):  # noqa: F811
    x = torch.randn((1, 1, 256), generator=torch.Generator().manual_seed(0)).expand(4, 1, 256).contiguous()
    x[..., 200:] = -math.inf
    out = torch.zeros((4, 1), dtype=torch.uint8, device="cuda")
    codec.sample_bytes(dev(x), torch.tensor([[-1.0], [1.0], [5.0], [math.nan]], device="cuda"), out)
    assert out[:, 0].tolist() == [0, 199, 199, 0]


def test_a_share_of_each(codec):  # noqa: F811
    """Equally spaced numbers give every byte its share of them, to within one."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn((1, 1, 256), generator=g)
    n = 20000
    u = (torch.arange(n).view(1, n) + 0.5) / n
    out = torch.zeros((1, n), dtype=torch.uint8, device="cuda")
    codec.sample_bytes(dev(x).expand(1, n, 256), dev(u), out)
    share = torch.bincount(out[0].long().cpu(), minlength=256).double()
    assert (share - torch.softmax(x[0, 0].double(), -1) * n).abs().max() <= 1.01


@pytest.mark.parametrize("how", [dict(), dict(top_k=30), dict(top_p=0.5), dict(top_k=30, top_p=0.5)])
def test_an_infinite_temperature(codec, how):  # noqa: F811
    """Every byte that is not ruled out is as likely as the others."""
    n = 600
    x = torch.full((1, n, 256), -math.inf)
    x[..., 100:200] = torch.randn((100,), generator=torch.Generator().manual_seed(4))
    u = (torch.arange(n, dtype=torch.float64) / n).float().view(1, n)
    for settings in (dict(temperature=math.inf, **how),
                     dict(d_params=torch.tensor([[math.inf, how.get("top_k", 0), how.get("top_p", 1.0),
                                                  0.0]], device="cuda"))):
        out = torch.full((1, n), 7, dtype=torch.uint8, device="cuda")
        logp = torch.full((1, n), 7.5, device="cuda")
        codec.sample_bytes(dev(x), dev(u), out, d_logp=logp, **settings)
        kept = (30 if "top_k" in how else 100) * (0.5 if "top_p" in how else 1)
        ranked = torch.sort(x[0, 0], descending=True)[1][:int(kept)].sort()[0]
        share = torch.arange(1, len(ranked) + 1, dtype=torch.float64)
        want = ranked[(share <= u[0].double()[:, None] * kept).sum(1)]
        assert torch.equal(out[0].cpu().long(), want)
        # a logarithm's value, rounded once
        assert (logp.cpu().double() + math.log(kept)).abs().max() <= 2.0 ** -24 * math.log(kept)


def test_capture(codec):  # noqa: F811
    x, u = torch.randn((9, 1, 256), device="cuda"), torch.rand((9, 1), device="cuda")
    out, logp = torch.zeros((9, 1), dtype=torch.uint8, device="cuda"), torch.zeros((9, 1), device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        codec.set_stream(torch.cuda.current_stream().cuda_stream)
        codec.sample_bytes(x, u, out, d_logp=logp, top_p=0.8)
    codec.set_stream(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        x.normal_()
        u.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), logp.clone()
        codec.sample_bytes(x, u, out, d_logp=logp, top_p=0.8)
        torch.cuda.synchronize()
        assert torch.equal(got[0], out) and torch.equal(got[1], logp)


def test_refusals(codec):  # noqa: F811
    x, u = torch.zeros((2, 3, 256), device="cuda"), torch.zeros((2, 3), device="cuda")
    out = torch.zeros((2, 3), dtype=torch.uint8, device="cuda")
    for call, why in [
            (lambda: codec.sample_bytes(x[..., :255], u, out), "logits"),
            (lambda: codec.sample_bytes(x, u[:, :2], out), "uniform"),
            (lambda: codec.sample_bytes(x, u, out[:, :2]), "logits"),
            (lambda: codec.sample_bytes(x, u, out.float()), "uint8"),
            (lambda: codec.sample_bytes(x, u, out[:1].expand(2, 3)), "overlap"),
            (lambda: codec.sample_bytes(x, u, out, d_logp=u), "input"),
            (lambda: codec.sample_bytes(x, u, out, temperature=math.nan), "NaN"),
            (lambda: codec.sample_bytes(x, u, out, d_params=torch.zeros((3, 4), device="cuda")), "params"),
            (lambda: codec.sample_bytes(x.cpu(), u, out), "cpu")]:
        with pytest.raises((boa_hip.BoaError, ValueError), match=why):
            call()
