"""The training operators just past the sizes at which they take another path:
rows stored past the L2s (over 32 MiB), four vectors a thread in the embedding
(from 524,288 vectors), as many blocks as the loss launches at most, more
chunks of the embedding's gradient than fit LDS at once (over 2,097,152 rows),
and every row tensor of the scan with 2^31 elements between its lanes."""
import math

import pytest
import torch

import boa_hip
import training_ref as ref
from test_gpu_training import (BF16, F32, ROWS_IN, SKIP, codec, dev, empty, far, lens_of,  # noqa: F401
                               place, run_scan, scan_inputs, tokens_of, work, zeroed)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lanes,T,width,layout,dtype", [
    (33, 2003, 256, "dense", BF16), (33, 2003, 256, "wide", BF16), (33, 2003, 256, "time", BF16),
    (17, 2003, 256, "dense", F32), (129, 1031, 64, "wide", F32), (9, 2003, 255, "odd", BF16),
    (9, 2003, 255, "odd", F32), (40, 431, 256, "dense", BF16)])
def test_embed_of_many_rows(codec, lanes, T, width, layout, dtype):  # noqa: F811
    """One product and one rounding: the same bits as torch's."""
    g = torch.Generator().manual_seed(lanes + T + width)
    tok, table = tokens_of("any", lanes, T, g), torch.randn((256, width), generator=g).to(dtype)
    lens = lens_of("ragged", lanes, T, g)
    live = dev(ref.mask(lens, lanes, T))
    out = empty(lanes, T, width, dtype, layout)
    codec.embed(dev(tok), dev(table), out, scale=0.37, d_lens=dev(lens))
    scale = torch.tensor(0.37, dtype=F32, device="cuda")
    want = (dev(table).float() * scale).to(dtype)[dev(tok).long()]
    want[~live] = SKIP
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embed_grad_of_many_rows(codec, dtype):  # noqa: F811
    lanes, T, width = 7, 300007, 4
    assert lanes * T > 1024 * 2048
    g = torch.Generator().manual_seed(3)
    tok = tokens_of("sparse", lanes, T, g)
    dout = torch.randn((lanes, T, width), generator=g).to(dtype)
    lens = torch.tensor([T, T - 1, T, 5, 0, T, T], dtype=torch.int32)
    live = ref.mask(lens, lanes, T)
    held = dout.clone()
    held[~live] = math.nan
    grad = torch.full((256, width), SKIP, device="cuda")
    args = (dev(tok), dev(held), grad, work(boa_hip.embed_grad_work_bytes(lanes, T, width)))
    codec.embed_grad(*args, scale=2.5, d_lens=dev(lens))
    first = grad.clone()
    ref.check("dtable", first.cpu(), ref.embed_grad(tok, dout, 2.5, live))
    codec.embed_grad(*args, scale=2.5, d_lens=dev(lens))
    assert torch.equal(first, grad), "two calls differ"


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lanes,T,dtype,layout", [
    (33, 2003, BF16, "dense"), (17, 2003, F32, "wide"), (17, 2003, F32, "odd")])
def test_loss_of_many_rows(codec, lanes, T, dtype, layout, in_place):  # noqa: F811
    g = torch.Generator().manual_seed(lanes + T)
    x = (torch.randn((lanes, T, 256), generator=g) * 3).to(dtype)
    x[..., 250:] = -math.inf
    tgt, bias = tokens_of("any", lanes, T, g).clamp(max=249), torch.randn(256, generator=g)
    lens = lens_of("ragged", lanes, T, g)
    live = ref.mask(lens, lanes, T)
    held = x.clone()
    held[~live] = math.nan
    logits = place(held, layout, math.nan)
    del held
    dx = logits if in_place else empty(lanes, T, 256, dtype, layout)
    loss = torch.full((lanes, T), SKIP, device="cuda")
    total, dbias = torch.zeros(1, device="cuda"), torch.zeros(256, device="cuda")
    codec.next_byte_loss(logits, dev(tgt), loss, work(boa_hip.next_byte_loss_work_bytes(lanes, T)),
                         d_bias=dev(bias), d_total=total, d_dlogits=dx, d_dbias=dbias, scale=0.125,
                         d_lens=dev(lens))
    zeroed(dx, live, "dlogits")
    sums = None
    for i in range(0, lanes, 4):  # the 64-bit form in parts, on the GPU
        part = slice(i, i + 4)
        on = dev(live[part])
        got = ref.loss(dev(x[part]), dev(bias), dev(tgt[part]), 0.125, on)
        wl, wt, wx, wb = (ref.V(v.val.cpu(), v.err.cpu()) for v in got)
        ref.check("loss", loss[part].cpu()[live[part]], wl[live[part]])
        ref.check("dlogits", dx[part].cpu(), wx, dtype)
        sums = (wt, wb) if sums is None else (sums[0] + wt, sums[1] + wb)
    assert (loss.cpu()[~live] == SKIP).all()
    ref.check("total", total.cpu(), sums[0])
    ref.check("dbias", dbias.cpu(), sums[1])


@pytest.mark.parametrize("T,ch", [(21, 64), (21, 130), (1, 64)])
def test_scan_of_far_lanes(codec, T, ch):  # noqa: F811
    """Every row tensor of the scan and of its gradient in turn: the same bits
    as with the lanes side by side (64 channels and more store dB and dC in
    different kernels)."""
    lanes, n = 2, 16
    s, _ = scan_inputs(lanes, T, ch, n, BF16, "full")
    near, _ = run_scan(codec, s, None, "dense")
    d = {k: v.cuda() for k, v in s.items()}
    names = ("u", "delta", "z", "B", "C", "A", "D", "delta_bias")
    w = work(boa_hip.selective_scan_work_bytes(lanes, T, ch, n, grad=True))
    rows = {"du": ch, "ddelta": ch, "dz": ch, "dB": n, "dC": n}
    for name in (*ROWS_IN, "out", *rows):
        e = dict(d)
        o = {"out": torch.zeros((lanes, T, ch), dtype=BF16, device="cuda")}
        o.update({k: torch.zeros((lanes, T, v), dtype=BF16, device="cuda") for k, v in rows.items()})
        if name in e:
            e[name] = far(s[name])
        else:
            o[name] = far(o[name])
        state, dstate = (torch.zeros((lanes, ch, n), device="cuda") for _ in range(2))
        dA, dD, db = (torch.zeros(k, device="cuda") for k in ((ch, n), (ch,), (ch,)))
        saved = torch.zeros(boa_hip.selective_scan_saved_floats(lanes, T, ch, n), device="cuda")
        args = [e[k] for k in names]
        codec.selective_scan(*args, o["out"], w, d_state_in=e["state_in"], d_state_out=state,
                             d_saved=saved)
        codec.selective_scan_grad(*args, saved, e["dout"], *[o[k] for k in rows], dA, dD, db, w,
                                  d_state_in=e["state_in"], d_dstate_out=e["dstate_out"],
                                  d_dstate_in=dstate)
        o.update(state_out=state, dstate_in=dstate, dA=dA, dD=dD, ddelta_bias=db)
        for k, v in o.items():
            assert torch.equal(v, near[k]), (name, k)
        del e, o
