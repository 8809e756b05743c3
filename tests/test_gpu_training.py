"""The training operators on the GPU against their 64-bit forms
(training_ref.py, whose error bounds are the tolerances): sizes from one row
up, odd widths and channel counts, lanes of length 0, strided and unaligned
rows, masked logits, refusals, streams and graphs."""
import math

import numpy as np
import pytest
import torch

import boa_hip
import training_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
SKIP = 7.5  # what outputs hold before a call


@pytest.fixture(scope="module")
def codec():
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    c = boa_hip.Codec(64, 1, 16, 1)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    return c


def work(n):
    # whatever a workspace holds must not matter
    return torch.full((max(n, 1),), 0xFF, dtype=torch.uint8, device="cuda")


def lens_of(kind, lanes, T, g):
    if kind == "full":
        return None
    n = torch.randint(0, T + 1, (lanes,), generator=g, dtype=torch.int32)
    n[0] = T + 5  # taken as T
    if lanes > 1:
        n[-1] = 0
    if lanes > 2:
        n[1] = -3  # taken as 0
    return n


def place(t, layout, fill=SKIP):
    """t [lanes, T, width] on the GPU with the strides of a layout."""
    lanes, T, width = t.shape
    if layout == "dense":
        buf = torch.full((lanes, T, width), fill, dtype=t.dtype, device="cuda")
        v = buf
    elif layout == "wide":  # beside other columns, as a slice of a product's rows
        buf = torch.full((lanes, T, width + 24), fill, dtype=t.dtype, device="cuda")
        v = buf[..., 8:8 + width]
    elif layout == "odd":  # unaligned rows
        buf = torch.full((lanes, T, width + 3), fill, dtype=t.dtype, device="cuda")
        v = buf[..., 1:1 + width]
    else:  # positions outermost
        buf = torch.full((T, lanes, width), fill, dtype=t.dtype, device="cuda")
        v = buf.transpose(0, 1)
    v.copy_(t)
    return v


def empty(lanes, T, width, dtype, layout):
    return place(torch.full((lanes, T, width), SKIP, dtype=dtype), layout)


def dev(x):
    return None if x is None else x.cuda()


def untouched(t, live, name):
    """rows past a lane's length hold what they held"""
    past = t.detach().float().cpu()[~live]
    assert (past == SKIP).all(), f"{name}: rows past the lanes' lengths were written"


def zeroed(t, live, name):
    past = t.detach().float().cpu()[~live]
    assert (past == 0).all(), f"{name}: gradients past the lanes' lengths are not zero"


def tokens_of(kind, lanes, T, g):
    if kind == "same":
        return torch.full((lanes, T), 65, dtype=torch.uint8)
    if kind == "ends":
        return torch.randint(0, 2, (lanes, T), generator=g, dtype=torch.uint8) * 255
    t = torch.randint(0, 256, (lanes, T), generator=g, dtype=torch.uint8)
    if kind == "sparse":
        t = t * (torch.rand((lanes, T), generator=g) < 0.1)
    return t


# ---------------------------------------------------------------- embedding
EMBED = [(1, 1, 64, "dense", "full"), (1, 1, 1, "dense", "full"), (5, 1, 80, "dense", "full"),
         (3, 37, 64, "dense", "ragged"), (4, 33, 100, "wide", "ragged"), (3, 19, 7, "odd", "ragged"),
         (2, 65, 512, "time", "ragged"), (7, 11, 512, "odd", "full"), (2, 300, 256, "wide", "full"),
         (40, 301, 256, "dense", "ragged")]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lanes,T,width,layout,kind", EMBED)
def test_embed(codec, lanes, T, width, layout, kind, dtype):
    g = torch.Generator().manual_seed(lanes * 1000 + T + width)
    tok = tokens_of("any", lanes, T + 2, g)
    table = torch.randn((256, width), generator=g).to(dtype)
    lens = lens_of(kind, lanes, T, g)
    live = ref.mask(lens, lanes, T)
    out = empty(lanes, T, width, dtype, layout)
    codec.embed(dev(tok)[:, 1:T + 1], dev(table), out, scale=0.37, d_lens=dev(lens))
    want = ref.embed(tok[:, 1:T + 1], table, 0.37)
    ref.check("out", out.cpu()[live], want[live], dtype)
    untouched(out, live, "out")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lanes,T,width,layout,kind,data", [
    (1, 1, 64, "dense", "full", "any"), (1, 1, 1, "odd", "full", "any"),
    (3, 21, 80, "dense", "ragged", "any"), (1, 64, 64, "dense", "full", "same"),
    (5, 200, 64, "wide", "ragged", "sparse"), (3, 500, 256, "dense", "full", "same"),
    (2, 333, 512, "dense", "ragged", "any"), (2, 333, 511, "odd", "ragged", "ends"),
    (9, 130, 7, "time", "ragged", "any"), (4, 1000, 100, "wide", "full", "ends"),
    (17, 1201, 16, "dense", "ragged", "sparse"), (3, 11003, 64, "dense", "full", "any"),
    (1, 300001, 4, "dense", "full", "sparse"), (600, 437, 8, "dense", "ragged", "same")])
def test_embed_grad(codec, lanes, T, width, layout, kind, data, dtype):
    g = torch.Generator().manual_seed(lanes * 1000 + T + width)
    tok = tokens_of(data, lanes, T, g)
    dout = torch.randn((lanes, T, width), generator=g).to(dtype)
    lens = lens_of(kind, lanes, T, g)
    live = ref.mask(lens, lanes, T)
    held = dout.clone()
    held[~live] = math.nan  # never read
    grad = torch.full((256, width), SKIP, device="cuda")
    n = boa_hip.embed_grad_work_bytes(lanes, T, width)
    args = (dev(tok), place(held, layout, math.nan), grad, work(n))
    codec.embed_grad(*args, scale=2.5, d_lens=dev(lens))
    first = grad.clone()
    ref.check("dtable", first.cpu(), ref.embed_grad(tok, dout, 2.5, live))
    codec.embed_grad(*args, scale=2.5, d_lens=dev(lens))
    assert torch.equal(first, grad), "two calls differ"


# --------------------------------------------------------------------- loss
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lanes,T,layout,kind,masked", [
    (1, 1, "dense", "full", False), (3, 1, "wide", "ragged", True), (1, 64, "dense", "full", True),
    (5, 13, "dense", "ragged", False), (5, 130, "odd", "ragged", True),
    (7, 91, "time", "ragged", True), (33, 200, "dense", "ragged", False)])
def test_loss(codec, lanes, T, layout, kind, masked, dtype):
    g = torch.Generator().manual_seed(lanes * 1000 + T)
    x = (torch.randn((lanes, T, 256), generator=g) * 3).to(dtype)
    tgt = tokens_of("any", lanes, T + 1, g)
    x[0, 0, int(tgt[0, 1])] = 40.0  # nearly certain
    if masked:
        x[..., 200:] = -math.inf
        x[-1, -1, 1:200] = torch.finfo(dtype).min
        tgt = tgt.clamp(max=199)
    bias = torch.randn(256, generator=g)
    lens = lens_of(kind, lanes, T, g)
    live = ref.mask(lens, lanes, T)
    held = x.clone()
    held[~live] = math.nan
    loss = torch.full((lanes, T), SKIP, device="cuda")
    total, dbias = torch.zeros(1, device="cuda"), torch.zeros(256, device="cuda")
    dx = empty(lanes, T, 256, dtype, layout)
    codec.next_byte_loss(place(held, layout, math.nan), dev(tgt)[:, 1:], loss,
                         work(boa_hip.next_byte_loss_work_bytes(lanes, T)), d_bias=dev(bias),
                         d_total=total, d_dlogits=dx, d_dbias=dbias, scale=0.125,
                         d_lens=dev(lens))
    wl, wt, wx, wb = ref.loss(x, bias, tgt[:, 1:], 0.125, live)
    ref.check("loss", loss.cpu()[live], wl[live])
    untouched(loss, live, "loss")
    ref.check("total", total, wt)
    ref.check("dlogits", dx, wx, dtype)
    zeroed(dx, live, "dlogits")
    ref.check("dbias", dbias, wb)


def test_loss_in_place_and_parts(codec):
    """dlogits over logits; without the optional outputs; no bias."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn((6, 50, 256), generator=g)
    tgt = tokens_of("any", 6, 50, g)
    live = ref.mask(None, 6, 50)
    w = work(boa_hip.next_byte_loss_work_bytes(6, 50))
    loss = torch.zeros((6, 50), device="cuda")
    codec.next_byte_loss(x.cuda(), dev(tgt), loss, w)
    want = ref.loss(x, None, tgt, 1.0, live)
    ref.check("loss", loss, want[0])
    buf = x.cuda()
    codec.next_byte_loss(buf, dev(tgt), loss, w, d_dlogits=buf)
    ref.check("dlogits", buf, want[2])
    total = torch.zeros(1, device="cuda")
    codec.next_byte_loss(x.cuda(), dev(tgt), loss, w, d_total=total)
    ref.check("total", total, want[1])


def test_loss_of_impossible_rows(codec):
    """A target that is ruled out, a row of nothing, a NaN: each in its own row."""
    x = torch.zeros((1, 6, 256))
    x[0, 1, 9] = -math.inf          # the target
    x[0, 2] = -math.inf             # everything
    x[0, 3, 5] = math.nan
    x[0, 4] = torch.finfo(F32).min  # the type's lowest value everywhere: uniform
    tgt = torch.full((1, 6), 9, dtype=torch.uint8)
    loss, dx = torch.zeros((1, 6), device="cuda"), torch.zeros((1, 6, 256), device="cuda")
    codec.next_byte_loss(x.cuda(), dev(tgt), loss, d_dlogits=dx)
    loss, dx = loss.cpu()[0], dx.cpu()[0]
    assert loss[1] == math.inf and loss[2] == math.inf and math.isnan(loss[3])
    assert abs(dx[1, 9].item() + 1.0) <= 2.0 ** -22 and dx[1, 8] > 0
    assert (dx[2] == 0).all() and dx[3].isnan().all()
    for r in (0, 4, 5):  # log 256, in fp32
        assert abs(loss[r].item() - math.log(256)) <= 8 * 2.0 ** -24 * math.log(256)
        assert dx[r].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_loss_of_a_nan_among_ruled_out_bytes(codec, dtype):
    """A NaN is not ruled out: its row's loss is NaN wherever it stands."""
    x = torch.full((1, 256, 256), -math.inf)
    x[0, torch.arange(256), torch.arange(256)] = math.nan
    tgt = torch.full((1, 256), 9, dtype=torch.uint8)
    loss = torch.zeros((1, 256), device="cuda")
    codec.next_byte_loss(x.to(dtype).cuda(), dev(tgt), loss,
                         work(boa_hip.next_byte_loss_work_bytes(1, 256)))
    assert loss.isnan().all()


def test_loss_of_near_certainty(codec):
    """Losses far under fp32's step at 1 keep their digits."""
    x = torch.zeros((1, 4, 256))
    tgt = torch.zeros((1, 4), dtype=torch.uint8)
    for r, v in enumerate((10.0, 20.0, 30.0, 60.0)):
        x[0, r, 0] = v
    loss, dx = torch.zeros((1, 4), device="cuda"), torch.zeros((1, 4, 256), device="cuda")
    codec.next_byte_loss(x.cuda(), dev(tgt), loss, d_dlogits=dx)
    want = ref.loss(x, None, tgt, 1.0, ref.mask(None, 1, 4))
    ref.check("loss", loss, want[0])
    ref.check("dlogits", dx, want[2])
    assert loss[0, 2].item() == pytest.approx(255 * math.exp(-30), rel=1e-4)


# --------------------------------------------------------------------- scan
def scan_inputs(lanes, T, ch, n, dtype, kind, state=True, seed=0):
    g = torch.Generator().manual_seed(seed + lanes * 1000 + T * 7 + ch)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    s = {"u": r(lanes, T, ch).to(dtype), "delta": r(lanes, T, ch).to(dtype),
         "z": (r(lanes, T, ch) * 2).to(dtype), "B": r(lanes, T, n).to(dtype),
         "C": r(lanes, T, n).to(dtype), "A": -torch.exp(r(ch, n)),
         "D": r(ch), "delta_bias": r(ch) - 2.0, "dout": r(lanes, T, ch).to(dtype)}
    if state:
        s["state_in"], s["dstate_out"] = r(lanes, ch, n), r(lanes, ch, n)
    return s, lens_of(kind, lanes, T, g)


ROWS_IN = ("u", "delta", "z", "B", "C", "dout")


def run_scan(codec, s, lens, layout, grad=True):
    lanes, T, ch = s["u"].shape
    n, dtype = s["A"].shape[1], s["u"].dtype
    live = ref.mask(lens, lanes, T)
    d = {}
    for k, v in s.items():
        if k in ROWS_IN:
            held = v.clone()
            held[~live] = math.nan
            d[k] = place(held, layout, math.nan)
        else:
            d[k] = v.cuda()
    args = [d[k] for k in ("u", "delta", "z", "B", "C", "A", "D", "delta_bias")]
    out = empty(lanes, T, ch, dtype, layout)
    state = torch.full((lanes, ch, n), SKIP, device="cuda")
    saved = torch.full((boa_hip.selective_scan_saved_floats(lanes, T, ch, n),), math.nan,
                       device="cuda")
    w = work(boa_hip.selective_scan_work_bytes(lanes, T, ch, n))
    codec.selective_scan(*args, out, w, d_state_in=d.get("state_in"), d_state_out=state,
                         d_lens=dev(lens), d_saved=saved if grad else None)
    got = {"out": out, "state_out": state}
    if grad:
        rows = {"du": ch, "ddelta": ch, "dz": ch, "dB": n, "dC": n}
        for k, width in rows.items():
            got[k] = empty(lanes, T, width, dtype, layout)
        got["dA"] = torch.full((ch, n), SKIP, device="cuda")
        got["dD"], got["ddelta_bias"] = (torch.full((ch,), SKIP, device="cuda") for _ in range(2))
        got["dstate_in"] = torch.full((lanes, ch, n), SKIP, device="cuda")
        w = work(boa_hip.selective_scan_work_bytes(lanes, T, ch, n, grad=True))
        codec.selective_scan_grad(*args, saved, d["dout"],
                                  *[got[k] for k in (*rows, "dA", "dD", "ddelta_bias")], w,
                                  d_state_in=d.get("state_in"), d_dstate_out=d.get("dstate_out"),
                                  d_dstate_in=got["dstate_in"], d_lens=dev(lens))
    return got, live


SCAN = [(1, 1, 1, 16, "dense", "full"), (2, 1, 64, 32, "dense", "full"),
        (3, 1, 130, 16, "wide", "ragged"), (2, 16, 64, 16, "dense", "full"),
        (2, 17, 128, 16, "dense", "ragged"), (3, 33, 160, 16, "wide", "ragged"),
        (3, 31, 67, 16, "odd", "ragged"), (2, 40, 66, 32, "odd", "ragged"),
        (4, 35, 192, 32, "time", "ragged"), (2, 100, 128, 16, "time", "full"),
        (70, 5, 32, 16, "dense", "ragged"), (1, 333, 64, 16, "dense", "full"),
        (2, 150, 64, 32, "wide", "ragged"), (1, 1201, 20, 16, "dense", "full"),
        (3, 700, 64, 32, "dense", "ragged"),
        (520, 19, 16, 16, "dense", "ragged"),    # whole lanes: no segments
        (264, 17, 12, 32, "time", "ragged"),
        (1, 4300, 4, 16, "dense", "full"),       # as many segments as there are
        (2, 5, 4096, 16, "dense", "full"), (1, 18, 4095, 32, "odd", "full")]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lanes,T,ch,n,layout,kind", SCAN)
def test_scan(codec, lanes, T, ch, n, layout, kind, dtype):
    s, lens = scan_inputs(lanes, T, ch, n, dtype, kind, state=lanes != 70)
    got, live = run_scan(codec, s, lens, layout)
    out, state, kept = ref.scan(s, live)
    ref.check("out", got["out"].cpu()[live], out[live], dtype)
    untouched(got["out"], live, "out")
    ref.check("state_out", got["state_out"], state)
    for k, want in ref.scan_grad(s, live, kept).items():
        ref.check(k, got[k], want, got[k].dtype)
    for k in ("du", "ddelta", "dz", "dB", "dC"):
        zeroed(got[k], live, k)


def test_scan_without_gradient_is_the_same(codec):
    s, lens = scan_inputs(3, 50, 128, 16, F32, "ragged")
    a, live = run_scan(codec, s, lens, "dense", grad=True)
    b, _ = run_scan(codec, s, lens, "dense", grad=False)
    assert torch.equal(a["out"], b["out"]) and torch.equal(a["state_out"], b["state_out"])


def test_scan_twice_is_the_same(codec):
    s, lens = scan_inputs(5, 77, 160, 16, BF16, "ragged")
    a, _ = run_scan(codec, s, lens, "dense")
    b, _ = run_scan(codec, s, lens, "dense")
    for k in a:
        assert torch.equal(a[k], b[k]), k


def test_scan_in_steps(codec):
    """A sequence in pieces, states handed on (in place), as decode steps and
    truncated training do: every piece within the bounds of the whole."""
    s, _ = scan_inputs(3, 41, 128, 16, F32, "full")
    live = ref.mask(None, 3, 41)
    want, state, _ = ref.scan(s, live)
    d = {k: v.cuda() for k, v in s.items()}
    h = d["state_in"].clone()
    out = torch.zeros((3, 41, 128), device="cuda")
    t = 0
    for n in (1, 1, 20, 1, 16, 2):
        cut = [d[k][:, t:t + n] for k in ("u", "delta", "z", "B", "C")]
        codec.selective_scan(*cut, d["A"], d["D"], d["delta_bias"], out[:, t:t + n],
                             work(boa_hip.selective_scan_work_bytes(3, n, 128, 16)),
                             d_state_in=h, d_state_out=h)
        t += n
    assert t == 41
    ref.check("out", out, want)
    ref.check("state", h, state)


# lanes that are cut into 2 to 32 segments, with more blocks than start at once
@pytest.mark.parametrize("lanes,T,ch,n", [(3, 500, 640, 16), (2, 70, 64, 32), (7, 333, 1024, 32)])
def test_scan_states_in_place(codec, lanes, T, ch, n):
    """state_out over state_in and dstate_in over dstate_out: what a lane's last
    segment stores is not what its other segments start from."""
    s, lens = scan_inputs(lanes, T, ch, n, F32, "ragged")
    live = ref.mask(lens, lanes, T)
    want, state, kept = ref.scan(s, live)
    d = {k: v.cuda() for k, v in s.items()}
    args = [d[k] for k in ("u", "delta", "z", "B", "C", "A", "D", "delta_bias")]
    out, h, g = torch.zeros_like(d["u"]), d["state_in"].clone(), d["dstate_out"].clone()
    saved = torch.empty(boa_hip.selective_scan_saved_floats(lanes, T, ch, n), device="cuda")
    codec.selective_scan(*args, out, work(boa_hip.selective_scan_work_bytes(lanes, T, ch, n)),
                         d_state_in=h, d_state_out=h, d_lens=dev(lens), d_saved=saved)
    ref.check("out", out.cpu()[live], want[live])
    ref.check("state", h, state)
    grads = {k: torch.empty_like(d[k]) for k in ("u", "delta", "z", "B", "C", "A", "D",
                                                 "delta_bias")}
    codec.selective_scan_grad(*args, saved, d["dout"], *grads.values(),
                              work(boa_hip.selective_scan_work_bytes(lanes, T, ch, n, grad=True)),
                              d_state_in=d["state_in"], d_dstate_out=g, d_dstate_in=g,
                              d_lens=dev(lens))
    for k, v in ref.scan_grad(s, live, kept).items():
        ref.check(k, g if k == "dstate_in" else grads[k[1:]], v)


def test_scan_extremes(codec):
    """Decays of 0 and 1, gates shut and open wide, delta of 0 and large."""
    s, _ = scan_inputs(2, 20, 64, 16, F32, "full")
    s["delta"][:, 3] = -200.0   # delta = 0
    s["delta"][:, 9] = 60.0     # the state is forgotten
    s["z"][:, 5] = -120.0
    s["z"][:, 6] = 120.0
    s["A"][:, 0] = 0.0          # never forgets
    s["A"][:, 1] = -1000.0
    got, live = run_scan(codec, s, None, "dense")
    for k, v in got.items():
        assert torch.isfinite(v).all(), k
    out, state, kept = ref.scan(s, live)
    ref.check("out", got["out"], out)
    ref.check("state_out", got["state_out"], state)
    for k, want in ref.scan_grad(s, live, kept).items():
        ref.check(k, got[k], want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_of_one_lane_alone(codec, dtype):
    """A lane's results do not depend on the lanes beside it, nor on NaN there."""
    s, _ = scan_inputs(4, 40, 96, 16, dtype, "full")
    a, _ = run_scan(codec, s, None, "dense")
    t = {k: v.clone() for k, v in s.items()}
    t["u"][1, 7] = math.nan
    t["B"][3] = math.inf
    b, _ = run_scan(codec, t, None, "dense")
    for k in ("out", "state_out", "du", "ddelta", "dz", "dB", "dC", "dstate_in"):
        assert torch.equal(a[k][0], b[k][0]) and torch.equal(a[k][2], b[k][2]), k


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [16, 32])
def test_scan_past_the_end_of_infinite_states(codec, n, dtype):
    """Gradients past a lane's length are zero whatever the lane holds."""
    s, _ = scan_inputs(3, 45, 70, n, dtype, "full")
    s["state_in"][0, 5, 3] = math.inf
    s["dstate_out"][1, 9, 2] = math.nan
    s["u"][2, 4, 60] = -math.inf
    got, live = run_scan(codec, s, torch.tensor([21, 35, 5], dtype=torch.int32), "wide")
    for k in ("du", "ddelta", "dz", "dB", "dC"):
        zeroed(got[k], live, k)
    untouched(got["out"], live, "out")


@pytest.mark.parametrize("T", [1, 3, 40])
def test_scan_that_forgets_at_once(codec, T):
    """The largest decays: each state is its last position's, in lanes that end
    inside a tile or hold nothing as well."""
    s, _ = scan_inputs(3, T, 64, 16, F32, "full")
    s["A"][:] = -torch.finfo(F32).max
    s["A"][:, 1] = -math.inf
    lens = torch.tensor([T, max(T - 1, 1), 0], dtype=torch.int32)
    got, live = run_scan(codec, s, lens, "dense", grad=False)
    # with any large decay the older positions' part is below what fp64 tells apart
    s["A"][:] = -1e6
    out, state, _ = ref.scan(s, live)
    ref.check("out", got["out"].cpu()[live], out[live])
    ref.check("state_out", got["state_out"], state)


# ------------------------------------------------------------- far addresses
def far(t, dtype=None, fill=SKIP):
    """[2, T, width] with 2^31 + 16 elements between the lanes."""
    lanes, T, width = t.shape
    step = (1 << 31) + 16
    buf = torch.empty(step + T * width, dtype=t.dtype, device="cuda")
    v = torch.as_strided(buf, (lanes, T, width), (step, width, 1))
    v.copy_(t)
    return v


def test_far_lanes(codec):
    """Offsets that pass 32 bits: every row tensor in turn."""
    g = torch.Generator().manual_seed(9)
    lanes, T, width = 2, 21, 64
    tok = tokens_of("any", lanes, T, g)
    live = ref.mask(None, lanes, T)
    table = torch.randn((256, width), generator=g).to(BF16)
    out = far(torch.zeros((lanes, T, width), dtype=BF16))
    codec.embed(dev(tok), dev(table), out)
    ref.check("out", out, ref.embed(tok, table, 1.0), BF16)
    del out
    dout = torch.randn((lanes, T, width), generator=g).to(BF16)
    dtable = torch.zeros(256 * width + 1, device="cuda")[1:].view(256, width)  # unaligned
    n = boa_hip.embed_grad_work_bytes(lanes, T, width)
    codec.embed_grad(dev(tok), far(dout), dtable, work(n))
    ref.check("dtable", dtable, ref.embed_grad(tok, dout, 1.0, live))
    x = torch.randn((lanes, T, 256), generator=g).to(BF16)
    loss = torch.zeros((lanes, T), device="cuda")
    dx = far(torch.zeros((lanes, T, 256), dtype=BF16))
    codec.next_byte_loss(far(x), dev(tok), loss, work(boa_hip.next_byte_loss_work_bytes(lanes, T)),
                         d_dlogits=dx)
    want = ref.loss(x, None, tok, 1.0, live)
    ref.check("loss", loss, want[0])
    ref.check("dlogits", dx, want[2], BF16)
    del dx
    s, _ = scan_inputs(lanes, T, 64, 16, BF16, "full")
    near, _ = run_scan(codec, s, None, "dense")
    d = {k: v.cuda() for k, v in s.items()}
    for name in ROWS_IN[:5]:
        e = dict(d, **{name: far(s[name])})
        o, st = torch.zeros((lanes, T, 64), dtype=BF16, device="cuda"), torch.zeros_like(d["state_in"])
        codec.selective_scan(*[e[k] for k in ("u", "delta", "z", "B", "C", "A", "D", "delta_bias")],
                             o, work(boa_hip.selective_scan_work_bytes(lanes, T, 64, 16)),
                             d_state_in=d["state_in"], d_state_out=st)
        assert torch.equal(o, near["out"]) and torch.equal(st, near["state_out"]), name
        del e


# ---------------------------------------------------------- used as they are
def _predictor(seed, lanes, T, d, ch, n):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    w = {"table": r(256, d), "w_in": r(d, 3 * ch + 2 * n) / math.sqrt(d), "A": -torch.exp(r(ch, n)),
         "D": r(ch), "delta_bias": r(ch) - 2, "w_out": r(ch, 256) / math.sqrt(ch), "bias": r(256)}
    return w, tokens_of("any", lanes, T + 1, g)


def _step(codec, w, data, d, ch, n, out):
    """One training step of embedding -> product -> scan -> product -> loss and
    back, into the tensors of `out` (allocated at the first call)."""
    lanes, T = data.shape[0], data.shape[1] - 1
    tok, tgt = data[:, :-1], data[:, 1:]
    if not out:
        z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
        out.update(x=z(lanes, T, d), p=z(lanes, T, 3 * ch + 2 * n), y=z(lanes, T, ch),
                   logits=z(lanes, T, 256), loss=z(lanes, T), total=z(1), bias=z(256),
                   dp=z(lanes, T, 3 * ch + 2 * n), A=z(ch, n), D=z(ch), delta_bias=z(ch),
                   table=z(256, d), dx=z(lanes, T, d), dy=z(lanes, T, ch), w_in=z(d, 3 * ch + 2 * n),
                   w_out=z(ch, 256),
                   saved=z(boa_hip.selective_scan_saved_floats(lanes, T, ch, n)),
                   work=work(max(boa_hip.embed_grad_work_bytes(lanes, T, d),
                                 boa_hip.selective_scan_work_bytes(lanes, T, ch, n, grad=True),
                                 boa_hip.selective_scan_work_bytes(lanes, T, ch, n),
                                 boa_hip.next_byte_loss_work_bytes(lanes, T))))
    o, wk = out, out["work"]
    parts = lambda p: (p[..., :ch], p[..., ch:2 * ch], p[..., 2 * ch:3 * ch],  # noqa: E731
                       p[..., 3 * ch:3 * ch + n], p[..., 3 * ch + n:])
    codec.embed(tok, w["table"], o["x"])
    torch.mm(o["x"].view(-1, d), w["w_in"], out=o["p"].view(lanes * T, -1))
    args = (*parts(o["p"]), w["A"], w["D"], w["delta_bias"])
    codec.selective_scan(*args, o["y"], wk, d_saved=o["saved"])
    torch.mm(o["y"].view(-1, ch), w["w_out"], out=o["logits"].view(-1, 256))
    codec.next_byte_loss(o["logits"], tgt, o["loss"], wk, d_bias=w["bias"], d_total=o["total"],
                         d_dlogits=o["logits"], d_dbias=o["bias"], scale=1.0 / (lanes * T))
    dl = o["logits"].view(-1, 256)
    torch.mm(o["y"].view(-1, ch).t(), dl, out=o["w_out"])
    torch.mm(dl, w["w_out"].t(), out=o["dy"].view(-1, ch))
    codec.selective_scan_grad(*args, o["saved"], o["dy"], *parts(o["dp"]), o["A"], o["D"],
                              o["delta_bias"], wk)
    dp = o["dp"].view(lanes * T, -1)
    torch.mm(o["x"].view(-1, d).t(), dp, out=o["w_in"])
    torch.mm(dp, w["w_in"].t(), out=o["dx"].view(-1, d))
    codec.embed_grad(tok, o["dx"], o["table"], wk)
    return {k: o[k] for k in w} | {"total": o["total"]}


def _step64(w, data, ch, n):
    """The same in 64 bits through torch's own differentiation."""
    w = {k: v.double().cpu().requires_grad_() for k, v in w.items()}
    tok, tgt = data[:, :-1].long(), data[:, 1:].long()
    p = w["table"][tok] @ w["w_in"]
    u, x, z, B, C = torch.split(p, [ch, ch, ch, n, n], -1)
    delta = torch.nn.functional.softplus(x + w["delta_bias"], threshold=1e9)
    h, ys = torch.zeros((tok.shape[0], ch, n), dtype=torch.float64), []
    for t in range(tok.shape[1]):
        h = torch.exp(delta[:, t, :, None] * w["A"]) * h \
            + (delta[:, t] * u[:, t])[..., None] * B[:, t, None, :]
        ys.append((h * C[:, t, None, :]).sum(-1))
    y = (torch.stack(ys, 1) + w["D"] * u) * z * torch.sigmoid(z)
    logp = torch.log_softmax(y @ w["w_out"] + w["bias"], -1)
    total = -logp.gather(-1, tgt[..., None]).sum()
    (total / tok.numel()).backward()
    return {k: v.grad for k, v in w.items()} | {"total": total.detach().view(1)}


def _close(got, want):
    for k in want:
        off = (got[k].double().cpu() - want[k]).norm() / want[k].norm()
        # thousands of fp32 roundings a sum, each 2^-24 of its terms, over a
        # chain of six operators: 2^-24 * 6 * sqrt(rows) of the norm and less
        assert off <= 2.0 ** -24 * 6 * 64, f"{k}: {off:.3g}"


def test_training_step(codec):
    d, ch, n, lanes, T = 64, 128, 16, 6, 90
    w, data = _predictor(0, lanes, T, d, ch, n)
    got = _step(codec, {k: v.cuda() for k, v in w.items()}, data.cuda(), d, ch, n, {})
    _close(got, _step64(w, data, ch, n))


def test_training_step_in_a_graph(codec):
    """Captured once, replayed on other data with eager work between the
    replays; every replay against the eager call."""
    d, ch, n, lanes, T = 64, 128, 16, 5, 70
    w, _ = _predictor(0, lanes, T, d, ch, n)
    wg = {k: v.cuda() for k, v in w.items()}
    datas = [_predictor(s, lanes, T, d, ch, n)[1].cuda() for s in range(4)]
    data = datas[0].clone()
    out, eager = {}, {}
    side = torch.cuda.Stream()
    own = boa_hip.Codec(64, 1, 16, 1)
    own.set_stream(side.cuda_stream)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(own, wg, data, d, ch, n, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = _step(own, wg, data, d, ch, n, out)
    for i in (1, 2, 3, 1):
        data.copy_(datas[i])
        graph.replay()
        torch.cuda.synchronize()
        res = {k: v.clone() for k, v in got.items()}
        want = _step(codec, wg, datas[i], d, ch, n, eager)
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(res[k], want[k]), (i, k)


def test_two_contexts_on_two_streams():
    """Calls that overlap in time, each with its own workspace."""
    a = [scan_inputs(4, 200, 128, 16, F32, "full", seed=s)[0] for s in range(2)]
    codecs, streams, got = [], [], []
    want = []
    for s in a:
        c = boa_hip.Codec(64, 1, 16, 1)
        c.set_stream(torch.cuda.current_stream().cuda_stream)
        want.append(run_scan(c, s, None, "dense")[0])
    torch.cuda.synchronize()
    for s in a:
        st = torch.cuda.Stream()
        c = boa_hip.Codec(64, 1, 16, 1)
        c.set_stream(st.cuda_stream)
        codecs.append(c)
        streams.append(st)
        with torch.cuda.stream(st):
            got.append(run_scan(c, s, None, "dense")[0])
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        for k in x:
            assert torch.equal(x[k], y[k]), k


# ----------------------------------------------------------------- refusals
def refused(fn, word):
    with pytest.raises((boa_hip.BoaError, ValueError)) as e:
        fn()
    assert word in str(e.value), str(e.value)


def test_refusals(codec):
    z = lambda *s, **k: torch.zeros(s, device="cuda", **k)  # noqa: E731
    tok = z(2, 3, dtype=torch.uint8)
    table, out = z(256, 64), z(2, 3, 64)
    refused(lambda: codec.embed(tok.cpu(), table, out), "tokens is on")
    refused(lambda: codec.embed(tok, table.bfloat16(), out), "table")
    refused(lambda: codec.embed(tok, z(255, 64), out), "table")
    refused(lambda: codec.embed(tok, z(256, 513), z(2, 3, 513)), "width")
    refused(lambda: codec.embed(tok, table, z(2, 4, 64)), "out")
    refused(lambda: codec.embed(tok, table, z(2, 3, 64, dtype=torch.float16)), "out")
    refused(lambda: codec.embed(tok, table, z(2, 1, 64).expand(2, 3, 64)), "rows overlap")
    refused(lambda: codec.embed(tok, table, z(2, 64, 3).transpose(1, 2)), "dense")
    refused(lambda: codec.embed(tok.t(), table, z(3, 2, 64)), "dense")
    refused(lambda: codec.embed(tok, table, out, d_lens=z(2)), "lens")
    refused(lambda: codec.embed(tok, table, out, d_lens=z(3, dtype=torch.int32)), "lens")
    refused(lambda: codec.embed(z(2, 0, dtype=torch.uint8), table, z(2, 0, 64)), "T")
    refused(lambda: codec.embed(z(0, 2, dtype=torch.uint8), table, z(0, 2, 64)), "lanes")
    big = z(40, 100, dtype=torch.uint8)
    refused(lambda: codec.embed_grad(big, z(40, 100, 64), table), "workspace")
    n = boa_hip.embed_grad_work_bytes(40, 100, 64)
    refused(lambda: codec.embed_grad(big, z(40, 100, 64), table, work(n)[:-1]), "workspace")
    refused(lambda: codec.embed_grad(big, z(40, 100, 64), table, work(n + 8)[8:]), "aligned")
    refused(lambda: codec.embed_grad(big, z(40, 100, 64), z(256, 65), work(n)), "dtable")

    logits, loss = z(2, 3, 256), z(2, 3)
    refused(lambda: codec.next_byte_loss(z(2, 3, 255), tok, loss), "logits")
    refused(lambda: codec.next_byte_loss(logits, tok, z(3, 2)), "loss")
    refused(lambda: codec.next_byte_loss(logits, tok, loss, d_dlogits=logits.bfloat16()), "dlogits")
    refused(lambda: codec.next_byte_loss(logits, tok, loss, d_bias=z(255)), "bias")
    refused(lambda: codec.next_byte_loss(z(40, 100, 256), big, z(40, 100)), "workspace")
    half = z(2, 6, 256)
    refused(lambda: codec.next_byte_loss(half[:, :3], tok, loss,
                                         d_dlogits=half.view(4, 3, 256)[:2]), "other strides")

    s, _ = scan_inputs(2, 5, 64, 16, F32, "full")
    d = {k: v.cuda() for k, v in s.items()}
    names = ("u", "delta", "z", "B", "C", "A", "D", "delta_bias")

    def scan(out=None, w=None, **change):
        e = dict(d, **change)
        codec.selective_scan(*[e[k] for k in names], z(2, 5, 64) if out is None else out, w,
                             d_state_in=e["state_in"], d_saved=e.get("saved"),
                             d_state_out=e.get("state_out"))

    refused(lambda: scan(A=z(64, 24), B=z(2, 5, 24), C=z(2, 5, 24), state_in=z(2, 64, 24)), "d_state")
    refused(lambda: scan(B=z(2, 5, 32)), "B")
    refused(lambda: scan(z=d["z"].bfloat16()), "z")
    refused(lambda: scan(state_in=z(2, 64, 32)), "state_in")
    refused(lambda: scan(saved=z(10)), "saved")
    refused(lambda: scan(saved=z(4097)[1:]), "aligned")
    refused(lambda: scan(state_out=z(2049)[1:].view(2, 64, 16)), "aligned")
    refused(lambda: scan(out=d["u"]), "input")
    refused(lambda: scan(out=z(1, 5, 64).expand(2, 5, 64)), "rows overlap")
    wide = torch.empty(((1 << 25) + 1) * 4 + 128, device="cuda")
    refused(lambda: scan(u=torch.as_strided(wide, (2, 5, 64), (64, (1 << 25) + 1, 1))), "2^25")
    del wide
    saved = z(boa_hip.selective_scan_saved_floats(2, 5, 64, 16))
    g = [z(2, 5, 64), z(2, 5, 64), z(2, 5, 64), z(2, 5, 16), z(2, 5, 16), z(64, 16), z(64), z(64)]
    a = [d[k] for k in names]
    refused(lambda: codec.selective_scan_grad(*a, saved, d["dout"], *g), "workspace")
    w = work(boa_hip.selective_scan_work_bytes(2, 5, 64, 16, grad=True))
    refused(lambda: codec.selective_scan_grad(*a, None, d["dout"], *g, w), "saved")
    refused(lambda: codec.selective_scan_grad(*a, saved, d["dout"], d["u"], *g[1:], w), "input")
    refused(lambda: codec.selective_scan_grad(*a, saved, d["dout"], d["dout"], *g[1:], w), "input")
    # a refused call leaves the context usable
    codec.embed(tok, table, out)
    torch.cuda.synchronize()
    assert (out == 0).all()
