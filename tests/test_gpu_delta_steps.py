"""Steps of the gated delta rule: few positions in one call are the same bits as
one position a call, and a predictor in fp32 that is served byte by byte gives
what it gives for the whole prompt at once."""
import pytest
import torch

import boa_hip
import training_ref
from test_gpu_delta import inputs
from test_gpu_training import BF16, F32, codec, dev, empty, lens_of, place, work  # noqa: F401
from training_ref import U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lanes,T,heads,hv,dk,dv,layout,kind,data", [
    (3, 12, 1, 2, 64, 64, "dense", "full", "plain"), (5, 12, 2, 4, 128, 128, "wide", "ragged", "reset"),
    (4, 7, 1, 3, 80, 80, "odd", "ragged", "same"), (300, 5, 1, 1, 33, 20, "time", "ragged", "none"),
    (70, 12, 4, 4, 64, 128, "dense", "ragged", "tiny")])
def test_few_positions_are_single_steps(codec, lanes, T, heads, hv, dk, dv, layout, kind, data, dtype):  # noqa: F811
    s, g = inputs(lanes, T, heads, hv, dk, dv, dtype, data)
    lens = lens_of(kind, lanes, T, g)
    x = {n: place(s[n], layout) for n in ("q", "k", "v", "g", "beta")}
    at_once = torch.empty((lanes, hv, dk, dv), device="cuda")
    out, steps = empty(lanes, T, hv * dv, dtype, layout), empty(lanes, T, hv * dv, dtype, layout)
    codec.delta_rule(*x.values(), out, heads=heads, scale=0.3, d_state_in=dev(s["state_in"]),
                     d_state_out=at_once, d_lens=dev(lens))
    state = dev(s["state_in"])
    for t in range(T):
        on = None if lens is None else (lens > t).int().cuda()
        codec.delta_rule(*[v[:, t:t + 1] for v in x.values()], steps[:, t:t + 1], heads=heads, scale=0.3,
                         d_state_in=state, d_state_out=state, d_lens=on)
    assert torch.equal(out, steps) and torch.equal(state, at_once)


@pytest.mark.parametrize("T", [5, 12, 64, 90, 700])
def test_served_in_fp32(codec, T):  # noqa: F811
    """Blocks of norm, product, rule and product with fp32 rows: a prompt of T
    bytes and 15 steps after it, and all of it at once."""
    lanes, steps, d, h, hv, dk, dv = 3, 15, 80, 1, 2, 48, 64
    g = torch.Generator().manual_seed(T)
    r = lambda *n: torch.randn(n, generator=g).cuda()  # noqa: E731
    n = 2 * h * dk + hv * dv + 2 * hv
    blocks = [(1 + 0.2 * r(d), r(d, n) / d ** 0.5, r(hv * dv, d) / (hv * dv) ** 0.5) for _ in range(2)]
    table, last, head = r(256, d), 1 + 0.2 * r(d), r(d, 256) / d ** 0.5
    tok = torch.randint(0, 256, (lanes, T + steps), generator=g, dtype=torch.uint8).cuda()

    def run(tok, states):
        rows = lambda w: torch.zeros((lanes, tok.shape[1], w), device="cuda")  # noqa: E731
        x, y, add = rows(d), rows(d), None
        codec.embed(tok, table, x)
        wk = work(boa_hip.delta_rule_work_bytes(lanes, tok.shape[1], h, hv, dk, dv))
        for (norm, opens, closes), state in zip(blocks, states):
            codec.rms_norm(x, y, d_weight=norm, d_residual=add, d_sum=None if add is None else x)
            z = y @ opens
            q, k, v = z[..., :dk], z[..., dk:2 * dk], z[..., 2 * dk:2 * dk + hv * dv]
            decay = -torch.nn.functional.softplus(z[..., -2 * hv:-hv]) * 0.05
            o = rows(hv * dv)
            codec.delta_rule(q, k, v, decay, torch.sigmoid(z[..., -hv:]), o, wk, heads=h,
                             scale=dk ** -0.5, d_state_in=state, d_state_out=state)
            add = o @ closes
        codec.rms_norm(x, y, d_weight=last, d_residual=add)
        return y @ head

    new = lambda: [torch.zeros((lanes, hv, dk, dv), device="cuda") for _ in blocks]  # noqa: E731
    whole, parts = new(), new()
    want = run(tok, whole)
    got = [run(tok[:, :T].contiguous(), parts)]
    got += [run(tok[:, t:t + 1].contiguous(), parts) for t in range(T, T + steps)]
    # eight operators on either side whose sums, of 128 terms at most, may be in
    # another order: less than 64 U of the norm each; a chunk's inverse may enlarge
    # them by its own size, 8 for keys that are not alike
    limit = U * 64 * 16 * 8
    for a, b in [(torch.cat(got, 1), want)] + list(zip(parts, whole)):
        off = (a.double() - b.double()).norm() / b.double().norm()
        assert off <= limit, (off.item(), limit)
