"""The training operators as the model uses them: mambav1's forward pass put
together from the embedding, the selective scan and torch's products, against
the codec's own forward pass of the same weights."""
import numpy as np
import pytest
import torch

import boa_hip
import synth

pytestmark = pytest.mark.gpu


def _model(weights, codec, d, L, ds, pieces):
    """Logits of the pieces [lanes, T] one after the other, states handed on."""
    w = {k: torch.from_numpy(v).cuda() for k, v in weights}
    di, r, _ = synth.dims(d, ds)
    lanes = pieces[0].shape[0]
    zeros = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    states = [zeros(lanes, di, ds) for _ in range(L)]
    before = [zeros(lanes, 3, di) for _ in range(L)]  # the conv's last inputs

    def norm(x, p):
        return torch.nn.functional.layer_norm(x, (d,), w[p + "weight"], w[p + "bias"], 1e-5)

    def linear(x, p):
        return x @ w[p + "weight"].t() + w.get(p + "bias", 0.0)

    logits = []
    for tok in pieces:
        T = tok.shape[1]
        x = zeros(lanes, T, d)
        codec.embed(tok, w["embedding.weight"], x)
        work = zeros(boa_hip.selective_scan_work_bytes(lanes, T, di, ds)).byte()
        for i in range(L):
            p, m = f"blocks.{i}.", f"blocks.{i}.mamba."
            xz = linear(norm(x, p + "ln1."), m + "in_proj.")
            seq = torch.cat([before[i], xz[..., :di]], 1)
            before[i] = seq[:, -3:].clone()
            taps = w[m + "conv1d.weight"][:, 0]
            u = w[m + "conv1d.bias"] + sum(seq[:, k:k + T] * taps[:, k] for k in range(4))
            u = torch.nn.functional.silu(u)
            dbc = u @ w[m + "x_proj.weight"].t()
            y = zeros(lanes, T, di)
            codec.selective_scan(u, dbc[..., :r] @ w[m + "dt_proj.weight"].t(), xz[..., di:],
                                 dbc[..., r:r + ds], dbc[..., r + ds:], -torch.exp(w[m + "A_log"]),
                                 w[m + "D"], w[m + "dt_proj.bias"], y, work, d_state_in=states[i],
                                 d_state_out=states[i])
            h = linear(norm(linear(y, m + "out_proj."), p + "ln2."), p + "ff.0.")
            x = linear(torch.nn.functional.gelu(h, approximate="tanh"), p + "ff.2.") + x
        logits.append(linear(torch.relu(linear(x, "head.0.")), "head.2."))
    return torch.cat(logits, 1)


@pytest.mark.parametrize("d,L,ds", [(64, 2, 16), (80, 3, 16), (256, 2, 16), (512, 1, 32)])
def test_operators_make_the_codecs_forward_pass(make_weights, d, L, ds):
    lanes, cuts = 5, (37, 1, 1, 20)
    weights = synth.random_weight_tensors(d, L, ds, seed=0)
    rng = np.random.default_rng(d)
    pieces = [torch.from_numpy(rng.integers(0, 256, (lanes, n), dtype=np.uint8)).cuda() for n in cuts]
    codec = boa_hip.Codec(d, L, ds, lanes)
    codec.set_stream(torch.cuda.current_stream().cuda_stream)
    codec.load_weights(str(make_weights(d, L, ds)))
    codec.reset_state(lanes)
    want = []
    for tok in pieces:
        out = torch.zeros((lanes, tok.shape[1], 256), device="cuda")
        codec.forward_chunk(tok.contiguous(), lanes, tok.shape[1], out)
        want.append(out)
    want = torch.cat(want, 1)
    got = _model(weights, codec, d, L, ds, pieces)
    # ten operators a layer and three around them, thousands of fp32 roundings
    # a sum, each 2^-24 of its terms: of the norm, less than 2^-24 * 64 each
    off = (got - want).norm() / want.norm()
    assert off <= 2.0 ** -24 * 64 * (10 * L + 3), off.item()
