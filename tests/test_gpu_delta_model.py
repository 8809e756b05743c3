"""A gated-delta-rule byte predictor put together from its operators: served byte
by byte after a prompt (norm and product in 8 bits, the rule, the choice of a
byte) and trained for a step (embedding, norm, the rule, loss, and back)."""
import math

import pytest
import torch

import boa_hip
import delta_ref
from test_gpu_training import BF16, F32, codec, dev, work  # noqa: F401
from training_ref import U

pytestmark = pytest.mark.gpu

D, H, HV, DK, DV = 80, 1, 2, 48, 64
N = 2 * H * DK + HV * DV + 2 * HV  # q, k, v, log decay and beta of each head of v
EPS = 1e-5


class Served:
    """Blocks of norm -> product -> rule -> product, residuals between them."""

    def __init__(self, codec, dtype, lanes, layers=2):  # noqa: F811
        g = torch.Generator().manual_seed(5)
        self.codec, self.dtype, self.lanes = codec, dtype, lanes
        self.table = torch.randn((256, D), generator=g).to(dtype).cuda()
        self.norms = [dev(1 + 0.2 * torch.randn((D,), generator=g)) for _ in range(layers + 1)]

        def weight(n, k):
            w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8).cuda()
            packed = work(boa_hip.int8_pack_bytes(n, k))
            codec.int8_pack(w, packed)
            return w, packed, dev((0.5 + torch.rand((n,), generator=g)) / 64 / k ** 0.5)

        self.opens = [weight(N, D) for _ in range(layers)]
        self.closes = [weight(D, HV * DV) for _ in range(layers)]
        self.head = weight(256, D)
        self.states = [torch.zeros((lanes, HV, DK, DV), device="cuda") for _ in range(layers)]

    def product(self, x8, s8, weight, T):
        w, packed, scale = weight
        out = torch.zeros((self.lanes, T, w.shape[0]), dtype=self.dtype, device="cuda")
        self.codec.int8_matmul(x8, s8, packed, scale, out)
        return out

    def run(self, tokens, uniform, out):
        """Chooses a byte after each position; what the last product read, and logits."""
        T = tokens.shape[1]
        rows = lambda n, dt=self.dtype: torch.zeros((self.lanes, T, n), dtype=dt, device="cuda")  # noqa: E731
        x, add = rows(D), None
        self.codec.embed(tokens, self.table, x)
        x8, s8 = rows(D, torch.int8), torch.zeros((self.lanes, T), device="cuda")
        o8 = rows(HV * DV, torch.int8)
        wk = work(boa_hip.delta_rule_work_bytes(self.lanes, T, H, HV, DK, DV))
        for i, state in enumerate(self.states):
            self.codec.rms_norm(x, d_weight=self.norms[i], d_residual=add, d_sum=x if i else None,
                                d_out8=x8, d_scale8=s8, eps=EPS)
            y = self.product(x8, s8, self.opens[i], T)
            q, k, v = y[..., :DK], y[..., DK:2 * DK], y[..., 2 * DK:2 * DK + HV * DV]
            decay = -torch.nn.functional.softplus(y[..., -2 * HV:-HV].float())
            beta = torch.sigmoid(y[..., -HV:].float())
            o = rows(HV * DV)
            self.codec.delta_rule(q, k, v, decay, beta, o, wk, heads=H, scale=DK ** -0.5,
                                  unit_qk=True, d_state_in=state, d_state_out=state)
            self.codec.int8_rows(o, o8, s8)
            add = self.product(o8, s8, self.closes[i], T)
        self.codec.rms_norm(x, d_weight=self.norms[-1], d_residual=add, d_sum=x, d_out8=x8,
                            d_scale8=s8, eps=EPS)
        logits = self.product(x8, s8, self.head, T)
        self.codec.sample_bytes(logits, uniform, out, temperature=0.9, top_k=50, top_p=0.95)
        return x8, s8, logits


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_served_steps_are_the_prompt(codec, dtype):  # noqa: F811
    """A prompt of 90 bytes and 15 steps after it, and the same bytes at once."""
    lanes, T, steps = 5, 90, 15
    g = torch.Generator().manual_seed(1)
    tok = torch.randint(0, 256, (lanes, T + steps), generator=g, dtype=torch.uint8).cuda()
    u = torch.rand((lanes, T + steps), generator=g).cuda()
    whole, parts = Served(codec, dtype, lanes), Served(codec, dtype, lanes)
    at_once = torch.zeros((lanes, T + steps), dtype=torch.uint8, device="cuda")
    x8, s8, want = whole.run(tok, u, at_once)
    out = torch.zeros_like(at_once)
    got = [parts.run(tok[:, :T].contiguous(), u[:, :T].contiguous(), out[:, :T])]
    for t in range(T, T + steps):
        got.append(parts.run(tok[:, t:t + 1].contiguous(), u[:, t:t + 1].contiguous(), out[:, t:t + 1]))
    y8, logits = torch.cat([p[0] for p in got], 1), torch.cat([p[2] for p in got], 1)
    # between the two the rule's sums are in another order; a value next to a border
    # of two steps of 1 / 127 of its row's largest may go either way, and in the
    # second block everything may then differ by some of those steps.  They are one
    # in 254 of a value at most, of each of the five roundings to 8 bits (two a
    # block, one at the end), and bf16's four a block of 2^-9 are less: a tenth of
    # the whole, taken over the whole
    off = (logits.float() - want.float()).norm() / want.float().norm()
    assert off <= 0.1, off.item()
    assert (y8 == x8).float().mean() > 0.5
    # and what is chosen is what those logits say
    assert (out[:, :T + steps] == at_once).float().mean() > 0.5
    again = torch.zeros_like(out)
    codec.sample_bytes(logits, u, again, temperature=0.9, top_k=50, top_p=0.95)
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_served_step_in_a_graph(codec, dtype):  # noqa: F811
    lanes = 3
    model, same = Served(codec, dtype, lanes), Served(codec, dtype, lanes)
    tok = torch.zeros((lanes, 1), dtype=torch.uint8, device="cuda")
    u, out = torch.rand((lanes, 1), device="cuda"), torch.zeros((lanes, 1), dtype=torch.uint8, device="cuda")
    model.run(tok, u, out), same.run(tok, u, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        codec.set_stream(torch.cuda.current_stream().cuda_stream)
        _, _, logits = model.run(tok, u, out)
    codec.set_stream(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        tok.random_(0, 256), u.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.zeros_like(out)
        _, _, want = same.run(tok, u, eager)
        torch.cuda.synchronize()
        assert torch.equal(logits, want) and torch.equal(out, eager)
        assert all(torch.equal(a, b) for a, b in zip(model.states, same.states))


def test_a_training_step(codec):  # noqa: F811
    """Loss and gradients of the embedding and the norm's weight against autograd
    in 64 bits."""
    lanes, T = 3, 70
    g = torch.Generator().manual_seed(2)
    r = lambda *n: torch.randn(n, generator=g)  # noqa: E731
    tok = torch.randint(0, 256, (lanes, T), generator=g, dtype=torch.uint8)
    nxt = torch.randint(0, 256, (lanes, T), generator=g, dtype=torch.uint8)
    p = {"table": r(256, D), "norm": 1 + 0.2 * r(D), "open": r(D, N) / D ** 0.5,
         "head": r(HV * DV, 256) / (HV * DV) ** 0.5}
    scale = 1 / math.sqrt(DK)

    # 64 bits
    e = {n: t.double().requires_grad_() for n, t in p.items()}
    x = e["table"][tok.long()]
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * e["norm"] @ e["open"]
    q, k, v = (y[..., a:b] for a, b in ((0, DK), (DK, 2 * DK), (2 * DK, 2 * DK + HV * DV)))
    q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + delta_ref.EPS) for t in (q, k))
    decay = -torch.nn.functional.softplus(y[..., -2 * HV:-HV])
    beta, v = torch.sigmoid(y[..., -HV:]), v.reshape(lanes, T, HV, DV)
    S, outs = torch.zeros((lanes, HV, DK, DV), dtype=torch.float64), []
    for t in range(T):
        S = S * torch.exp(decay[:, t])[..., None, None]
        err = v[:, t] - (S * k[:, t, None, :, None]).sum(2)
        S = S + (beta[:, t, :, None, None] * k[:, t, None, :, None]) * err[..., None, :]
        outs.append((S * q[:, t, None, :, None]).sum(2) * scale)
    z = torch.stack(outs, 1).reshape(lanes, T, HV * DV) @ e["head"]
    nll = torch.nn.functional.cross_entropy(z.view(-1, 256), nxt.view(-1).long(), reduction="sum")
    nll.backward()

    # here
    w = {n: dev(t) for n, t in p.items()}
    zeros = lambda *n: torch.zeros(n, device="cuda")  # noqa: E731
    x, n1 = zeros(lanes, T, D), zeros(lanes, T, D)
    codec.embed(dev(tok), w["table"], x)
    codec.rms_norm(x, n1, d_weight=w["norm"], eps=EPS)
    n1.requires_grad_()
    y = n1 @ w["open"]
    decay = -torch.nn.functional.softplus(y[..., -2 * HV:-HV])
    beta = torch.sigmoid(y[..., -HV:])
    q, k, v = (y[..., a:b] for a, b in ((0, DK), (DK, 2 * DK), (2 * DK, 2 * DK + HV * DV)))
    sizes = (lanes, T, H, HV, DK, DV)
    o, saved = zeros(lanes, T, HV * DV), zeros(boa_hip.delta_rule_saved_floats(*sizes))
    wk = work(boa_hip.delta_rule_work_bytes(*sizes, grad=True))
    rows = [t.detach() for t in (q, k, v, decay, beta)]
    how = dict(heads=H, scale=scale, unit_qk=True)
    codec.delta_rule(*rows, o, wk, d_saved=saved, **how)
    logits = o @ w["head"]
    loss, total, dz = zeros(lanes, T), zeros(1), zeros(lanes, T, 256)
    codec.next_byte_loss(logits, dev(nxt), loss, work(boa_hip.next_byte_loss_work_bytes(lanes, T)),
                         d_total=total, d_dlogits=dz)
    grads = [torch.zeros_like(t) for t in rows]
    codec.delta_rule_grad(*rows, saved, dz @ w["head"].t(), *grads, wk, **how)
    dn, = torch.autograd.grad([q, k, v, decay, beta], [n1], grads)
    dx, dnorm, dtable = zeros(lanes, T, D), zeros(D), zeros(256, D)
    codec.rms_norm_grad(x, dn, dx, work(boa_hip.rms_norm_grad_work_bytes(lanes, T, D)),
                        d_weight=w["norm"], d_dweight=dnorm, eps=EPS)
    codec.embed_grad(dev(tok), dx, dtable, work(boa_hip.embed_grad_work_bytes(lanes, T, D)))

    # ten operators there and ten back; a sum's roundings, of 256 terms at most and
    # over 70 positions, are of the norm less than 2^-24 * 64 each; a chunk's
    # inverse, of a matrix whose entries are below 1, may enlarge them by its own
    # size, 8 for keys that are not alike
    limit = U * 64 * 20 * 8
    assert abs(loss.double().sum().item() - nll.item()) <= limit * nll.item()
    for name, got in (("table", dtable), ("norm", dnorm)):
        want = e[name].grad
        off = (got.cpu().double() - want).norm() / want.norm()
        assert off <= limit, (name, off.item(), limit)
