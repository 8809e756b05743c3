"""The gated delta rule and its gradient in 64 bits, and bounds on what fp32
arithmetic may be off by.

Values come from the recurrence, position by position, gradients from
differentiating it (torch's autograd in 64 bits).  The bounds come from the
formulas in chunks of 64 positions, carried in `M`: a matrix with an error
bound, where a sum of n products adds (n + 4) U of the sum of their magnitudes
(n + 3 roundings whatever the order, and operands taken apart into bfloat16
parts whose products of less than 2^-24 are left out), and an elementwise
operation its operands' errors and half a step of its result.  The inverse of
1 + A adds |T| (error of A + 3 n U (1 + |A|)) |T|, from substitution in rows
and blocks.
"""
import torch

from training_ref import U

C, EPS = 64, 1e-6


class M:
    def __init__(self, val, err=None):
        self.val, self.err = val, torch.zeros_like(val) if err is None else err

    def __matmul__(self, o):
        n = self.val.shape[-1]
        a, b = self.val.abs(), o.val.abs()
        return M(self.val @ o.val, a @ o.err + self.err @ b + self.err @ o.err
                 + (n + 4) * U * (a @ b))

    def __mul__(self, o):
        o = o if isinstance(o, M) else M(torch.as_tensor(o, dtype=torch.float64))
        p = self.val * o.val
        return M(p, self.val.abs() * o.err + o.val.abs() * self.err + self.err * o.err
                 + U * p.abs())

    def __add__(self, o):
        s = self.val + o.val
        return M(s, self.err + o.err + U * s.abs())

    def __neg__(self):
        return M(-self.val, self.err)

    def __sub__(self, o):
        return self + -o

    def sum(self, dim):
        n = self.val.shape[dim]
        return M(self.val.sum(dim, keepdim=True), self.err.sum(dim, keepdim=True)
                 + n * U * self.val.abs().sum(dim, keepdim=True))

    @property
    def t(self):
        return M(self.val.transpose(-1, -2), self.err.transpose(-1, -2))

    def only(self, mask):
        return M(self.val * mask, self.err * mask)


def function(val, steps=4):
    """a value off by a few half-steps of itself"""
    return M(val, steps * U * val.abs())


def recurrence(s, heads, scale, unit, live, grad=False):
    """(values, gradients): dicts of 64-bit tensors shaped as the rows."""
    names = ["q", "k", "v", "g", "beta"] + (["state_in"] if s.get("state_in") is not None else [])
    x = {n: s[n].detach().double().requires_grad_(grad) for n in names}
    lanes, T, hv = s["g"].shape
    dk, dv = s["q"].shape[2] // heads, s["v"].shape[2] // hv

    def wide(t):
        t = t.view(lanes, T, heads, dk)
        if unit:
            t = t / torch.sqrt((t * t).sum(-1, keepdim=True) + EPS)
        return t.repeat_interleave(hv // heads, 2)

    q, k, v = wide(x["q"]), wide(x["k"]), x["v"].view(lanes, T, hv, dv)
    S = x["state_in"] if "state_in" in x else torch.zeros((lanes, hv, dk, dv), dtype=torch.float64)
    outs = []
    for t in range(T):
        on = live[:, t, None, None, None]
        kept = S * torch.exp(x["g"][:, t])[..., None, None]
        e = v[:, t] - (kept * k[:, t, :, :, None]).sum(2)
        new = kept + (x["beta"][:, t, :, None] * k[:, t])[..., None] * e[..., None, :]
        S = torch.where(on, new, S)
        outs.append((S * q[:, t, :, :, None]).sum(2) * scale)
    out = torch.stack(outs, 1).reshape(lanes, T, hv * dv) * live[..., None]
    got = {"out": out.detach(), "state_out": S.detach()}
    if not grad:
        return got, None
    total = (out * s["dout"].double() * live[..., None]).sum()
    if s.get("dstate_out") is not None:
        total = total + (S * s["dstate_out"].double()).sum()
    gs = torch.autograd.grad(total, [x[n] for n in names], allow_unused=True)
    grads = {"d" + n: (torch.zeros_like(x[n]) if gi is None else gi) for n, gi in zip(names, gs)}
    return got, grads


def _segment(lanes, hv, T, dk, dv):
    """chunks of a segment: few long sequences are cut, each segment taken from a
    zero state and from the identity first"""
    chunks, wide = -(-T // C), 64 if dk <= 64 else 128
    n = int((16 * chunks) ** 0.5)
    n = min(n, 256 // (lanes * hv * (-(-dv // 64) + wide // 64)))
    return chunks if chunks < 8 or n < 3 else -(-chunks // n)


def _firsts(S, step, free, dk, chunks, each, back):
    """The segments' first states from the first one's: step(c, S) is a chunk's,
    free(c, S) without what it adds."""
    order = range(0, chunks, each)
    firsts = {}
    for at in (reversed(order) if back else order):
        firsts[at] = S
        local = M(torch.zeros_like(S.val))
        eye = torch.eye(dk, dtype=torch.float64).expand(*S.val.shape[:-2], dk, dk)
        move = M(eye)
        inside = range(at, min(at + each, chunks))
        for c in inside:  # the moves are the forward pass's, whichever way they are used
            move = free(c, move)
        for c in (reversed(inside) if back else inside):
            local = step(c, local)
        S = (move.t if back else move) @ S + local
    return firsts


def _chunked(t, heads, live):
    lanes, T, width = t.shape
    n = -(-T // C)
    p = torch.zeros((lanes, n * C, width), dtype=torch.float64)
    p[:, :T] = torch.where(live[..., None], t.double(), torch.zeros((), dtype=torch.float64))
    return p.view(lanes, n, C, heads, width // heads).permute(0, 3, 1, 2, 4)


def bounds(s, heads, scale, unit, live, grad=False):
    """Error bounds of fp32 results, shaped as the rows."""
    lanes, T, hv = s["g"].shape
    group, dk = hv // heads, s["q"].shape[2] // heads
    dv = s["v"].shape[2] // hv

    def rows(t):  # [lanes, h, n, C, d] -> [lanes, T, h d]
        return t.permute(0, 2, 3, 1, 4).reshape(lanes, -1, t.shape[1] * t.shape[4])[:, :T]

    def unit_of(t):
        t = _chunked(t, heads, live).repeat_interleave(group, 1)
        r = 1 / torch.sqrt((t * t).sum(-1, keepdim=True) + EPS) if unit else torch.ones_like(t[..., :1])
        r = M(r, (dk + 4) * U * r if unit else None)
        return M(t) * r, r

    (q, rq), (k, rk) = unit_of(s["q"]), unit_of(s["k"])
    v, beta = M(_chunked(s["v"], hv, live)), M(_chunked(s["beta"], hv, live))
    g = _chunked(torch.clamp(s["g"].double(), min=-1e4), hv, live)
    G = g.cumsum(3)
    low = torch.ones((C, C), dtype=torch.float64).tril()
    D = function(torch.exp(torch.where(low > 0, G - G.transpose(-1, -2), torch.zeros(()).double()))
                 * low)
    since, left = function(torch.exp(G)), function(torch.exp(G[:, :, :, -1:] - G))
    kk = ((k @ k.t) * D).only(low.tril(-1))
    A = kk * beta
    P = ((q @ k.t) * D * scale).only(low)
    eye = torch.eye(C, dtype=torch.float64)
    inv = torch.linalg.inv(eye + A.val)
    T_ = M(inv, inv.abs() @ (A.err + 3 * C * U * (eye + A.val.abs())) @ inv.abs())
    W, Un = T_ @ (k * beta * since), T_ @ (v * beta)
    n = g.shape[2]
    at = lambda m, c: M(m.val[:, :, c], m.err[:, :, c])  # noqa: E731
    stack = lambda ms: M(torch.stack([m.val for m in ms], 2),  # noqa: E731
                         torch.stack([m.err for m in ms], 2))
    S = M(s["state_in"].double() if s.get("state_in") is not None
          else torch.zeros((lanes, hv, dk, dv), dtype=torch.float64))
    kl, all_ = k * left, at(since, slice(None))
    all_ = M(since.val[:, :, :, -1:], since.err[:, :, :, -1:])
    each = _segment(lanes, hv, T, dk, dv)
    zero = M(torch.zeros((), dtype=torch.float64))

    def step(c, S, add=True):
        N = (at(Un, c) if add else zero) - at(W, c) @ S
        return S * at(all_, c) + at(kl, c).t @ N

    free = lambda c, S: step(c, S, False)  # noqa: E731
    firsts = {} if each == n else _firsts(S, step, free, dk, n, each, False)
    Ss, Ns = [], []
    for c in range(n):
        S = firsts.get(c, S)
        Ss.append(S)
        Ns.append(at(Un, c) - at(W, c) @ S)
        S = S * at(all_, c) + at(kl, c).t @ Ns[-1]
    S0, N = stack(Ss), stack(Ns)
    qs = q * since * scale
    got = {"out": rows((qs @ S0 + P @ N).err), "state_out": S.err}
    if not grad:
        return got, None
    dO = M(_chunked(s["dout"], hv, live))
    dN = P.t @ dO
    dS = M(s["dstate_out"].double() if s.get("dstate_out") is not None
           else torch.zeros((lanes, hv, dk, dv), dtype=torch.float64))
    def back(c, dS):
        d = at(dN, c) + at(kl, c) @ dS
        return dS * at(all_, c) + at(qs, c).t @ at(dO, c) - at(W, c).t @ d

    lasts = {} if each == n else _firsts(dS, back, free, dk, n, each, True)
    dSs, dNs = [], []
    for c in reversed(range(n)):
        if c == n - 1 or (c + 1) % each == 0:
            dS = lasts.get(c // each * each, dS)
        dSs.append(dS)
        dNs.append(at(dN, c) + at(kl, c) @ dS)
        dS = dS * at(all_, c) + at(qs, c).t @ at(dO, c) - at(W, c).t @ dNs[-1]
    dS0, dN = stack(dSs[::-1]), stack(dNs[::-1])
    dR = T_.t @ dN
    dA, dP = (-(dR @ N.t)).only(low.tril(-1)), (dO @ N.t).only(low)
    os, ns, rs = dO @ S0.t, N @ dS0.t, dR @ S0.t
    e1, e2 = dP * D * scale, dA * D * beta
    dq = os * since * scale + e1 @ k
    dkey = e1.t @ q + (e2 + e2.t) @ k + ns * left - rs * since * beta
    drow = (rs * k).sum(-1) * since
    dbeta = (dR * v).sum(-1) - drow + (dA * kk).sum(-1)
    m = dA * A + dP * P
    last = (ns * k).sum(-1) * left
    dG = m.sum(-1) - m.sum(-2).t - last + (os * qs).sum(-1) - drow * beta
    tail = last.sum(-2) + all_ * M((dS0 * S0).sum(-1).sum(-2).val, (dS0 * S0).sum(-1).sum(-2).err)
    dG = M(dG.val + 0, dG.err)
    dG.val[:, :, :, -1:] += tail.val
    dG.err[:, :, :, -1:] += tail.err + U * tail.val.abs()
    dg = dG.err.flip(3).cumsum(3).flip(3) + C * U * dG.val.abs().flip(3).cumsum(3).flip(3)

    def through(d, u, r):  # the heads that share a row, then the division by its length
        view = lambda t: t.reshape(lanes, heads, group, n, C, -1)  # noqa: E731
        d = M(view(d.val), view(d.err)).sum(2)
        u, r = M(view(u.val)[:, :, :1], view(u.err)[:, :, :1]), M(view(r.val)[:, :, :1],
                                                                  view(r.err)[:, :, :1])
        if unit:
            d = (d - u * (u * d).sum(-1)) * r
        return rows(d.err[:, :, 0])

    grads = {"dq": through(dq, q, rq), "dk": through(dkey, k, rk), "dv": rows((dR * beta).err),
             "dg": rows(dg), "dbeta": rows(dbeta.err), "dstate_in": dS.err}
    return got, grads


def check(name, got, want, err, dtype=None):
    """got within the bound (and, stored in bfloat16, half a step) of want"""
    dtype = dtype or got.dtype
    tol = err + U * want.abs() + 2.0 ** -126
    if dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (want.abs() + err)
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all().item(), f"{name}: not finite"
    worst = (off / tol).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} times its bound (largest error {off.max().item():.3g})"
