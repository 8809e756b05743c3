"""The training operators in 64 bits, each value with a bound on what fp32
arithmetic may be off by.

`V` carries a float64 value and an error bound through the formulas: every
fp32 operation adds half a step of its result (U = 2^-24 of it), a function
the error of its argument and a few steps of its own, a sum of n terms n
half-steps of the sum of their magnitudes (whatever its order).  So a test
states its formula once and gets its tolerance from it; what is stored in
bf16 adds half a step (2^-8) at the end.
"""
import math

import torch

U = 2.0 ** -24


class V:
    def __init__(self, val, err=None):
        self.val = val
        self.err = torch.zeros_like(val) if err is None else err

    def __add__(self, o):
        o = of(o, self.val)
        s = self.val + o.val
        return V(s, self.err + o.err + U * s.abs())

    def __mul__(self, o):
        o = of(o, self.val)
        p = self.val * o.val
        return V(p, self.val.abs() * o.err + o.val.abs() * self.err + self.err * o.err
                 + U * p.abs())

    __radd__, __rmul__ = __add__, __mul__

    def __neg__(self):
        return V(-self.val, self.err)

    def __sub__(self, o):
        return self + -of(o, self.val)

    def __getitem__(self, i):
        return V(self.val[i], self.err[i])

    def sum(self, dim):
        dims = (dim,) if isinstance(dim, int) else dim
        n = math.prod(self.val.shape[d] for d in dims)
        return V(self.val.sum(dims), self.err.sum(dims) + n * U * self.val.abs().sum(dims))

    def exp(self):  # the argument in base 2: three roundings; the function: two
        e = torch.exp(self.val)
        return V(e, torch.exp(self.val + self.err + 3 * U * self.val.abs()) * (1 + 2 * U) - e)

    def sigmoid(self):  # 1 / (1 + e^-x): slope at most its value or 1 - its value
        s = torch.sigmoid(self.val)
        return V(s, s * ((1 - s) * (torch.expm1(self.err + 3 * U * self.val.abs()) + 2 * U)
                         + 4 * U))

    def softplus(self):  # log(1 + e^x); slope sigmoid(x) <= softplus(x)
        s = torch.nn.functional.softplus(self.val, threshold=1e9)
        slope = torch.sigmoid(self.val)
        # e^-|x| off by 3 |x| + 2 half-steps, the series and its quotient by 16
        return V(s, slope * self.err + torch.exp(-self.val.abs()) * (3 * self.val.abs() + 2) * U
                 + 16 * U * s)


def of(x, like):
    if isinstance(x, V):
        return x
    return V(torch.as_tensor(x, dtype=torch.float64).expand_as(like) if not torch.is_tensor(x)
             else x.double())


def stack(vs, dim):
    return V(torch.stack([v.val for v in vs], dim), torch.stack([v.err for v in vs], dim))


def stored(v, dtype):
    """(value, tolerance) of v stored as dtype; plus the least normal number,
    under which fp32 and bf16 have other steps."""
    tol = v.err + 2.0 ** -126
    if dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (v.val.abs() + v.err)
    return v.val, tol


def check(name, got, want, dtype=None):
    """got within the bound of want (a V), finite wherever want is."""
    val, tol = stored(want, dtype or got.dtype)
    off = (got.double().cpu() - val).abs()
    worst = (off / tol).max().item() if off.numel() else 0.0
    assert torch.isfinite(got).all().item(), f"{name}: not finite"
    assert worst <= 1.0, f"{name}: {worst:.3g} times its bound (largest error {off.max().item():.3g})"


def mask(lens, lanes, T):
    m = torch.ones((lanes, T), dtype=torch.bool)
    if lens is not None:
        for i, n in enumerate(lens.tolist()):
            m[i, max(0, min(n, T)):] = False
    return m


# ---------------------------------------------------------------- embedding
def embed(tokens, table, scale):
    return V(table.double()[tokens.long()]) * V(torch.tensor(scale, dtype=torch.float32).double())


def embed_grad(tokens, dout, scale, live):
    """sums by byte: at most as many roundings as there are rows of it"""
    out = []
    for v in range(256):
        d = dout[(tokens == v) & live].double()
        out.append(V(d.sum(0), len(d) * U * d.abs().sum(0)))
    return stack(out, 0) * V(torch.tensor(scale, dtype=torch.float32).double())


# --------------------------------------------------------------------- loss
def loss(logits, bias, targets, scale, live):
    """loss, total, dlogits, dbias; rows that are not live are zero."""
    x = V(logits.double())
    if bias is not None:
        x = x + V(bias.double())
    ninf = -math.inf
    x.err = torch.where(x.val == ninf, torch.zeros_like(x.err), x.err)
    top = x.val.amax(-1, keepdim=True)
    d = V(x.val - top, x.err + x.err.gather(-1, x.val.argmax(-1, keepdim=True))
          + U * (x.val - top).abs())
    gone = x.val == ninf
    d = V(torch.where(gone, torch.zeros_like(d.val), d.val),
          torch.where(gone, torch.zeros_like(d.err), d.err))
    e = d.exp()
    e = V(torch.where(gone, torch.zeros_like(e.val), e.val),
          torch.where(gone, torch.zeros_like(e.err), e.err))
    first = torch.nn.functional.one_hot(x.val.argmax(-1), 256).bool()
    rest = V(e.val * ~first, e.err * ~first).sum(-1)
    # log1p: slope 1 / (1 + rest), its own arithmetic 8 half-steps of it
    lp = torch.log1p(rest.val)
    lp = V(lp, rest.err / (1 + rest.val) + 8 * U * lp)
    hit = targets.long()[..., None]
    dt = d[...].val.gather(-1, hit)[..., 0]
    out = lp - V(dt, d.err.gather(-1, hit)[..., 0])
    total = rest + torch.ones_like(rest.val)
    inv = V(float(torch.tensor(scale, dtype=torch.float32)) / total.val,
            abs(scale) / total.val * (total.err / total.val + 2 * U))
    inv = V(inv.val[..., None].expand_as(e.val), inv.err[..., None].expand_as(e.val))
    one = torch.nn.functional.one_hot(targets.long(), 256).bool()
    at = V(e.val - total.val[..., None], e.err + total.err[..., None]
           + U * (e.val - total.val[..., None]).abs())
    # the largest logit's own gradient is minus the others' share
    both = one & first
    at = V(torch.where(both, -rest.val[..., None].expand_as(e.val), at.val),
           torch.where(both, rest.err[..., None].expand_as(e.val), at.err))
    grad = V(torch.where(one, at.val, e.val), torch.where(one, at.err, e.err)) * inv
    zero = lambda v, m: V(v.val * m, v.err * m)  # noqa: E731
    out, grad = zero(out, live), zero(grad, live[..., None])
    # the total is summed in 64 bits and rounded once
    tot = V(out.val.sum().view(1), out.err.sum().view(1) + U * out.val.sum().abs().view(1))
    return out, tot, grad, grad.sum((0, 1))


# --------------------------------------------------------------------- scan
def scan(s, live):
    """Forward of the inputs s (float tensors; state_in may be None): out,
    state_out and what the gradient needs."""
    w = {k: V(v.double()) for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    lanes, T, ch = s["u"].shape
    A = w["A"]
    n = A.val.shape[1]
    h = w.get("state_in") or V(torch.zeros((lanes, ch, n), dtype=torch.float64))
    x = w["delta"] + w["delta_bias"]
    delta = x.softplus()
    hs, ys, decays = [h], [], []
    for t in range(T):
        d = delta[:, t, :, None]
        a = (V(d.val.expand(lanes, ch, n), d.err.expand(lanes, ch, n)) * A).exp()
        du = delta[:, t] * w["u"][:, t]
        new = a * hs[-1] + du[:, :, None] * w["B"][:, t, None, :]
        on = live[:, t, None, None]
        hs.append(V(torch.where(on, new.val, hs[-1].val), torch.where(on, new.err, hs[-1].err)))
        ys.append((hs[-1] * w["C"][:, t, None, :]).sum(2) + w["D"] * w["u"][:, t])
        decays.append(a)
    y = stack(ys, 1)
    gate = w["z"].sigmoid()
    out = y * (w["z"] * gate)
    return out, hs[-1], dict(w=w, x=x, delta=delta, hs=hs, y=y, gate=gate, decays=decays)


def scan_grad(s, live, kept):
    w, x, delta, hs, y, sig = (kept[k] for k in ("w", "x", "delta", "hs", "y", "gate"))
    lanes, T, ch = s["u"].shape
    n = s["A"].shape[1]
    on = live[..., None].double()
    z, u, dout = w["z"], w["u"], w["dout"]
    zero = lambda v, m: V(v.val * m, v.err * m)  # noqa: E731
    dy = zero(dout * (z * sig), on)
    g = w.get("dstate_out") or V(torch.zeros((lanes, ch, n), dtype=torch.float64))
    cols = {k: [] for k in ("I", "M", "dB", "dC", "dA")}
    for t in reversed(range(T)):
        m4 = live[:, t, None, None].double()
        a = kept["decays"][t]
        dh = g + w["C"][:, t, None, :] * dy[:, t, :, None]
        nxt = a * dh
        m = zero(nxt * hs[t], m4)
        d = delta[:, t, :, None]
        cols["dA"].append(m * d)
        cols["M"].append((m * w["A"]).sum(2))
        cols["I"].append(zero((dh * w["B"][:, t, None, :]).sum(2), live[:, t, None].double()))
        du = (delta[:, t] * u[:, t])[:, :, None]
        cols["dB"].append(zero((dh * du).sum(1), live[:, t, None].double()))
        cols["dC"].append((hs[t + 1] * dy[:, t, :, None]).sum(1))
        keep = live[:, t, None, None]
        g = V(torch.where(keep, nxt.val, g.val), torch.where(keep, nxt.err, g.err))
    I, M, dB, dC, dA = (stack(cols[k][::-1], 1) for k in ("I", "M", "dB", "dC", "dA"))
    dx = zero((M + u * I) * x.sigmoid(), on)
    one = torch.ones_like(z.val)
    return {
        "du": dy * w["D"] + delta * I, "ddelta": dx,
        "dz": zero(dout * y * (sig * (z * (V(one) - sig) + one)), on),
        "dB": dB, "dC": dC, "dA": dA.sum((0, 1)), "dD": (dy * u).sum((0, 1)),
        "ddelta_bias": dx.sum((0, 1)), "dstate_in": g}
