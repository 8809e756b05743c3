"""What the gated delta rule may be off by where bounds on single elements say
little: errors that are carried on from chunk to chunk.

With unit keys and betas up to 1 a position's move, e^g (1 - beta k k^T), makes
no state longer, so the errors that chunks add are summed, not multiplied, and a
result's error as a norm stays near that of a single chunk.  How large that is,
the same formulas in chunks say when torch computes them in fp32 on the CPU: off
by `off32` of the norm.  A limit is 12 off32 + 256 U:
 - 12, about sqrt(128): torch adds a sum of up to 128 products in blocks, the
   matrix instructions add them one after the other, with that many more
   roundings between, of random signs;
 - 256 U: a chain of up to 22 segments, each a product of d_k (sqrt(128) < 12)
   roundings that the chunks alone do not have.
Rows in bfloat16 add half a step of each element, at most 2^-8 of the norm.
"""
import torch

import delta_ref as ref
from training_ref import U

C = ref.C


def chunked(s, heads, scale, live, dtype, each=None, mode=None):
    """The rule in chunks, differentiable, in `dtype`.  each, mode: sequences in
    segments of that many chunks whose moves M (state before -> after) are
    mistaken: "drop" and "across" (M^T) for the states, "back drop" and "back
    across" for their gradients alone."""
    lanes, T, hv = s["g"].shape
    group, dk = hv // heads, s["q"].shape[2] // heads

    def unit(t):
        t = cut(t, heads).repeat_interleave(group, 1)
        return t / torch.sqrt((t * t).sum(-1, keepdim=True) + ref.EPS)

    n = -(-T // C)

    def cut(t, h):
        t = torch.where(live[..., None], t.to(dtype if t.dtype != torch.float64 else t.dtype),
                        torch.zeros((), dtype=t.dtype if t.dtype == torch.float64 else dtype))
        t = torch.cat([t, torch.zeros((lanes, n * C - T, t.shape[2]), dtype=t.dtype)], 1)
        return t.view(lanes, n, C, h, -1).permute(0, 3, 1, 2, 4)

    q, k, v, beta = unit(s["q"]), unit(s["k"]), cut(s["v"], hv), cut(s["beta"], hv)
    G = cut(s["g"].double(), hv).cumsum(3)
    low = torch.ones((C, C), dtype=dtype).tril()
    D = torch.exp(torch.where(low > 0, G - G.transpose(-1, -2), torch.zeros_like(G))).to(dtype) * low
    since, left = torch.exp(G).to(dtype), torch.exp(G[:, :, :, -1:] - G).to(dtype)
    A = (k @ k.transpose(-1, -2)) * D * low.tril(-1) * beta
    P = (q @ k.transpose(-1, -2)) * D * scale
    one = torch.eye(C, dtype=dtype) + A

    def solve(c, x):
        return torch.linalg.solve_triangular(one[:, :, c], x, upper=False, unitriangular=True)

    def step(c, S, add):
        r = -(k[:, :, c] @ S) * (beta * since)[:, :, c]
        if add:
            r = r + v[:, :, c] * beta[:, :, c]
        N = solve(c, r)
        return S * since[:, :, c, -1:], N, (k * left)[:, :, c].transpose(-1, -2) @ N

    S, outs = s["state_in"].to(dtype), []
    for at in range(0, n, each or n):
        inside = range(at, min(at + (each or n), n))
        first = S
        for c in inside:
            kept, N, new = step(c, S, True)
            outs.append((q[:, :, c] @ S) * (since[:, :, c] * scale) + P[:, :, c] @ N)
            S = kept + new
        if mode:
            local, M = torch.zeros_like(first), torch.eye(dk, dtype=dtype).expand(*S.shape[:2], dk, dk)
            for c in inside:
                kept, _, new = step(c, local, True)
                local = kept + new
                kept, _, new = step(c, M, False)
                M = (kept + new).detach()
            right, across = M @ first, M.transpose(-1, -2) @ first
            S = local + {"right": right, "drop": 0, "across": across, "back drop": right.detach(),
                         "back across": (right - across).detach() + across}[mode]
    out = torch.stack(outs, 2).permute(0, 2, 3, 1, 4).reshape(lanes, n * C, -1)[:, :T]
    return {"out": out * live[..., None], "state_out": S}


def results(f, s, grad):
    """f's outputs of s and, if `grad`, the gradients with those of s's outputs"""
    names = ["q", "k", "v", "g", "beta", "state_in"]
    x = {n: s[n].detach().clone().requires_grad_(grad) for n in names}
    got = f(x)
    if not grad:
        return {n: t.detach() for n, t in got.items()}
    total = sum((got[n] * s[d].to(got[n].dtype)).sum() for n, d in (("out", "dout"),
                                                                    ("state_out", "dstate_out")))
    grads = torch.autograd.grad(total, [x[n] for n in names], allow_unused=True)
    return {**{n: t.detach() for n, t in got.items()},
            **{"d" + n: torch.zeros_like(x[n]) if g is None else g for n, g in zip(names, grads)}}


def off(got, want):
    """[lanes]: the norm of what a lane's result is off by, as a share of its own"""
    d = (got.double() - want.double()).flatten(1).norm(dim=1)
    n = want.double().flatten(1).norm(dim=1)
    return torch.where(n > 0, d / n.clamp_min(1e-300), d)


def limits(s, heads, scale, live, want, grad=True):
    """name -> [lanes]: what each result may be off by"""
    at32 = {n: s[n].float() for n in s}
    got = results(lambda x: chunked(x, heads, scale, live, torch.float32), at32, grad)
    return {n: 12 * off(got[n], want[n]) + 256 * U for n in got}


def exact(s, heads, scale, live, grad=True):
    got, grads = ref.recurrence(s, heads, scale, True, live, grad)
    return {**got, **(grads or {})}


SHAPES = [  # lanes, T, heads, v heads, d_k, d_v, layout, lens, kind
    # cut into segments through which the states live on
    (1, 600, 1, 2, 64, 64, "dense", "full", "long"), (2, 1100, 1, 2, 33, 80, "odd", "ragged", "long"),
    (3, 700, 1, 1, 80, 70, "wide", "ragged", "long"), (1, 900, 2, 2, 128, 128, "dense", "full", "long"),
    (2, 640, 1, 2, 128, 64, "time", "ragged", "long"),
    # the same key again and again, and states that nothing makes shorter
    (3, 700, 1, 2, 80, 70, "wide", "ragged", "same"), (1, 900, 2, 2, 128, 128, "dense", "full", "none"),
    (1, 63, 1, 1, 64, 64, "dense", "full", "same"), (3, 129, 2, 4, 128, 128, "dense", "ragged", "same"),
    (70, 150, 2, 4, 33, 20, "dense", "ragged", "long"), (5, 200, 2, 2, 64, 128, "odd", "ragged", "none")]


def inputs(lanes, T, heads, hv, dk, dv, dtype, kind):
    g = torch.Generator().manual_seed(lanes * 1000 + T + dk + 3 * dv)
    r = lambda *n: torch.randn(n, generator=g)  # noqa: E731
    s = {"q": r(lanes, T, heads * dk), "k": r(lanes, T, heads * dk), "v": r(lanes, T, hv * dv),
         "g": -torch.exp(r(lanes, T, hv)) * 1e-3, "beta": 0.02 + 0.08 * torch.rand((lanes, T, hv), generator=g),
         "state_in": r(lanes, hv, dk, dv), "dout": r(lanes, T, hv * dv) * 0.1,
         "dstate_out": r(lanes, hv, dk, dv)}
    if kind == "same":
        s["k"] = s["k"][:, :1].expand(lanes, T, heads * dk) + 1e-3 * s["k"]
        s["beta"] = torch.ones_like(s["beta"])
        s["g"] = s["g"] * 0.1
    elif kind == "none":
        s["g"] = torch.zeros_like(s["g"])
        s["beta"] = torch.sigmoid(r(lanes, T, hv)) * (torch.rand((lanes, T, hv), generator=g) < 0.5)
    for n in ("q", "k", "v", "dout"):
        s[n] = s[n].to(dtype)
    return s, g
