"""Performance cases of the training operators: embedding, gated linear
recurrence (the selective scan) and next-byte loss, each with its gradient.

A case is one pass of one of five paths over rows = `lanes` x `T` (byte
sequences side by side, a row for each byte):

  embed       tokens -> scaled rows of the embedding table
  embed_grad  gradient of those rows -> gradient of the table
  scan        the recurrence forward, state in and out (T = 1: one decode step)
  scan_train  the recurrence forward and its gradients, as a training step
              runs them
  loss        logits and next bytes -> loss of every row, its sum, the
              gradients of the logits and of the head's bias

`precision` is the type of the row tensors ("fp32" or "bf16"); weights, states
and the gradients of weights are float32.  `ragged` cases have lanes of
different lengths, one of them empty: rows past a lane's length keep what the
output held (zero here), and their gradients are zero.
"""
import importlib
import math

import torch

own = False

# widths of the repository's models: (d_model, channels of the recurrence, d_state)
_WIDTHS = {"d64": (64, 128, 16), "d80": (80, 160, 16), "d256": (256, 512, 16),
           "d512": (512, 1024, 32)}


def _case(name, path, model, lanes, T, precision, ragged=False, data="records", masked=False):
    c = {"path": path, "model": model, "lanes": lanes, "T": T, "precision": precision,
         "ragged": ragged, "data": data, "masked": masked}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one byte of every stream that is decoded live
        _case("embed_step", "embed", "d64", 64, 1, "fp32"),
        # a training batch of whole chunks
        _case("embed_d256_bf16", "embed", "d256", 250, 2085, "bf16", ragged=True),
        # a few short texts
        _case("embed_grad_d256", "embed_grad", "d256", 37, 219, "fp32"),
        # a large batch in which most bytes are zero, as in sparse records
        _case("embed_grad_d256_sparse", "embed_grad", "d256", 1000, 521, "fp32", ragged=True,
              data="sparse"),
        # a decode step of a thousand lanes, state in and out
        _case("scan_step_d256", "scan", "d256", 1000, 1, "fp32"),
        # scoring one long text: a single sequence
        _case("scan_long_d64", "scan", "d64", 1, 16001, "fp32"),
        # fitting the small model to a few texts
        _case("scan_train_d64", "scan_train", "d64", 4, 257, "fp32"),
        # a training batch of the headline model in either precision
        _case("scan_train_d256", "scan_train", "d256", 16, 1041, "fp32", ragged=True),
        _case("scan_train_d256_bf16", "scan_train", "d256", 32, 1024, "bf16"),
        # the large model with 32 states a channel
        _case("scan_train_d512_bf16", "scan_train", "d512", 4, 777, "bf16", ragged=True),
        # the loss of a few bytes, and of a large batch whose alphabet is known
        _case("loss_small", "loss", "d64", 8, 9, "fp32"),
        _case("loss_large", "loss", "d256", 1000, 521, "fp32", ragged=True, masked=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    path = rng.choice(["embed", "embed_grad", "scan", "scan", "scan_train", "scan_train", "loss"])
    model = rng.choice(sorted(_WIDTHS))
    width, channels, n = _WIDTHS[model]
    precision = rng.choice(["fp32", "bf16"])
    data = rng.choice(["records", "sparse"])
    if path in ("scan", "scan_train"):
        rows = 32 * 1024 * 512 * 16 // (channels * n)  # as many states as the largest listed case
        lanes = _log_int(rng, 1, 256)
        T = 1 if path == "scan" and rng.random() < 0.25 else _log_int(
            rng, 2, max(2, min(16384, rows // lanes)))
    else:
        rows = 500000 if path == "loss" else 500000 * 256 // max(width, 256)
        lanes = _log_int(rng, 1, 1000)
        T = _log_int(rng, 1, max(1, min(65536, rows // lanes)))
    return _case(None, path, model, lanes, T, precision, ragged=lanes > 1 and rng.random() < 0.5,
                 data=data, masked=path == "loss" and rng.random() < 0.5)


# ------------------------------------------------------------------ inputs
def _tokens(case, g, extra):
    """[lanes, T + extra] bytes: little-endian float32 records as an instrument
    writes them, or records of which seven in eight are zero."""
    lanes, T = case["lanes"], case["T"] + extra
    k = (lanes * T + 3) // 4
    v = torch.round(torch.randn((k,), generator=g, device="cuda") * 1000) / 1000
    if case["data"] == "sparse":
        v = v * (torch.rand((k,), generator=g, device="cuda") < 0.125)
    return v.view(torch.uint8)[:lanes * T].view(lanes, T)


def _lens(case, g):
    if not case["ragged"]:
        return None
    lanes, T = case["lanes"], case["T"]
    n = torch.randint(0, T + 1, (lanes,), generator=g, device="cuda", dtype=torch.int32)
    n[0] = T
    n[-1] = 0
    return n


def _type(case):
    return torch.bfloat16 if case["precision"] == "bf16" else torch.float32


def prepare(case, seed):
    width, channels, n = _WIDTHS[case["model"]]
    lanes, T, path, dt = case["lanes"], case["T"], case["path"], _type(case)
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    s = {"case": case, "lens": _lens(case, g)}
    if path in ("embed", "embed_grad"):
        s["tokens"] = _tokens(case, g, 0)
        s["scale"] = math.sqrt(width)
        if path == "embed":
            s["table"] = (randn(256, width) / math.sqrt(width)).to(dt)
        else:
            s["dout"] = (randn(lanes, T, width) * 1e-2).to(dt)
    elif path == "loss":
        s["targets"] = _tokens(case, g, 1)[:, 1:]  # the byte after each of a chunk's
        s["logits"] = (randn(lanes, T, 256) * 2).to(dt)
        if case["masked"]:  # bytes that the records' format rules out
            s["logits"][:, :, 250:] = -math.inf
            s["targets"].clamp_(max=249)
        s["bias"] = randn(256) * 0.1
        s["scale"] = 1.0 / (lanes * T)
    else:
        # u beside z and B beside C, as the products before the scan leave them
        r = width // 16
        xz = randn(lanes, T, 2 * channels).to(dt)
        dbc = randn(lanes, T, r + 2 * n).to(dt)
        s["u"], s["z"] = xz[..., :channels], xz[..., channels:]
        s["B"], s["C"] = dbc[..., r:r + n], dbc[..., r + n:]
        s["delta"] = (randn(lanes, T, channels) * 0.5).to(dt)
        first = torch.exp(math.log(1e-3) + math.log(100.0)
                          * torch.rand((channels,), generator=g, device="cuda"))
        s["delta_bias"] = first + torch.log(-torch.expm1(-first))
        s["A"] = -torch.exp(torch.log(torch.arange(1, n + 1, device="cuda").float())
                            + 0.1 * randn(channels, n))
        s["D"] = 1 + 0.1 * randn(channels)
        s["state_in"] = randn(lanes, channels, n) * 0.1
        if path == "scan_train":
            s["dout"] = (randn(lanes, T, channels) * 1e-2).to(dt)
            s["dstate_out"] = randn(lanes, channels, n) * 1e-2
    if own:
        _own_state(s)
    return s


def _own_state(s):
    """What a program of this library keeps between calls: a context, outputs and workspaces."""
    boa = importlib.import_module("boa-constrictor_amd.boa_hip")
    case = s["case"]
    width, channels, n = _WIDTHS[case["model"]]
    lanes, T, path, dt = case["lanes"], case["T"], case["path"], _type(case)

    def zeros(*shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    s["codec"] = boa.Codec(64, 1, 16, max_lanes=1)
    s["codec"].set_stream(torch.cuda.current_stream().cuda_stream)
    work = 0
    if path == "embed":
        s["out"] = zeros(lanes, T, width, dtype=dt)
    elif path == "embed_grad":
        s["dtable"] = zeros(256, width)
        work = boa.embed_grad_work_bytes(lanes, T, width)
    elif path == "loss":
        s["loss"], s["total"] = zeros(lanes, T), zeros(1)
        s["dlogits"], s["dbias"] = zeros(lanes, T, 256, dtype=dt), zeros(256)
        work = boa.next_byte_loss_work_bytes(lanes, T)
    else:
        s["out"] = zeros(lanes, T, channels, dtype=dt)
        s["state_out"] = zeros(lanes, channels, n)
        work = boa.selective_scan_work_bytes(lanes, T, channels, n, grad=path == "scan_train")
        if path == "scan_train":
            s["saved"] = zeros(boa.selective_scan_saved_floats(lanes, T, channels, n))
            dxz = zeros(lanes, T, 2 * channels, dtype=dt)
            ddbc = zeros(lanes, T, width // 16 + 2 * n, dtype=dt)
            s["du"], s["dz"] = dxz[..., :channels], dxz[..., channels:]
            s["dB"], s["dC"] = ddbc[..., -2 * n:-n], ddbc[..., -n:]
            s["ddelta"] = zeros(lanes, T, channels, dtype=dt)
            s["dA"], s["dD"], s["ddelta_bias"] = zeros(channels, n), zeros(channels), zeros(channels)
            s["dstate_in"] = zeros(lanes, channels, n)
    s["work"] = zeros(work, dtype=torch.uint8)


# ---------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    return {"embed": _embed, "embed_grad": _embed_grad, "loss": _loss, "scan": _scan,
            "scan_train": _scan}[state["case"]["path"]](state)


def _run_own(s):
    path, codec = s["case"]["path"], s["codec"]
    if path == "embed":
        codec.embed(s["tokens"], s["table"], s["out"], scale=s["scale"], d_lens=s["lens"])
        return s["out"]
    if path == "embed_grad":
        codec.embed_grad(s["tokens"], s["dout"], s["dtable"], s["work"], scale=s["scale"],
                         d_lens=s["lens"])
        return s["dtable"]
    if path == "loss":
        codec.next_byte_loss(s["logits"], s["targets"], s["loss"], s["work"], d_bias=s["bias"],
                             d_total=s["total"], d_dlogits=s["dlogits"], d_dbias=s["dbias"],
                             scale=s["scale"], d_lens=s["lens"])
        return {k: s[k] for k in ("loss", "total", "dlogits", "dbias")}
    args = [s[k] for k in ("u", "delta", "z", "B", "C", "A", "D", "delta_bias")]
    codec.selective_scan(*args, s["out"], s["work"], d_state_in=s["state_in"],
                         d_state_out=s["state_out"], d_lens=s["lens"], d_saved=s.get("saved"))
    names = ["out", "state_out"]
    if path == "scan_train":
        grads = ["du", "ddelta", "dz", "dB", "dC", "dA", "dD", "ddelta_bias"]
        codec.selective_scan_grad(*args, s["saved"], s["dout"], *[s[k] for k in grads], s["work"],
                                  d_state_in=s["state_in"], d_dstate_out=s["dstate_out"],
                                  d_dstate_in=s["dstate_in"], d_lens=s["lens"])
        names += grads + ["dstate_in"]
    return {k: s[k] for k in names}


# ------------------------------------------------- the operators' plain form
def _mask(s):
    """[lanes, T, 1]: 1 where a row lies within its lane's length."""
    case = s["case"]
    if s["lens"] is None:
        return torch.ones((case["lanes"], case["T"], 1), device="cuda")
    return (torch.arange(case["T"], device="cuda") < s["lens"][:, None]).float()[..., None]


def _embed(s):
    rows = s["table"].float()[s["tokens"].long()] * s["scale"]
    return (rows * _mask(s)).to(s["table"].dtype)


def _embed_grad(s):
    # a product with the bytes' 256 truth values, in 64 bits: a sum may run over most rows
    d = (s["dout"].double() * _mask(s)).view(-1, s["dout"].shape[-1])
    hit = s["tokens"].reshape(-1)[:, None] == torch.arange(256, device="cuda")
    return (torch.matmul(hit.double().t(), d) * s["scale"]).float()


def _loss(s):
    on = _mask(s)
    x = s["logits"].float() + s["bias"]
    x = x - x.amax(-1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(-1, keepdim=True)
    hit = s["targets"].long()[..., None]
    loss = (torch.log(total) - x.gather(-1, hit)) * on
    grad = e / total
    grad.scatter_add_(-1, hit, torch.full_like(loss, -1.0))
    grad = grad * on * s["scale"]
    return {"loss": loss[..., 0], "total": loss.double().sum().float().view(1),
            "dlogits": grad.to(s["logits"].dtype), "dbias": grad.sum((0, 1))}


def _recurrence(a, b):
    """h[:, t] = a[:, t] h[:, t - 1] + b[:, t] from h[:, -1] = 0, by doubling spans."""
    k, T = 1, a.shape[1]
    while k < T:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return b


def _scan(s):
    on, dt = _mask(s), s["u"].dtype
    u, z, B, C = (s[k].float() * on for k in ("u", "z", "B", "C"))
    x = s["delta"].float() + s["delta_bias"]
    delta = (torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))) * on
    decay = torch.exp(delta[..., None] * s["A"])
    enter = (delta * u)[..., None] * B[:, :, None, :]
    enter[:, 0] += decay[:, 0] * s["state_in"]
    h = _recurrence(decay, enter)
    del enter
    y = (h * C[:, :, None, :]).sum(-1) + s["D"] * u
    gate = torch.sigmoid(z)
    got = {"out": (y * z * gate).to(dt), "state_out": h[:, -1].contiguous()}
    if s["case"]["path"] == "scan":
        return got
    dout = s["dout"].float() * on
    dy = dout * z * gate
    # dh[t] = C[t] dy[t] + decay[t + 1] dh[t + 1], from the last row to the first
    right = torch.cat([torch.ones_like(decay[:, :1]), decay[:, 1:].flip(1)], 1)
    enter = (C[:, :, None, :] * dy[..., None]).flip(1)
    enter[:, 0] += s["dstate_out"]
    dh = _recurrence(right, enter).flip(1)
    del right, enter
    into = (dh * B[:, :, None, :]).sum(-1)
    before = torch.cat([s["state_in"][:, None], h[:, :-1]], 1)
    m = dh * before * decay
    del before
    ddelta = ((m * s["A"]).sum(-1) + into * u) * torch.sigmoid(x) * on
    got.update(
        du=(dy * s["D"] + into * delta).to(dt), ddelta=ddelta.to(dt),
        dz=(dout * y * gate * (1 + z * (1 - gate))).to(dt),
        dB=((dh * (delta * u)[..., None]).sum(2) * on).to(dt),
        dC=((h * dy[..., None]).sum(2) * on).to(dt),
        dA=(m * delta[..., None]).sum((0, 1)), dD=(dy * u).sum((0, 1)),
        ddelta_bias=ddelta.sum((0, 1)), dstate_in=dh[:, 0] * decay[:, 0])
    return got


# ----------------------------------------------------------- what it needs
def work(case):
    """Each input read and each output written once; multiplications and
    additions (and an exponential as one operation) of the formulas."""
    width, channels, n = _WIDTHS[case["model"]]
    lanes, rows, path = case["lanes"], case["lanes"] * case["T"], case["path"]
    size = 2 if case["precision"] == "bf16" else 4
    if path == "embed":
        return {"bytes": rows * (1 + width * size) + 256 * width * size, "flops": rows * width}
    if path == "embed_grad":
        return {"bytes": rows * (1 + width * size) + 256 * width * 4, "flops": rows * width}
    if path == "loss":
        return {"bytes": rows * (1 + 4 + 2 * 256 * size), "flops": rows * 256 * 8}
    states = 4 * lanes * channels * n
    moved = rows * size * (4 * channels + 2 * n) + 2 * states + 4 * channels * (n + 2)
    flops = rows * channels * (7 * n + 20)
    if path == "scan_train":
        moved += rows * size * (7 * channels + 4 * n) + 2 * states + 8 * channels * (n + 2)
        flops += rows * channels * (21 * n + 40)
    return {"bytes": moved, "flops": flops}


# -------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    lanes, T, path = case["lanes"], case["T"], case["path"]
    lens = [T] * lanes if s["lens"] is None else s["lens"].tolist()
    valid = torch.zeros((lanes, T), dtype=torch.bool, device="cuda")
    for i, k in enumerate(lens):
        valid[i, :k] = True
    if path == "embed":
        out = torch.zeros((lanes, T, s["table"].shape[1]), dtype=torch.float64, device="cuda")
        for v in range(256):
            out[(s["tokens"] == v) & valid] = s["table"][v].double() * s["scale"]
        return out
    if path == "embed_grad":
        return torch.stack([s["dout"][(s["tokens"] == v) & valid].double().sum(0) * s["scale"]
                            for v in range(256)])
    if path == "loss":
        logp = torch.log_softmax((s["logits"].double() + s["bias"].double()), -1)
        pick = torch.nn.functional.one_hot(s["targets"].long(), 256).bool()
        loss = -logp[pick].view(lanes, T)
        loss[~valid] = 0
        grad = (torch.exp(logp) - pick.double()) * s["scale"]
        grad[~valid] = 0
        return {"loss": loss, "total": loss.sum().view(1), "dlogits": grad,
                "dbias": grad.view(-1, 256).sum(0)}
    return _exact_scan(s, valid)


def _exact_scan(s, valid):
    w = {k: v.double() for k, v in s.items()
         if isinstance(v, torch.Tensor) and v.is_floating_point()}
    u, z, B, C, A, D = (w[k] for k in ("u", "z", "B", "C", "A", "D"))
    x = w["delta"] + w["delta_bias"]
    delta = torch.logaddexp(x, torch.zeros_like(x))
    T, on = u.shape[1], valid.double()
    hs, ys = [w["state_in"]], []
    for t in range(T):
        d = delta[:, t, :, None]
        new = torch.exp(d * A) * hs[-1] + d * u[:, t, :, None] * B[:, t, None, :]
        hs.append(torch.where(valid[:, t, None, None], new, hs[-1]))
        ys.append(torch.matmul(hs[-1], C[:, t, :, None])[..., 0] + D * u[:, t])
    y = torch.stack(ys, 1)
    silu = torch.nn.functional.silu(z)
    got = {"out": y * silu * on[..., None], "state_out": hs[-1]}
    if s["case"]["path"] == "scan":
        return got
    dy = w["dout"] * silu
    sig = torch.sigmoid(z)
    dh, dA = w["dstate_out"], torch.zeros_like(A)
    into, through, dB, dC = [], [], [], []
    for t in reversed(range(T)):
        here, d = valid[:, t, None, None], delta[:, t, :, None]
        full = dh + dy[:, t, :, None] * C[:, t, None, :]
        a = torch.exp(d * A)
        m = full * a * hs[t] * on[:, t, None, None]
        dA += (m * d).sum(0)
        through.append((m * A).sum(-1))
        into.append(torch.matmul(full, B[:, t, :, None])[..., 0] * on[:, t, None])
        dB.append(torch.matmul((delta * u)[:, t, None, :], full)[:, 0] * on[:, t, None])
        dC.append(torch.matmul(dy[:, t, None, :], hs[t + 1])[:, 0] * on[:, t, None])
        dh = torch.where(here, full * a, dh)
    into, through, dB, dC = (torch.stack(v[::-1], 1) for v in (into, through, dB, dC))
    dx = (through + into * u) * torch.sigmoid(x) * on[..., None]
    dy = dy * on[..., None]
    got.update(
        du=dy * D + into * delta, ddelta=dx,
        dz=w["dout"] * y * sig * (1 + z * (1 - sig)) * on[..., None], dB=dB, dC=dC, dA=dA,
        dD=(dy * u).sum((0, 1)), ddelta_bias=dx.sum((0, 1)), dstate_in=dh)
    return got
