"""Cases of the gated linear recurrence and of the group norm with an activation: what is measured, and its plain form.

A case is a dict of plain values.  ``listed()`` names the representative ones, ``draw(rng)`` gives one more of the same
ranges, ``prepare`` makes what a user's program has in hand, ``run`` is one pass (through the package's entry points where
``own`` is true, else through elementary torch operations), ``work`` the bytes and operations that a pass cannot do
without, ``exact`` the same outputs from the definitions in 64 bits.

Gated linear recurrence over the steps t of x, f (B, L, D), one state per sequence and channel:
    h_t = (1 - l_t) h_{t-1} + l_t x_t                  l = sigmoid(-f)            (tied gates)
    h_t = (1 - l_t) h_{t-1} + sigmoid(i_t) x_t                                    (an input gate of its own)
    y_t = h_t
A step with its reset flag set starts from a zero state; a padded step leaves the state as it is and gives y = 0.

Group norm over a sequence, channels last, x (B, L, D) in G groups of D / G channels: mean and variance of a group over its
channels and the steps that are not padded; y = silu((x - mean) / sqrt(var + eps) * (1 + weight) + bias), 0 where padded.

Operators
  step        one token of every sequence: x, f (B, D) and the state -> y, the new state
  scan        whole sequences, inference: y and the state after the last step
  train       the same with the gradients of x, the gates and the state that came in
  norm        group norm + SiLU, inference
  norm_train  the same with the gradients of x, weight and bias
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5


def _rec(name, op, dtype, batch, length, dim, gate=False, pad=0.0, docs=0, reverse=False, layout="plain", state=True):
    """gate: an input gate of its own; pad: largest padded share of a sequence; docs: mean length of the documents that a
    sequence packs (0: one); layout: plain (B, L, D), sliced (columns of one projection's output) or time (L, B, D);
    state: whether a state comes in."""
    case = {"op": op, "dtype": dtype, "batch": batch, "length": length, "dim": dim, "gate": gate, "pad": pad, "docs": docs,
            "reverse": reverse, "layout": layout, "state": state}
    return dict(case, name=name) if name else case


def _norm(name, op, dtype, batch, length, dim, groups, pad=0.0):
    case = {"op": op, "dtype": dtype, "batch": batch, "length": length, "dim": dim, "groups": groups, "pad": pad}
    return dict(case, name=name) if name else case


def listed():
    return [
        # interactive decoding: a few sequences, one token each; latency
        _rec("step_few", "step", "bf16", 4, 1, 512),
        # batched decoding at the serving width, gates of their own
        _rec("step_batched", "step", "bf16", 64, 1, 2048, gate=True),
        # prefill of one short prompt behind an earlier turn's state
        _rec("scan_prompt", "scan", "bf16", 1, 300, 1024, layout="sliced"),
        # a language model's layer on a padded batch, operands where the projection left them
        _rec("scan_lm", "scan", "bf16", 8, 4096, 1024, pad=0.5, layout="sliced"),
        # one long context: the time axis is all there is to split
        _rec("scan_long", "scan", "bf16", 1, 65536, 2048, state=False),
        # the backward direction of a bidirectional encoder, fp32, ragged sizes, time-major
        _rec("scan_encoder_fp32", "scan", "fp32", 4, 2805, 1001, gate=True, pad=0.3, reverse=True, layout="time", state=False),
        # pre-training: documents packed into sequences
        _rec("train_lm", "train", "bf16", 8, 4096, 2048, docs=700, state=False),
        # the continued half of a long sequence, an input gate of its own, padded
        _rec("train_gated_fp16", "train", "fp16", 2, 16384, 1024, gate=True, pad=0.4),
        # a small padded batch in fp32, groups of three channels
        _norm("norm_small_fp32", "norm", "fp32", 2, 300, 96, 32, pad=0.5),
        # feature maps of 64 x 64 positions
        _norm("norm_maps", "norm", "bf16", 16, 4096, 512, 32),
        # training of an encoder layer on padded batches
        _norm("norm_train_encoder", "norm_train", "bf16", 32, 1024, 1024, 32, pad=0.25),
        # training on long sequences: a group does not fit one multiprocessor
        _norm("norm_train_long", "norm_train", "fp16", 2, 32768, 1024, 16),
    ]


# bytes of the activations of the largest listed case of each operator
_CAP = {"step": 64 * 2048 * 5 * 2, "scan": 65536 * 2048 * 3 * 2, "train": 8 * 4096 * 2048 * 6 * 2, "norm": 16 * 4096 * 512 * 2 * 2,
        "norm_train": 2 * 32768 * 1024 * 4 * 2}


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _arrays(case):
    """activations read or written by a pass"""
    gates = 3 if case.get("gate") else 2
    return {"step": gates + 1, "scan": gates + 1, "train": 2 * gates + 2, "norm": 2, "norm_train": 4}[case["op"]]


def draw(rng):
    op = rng.choice(["step", "scan", "scan", "train", "train", "norm", "norm_train", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    pad = round(rng.uniform(0.05, 1.0), 3) if rng.random() < 0.4 else 0.0
    if op.startswith("norm"):
        size = rng.choice([_spread(rng, 1, 256), 8 * _spread(rng, 1, 16)])
        groups = _spread(rng, 1, 64)
        case = _norm(None, op, dtype, 1, 1, size * groups, groups, pad)
        longest = 32768
    else:
        dim = rng.choice([_spread(rng, 8, 8192), 8 * _spread(rng, 4, 512)])
        case = _rec(None, op, dtype, 1, 1, dim, gate=rng.random() < 0.4, pad=0.0 if op == "step" else pad,
                    docs=_spread(rng, 2, 5000) if op != "step" and rng.random() < 0.35 else 0,
                    reverse=op != "step" and rng.random() < 0.3,
                    layout="plain" if op == "step" else rng.choice(["plain", "plain", "sliced", "time"]),
                    state=op == "step" or rng.random() < 0.6)
        longest = 65536
    least = -(-32 // size) if op.startswith("norm") else 1   # (a group of fewer values has hardly a variance)
    room = _CAP[op] // (_arrays(case) * SIZE[dtype] * case["dim"])   # sequences x steps
    if op == "step":
        case["batch"] = _spread(rng, 1, max(1, min(512, room)))
        return case
    rows = _spread(rng, max(1, room // 512), max(1, room))
    case["length"] = _spread(rng, least, max(least, min(longest, rows)))
    case["batch"] = max(1, min(256, rows // case["length"]))
    return case


def _seeded(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(case, gen):
    """steps of each sequence that are not padded; with pad near 1 down to none"""
    b, n = case["batch"], case["length"]
    keep = (1 - case["pad"] * torch.rand(b, generator=gen, device="cuda")) * n
    return keep.round().to(torch.int64)


def prepare(case, seed):
    gen = _seeded(seed)
    dt = DTYPES[case["dtype"]]
    b, n, d = case["batch"], case["length"], case["dim"]
    st = {"case": case, "mask": None, "reset": None}

    def normal(*size, dtype=dt, scale=1.0, shift=0.0):
        return torch.randn(*size, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).add_(shift).to(dtype)

    if case["pad"] > 0:
        st["mask"] = torch.arange(n, device="cuda")[None, :] >= _lengths(case, gen)[:, None]
    if case["op"].startswith("norm"):
        st["x"] = normal(b, n, d)
        st["x"] += normal(d, scale=0.5)
        st["weight"] = normal(d, dtype=torch.float32, scale=0.1)
        st["bias"] = normal(d, dtype=torch.float32, scale=0.1)
        if case["op"] == "norm_train":
            st["dy"] = normal(b, n, d)
            st["x"].requires_grad_()
        if own:
            import fairseq_apollo_b200 as M
            norm = M.GroupNorm(d, case["groups"], eps=EPS, activation="silu").cuda()
            with torch.no_grad():
                norm.weight.copy_(st["weight"])
                norm.bias.copy_(st["bias"])
            st["norm"] = norm
        return st

    # the forget gates of a trained layer stand mostly open: a state lasts from a few steps to a few thousand
    span = normal(d, dtype=torch.float32, scale=1.5, shift=3.0)
    shape = (b, d) if case["op"] == "step" else (b, n, d)
    gates = 3 if case["gate"] else 2
    z = normal(*shape[:-1], gates * d) if case["layout"] == "sliced" else None
    parts = []
    for k in range(gates):
        if z is not None:
            t = z[..., k * d:(k + 1) * d]
        elif case["layout"] == "time":
            t = normal(n, b, d).transpose(0, 1)
        else:
            t = normal(*shape)
        if k == 1:
            t += span.to(dt)
        parts.append(t)
    st["x"], st["f"], st["i"] = parts[0], parts[1], parts[2] if case["gate"] else None
    st["h"] = normal(b, d, dtype=torch.float32) if case["state"] else None
    if case["docs"]:
        st["reset"] = torch.rand(b, n, generator=gen, device="cuda") < 1.0 / case["docs"]
    if case["op"] == "train":
        st["dy"] = normal(b, n, d)
        st["dh"] = normal(b, d, dtype=torch.float32)
        for key in ("x", "f", "i", "h"):
            if st[key] is not None:
                st[key] = st[key].detach().requires_grad_()
    return st


# ------------------------------------------------------------------------------- the framework's operators
def _run_own(st):
    import fairseq_apollo_b200 as M
    case = st["case"]
    op = case["op"]
    if op == "step":
        return list(M.ops.gated_recurrence_step(st["x"], st["f"], st["i"], st["h"]))
    if op == "scan":
        with torch.no_grad():
            return list(M.gated_recurrence(st["x"], st["f"], st["i"], padding_mask=st["mask"], reset_mask=st["reset"],
                                           h_in=st["h"], want_state=True, reverse=case["reverse"]))
    if op == "train":
        y, h = M.gated_recurrence(st["x"], st["f"], st["i"], padding_mask=st["mask"], reset_mask=st["reset"], h_in=st["h"],
                                  want_state=True, reverse=case["reverse"])
        wrt = [t for t in (st["x"], st["f"], st["i"], st["h"]) if t is not None]
        return [y, h] + list(torch.autograd.grad([y, h], wrt, [st["dy"], st["dh"]]))
    norm = st["norm"]
    if op == "norm":
        with torch.no_grad():
            return [norm(st["x"], st["mask"])]
    y = norm(st["x"], st["mask"])
    return [y] + list(torch.autograd.grad(y, [st["x"], norm.weight, norm.bias], st["dy"]))


# ------------------------------------------------------------------------------------------ the plain form
def _plain_scan(a, c):
    """c_t + a_t c_{t-1} + a_t a_{t-1} c_{t-2} + ... along dim 1, in place, by doubling the reach"""
    k, n = 1, c.shape[1]
    while k < n:
        c[:, k:] = c[:, k:] + a[:, k:] * c[:, :-k]
        a[:, k:] = a[:, k:] * a[:, :-k]
        k *= 2
    return c


def _turn(t, reverse):
    return t.flip(1) if reverse and t is not None else t


def _plain_gates(st):
    """(decay a, decay's slope, written value c, x, leak l, input gate s or None, pad, reset), fp32, in the order of the walk"""
    rev = st["case"]["reverse"]
    x, f = _turn(st["x"].detach().float(), rev), _turn(st["f"].detach().float(), rev)
    leak, keep = torch.sigmoid(-f), torch.sigmoid(f)
    s = None if st["i"] is None else torch.sigmoid(_turn(st["i"].detach().float(), rev))
    c = (leak if s is None else s) * x
    a = keep.clone()
    pad = None if st["mask"] is None else _turn(st["mask"], rev)[..., None]
    reset = None if st["reset"] is None else _turn(st["reset"], rev)[..., None]
    if pad is not None:
        a.masked_fill_(pad, 1.0)
        c.masked_fill_(pad, 0.0)
    if reset is not None:
        a.masked_fill_(reset, 0.0)
    return a, keep * leak, c, x, leak, s, pad, reset


def _plain_recurrence(st):
    case = st["case"]
    dt, rev = DTYPES[case["dtype"]], case["reverse"]
    if case["op"] == "step":
        x, f = st["x"].float(), st["f"].float()
        gate = torch.sigmoid(-f) if st["i"] is None else torch.sigmoid(st["i"].float())
        h = torch.sigmoid(f) * st["h"] + gate * x
        return [h.to(dt), h]
    a, slope, c, x, leak, s, pad, reset = _plain_gates(st)
    h0 = None if st["h"] is None else st["h"].detach()
    h = c.clone()
    if h0 is not None:
        h[:, 0] = h[:, 0] + a[:, 0] * h0
    h = _plain_scan(a.clone(), h)
    y = h if pad is None else h.masked_fill(pad, 0.0)
    out = [_turn(y, rev).to(dt), h[:, -1].clone()]
    if case["op"] == "scan":
        return out
    # gradients: g_t = dy_t + a_{t+1} g_{t+1}, the state's gradient entering behind the last step
    dy = _turn(st["dy"].float(), rev)
    g = dy.clone() if pad is None else dy.masked_fill(pad, 0.0)
    g[:, -1] = g[:, -1] + st["dh"]
    ahead = torch.zeros_like(a)
    ahead[:, :-1] = a[:, 1:]
    g = _plain_scan(ahead.flip(1), g.flip(1)).flip(1)
    before = torch.zeros_like(h)
    before[:, 1:] = h[:, :-1]
    if h0 is not None:
        before[:, 0] = h0
    if reset is not None:
        before.masked_fill_(reset, 0.0)
    if s is None:
        grads = [leak * g, slope * (before - x) * g]
    else:
        grads = [s * g, slope * before * g, s * (1 - s) * x * g]
    if pad is not None:
        grads = [t.masked_fill(pad, 0.0) for t in grads]
    out += [_turn(t, rev).to(dt) for t in grads]
    if h0 is not None:
        out.append(a[:, 0] * g[:, 0])
    return out


def _plain_norm(st):
    case = st["case"]
    b, n, d, g = case["batch"], case["length"], case["dim"], case["groups"]
    dt = DTYPES[case["dtype"]]
    x = st["x"].detach().float().view(b, n, g, d // g)
    live = torch.ones(b, n, 1, 1, device=x.device) if st["mask"] is None else (~st["mask"]).float().view(b, n, 1, 1)
    size = (live.sum(1, keepdim=True) * (d // g)).clamp(min=1)
    mean = (x * live).sum((1, 3), keepdim=True) / size
    off = (x - mean) * live
    rstd = torch.rsqrt((off * off).sum((1, 3), keepdim=True) / size + EPS)
    xn = off * rstd
    w, c = (1 + st["weight"]).view(1, 1, g, -1), st["bias"].view(1, 1, g, -1)
    z = xn * w + c
    gate = torch.sigmoid(z)
    y = (z * gate * live).view(b, n, d).to(dt)
    if case["op"] == "norm":
        return [y]
    dz = st["dy"].float().view(b, n, g, d // g) * live * gate * (1 + z * (1 - gate))
    dn = dz * w
    dx = rstd * (dn - live * (dn.sum((1, 3), keepdim=True) + xn * (dn * xn).sum((1, 3), keepdim=True)) / size)
    return [y, dx.view(b, n, d).to(dt), (dz * xn).sum((0, 1)).view(d), dz.sum((0, 1)).view(d)]


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_norm(state) if state["case"]["op"].startswith("norm") else _plain_recurrence(state)


def work(case):
    values = case["batch"] * case["length"] * case["dim"]
    nbytes = _arrays(case) * values * SIZE[case["dtype"]]
    if case["pad"] > 0:
        nbytes += case["batch"] * case["length"]
    if case["op"].startswith("norm"):
        nbytes += 8 * case["dim"] * (2 if case["op"] == "norm_train" else 1)
        return {"bytes": nbytes, "flops": values * (12 if case["op"] == "norm" else 40)}
    if case["docs"]:
        nbytes += case["batch"] * case["length"]
    states = (1 + bool(case["state"])) * (2 if case["op"] == "train" else 1)
    nbytes += states * 4 * case["batch"] * case["dim"]
    return {"bytes": nbytes, "flops": values * (7 if case["op"] != "train" else 24) + (values * 4 if case["gate"] else 0)}


# ---------------------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(case, st) if case["op"].startswith("norm") else _exact_recurrence(case, st)


def _exact_recurrence(case, st):
    """step after step, time first; the elementwise parts of all steps at once"""
    f64 = torch.float64
    rev = case["reverse"]

    def wide(t):
        if t is None:
            return None
        t = t.detach()
        t = (t[:, None] if case["op"] == "step" else t).transpose(0, 1).to(f64)
        return t.flip(0) if rev else t

    def back(t):
        t = (t.flip(0) if rev else t).transpose(0, 1)
        return t[:, 0] if case["op"] == "step" else t

    def flags(t):
        return None if t is None else (t.t().flip(0) if rev else t.t())[..., None]

    x, f, i = wide(st["x"]), wide(st["f"]), wide(st["i"])
    n, b, d = x.shape
    pad, cut = flags(st["mask"]), flags(st["reset"])
    keep, leak = 1 / (1 + torch.exp(-f)), 1 / (1 + torch.exp(f))
    into = leak if i is None else 1 / (1 + torch.exp(-i))
    flow, enter = keep, into * x
    if pad is not None:
        flow, enter = torch.where(pad, 1.0, flow), torch.where(pad, 0.0, enter)
    if cut is not None:
        flow = torch.where(cut, 0.0, flow)
    h = torch.zeros(b, d, dtype=f64, device=x.device) if st["h"] is None else st["h"].detach().to(f64)
    states = torch.empty(n + 1, b, d, dtype=f64, device=x.device)
    states[0] = h
    for t in range(n):
        torch.addcmul(enter[t], flow[t], states[t], out=states[t + 1])
    y = states[1:] if pad is None else torch.where(pad, 0.0, states[1:])
    if case["op"] == "step":
        return [back(y), states[n]]
    if case["op"] == "scan":
        return [back(y), states[n].clone()]
    dy = wide(st["dy"])
    g = torch.empty_like(states)   # g[t]: the gradient of the state behind step t - 1
    g[n] = st["dh"].to(f64)
    for t in range(n - 1, -1, -1):
        if pad is None:
            g[t + 1] += dy[t]
        else:
            g[t + 1] += torch.where(pad[t], 0.0, dy[t])
        torch.mul(flow[t], g[t + 1], out=g[t])
    dh = g[1:]
    prev = states[:n] if cut is None else torch.where(cut, 0.0, states[:n])
    grads = [dh * into, dh * keep * leak * (prev - x if i is None else prev)]
    if i is not None:
        grads.append(dh * into * (1 / (1 + torch.exp(i))) * x)
    if pad is not None:
        grads = [torch.where(pad, 0.0, t) for t in grads]
    out = [back(y), states[n].clone()] + [back(t) for t in grads]
    return out if st["h"] is None else out + [g[0]]


def _exact_norm(case, st):
    f64 = torch.float64
    b, n, d, groups = case["batch"], case["length"], case["dim"], case["groups"]
    wide = d // groups
    weight, bias = 1 + st["weight"].to(f64), st["bias"].to(f64)
    train = case["op"] == "norm_train"
    y = torch.zeros(b, n, d, dtype=f64, device="cuda")
    dx = torch.zeros_like(y) if train else None
    dw, db = (torch.zeros(d, dtype=f64, device="cuda") for _ in range(2))
    ends = [n] * b if st["mask"] is None else (~st["mask"]).sum(1).tolist()   # (padding is on the right)
    for s, end in enumerate(ends):
        if end == 0:
            continue
        x = st["x"].detach()[s, :end].to(f64).reshape(end, groups, wide)
        mean = x.mean((0, 2), keepdim=True)
        std = ((x - mean).square().mean((0, 2), keepdim=True) + EPS).sqrt()
        xn = (x - mean) / std
        z = xn.reshape(end, d) * weight + bias
        sig = 1 / (1 + torch.exp(-z))
        y[s, :end] = z * sig
        if train:
            dz = st["dy"][s, :end].to(f64) * (sig + z * sig * (1 - sig))
            dw += (dz * xn.reshape(end, d)).sum(0)
            db += dz.sum(0)
            dn = (dz * weight).reshape(end, groups, wide)
            part = dn - dn.mean((0, 2), keepdim=True) - xn * (dn * xn).mean((0, 2), keepdim=True)
            dx[s, :end] = (part / std).reshape(end, d)
    return [y, dx, dw, db] if train else [y]
