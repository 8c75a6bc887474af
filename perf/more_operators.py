"""Cases of linear attention with a decay for each head and of the root-mean-square norm with a residual: what is measured, and
its plain form.

A case is a dict of plain values.  ``listed()`` names the representative ones, ``draw(rng)`` gives one more of the same
ranges, ``prepare`` makes what a user's program has in hand, ``run`` is one pass (through the package's entry points where
``own`` is true, else through elementary torch operations), ``work`` the bytes and operations that a pass cannot do
without, ``exact`` the same outputs from the definitions in 64 bits.

Decayed attention over the steps t of q, k (B, L, H, K), v (B, L, H, V) and gates f (B, L, H), one state (K, V) per sequence and head:
    S_t = a_t S_{t-1} + k_t v_t^T      y_t = scale S_t^T q_t      a = sigmoid(f)
A step with its reset flag set starts from a zero state; a padded step leaves the state as it is and gives y = 0.

Root-mean-square norm of x (B, L, D) in G groups of D / G channels: r = x + residual, rounded to x's type,
y = r / sqrt(mean(r^2) + eps) * (1 + weight), the mean over a group's channels.

Operators
  step        one token of every sequence: q, k (B, H, K), v (B, H, V), f (B, H) and the state -> y, the new state
  scan        whole sequences, inference: y and the state after the last step
  train       the same with the gradients of q, k, v, f and the state that came in
  norm        the norm, inference: y, and r where there is a residual
  norm_train  the same with the gradients of x, the residual and weight
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5


def _att(name, op, dtype, batch, length, heads, keys, values, pad=0.0, docs=0, reverse=False, layout="plain", state=True):
    """pad: largest padded share of a sequence; docs: mean length of the documents that a sequence packs (0: one); layout: plain
    (B, L, H, .), sliced (columns of one projection's output) or time (L, B, H, .); state: whether a state comes in."""
    case = {"op": op, "dtype": dtype, "batch": batch, "length": length, "heads": heads, "keys": keys, "values": values, "pad": pad,
            "docs": docs, "reverse": reverse, "layout": layout, "state": state}
    return dict(case, name=name) if name else case


def _norm(name, op, dtype, batch, length, dim, groups=1, residual=True):
    case = {"op": op, "dtype": dtype, "batch": batch, "length": length, "dim": dim, "groups": groups, "residual": residual}
    return dict(case, name=name) if name else case


def listed():
    return [
        # interactive decoding: a few sequences, one token each; latency
        _att("step_few", "step", "bf16", 4, 1, 8, 64, 64),
        # batched decoding at the serving width: the states are all there is to move
        _att("step_batched", "step", "bf16", 64, 1, 16, 128, 128),
        # prefill of one short prompt behind an earlier turn's state
        _att("scan_prompt", "scan", "bf16", 1, 300, 16, 64, 64, layout="sliced"),
        # a language model's layer on a padded batch, operands where the projection left them
        _att("scan_lm", "scan", "bf16", 8, 4096, 16, 64, 64, pad=0.5, layout="sliced"),
        # one long context: few heads, the time axis is all there is to split
        _att("scan_long", "scan", "bf16", 1, 65536, 16, 128, 128, state=False),
        # the backward direction of a bidirectional encoder, fp32, ragged sizes, time-major
        _att("scan_encoder_fp32", "scan", "fp32", 4, 2805, 7, 50, 83, pad=0.3, reverse=True, layout="time", state=False),
        # pre-training: documents packed into sequences
        _att("train_lm", "train", "bf16", 8, 4096, 16, 128, 128, docs=700, state=False),
        # the continued half of long padded sequences, keys narrower than values
        _att("train_narrow_fp16", "train", "fp16", 2, 16384, 16, 64, 128, pad=0.4),
        # each head's output of a small fp32 batch
        _norm("norm_heads_fp32", "norm", "fp32", 2, 300, 512, groups=8, residual=False),
        # in front of a layer at the width of the long-context configuration
        _norm("norm_residual", "norm", "bf16", 8, 4096, 2048),
        # training, the residual stream of an ordinary batch
        _norm("norm_train_residual", "norm_train", "bf16", 16, 4096, 1024),
        # training, heads of a long sequence's output
        _norm("norm_train_heads", "norm_train", "fp16", 2, 32768, 1024, groups=16, residual=False),
    ]


def _values(case):
    """activation values that a pass reads and writes"""
    rows = case["batch"] * case["length"]
    if case["op"].startswith("norm"):
        arrays = 2 + 2 * case["residual"]                 # x, residual, y, r
        if case["op"] == "norm_train":
            arrays += 2 + case["residual"]                # dy, dr, dx (which is the residual's gradient too)
        return rows * case["dim"] * arrays
    one = 2 * case["keys"] + 2 * case["values"] + 1       # q, k, v, f, y
    if case["op"] == "train":
        one += case["values"] + 2 * case["keys"] + case["values"] + 1   # dy, dq, dk, dv, df
    return rows * case["heads"] * one


def work(case):
    nbytes = _values(case) * SIZE[case["dtype"]]
    rows = case["batch"] * case["length"]
    if case["op"].startswith("norm"):
        values = rows * case["dim"]
        nbytes += 4 * case["dim"] * (2 if case["op"] == "norm_train" else 1)
        return {"bytes": nbytes, "flops": values * (5 if case["op"] == "norm" else 16)}
    per_head = case["keys"] * case["values"]
    nbytes += rows * ((case["pad"] > 0) + (case["docs"] > 0))
    states = (1 + bool(case["state"])) * (2 if case["op"] == "train" else 1)
    nbytes += states * 4 * case["batch"] * case["heads"] * per_head
    # a step by the recurrence: decay and outer product (3), y (2); backward: S again, R (3 each), dq, dk, dv (2 each), df (2)
    return {"bytes": nbytes, "flops": rows * case["heads"] * per_head * (5 if case["op"] != "train" else 19)}


_CAP = {}   # bytes of the largest listed case of each operator


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    if not _CAP:
        for c in listed():
            _CAP[c["op"]] = max(_CAP.get(c["op"], 0), work(c)["bytes"])
    op = rng.choice(["step", "step", "scan", "scan", "scan", "train", "train", "train", "norm", "norm_train", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op.startswith("norm"):
        groups = rng.choice([1, 1, _spread(rng, 2, 32)])
        size = rng.choice([_spread(rng, 16, 4096), 8 * _spread(rng, 2, 256)])
        case = _norm(None, op, dtype, 1, 1, min(8192, max(size, 4 * groups) // groups * groups), groups, residual=rng.random() < 0.6)
        longest = 32768
    else:
        heads = _spread(rng, 1, 32)
        dims = rng.choice([[64, 64], [128, 128], [64, 128], [8 * _spread(rng, 1, 32), 8 * _spread(rng, 1, 32)],
                           [_spread(rng, 1, 256), _spread(rng, 1, 256)]])
        pad = round(rng.uniform(0.05, 1.0), 3) if rng.random() < 0.4 else 0.0
        case = _att(None, op, dtype, 1, 1, heads, dims[0], dims[1], pad=0.0 if op == "step" else pad,
                    docs=_spread(rng, 2, 5000) if op != "step" and rng.random() < 0.35 else 0,
                    reverse=op != "step" and rng.random() < 0.3,
                    layout="plain" if op == "step" else rng.choice(["plain", "plain", "sliced", "time"]),
                    state=op == "step" or rng.random() < 0.6)
        longest = 65536 if op == "scan" else 16384
    if op == "step":
        case["batch"] = _spread(rng, 1, max(1, min(512, _CAP[op] // work(case)["bytes"])))
        return case
    room = int(_CAP[op] // (_values(case) * SIZE[dtype]))   # sequences x steps
    if not op.startswith("norm"):   # (the plain form keeps states and pairs of steps of every 64 steps in fp32)
        room = min(room, int(2.2e9 // (heads * (64 * 4 + dims[0] * dims[1] // 16))))
    rows = _spread(rng, max(1, room // 512), max(1, room))
    case["length"] = _spread(rng, 1, min(longest, rows))
    case["batch"] = max(1, min(256, rows // case["length"]))
    while case["batch"] > 1 and work(case)["bytes"] > _CAP[op]:   # (states that come and go)
        case["batch"] = max(1, case["batch"] * 3 // 4)
    return case


def _seeded(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    gen = _seeded(seed)
    dt = DTYPES[case["dtype"]]
    b, n = case["batch"], case["length"]
    st = {"case": case, "mask": None, "reset": None}

    def normal(*size, dtype=dt, scale=1.0, shift=0.0):
        return torch.randn(*size, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).add_(shift).to(dtype)

    if case["op"].startswith("norm"):
        d = case["dim"]
        st["x"] = normal(b, n, d)
        st["res"] = normal(b, n, d, scale=2.0) if case["residual"] else None
        st["weight"] = normal(d, dtype=torch.float32, scale=0.1)
        if case["op"] == "norm_train":
            st["dy"] = normal(b, n, d)
            st["dr"] = normal(b, n, d) if case["residual"] else None
            for key in ("x", "res", "weight"):
                if st[key] is not None:
                    st[key].requires_grad_()
        return st

    h, kd, vd = case["heads"], case["keys"], case["values"]
    st["scale"] = kd ** -0.5
    if case["pad"] > 0:
        keep = (1 - case["pad"] * torch.rand(b, generator=gen, device="cuda")) * n
        st["mask"] = torch.arange(n, device="cuda")[None, :] >= keep.round()[:, None]
    # heads of a trained layer remember from a few steps to some hundred, each step a little differently
    span = normal(h, dtype=torch.float32, scale=1.5, shift=3.0)
    widths = [h * kd, h * kd, h * vd, h]
    if case["op"] == "step":
        parts = [normal(b, w) for w in widths]
    elif case["layout"] == "sliced":
        parts = list(normal(b, n, sum(widths)).split(widths, dim=-1))
    elif case["layout"] == "time":
        parts = [normal(n, b, w).transpose(0, 1) for w in widths]
    else:
        parts = [normal(b, n, w) for w in widths]
    q, k, v = (p.unflatten(-1, (h, w // h)) for p, w in zip(parts[:3], widths))
    f = parts[3]
    f += span.to(dt)
    st.update(q=q, k=k, v=v, f=f)
    st["h"] = normal(b, h, kd, vd, dtype=torch.float32, scale=3.0) if case["state"] else None
    if case["docs"]:
        st["reset"] = torch.rand(b, n, generator=gen, device="cuda") < 1.0 / case["docs"]
    if case["op"] == "train":
        st["dy"] = normal(b, n, h, vd)
        st["dh"] = normal(b, h, kd, vd, dtype=torch.float32)
        for key in ("q", "k", "v", "f", "h"):
            if st[key] is not None:
                st[key] = st[key].detach().requires_grad_()
    return st


# ------------------------------------------------------------------------------- the framework's operators
def _run_own(st):
    import fairseq_apollo_b200 as M
    case = st["case"]
    op = case["op"]
    if op == "step":
        return list(M.ops.decayed_attention_step(st["q"], st["k"], st["v"], st["f"], st["h"], scale=st["scale"]))
    if op == "scan":
        with torch.no_grad():
            return list(M.decayed_attention(st["q"], st["k"], st["v"], st["f"], padding_mask=st["mask"], reset_mask=st["reset"],
                                            h_in=st["h"], scale=st["scale"], want_state=True, reverse=case["reverse"]))
    if op == "train":
        y, h = M.decayed_attention(st["q"], st["k"], st["v"], st["f"], padding_mask=st["mask"], reset_mask=st["reset"], h_in=st["h"],
                                   scale=st["scale"], want_state=True, reverse=case["reverse"])
        wrt = [t for t in (st["q"], st["k"], st["v"], st["f"], st["h"]) if t is not None]
        return [y, h] + list(torch.autograd.grad([y, h], wrt, [st["dy"], st["dh"]]))
    if op == "norm":
        with torch.no_grad():
            r = M.rms_norm(st["x"], st["weight"], residual=st["res"], num_groups=case["groups"], eps=EPS)
        return [r] if st["res"] is None else list(r)
    r = M.rms_norm(st["x"], st["weight"], residual=st["res"], num_groups=case["groups"], eps=EPS)
    if st["res"] is None:
        return [r] + list(torch.autograd.grad(r, [st["x"], st["weight"]], st["dy"]))
    return list(r) + list(torch.autograd.grad(list(r), [st["x"], st["res"], st["weight"]], [st["dy"], st["dr"]]))


# ------------------------------------------------------------------------------------------ the plain form
_C = 64   # steps of a chunk


def _chunks(t, reverse, n):
    """(B, L, H, .) -> (B, N, H, C, .) in the order of the walk, filled up with zeros"""
    t = t.detach()
    t = t.flip(1) if reverse else t
    fill = n * _C - t.shape[1]
    if fill:
        t = torch.cat([t, t.new_zeros(t.shape[0], fill, *t.shape[2:])], 1)
    return t.unflatten(1, (n, _C)).transpose(2, 3)


def _join(t, reverse, length):
    """and back"""
    t = t.transpose(2, 3).flatten(1, 2)[:, :length]
    return t.flip(1) if reverse else t


def _states(decay, added, first, back):
    """(N, ...) states in front of each chunk (``back``: behind it) and the one at the end, by doubling the reach; decay (B, N, H, 1, 1)"""
    if back:
        decay, added = decay.flip(1), added.flip(1)
    s = torch.cat([first[:, None], added], 1)                       # s[0] = first, s[c + 1] = decay[c] s[c] + added[c]
    a = torch.cat([torch.ones_like(decay[:, :1]), decay], 1)
    reach = 1
    while reach < s.shape[1]:
        s[:, reach:] = s[:, reach:] + a[:, reach:] * s[:, :-reach]
        a[:, reach:] = a[:, reach:] * a[:, :-reach]
        a[:, :reach] = 0
        reach *= 2
    front, last = s[:, :-1], s[:, -1]
    return (front.flip(1) if back else front), last


def _plain_step(st):
    q, k, v = (st[key].float() for key in ("q", "k", "v"))
    a = torch.sigmoid(st["f"].float())[..., None, None]
    s = a * st["h"] + k[..., :, None] * v[..., None, :]
    y = (q[..., :, None] * s).sum(-2) * st["scale"]
    return [y.to(st["q"].dtype), s]


def _plain_attention(st):
    case = st["case"]
    dt, rev, length = DTYPES[case["dtype"]], case["reverse"], case["length"]
    n = -(-length // _C)
    scale = st["scale"]
    q, k, v = (_chunks(st[key], rev, n).float() for key in ("q", "k", "v"))
    f = _chunks(st["f"][..., None], rev, n)[..., 0].double()         # (B, N, H, C); sums of logarithms in 64 bits
    pad = torch.zeros(case["batch"], length, 1, 1, dtype=torch.bool, device=f.device) if st["mask"] is None else st["mask"][..., None, None]
    pad = _chunks((~pad).float(), rev, n)[..., 0] == 0               # (B, N, 1, C), the filling too
    reset = None if st["reset"] is None else _chunks(st["reset"][..., None, None].float(), rev, n)[..., 0]
    g = torch.nn.functional.logsigmoid(f).masked_fill(pad, 0.0)
    if reset is not None:
        g = g.masked_fill(reset > 0, 0.0)
    G = g.cumsum(-1)
    i = torch.arange(_C, device=f.device)
    seen = (i[:, None] >= i[None, :]).expand(*G.shape[:2], 1, _C, _C)
    enter, leave = torch.exp(G).float(), torch.exp(G[..., -1:] - G).float()
    if reset is not None:
        part = reset.cumsum(-1)
        seen = seen & (part[..., :, None] == part[..., None, :])
        enter = enter * (part == 0)
        leave = leave * (part == part[..., -1:])
    D = torch.exp(G[..., :, None] - G[..., None, :]).masked_fill(~seen, 0.0).float()
    through = enter[..., -1]                                         # (B, N, H)
    k, v, q = (t.masked_fill(pad[..., None], 0.0) for t in (k, v, q))
    first = torch.zeros(q.shape[0], q.shape[2], q.shape[-1], v.shape[-1], device=q.device) if st["h"] is None else st["h"].detach()
    S0, last = _states(through[..., None, None], (k * leave[..., None]).transpose(-1, -2) @ v, first, False)
    P = (q @ k.transpose(-1, -2)) * scale
    y = (P * D) @ v + enter[..., None] * scale * (q @ S0)
    out = [_join(y, rev, length).to(dt), last]
    if case["op"] == "scan":
        return out
    dy = _chunks(st["dy"], rev, n).float().masked_fill(pad[..., None], 0.0)
    dP = (dy @ v.transpose(-1, -2)) * D
    R, dh = _states(through[..., None, None], (q * (enter * scale)[..., None]).transpose(-1, -2) @ dy, st["dh"], True)
    P0 = P * D
    dv = P0.transpose(-1, -2) @ dy + leave[..., None] * (k @ R)
    dq0 = enter[..., None] * scale * (dy @ S0.transpose(-1, -2))
    dq = scale * (dP @ k) + dq0
    dk0 = leave[..., None] * (v @ R.transpose(-1, -2))
    dk = scale * (dP.transpose(-1, -2) @ q) + dk0
    # d log a_t: what passes from a step before t to t or one behind it, inside the chunk, from outside, to outside, and through it
    W = (P * dP).masked_fill(i[:, None] == i[None, :], 0.0)
    across = (W.sum(-1) - W.sum(-2)).double() + (dq0 * q).sum(-1)
    over = (dk0 * k).sum(-1).double().cumsum(-1)
    da = across.flip(-1).cumsum(-1).flip(-1) + torch.cat([torch.zeros_like(over[..., :1]), over[..., :-1]], -1)
    da = da + (through * (S0 * R).sum((-1, -2)))[..., None]
    df = (da * torch.sigmoid(-f)).masked_fill(pad, 0.0)
    if reset is not None:
        df = df.masked_fill(reset > 0, 0.0)
    out += [_join(t, rev, length).to(dt) for t in (dq, dk, dv)] + [_join(df[..., None], rev, length)[..., 0].to(dt)]
    if st["h"] is not None:
        out.append(dh)
    return out


def _plain_norm(st):
    case = st["case"]
    g, dt = case["groups"], DTYPES[case["dtype"]]
    x = st["x"].detach()
    total = x if st["res"] is None else (x.float() + st["res"].detach().float()).to(dt)
    r = total.float().unflatten(-1, (g, -1))
    rstd = torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS)
    w = (1 + st["weight"].detach()).unflatten(-1, (g, -1))
    out = [(r * rstd * w).flatten(-2).to(dt)]
    if st["res"] is not None:
        out.append(total)
    if case["op"] == "norm":
        return out
    dy = st["dy"].float().unflatten(-1, (g, -1))
    dn = dy * w
    xn = r * rstd
    dx = rstd * (dn - xn * (dn * xn).mean(-1, keepdim=True))
    dx = dx.flatten(-2)
    if st["res"] is not None:
        dx = dx + st["dr"].float()
    dx = dx.to(dt)
    return out + [dx] * (1 + (st["res"] is not None)) + [(dy * xn).sum((0, 1)).flatten()]


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        op = state["case"]["op"]
        return _plain_norm(state) if op.startswith("norm") else _plain_step(state) if op == "step" else _plain_attention(state)


# --------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    """Step by step (attention), row by row (norm)."""
    st = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(st) if case["op"].startswith("norm") else _exact_attention(st)


def _exact_attention(st):
    case = st["case"]
    one = case["op"] == "step"
    q, k, v, f = (st[key].detach().double() for key in ("q", "k", "v", "f"))
    if one:
        q, k, v, f = (t[:, None] for t in (q, k, v, f))
    b, length, h, kd = q.shape
    vd = v.shape[-1]
    if b * h * kd * vd * 8 * length > (4e12 if case["op"] == "train" else 1e13):
        return None
    order = list(range(length))
    if case["reverse"]:
        order.reverse()
    a = torch.sigmoid(f)
    live = torch.ones(b, length, 1, device=q.device, dtype=torch.float64)
    fresh = torch.zeros(b, length, 1, dtype=torch.bool, device=q.device)
    if st["mask"] is not None:
        live = (~st["mask"]).double()[..., None]
        a = torch.where(st["mask"][..., None], 1.0, a)
    if st["reset"] is not None:
        fresh = st["reset"][..., None]
        a = torch.where(fresh, 0.0, a)
    q, k, v = (t * live[..., None] for t in (q, k, v))
    q = q * st["scale"]
    s = torch.zeros(b, h, kd, vd, device=q.device, dtype=torch.float64) if st["h"] is None else st["h"].detach().double()
    train = case["op"] == "train"
    y = torch.empty(b, length, h, vd, device=q.device, dtype=torch.float64)
    dq = torch.empty_like(q)
    dy = st["dy"].double() * live[..., None] if train else None
    for t in order:
        s = a[:, t, :, None, None] * s + k[:, t, :, :, None] * v[:, t, :, None, :]
        y[:, t] = torch.einsum("bhk,bhkv->bhv", q[:, t], s)
        if train:
            dq[:, t] = torch.einsum("bhkv,bhv->bhk", s, dy[:, t])
    if not train:
        return [y[:, 0], s] if one else [y, s]
    r = st["dh"].double()
    whole = (r * s).sum((-1, -2))
    dk, dv = torch.empty_like(k), torch.empty_like(v)
    da = torch.empty_like(a)
    for t in reversed(order):
        r = r + q[:, t, :, :, None] * dy[:, t, :, None, :]
        dk[:, t] = torch.einsum("bhkv,bhv->bhk", r, v[:, t])
        dv[:, t] = torch.einsum("bhkv,bhk->bhv", r, k[:, t])
        # <R_t, S_t> less what step t brought in itself is what came through its decay
        whole = whole + (q[:, t] * dq[:, t]).sum(-1) - (k[:, t] * dk[:, t]).sum(-1)
        da[:, t] = whole
        r = a[:, t, :, None, None] * r
        whole = torch.where(fresh[:, t], 0.0, whole)   # (nothing passes the first step of a document)
    df = (da * torch.sigmoid(-f) * live).masked_fill(fresh, 0.0)
    out = [y, s, dq * st["scale"] * live[..., None], dk * live[..., None], dv * live[..., None], df]
    return out + ([r] if st["h"] is not None else [])


def _exact_norm(st):
    case = st["case"]
    g = case["groups"]
    x = st["x"].detach()
    r = x.double() if st["res"] is None else (x.double() + st["res"].detach().double()).to(x.dtype).double()
    total = r
    b, n, d = r.shape
    r = r.reshape(b, n, g, d // g)
    w = (st["weight"].detach().double() + 1).reshape(g, d // g)
    size = torch.sqrt(torch.square(r).sum(-1, keepdim=True) / (d // g) + EPS)
    y = (r / size * w).reshape(b, n, d)
    out = [y] + ([] if st["res"] is None else [total])
    if case["op"] == "norm":
        return out
    dy = st["dy"].double().reshape(b, n, g, d // g)
    along = (dy * w * r).sum(-1, keepdim=True) / (d // g)
    dx = ((dy * w) / size - r * along / size ** 3).reshape(b, n, d)
    if st["res"] is not None:
        dx = dx + st["dr"].double()
    dw = (dy * r / size).sum((0, 1)).reshape(d)
    return out + [dx] * (1 + (st["res"] is not None)) + [dw]
