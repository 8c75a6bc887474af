"""Gated linear recurrence where gates stand nearly closed or nearly open: both sides of a gate to their last places.

Tolerances.  With u = 2^-24, the smaller side g of a gate (the leak where f >= 0, the decay where f < 0) is off by r g with
r = 2 u (4 + |f|) for the 16-bit types' approximate exponential and reciprocal, 8 u in fp32, and by 2^-125 where it is below 2^-126;
the larger side, 1 - g, then by r g <= r (1 - g) too.  In the 16-bit types a decay of more than e^-6 (fp16: e^-5) may be 1 - l instead:
the sum 1 + e, its reciprocal (2 u) and the difference leave it within 5 u of 1, so 5 u / k come to its r.  So with decay k, leak l and M_t = k M_{t-1} + (l or the input gate) |x_t|, the same
recurrence over absolute values, a step adds (r + 8 u) M_t to the state's error (its products and sums, the joining of segments), and
    E_t = k E_{t-1} + (r + 8 u) M_t + 2^-125 (M_{t-1} + |x_t|).
The gradient's recurrence likewise; products add their factors' bounds, df = k l (h_{t-1} - x) g having both sides as factors.
16-bit outputs add half a step, eps / 2 of their value, and the smallest subnormal.
"""
import pytest
import torch
from test_gated_recurrence import DTYPES, F64, U, close, cuda, inputs, run_all

LEAST = 2.0 ** -125
TAKEN_AS_DIFFERENCE = {torch.bfloat16: -6.0, torch.float16: -5.0}   # gates' arguments from here on


def tight(x, f, i=None, pad=None, reset=None, h_in=None, reverse=False, dy=None, dh=None):
    """outputs of the recurrence and the bounds of their errors, (value, bound) each"""
    half = torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float32 else 0.0
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    spread = 0.0 if x.dtype == torch.float32 else 1.0
    B, L, D = x.shape
    x_dtype = x.dtype

    def turn(t):
        return t.flip(1) if reverse else t

    def wide(t):
        return None if t is None else turn(t.detach().cpu().to(F64))

    def flags(t):
        return torch.zeros(B, L, 1, dtype=torch.bool) if t is None else turn((t != 0).cpu())[..., None]

    x, f, i, dy, pad, cut = wide(x), wide(f), wide(i), wide(dy), flags(pad), flags(reset)
    x, f = torch.where(pad, 0.0, x), torch.where(pad, 0.0, f)
    k, l = torch.sigmoid(f), torch.sigmoid(-f)
    r = 2 * U * (4 + spread * f.abs())
    if x_dtype in TAKEN_AS_DIFFERENCE:
        r = r + torch.where(f >= TAKEN_AS_DIFFERENCE[x_dtype], 5 * U / k, 0.0)
    if i is None:
        s, rs = l, 2 * U * (4 + spread * f.abs())
    else:
        i = torch.where(pad, 0.0, i)
        s, rs = torch.sigmoid(i), 2 * U * (4 + spread * i.abs())
    h = torch.zeros(B, D, dtype=F64) if h_in is None else h_in.detach().cpu().to(F64)
    m, e = h.abs(), torch.zeros(B, D, dtype=F64)
    rows = []
    for t in range(L):
        h, m, e = (torch.where(cut[:, t], 0.0, v) for v in (h, m, e))
        c = s[:, t] * x[:, t]
        m1 = k[:, t] * m + c.abs()
        e1 = k[:, t] * e + 8 * U * m1 + r[:, t] * k[:, t] * m + rs[:, t] * c.abs() + LEAST * (m + x[:, t].abs())
        new = [torch.where(pad[:, t], a, b) for a, b in ((h, k[:, t] * h + c), (m, m1), (e, e1))]
        rows.append([h, m, e] + new)
        h, m, e = new
    hp, mp, ep, hs, _, es = (torch.stack(v, 1) for v in zip(*rows))

    def out(v, err):
        v, err = torch.where(pad, 0.0, v), torch.where(pad, 0.0, err)
        return turn(v), turn(err * 1.01 + half * v.abs() + tiny)

    res = {"y": out(hs, es), "h": (h, e * 1.01 + tiny)}
    if dy is None:
        return res
    dy = torch.where(pad, 0.0, dy)
    q = torch.zeros(B, D, dtype=F64) if dh is None else dh.detach().cpu().to(F64)
    mq, eq = q.abs(), torch.zeros(B, D, dtype=F64)
    rows = [None] * L
    for t in range(L - 1, -1, -1):
        g, mg = q + dy[:, t], mq + dy[:, t].abs()
        eg = eq + U * mg
        rows[t] = (g, mg, eg)
        a = k[:, t]
        q, mq, eq = (torch.where(cut[:, t], 0.0, torch.where(pad[:, t], v, w)) for v, w in
                     ((q, a * g), (mq, a * mg), (eq, a * eg + (8 * U + r[:, t]) * a * mg + LEAST * mg)))
    g, mg, eg = (torch.stack(v, 1) for v in zip(*rows))
    eg = eg + 8 * U * mg   # (the joining of what flows in from behind a segment)
    if i is None:
        v, mv, ev = hp - x, mp + x.abs(), ep + U * (mp + x.abs())
    else:
        v, mv, ev = hp, mp, ep
    res["dx"] = out(s * g, s * (eg + (4 * U + rs) * mg) + LEAST * mg)
    res["df"] = out(k * l * v * g, k * l * (mv * eg + mg * ev + (8 * U + 2 * r) * mv * mg) + LEAST * mv * mg)
    if i is not None:
        n = torch.sigmoid(-i)
        res["di"] = out(s * n * x * g, x.abs() * (s * n * (eg + (8 * U + 2 * rs) * mg) + 2 * LEAST * mg))
    res["dh"] = (q, eq * 1.01 + 8 * U * mq + tiny)
    return res


def check_all(got, r, reverse=False):
    want = tight(r["x"], r["f"], r["i"], r["pad"], r["reset"], r["h_in"], reverse, r["dy"], r["dh"])
    for k, v in got.items():
        close(v, want[k], k)


def closed(B, L, D, dtype, gate, seed, low=-30.0, high=-6.0, scale=1.0, **kw):
    r = inputs(B, L, D, dtype, gate, seed, **kw)
    gen = torch.Generator().manual_seed(seed + 1)
    r["f"] = (low + (high - low) * torch.rand(B, L, D, generator=gen)).to(dtype)
    r["h_in"] = r["h_in"] * scale
    return r


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_closed_gates_keep_their_gradient(dtype, gate):
    """decays down to e^-30: df is their product, and a state of 10^6 leaves as such a decay says"""
    import fairseq_apollo_b200 as M
    for L, scale in ((1, 1.0), (1, 1e6), (3, 1e4), (40, 1e6), (300, 1.0)):
        for reverse in (False, True):
            r = closed(2, L, 66, dtype, gate, L, scale=scale, pad="any" if L == 40 else None, reset="docs" if L == 300 else None)
            got = run_all(M, r, reverse)
            check_all(got, r, reverse)
            if dtype == torch.float32:   # (0 behind resets and where padded only)
                want = tight(r["x"], r["f"], r["i"], r["pad"], r["reset"], r["h_in"], reverse, r["dy"], r["dh"])["df"][0]
                assert torch.equal(got["df"].cpu() != 0, want != 0)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gates_of_both_kinds(dtype, gate):
    """closed and open gates side by side and in turn, from decays of e^-80 to leaks of e^-80"""
    import fairseq_apollo_b200 as M
    for D in (64, 35):
        r = closed(2, 150, D, dtype, gate, 9, -80.0, 80.0, 1e3, reset="docs")
        check_all(run_all(M, r, False), r)
        r["f"][:, ::2] = 0.0
        r["f"][:, 1::4] = -0.0
        check_all(run_all(M, r, False), r)
        r = inputs(2, 150, D, dtype, gate, 10, "right")
        check_all(run_all(M, r, True), r, True)


@pytest.mark.gpu
@pytest.mark.parametrize("cluster", [1, 2, 4, 8, 16])
def test_closed_gates_over_every_split(cluster):
    import fairseq_apollo_b200 as M
    from fairseq_apollo_b200 import _lib
    try:
        _lib.set_option(8, cluster)
        for dtype, gate in ((torch.bfloat16, False), (torch.float32, True)):
            for L, low, high in ((700, -12.0, 3.0), (90, -30.0, -8.0)):
                r = closed(2, L, 70, dtype, gate, L, low, high, 1e5, reset="docs" if L == 700 else None)
                check_all(run_all(M, r, False), r)
    finally:
        _lib.set_option(8, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_single_steps(dtype, gate):
    """an old state leaves as far as its decay says, step by step"""
    import fairseq_apollo_b200 as M
    r = closed(3, 6, 70, dtype, gate, 4, scale=1e6)
    r["f"][:, 3:] = inputs(3, 3, 70, dtype, gate, 5)["f"]
    want = tight(r["x"], r["f"], r["i"], h_in=r["h_in"])
    state, ys = cuda(r["h_in"]), []
    for t in range(6):
        y, state = M.ops.gated_recurrence_step(*(None if r[k] is None else cuda(r[k][:, t]) for k in ("x", "f", "i")), state)
        ys.append(y)
    close(torch.stack(ys, 1), want["y"], "y")
    close(state, want["h"], "h")


# ------------------------------------------------------------ infinite, missing and very large values
def same_or_close(got, want, what, dtype=None):
    """within the bound where the 64-bit value is finite in the output's type, the same infinity or NaN elsewhere"""
    value, bound = want
    got = got.detach().cpu().to(F64)
    top = torch.finfo(dtype or torch.float32).max
    odd = ~(value.abs() <= top)
    assert torch.equal(got[odd].isnan(), value[odd].isnan()), what
    assert torch.equal(got[odd].nan_to_num(0.0, 1.0, -1.0).sign(), value[odd].nan_to_num(0.0, 1.0, -1.0).sign()), what
    assert not torch.isfinite(got[odd]).any(), what
    close(torch.where(odd, 0.0, got), (torch.where(odd, 0.0, value), torch.where(odd, 1.0, bound)), what)


def check_odd(got, r, reverse=False):
    want = tight(r["x"], r["f"], r["i"], r["pad"], r["reset"], r["h_in"], reverse, r["dy"], r["dh"])
    for k, v in got.items():
        same_or_close(v, want[k], k, v.dtype)


def odd_values(B, L, D, dtype, gate, seed, what, **kw):
    """ordinary inputs, some channels of which hold something that is not finite, at the ends and within segments"""
    r = inputs(B, L, D, dtype, gate, seed, **kw)
    inf, nan = float("inf"), float("nan")
    if what in ("state", "all"):
        r["h_in"][0, 1], r["h_in"][-1, 2], r["h_in"][0, D - 1] = inf, -inf, nan
        r["h_in"][0, 3] = inf
        r["x"][0, L // 2, 3] = -inf   # the other infinity: NaN from there
    if what in ("input", "all"):
        r["x"][0, L // 3, 5], r["x"][0, 0, 6], r["x"][-1, L - 1, 7] = inf, -inf, nan
    if what in ("gradient", "all"):
        r["dy"][0, L // 3, 9], r["dy"][0, 0, 10], r["dy"][-1, L - 1, 11], r["dy"][0, L - 1, 12] = inf, -inf, nan, inf
        r["dh"][0, 13], r["dh"][-1, 14], r["dh"][0, 12] = inf, -inf, -inf
    return r


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["state", "input", "gradient", "all"])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_values_stay(dtype, gate, what):
    """an infinite state, input or gradient stays what it is until a reset or the other infinity, through decays whose product is 0 in
    fp32 too, and changes nothing beside itself"""
    import fairseq_apollo_b200 as M
    for L, kw in ((1, {}), (2, {}), (45, {}), (45, {"pad": "any", "reset": "docs"}), (400, {"reset": "docs"}), (700, {})):
        for reverse in (False, True):
            r = odd_values(2, L, 66, dtype, gate, L + 1, what, **kw)
            check_odd(run_all(M, r, reverse), r, reverse)
    r = odd_values(2, 300, 32, dtype, gate, 3, what)
    r["f"] = (r["f"] - 3).clamp(max=0).to(dtype)
    check_odd(run_all(M, r, False), r)


@pytest.mark.gpu
@pytest.mark.parametrize("cluster", [1, 2, 4, 8, 16])
def test_infinite_values_over_every_split(cluster):
    import fairseq_apollo_b200 as M
    from fairseq_apollo_b200 import _lib
    _lib.device_error(reset=True)
    try:
        _lib.set_option(8, cluster)
        for dtype, gate in ((torch.bfloat16, False), (torch.float32, True), (torch.float16, True), (torch.float32, False)):
            for L, kw in ((700, {"reset": "docs"}), (2100, {}), (90, {"pad": "any"})):
                r = odd_values(2, L, 70, dtype, gate, L, "all", **kw)
                check_odd(run_all(M, r, L == 90), r, L == 90)
    finally:
        _lib.set_option(8, 0)
    assert _lib.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_values_in_single_steps(dtype, gate):
    import fairseq_apollo_b200 as M
    r = odd_values(3, 9, 66, dtype, gate, 5, "all")
    want = tight(r["x"], r["f"], r["i"], h_in=r["h_in"])
    state, ys = cuda(r["h_in"]), []
    for t in range(9):
        y, state = M.ops.gated_recurrence_step(*(None if r[k] is None else cuda(r[k][:, t]) for k in ("x", "f", "i")), state)
        ys.append(y)
    same_or_close(torch.stack(ys, 1), want["y"], "y", dtype)
    same_or_close(state, want["h"], "h")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_next_to_the_largest(dtype):
    """states and inputs whose difference is past fp32's range: the state between them is not"""
    import fairseq_apollo_b200 as M
    for L in (1, 2, 37, 300):
        r = inputs(2, L, 66, dtype, False, L)
        r["f"] = (r["f"] - 2).to(dtype)
        r["x"] = (3e38 * torch.randn(r["x"].shape, generator=torch.Generator().manual_seed(2)).sign()).to(dtype)
        r["h_in"] = 3e38 * r["h_in"].sign()
        r["dy"], r["dh"] = (r["dy"] * 0.1).to(dtype), r["dh"] * 0.1
        got = run_all(M, r, False)
        assert torch.isfinite(got["y"]).all() and torch.isfinite(got["h"]).all()
        check_odd(got, r)
    x, f = r["x"][:, 0], r["f"][:, 0]
    y, h = M.ops.gated_recurrence_step(cuda(x), cuda(f), None, cuda(r["h_in"]))
    want = tight(x[:, None], f[:, None], h_in=r["h_in"])
    close(h, want["h"], "h")
    close(y[:, None], want["y"], "y")
    # an input gate: h = 3e38 and a value of the same size add up to no more than that where both are held back
    big = torch.full((2, 66), 3e38)
    f, i = torch.full((2, 1, 66), -1.0).to(dtype), torch.full((2, 1, 66), -1.0).to(dtype)
    x = big[:, None].to(dtype)
    for h_in in (big, -big):
        want = tight(x, f, i, h_in=h_in)
        y, h = M.gated_recurrence(cuda(x), cuda(f), cuda(i), h_in=cuda(h_in), want_state=True)
        close(h, want["h"], "h")
        close(M.ops.gated_recurrence_step(cuda(x[:, 0]), cuda(f[:, 0]), cuda(i[:, 0]), cuda(h_in))[1], want["h"], "h")


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_values_in_other_memory_orders(dtype, gate):
    """rows on odd addresses, columns of wider rows, time first, channels not adjacent"""
    import fairseq_apollo_b200 as M

    def odd_columns(t):
        wide = torch.full(t.shape[:-1] + (t.shape[-1] + 9,), 7.0, dtype=t.dtype, device=t.device)
        wide[..., 5:5 + t.shape[-1]] = t
        return wide[..., 5:5 + t.shape[-1]]

    for D in (64, 65):
        for L, kw in ((300, {"pad": "right"}), (90, {"reset": "docs"})):
            r = odd_values(3, L, D, dtype, gate, D + L, "all", **kw)
            plain = run_all(M, r, False)
            check_odd(plain, r)
            for shape in (odd_columns, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                          lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
                got = run_all(M, r, False, shape)
                for k in plain:
                    assert torch.equal(plain[k].nan_to_num(3.0), got[k].nan_to_num(3.0)), k


@pytest.mark.gpu
def test_infinite_values_replayed():
    """captured, replayed with an infinity in the captured tensors and without again"""
    import fairseq_apollo_b200 as M
    r = inputs(2, 900, 64, torch.bfloat16, False, 6, None, "docs")
    x, f, h, cut = (cuda(r[k]) for k in ("x", "f", "h_in", "reset"))

    def call():
        with torch.no_grad():
            return M.gated_recurrence(x, f, reset_mask=cut, h_in=h, want_state=True)

    clean = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    keep = x.clone()
    for value in (float("inf"), None, float("nan"), None):
        x.copy_(keep)
        if value is not None:
            x[0, 10, 3] = value
        graph.replay()
        torch.cuda.synchronize()
        want = clean if value is None else call()
        assert all(torch.equal(a.nan_to_num(3.0), b.nan_to_num(3.0)) for a, b in zip(got, want))
        assert (value is None) == bool(torch.isfinite(got[0]).all())
