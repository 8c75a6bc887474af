"""Gated linear recurrence: forward, gradients, single steps, against the recurrence written out in 64 bits.

Tolerances.  With u = 2^-24 an fp32 pass rounds each product and sum of a step (at most 8 of them: the leak's sum and
reciprocal, the state's update, the decay's product, the joining of a state that comes in), relative to M_t, the same
recurrence over absolute values.  A leak is off by what its exponential is: relative (4 + |f|) 2 u for the 16-bit types'
approximate exponential and reciprocal, 4 * 2 u for fp32's; one below 2^-126 may be 0 (the exponential's overflow, or a
reciprocal that flushes): d_t = that times l_t, plus 2^-125.  Errors decay with the state, so
    E_t = (1 - l_t) E_{t-1} + 8 u M_t + d_t (M_{t-1} + |x_t|)
bounds the state's error, the mirrored recurrence the gradient's, and products add their factors' bounds.  An output of a
16-bit type adds half a step, eps / 2 of its value (and half the smallest subnormal).
"""
import ctypes

import pytest
import torch

U = 2.0 ** -24
F64 = torch.float64
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference(x, f, i=None, pad=None, reset=None, h_in=None, reverse=False, dy=None, dh=None):
    """All outputs and the bounds of their errors, (value, bound) each, from inputs of the tested type."""
    half = torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float32 else 0.0
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    slow = x.dtype == torch.float32

    def wide(t):
        return None if t is None else (t.flip(1) if reverse else t).detach().cpu().to(F64)

    def flags(t):
        return torch.zeros(B, L, 1, dtype=torch.bool) if t is None else ((t.flip(1) if reverse else t) != 0).cpu()[..., None]

    def back(t):
        return t.flip(1) if reverse else t

    B, L, D = x.shape
    x, f, i, dy = wide(x), wide(f), wide(i), wide(dy)
    pad, cut = flags(pad), flags(reset)
    x, f = torch.where(pad, 0.0, x), torch.where(pad, 0.0, f)
    i = None if i is None else torch.where(pad, 0.0, i)
    leak, keep = torch.sigmoid(-f), torch.sigmoid(f)
    s = None if i is None else torch.sigmoid(i)
    into = leak if s is None else s
    def gate_off(v, at):   # error of a gate of this value at this argument
        return 2 * U * (4 + (0 if slow else 1) * at.abs()) * v + 2.0 ** -125

    dl = gate_off(leak, f)
    ds = dl if i is None else gate_off(s, i)
    h = torch.zeros(B, D, dtype=F64) if h_in is None else h_in.detach().cpu().to(F64)
    m, e = h.abs(), torch.zeros(B, D, dtype=F64)
    hs, hp, ms, mp, es, ep = ([] for _ in range(6))
    for t in range(L):
        h = torch.where(cut[:, t], 0.0, h)
        m = torch.where(cut[:, t], 0.0, m)
        e = torch.where(cut[:, t], 0.0, e)
        hp.append(h), mp.append(m), ep.append(e)
        a, c = keep[:, t], into[:, t] * x[:, t]
        m1 = a * m + c.abs()
        e1 = a * e + 8 * U * m1 + dl[:, t] * m + ds[:, t] * x[:, t].abs()
        h = torch.where(pad[:, t], h, a * h + c)
        m = torch.where(pad[:, t], m, m1)
        e = torch.where(pad[:, t], e, e1)
        hs.append(h), ms.append(m), es.append(e)
    hs, hp, ms, mp, es, ep = (torch.stack(v, 1) for v in (hs, hp, ms, mp, es, ep))
    y = torch.where(pad, 0.0, hs)

    def out(v, err):
        return back(v), back(err * 1.01 + half * v.abs() + tiny)

    res = {"y": out(y, torch.where(pad, 0.0, es)), "h": (hs[:, -1], es[:, -1] + tiny)}
    if dy is None:
        return res
    dy = torch.where(pad, 0.0, dy)
    q = torch.zeros(B, D, dtype=F64) if dh is None else dh.detach().cpu().to(F64)
    mq, eq = q.abs(), torch.zeros(B, D, dtype=F64)
    gs, mg, eg = ([None] * L for _ in range(3))
    for t in range(L - 1, -1, -1):
        g, m1 = q + dy[:, t], mq + dy[:, t].abs()
        e1 = eq + U * m1
        gs[t], mg[t], eg[t] = g, m1, e1
        a = keep[:, t]
        q = torch.where(pad[:, t], q, a * g)
        mq = torch.where(pad[:, t], mq, a * m1)
        eq = torch.where(pad[:, t], eq, a * e1 + 8 * U * m1 + dl[:, t] * m1)
        q, mq, eq = (torch.where(cut[:, t], 0.0, v) for v in (q, mq, eq))
    g, mg, eg = (torch.stack(v, 1) for v in (gs, mg, eg))
    live = (~pad).to(F64)
    eg = eg + 8 * U * mg   # (the joining of what flows in from behind a segment)
    if s is None:
        val, top, off = hp - x, mp + x.abs(), ep + U * (mp + x.abs())
    else:
        val, top, off = hp, mp, ep
    # (the decay 1 - l as a factor is off by 2 u + dl absolutely, not relatively)
    fa = keep + 2 * U + dl
    df_err = (leak + dl) * (fa * top * eg + fa * mg * off + (8 * U + dl) * top * mg) + dl * fa * top * mg
    res["dx"] = out(live * into * g, live * (into * (eg + 4 * U * mg) + ds * mg))
    res["df"] = out(live * keep * leak * val * g, live * df_err)
    if s is not None:
        n = torch.sigmoid(-i)
        res["di"] = out(live * s * n * x * g, live * x.abs() * (s * n * (eg + 6 * U * mg) + (ds * n + s * gate_off(n, i)) * mg))
    res["dh"] = (q, eq + 8 * U * mq + tiny)
    return res


def close(got, want, what):
    value, bound = want
    got = got.detach().cpu().to(F64)
    assert got.shape == value.shape, (what, got.shape, value.shape)
    bad = ~((got - value).abs() <= bound)
    assert not bad.any(), "%s: %d of %d off, first at %s: %r, not %r +- %r" % (
        what, int(bad.sum()), bad.numel(), tuple(bad.nonzero()[0].tolist()), float(got[bad][0]), float(value[bad][0]), float(bound[bad][0]))


def inputs(B, L, D, dtype, gate, seed, pad=None, reset=None, state=True):
    gen = torch.Generator().manual_seed(seed)
    r = {"x": torch.randn(B, L, D, generator=gen), "f": torch.randn(B, L, D, generator=gen) * 2 + 2,
         "i": torch.randn(B, L, D, generator=gen) if gate else None, "dy": torch.randn(B, L, D, generator=gen)}
    r = {k: None if v is None else v.to(dtype) for k, v in r.items()}
    r["h_in"] = torch.randn(B, D, generator=gen) if state else None
    r["dh"] = torch.randn(B, D, generator=gen) if state else None
    n = torch.randint(0, L + 1, (B,), generator=gen)
    r["pad"] = {None: None, "right": torch.arange(L)[None] >= n[:, None], "left": torch.arange(L)[None] < n[:, None],
                "any": torch.rand(B, L, generator=gen) < 0.3, "all": torch.ones(B, L, dtype=torch.bool)}[pad]
    if r["pad"] is not None and B > 1 and pad == "right":
        r["pad"][-1] = True   # a sequence without a step
    r["reset"] = {None: None, "docs": torch.rand(B, L, generator=gen) < 0.1, "every": torch.ones(B, L, dtype=torch.bool)}[reset]
    return r


def cuda(t):
    return None if t is None else t.cuda()


def run_all(M, r, reverse, shape=lambda t: t):
    """inference and training on the GPU -> dict of outputs"""
    c = {k: cuda(v) for k, v in r.items()}
    x, f, i = (None if c[k] is None else shape(c[k]) for k in ("x", "f", "i"))
    with torch.no_grad():
        y0, h0 = M.gated_recurrence(x, f, i, c["pad"], c["reset"], c["h_in"], want_state=True, reverse=reverse)
    leaves = [t.detach().requires_grad_() for t in (x, f, i, c["h_in"]) if t is not None]
    at = iter(leaves)
    x1, f1 = next(at), next(at)
    i1 = next(at) if i is not None else None
    h1 = next(at) if c["h_in"] is not None else None
    y, h = M.gated_recurrence(x1, f1, i1, c["pad"], c["reset"], h1, want_state=True, reverse=reverse)
    for a, b in ((y0, y), (h0, h)):   # (NaN in the same places)
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
    outs, gs = ([y, h], [c["dy"], c["dh"]]) if c["dh"] is not None else ([y], [c["dy"]])
    grads = list(torch.autograd.grad(outs, leaves, gs))
    res = {"y": y, "h": h, "dx": grads.pop(0), "df": grads.pop(0)}
    if i is not None:
        res["di"] = grads.pop(0)
    if h1 is not None:
        res["dh"] = grads.pop(0)
    return res


def check_all(got, r, reverse, dtype):
    want = reference(r["x"], r["f"], r["i"], r["pad"], r["reset"], r["h_in"], reverse, r["dy"], r["dh"])
    for k, v in got.items():
        if k in ("y", "dx", "df", "di"):
            assert v.dtype == dtype
        close(v, want[k], k)


# --------------------------------------------------------------------------------------- without a GPU
def test_host_refuses_cpu_tensors():
    import fairseq_apollo_b200 as M
    x = torch.randn(2, 3, 4)
    for grad in (False, True):
        with pytest.raises(RuntimeError, match="CUDA"):
            M.gated_recurrence(x.clone().requires_grad_(grad), x)
    with pytest.raises(RuntimeError, match="CUDA"):
        M.ops.gated_recurrence_step(x[:, 0], x[:, 0])
    with pytest.raises(RuntimeError, match="CUDA"):
        M.GatedRecurrence(4)(x)


def test_abi_refusals():
    import fairseq_apollo_b200 as M
    from fairseq_apollo_b200 import _lib
    lib = _lib.lib()
    one, odd = ctypes.c_void_p(16), ctypes.c_void_p(18)
    s8, s14 = [4, 4] * 4, [4, 4] * 7

    def fwd(x=one, f=one, y=one, dtype=0, B=1, L=1, D=4, h=None):
        return lib.mega_gated_recurrence_fwd(x, f, None, y, dtype, B, L, D, *s8, None, None, h, None, None, 0, None)

    def bwd(dy=one, starts=one, i=None, di=None, dtype=0, B=1):
        return lib.mega_gated_recurrence_bwd(dy, one, one, i, one, one, di, dtype, B, 1, 4, *s14, None, None, starts, None, None, 0, None)

    assert fwd(x=None) == 1 and fwd(f=None) == 1 and fwd(y=None) == 1
    assert fwd(dtype=7) == 2 and fwd(B=0) == 3 and fwd(L=0) == 3 and fwd(D=-1) == 3
    assert fwd(x=odd) == 5 and fwd(h=odd) == 5 and fwd(x=ctypes.c_void_p(17), dtype=1) == 5
    assert fwd(B=65536) == 7
    assert bwd(dy=None) == 1 and bwd(starts=None) == 1 and bwd(i=one) == 1 and bwd(dtype=-1) == 2 and bwd(B=70000) == 7
    assert lib.mega_gated_recurrence_step(one, one, None, one, 0, 1, 4, 4, 4, 4, 4, None, None, None) == 1
    assert lib.mega_gated_recurrence_step(one, one, None, one, 0, 1, 0, 4, 4, 4, 4, None, one, None) == 3
    assert lib.mega_gated_recurrence_segment(9, 0) == 0
    for dt in range(3):
        assert lib.mega_gated_recurrence_segment(dt, 0) > 0 and lib.mega_gated_recurrence_segment(dt, 1) > 0


def test_reference_gradients_against_differences():
    """the formulas that the kernels are held to, by central differences in 64 bits"""
    for gate in (False, True):
        for reverse in (False, True):
            r = inputs(2, 9, 3, torch.float32, gate, 5, "any", "docs")
            want = reference(r["x"], r["f"], r["i"], r["pad"], r["reset"], r["h_in"], reverse, r["dy"], r["dh"])

            def value(**over):
                a = {k: (None if r[k] is None else r[k].to(F64)) for k in ("x", "f", "i", "h_in")}
                a.update(over)
                out = reference_f64(a["x"], a["f"], a["i"], r["pad"], r["reset"], a["h_in"], reverse)
                return (out[0] * r["dy"].to(F64)).sum() + (out[1] * r["dh"].to(F64)).sum()

            names = [("x", "dx"), ("f", "df"), ("h_in", "dh")] + ([("i", "di")] if gate else [])
            for name, grad in names:
                v = torch.randn(r[name].shape, generator=torch.Generator().manual_seed(1), dtype=F64)
                eps = 1e-5
                base = r[name].to(F64)
                diff = (value(**{name: base + eps * v}) - value(**{name: base - eps * v})) / (2 * eps)
                assert abs(float(diff - (want[grad][0] * v).sum())) < 1e-6 * (1 + abs(float(diff)))


def reference_f64(x, f, i, pad, reset, h, reverse):
    ts = range(x.shape[1] - 1, -1, -1) if reverse else range(x.shape[1])
    y = torch.zeros_like(x)
    for t in ts:
        if reset is not None:
            h = torch.where(reset[:, t, None], 0.0, h)
        a = torch.sigmoid(f[:, t])
        new = a * h + (1 - a if i is None else torch.sigmoid(i[:, t])) * x[:, t]
        dead = torch.zeros_like(new, dtype=torch.bool) if pad is None else pad[:, t, None].expand_as(new)
        h = torch.where(dead, h, new)
        y[:, t] = torch.where(dead, 0.0, h)
    return y, h


# ------------------------------------------------------------------------------------------- on the GPU
SHAPES = [(1, 1, 1), (2, 1, 64), (3, 5, 3), (2, 16, 64), (1, 17, 65), (2, 33, 130), (4, 127, 32), (2, 128, 64), (1, 129, 62),
          (5, 257, 96), (1, 1025, 200), (2, 2100, 72)]


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_64_bits(shape, dtype, gate):
    import fairseq_apollo_b200 as M
    B, L, D = shape
    r = inputs(B, L, D, dtype, gate, L * 3 + D, pad="right" if L % 2 else None, reset="docs" if D % 4 == 0 else None, state=L % 3 != 0)
    check_all(run_all(M, r, reverse=B % 2 == 0), r, B % 2 == 0, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("reset", [None, "docs", "every"])
@pytest.mark.parametrize("pad", [None, "right", "left", "any", "all"])
def test_masks(pad, reset, reverse):
    import fairseq_apollo_b200 as M
    for dtype, gate in ((torch.bfloat16, False), (torch.float32, True)):
        r = inputs(3, 301, 70, dtype, gate, 11, pad, reset)
        check_all(run_all(M, r, reverse), r, reverse, dtype)
        if r["pad"] is not None:   # a byte mask says the same
            r8 = dict(r, pad=r["pad"].to(torch.uint8) * 3, reset=None if r["reset"] is None else r["reset"].to(torch.int32))
            a, b = run_all(M, r, reverse), run_all(M, r8, reverse)
            assert all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("long", [(1, 40000, 16), (1, 9000, 520), (70, 600, 64), (300, 40, 128), (2, 20000, 33)])
def test_long_and_wide(long, gate):
    """the splits over time that few and many sequences take"""
    import fairseq_apollo_b200 as M
    r = inputs(*long, torch.bfloat16, gate, 3, "right" if long[0] == 70 else None, "docs" if long[1] == 9000 else None, state=long[0] != 2)
    check_all(run_all(M, r, False), r, False, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("cluster", [1, 2, 4, 8, 16])
def test_every_split_of_the_time_axis(cluster):
    """the same call over clusters of 1 to 8 blocks and by warps alone, padded, with documents, reversed; no wait gave up"""
    import fairseq_apollo_b200 as M
    from fairseq_apollo_b200 import _lib
    _lib.device_error(reset=True)
    try:
        _lib.set_option(8, cluster)
        for dtype, gate, D in ((torch.bfloat16, False, 64), (torch.float16, True, 70), (torch.float32, True, 65), (torch.float32, False, 128),
                               (torch.bfloat16, True, 33)):
            for L in (3, 700, 2049):
                r = inputs(2, L, D, dtype, gate, L + cluster, "any" if L == 700 else None, "docs" if L > 700 else None)
                check_all(run_all(M, r, L == 700), r, L == 700, dtype)
                assert _lib.last_kernel() == "gated_recurrence" + (" serial" if cluster == 16 else "")
    finally:
        _lib.set_option(8, 0)
    assert _lib.device_error() == 0


@pytest.mark.gpu
def test_gates_far_open_and_closed():
    """f up to +-200: leaks that vanish, states that are forgotten at once; everything stays finite"""
    import fairseq_apollo_b200 as M
    for dtype in DTYPES:
        for gate in (False, True):
            r = inputs(2, 200, 64, dtype, gate, 7)
            r["f"] = (r["f"] - 2).mul(50).clamp(-200, 200).to(dtype)
            if gate:
                r["i"] = r["i"].mul(60).to(dtype)
            got = run_all(M, r, False)
            assert all(torch.isfinite(v).all() for v in got.values())
            check_all(got, r, False, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [False, True])
def test_nothing_comes_out_of_padded_places_or_over_a_reset(gate):
    import fairseq_apollo_b200 as M
    for dtype in DTYPES:
        for pad in ("right", "any"):
            r = inputs(3, 150, 66, dtype, gate, 9, pad, "docs")
            clean = run_all(M, r, False)
            bad = dict(r)
            for k in ("x", "f", "i", "dy"):
                if r[k] is not None:
                    t = r[k].clone()
                    t[r["pad"]] = float("nan") if k != "f" else float("inf")
                    bad[k] = t
            dirty = run_all(M, bad, False)
            assert all(torch.equal(clean[k], dirty[k]) for k in clean)
        # a document that overflows, the next one untouched: forward as well as backward in time
        r = inputs(2, 300, 64, dtype, gate, 10)
        cut = torch.zeros(2, 300, dtype=torch.bool)
        cut[:, 137] = True
        r["reset"] = cut
        clean = run_all(M, r, False)
        bad = dict(r, x=r["x"].clone(), h_in=r["h_in"].clone(), dy=r["dy"].clone())
        bad["x"][:, 20] = float("nan")
        bad["h_in"][:] = float("inf")
        dirty = run_all(M, bad, False)
        assert torch.equal(clean["y"][:, 137:], dirty["y"][:, 137:]) and torch.equal(clean["h"], dirty["h"])
        assert torch.equal(clean["dx"][:, 137:], dirty["dx"][:, 137:]) and torch.equal(clean["df"][:, 137:], dirty["df"][:, 137:])
        bad = dict(r, dy=r["dy"].clone())
        bad["dy"][:, 200] = float("nan")
        dirty = run_all(M, bad, False)
        assert torch.equal(clean["dx"][:, :137], dirty["dx"][:, :137]) and torch.equal(clean["dh"], dirty["dh"])


@pytest.mark.gpu
def test_memory_orders_and_alignment():
    import fairseq_apollo_b200 as M

    def time_major(t):
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    def sliced(t):   # columns of a wider row, off the 16-byte boundaries
        wide = torch.full(t.shape[:-1] + (t.shape[-1] + 9,), 7.0, dtype=t.dtype, device=t.device)
        wide[..., 5:5 + t.shape[-1]] = t
        return wide[..., 5:5 + t.shape[-1]]

    def even(t):
        wide = torch.full(t.shape[:-1] + (t.shape[-1] + 16,), 7.0, dtype=t.dtype, device=t.device)
        wide[..., 8:8 + t.shape[-1]] = t
        return wide[..., 8:8 + t.shape[-1]]

    def length_last(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def flipped(t):   # every other step of a longer tensor
        wide = torch.zeros(t.shape[0], 2 * t.shape[1], t.shape[2], dtype=t.dtype, device=t.device)
        wide[:, ::2] = t
        return wide[:, ::2]

    for dtype in DTYPES:
        for D in (64, 70, 41):
            r = inputs(3, 140, D, dtype, True, 2, "any", "docs")
            plain = run_all(M, r, False)
            check_all(plain, r, False, dtype)
            for shape in (time_major, sliced, even, length_last, flipped):
                got = run_all(M, r, False, shape)
                assert all(torch.equal(plain[k], got[k]) for k in plain), (dtype, D, shape.__name__)
    # one sequence's gates for all of them, without a copy
    x = torch.randn(4, 50, 64, device="cuda")
    f = torch.randn(1, 50, 64, device="cuda")
    assert torch.equal(M.gated_recurrence(x, f.expand(4, 50, 64)), M.gated_recurrence(x, f.repeat(4, 1, 1)))
    xg, fg = x.clone().requires_grad_(), f.clone().requires_grad_()
    a = torch.autograd.grad(M.gated_recurrence(xg, fg.expand(4, 50, 64)).sum(), [xg, fg])
    b = torch.autograd.grad(M.gated_recurrence(xg, fg.repeat(4, 1, 1)).sum(), [xg, fg])
    assert torch.equal(a[0], b[0]) and torch.allclose(a[1], b[1], rtol=1e-5, atol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_operand(dtype, gate):
    """one tensor that holds the operands side by side: the same values, its gradient in one piece"""
    import fairseq_apollo_b200 as M
    from fairseq_apollo_b200 import functions
    for D in (64, 35):
        r = inputs(2, 77, D, dtype, gate, 4, "right", "docs")
        want = run_all(M, r, True)
        z = torch.cat([r["x"], r["f"]] + ([r["i"]] if gate else []), -1).cuda().requires_grad_()
        h_in = r["h_in"].cuda().requires_grad_()
        y, h = functions.gated_recurrence_packed(z, gate, r["pad"].cuda(), r["reset"].cuda(), h_in, True, True)
        dz, dh = torch.autograd.grad([y, h], [z, h_in], [r["dy"].cuda(), r["dh"].cuda()])
        assert torch.equal(y, want["y"]) and torch.equal(h, want["h"]) and torch.equal(dh, want["dh"])
        parts = dz.split(D, -1)
        assert torch.equal(parts[0], want["dx"]) and torch.equal(parts[1], want["df"])
        if gate:
            assert torch.equal(parts[2], want["di"])


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_and_pieces_equal_the_whole(dtype, gate):
    import fairseq_apollo_b200 as M
    for B, D in ((1, 1), (3, 70), (33, 512)):
        r = inputs(B, 12, D, dtype, gate, 8)
        x, f, i, h = (cuda(r[k]) for k in ("x", "f", "i", "h_in"))
        want = reference(r["x"], r["f"], r["i"], h_in=r["h_in"])
        ys, state = [], h.clone()
        for t in range(12):
            sl = [None if v is None else v[:, t] for v in (x, f, i)]
            before = state.clone()
            y, new = M.ops.gated_recurrence_step(*sl, state)
            assert torch.equal(state, before) and torch.equal(y, new.to(dtype))
            y2, same = M.ops.gated_recurrence_step(*sl, state, h_out=state)   # in place
            assert same is state or same.data_ptr() == state.data_ptr()
            assert torch.equal(state, new) and torch.equal(y2, y)
            ys.append(y)
        close(torch.stack(ys, 1), want["y"], "y")
        close(state, want["h"], "h")
        # in pieces of 5 with the state handed on
        h2, parts = h, []
        for k in range(0, 12, 5):
            y, h2 = M.gated_recurrence(x[:, k:k + 5], f[:, k:k + 5], None if i is None else i[:, k:k + 5], h_in=h2, want_state=True)
            parts.append(y)
        close(torch.cat(parts, 1), want["y"], "y")
        close(h2, want["h"], "h")
    y, h = M.ops.gated_recurrence_step(x[:, 0], f[:, 0])   # from nothing
    assert torch.equal(h, M.ops.gated_recurrence_step(x[:, 0], f[:, 0], None, torch.zeros_like(h))[1])


@pytest.mark.gpu
def test_truncated_backpropagation_through_states():
    """two chained calls have the gradients of one call over both"""
    import fairseq_apollo_b200 as M
    r = inputs(2, 90, 40, torch.float32, True, 21)
    x, f, i, h0, dy = (r[k].cuda() for k in ("x", "f", "i", "h_in", "dy"))
    leaves = [t.clone().requires_grad_() for t in (x, f, i, h0)]
    y1, h = M.gated_recurrence(leaves[0][:, :37], leaves[1][:, :37], leaves[2][:, :37], h_in=leaves[3], want_state=True)
    y2 = M.gated_recurrence(leaves[0][:, 37:], leaves[1][:, 37:], leaves[2][:, 37:], h_in=h)
    got = torch.autograd.grad([y1, y2], leaves, [dy[:, :37], dy[:, 37:]])
    want = reference(r["x"], r["f"], r["i"], h_in=r["h_in"], dy=r["dy"])
    for g, k in zip(got, ("dx", "df", "di", "dh")):
        close(g, want[k], k)


@pytest.mark.gpu
def test_state_alone_and_states_written_over():
    """a gradient through the state that leaves only; the state that came in, in 16 bits, overwritten before the backward"""
    import fairseq_apollo_b200 as M
    r = inputs(2, 50, 24, torch.float32, True, 31)
    leaves = [r[k].cuda().requires_grad_() for k in ("x", "f", "i", "h_in")]
    _, h = M.gated_recurrence(*leaves[:3], h_in=leaves[3], want_state=True)
    got = torch.autograd.grad(h, leaves, r["dh"].cuda())
    want = reference(r["x"], r["f"], r["i"], h_in=r["h_in"], dy=torch.zeros_like(r["dy"]), dh=r["dh"])
    for g, k in zip(got, ("dx", "df", "di", "dh")):
        close(g, want[k], k)
    state = r["h_in"].cuda().bfloat16()
    h0 = state.clone().requires_grad_()
    y, h = M.gated_recurrence(leaves[0], leaves[1], h_in=h0 * 1, want_state=True)
    assert torch.autograd.grad(y.sum(), h0, retain_graph=True)[0].dtype == torch.bfloat16
    y, h = M.gated_recurrence(leaves[0], leaves[1], h_in=state, want_state=True)
    state.copy_(h.detach())
    y.sum().backward()


@pytest.mark.gpu
def test_more_than_31_bits_of_values():
    """offsets past 2^31 values: the end of a long call, against the same steps by themselves behind the state before them"""
    import fairseq_apollo_b200 as M
    L, D, tail = 270000, 8192, 300
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(1, L, D, device="cuda", dtype=torch.bfloat16, generator=gen)
    f = torch.randn(1, L, D, device="cuda", dtype=torch.bfloat16, generator=gen)
    assert x.numel() > 2 ** 31
    with torch.no_grad():
        y, h = M.gated_recurrence(x, f, want_state=True)
        _, mid = M.gated_recurrence(x[:, :L - tail], f[:, :L - tail], want_state=True)
        z, end = M.gated_recurrence(x[:, L - tail:], f[:, L - tail:], h_in=mid, want_state=True)
    # (the same values joined at other places: states of size 1 within some 2^-21, outputs a bf16 step more)
    assert float((h - end).abs().max()) < 2.0 ** -20
    assert float((y[:, L - tail:].float() - z.float()).abs().max()) < 2.0 ** -7 * float(z.abs().max())
    del y, z
    xg, fg = x[:, L - 3 * tail:].clone(), f[:, L - 3 * tail:].clone()
    x.requires_grad_(), f.requires_grad_()
    y, h = M.gated_recurrence(x, f, want_state=True)
    dx, df = torch.autograd.grad(h, [x, f], torch.ones_like(h))
    xg.requires_grad_(), fg.requires_grad_()
    with torch.no_grad():
        _, mid = M.gated_recurrence(x[:, :L - 3 * tail], f[:, :L - 3 * tail], want_state=True)
    _, h = M.gated_recurrence(xg, fg, h_in=mid, want_state=True)
    a, b = torch.autograd.grad(h, [xg, fg], torch.ones_like(h))
    # (segments begin elsewhere, so sums differ in their last bits and a rounding to bf16 may go the other way: one step, eps of the
    # value.  dx is at most 1, df = q l (h - x) at most a quarter of |h| + |x| < 16)
    for full, part, top in ((dx, a, 1.0), (df, b, 4.0)):
        assert float((full[:, L - 3 * tail:].float() - part.float()).abs().max()) <= torch.finfo(torch.bfloat16).eps * top


@pytest.mark.gpu
def test_no_steps_no_sequences():
    import fairseq_apollo_b200 as M
    h = torch.randn(3, 8, device="cuda")
    x = torch.zeros(3, 0, 8, device="cuda")
    y, out = M.gated_recurrence(x, x, h_in=h, want_state=True)
    assert y.shape == (3, 0, 8) and torch.equal(out, h) and out.data_ptr() != h.data_ptr()
    assert (M.gated_recurrence(x, x, want_state=True)[1] == 0).all()
    e = torch.zeros(0, 5, 8, device="cuda")
    assert M.gated_recurrence(e, e).shape == (0, 5, 8)
    hg = h.clone().requires_grad_()
    xg = x.clone().requires_grad_()
    y, out = M.gated_recurrence(xg, x, h_in=hg, want_state=True)
    gx, gh = torch.autograd.grad([y, out], [xg, hg], [torch.zeros_like(y), torch.ones_like(out)])
    assert gx.shape == x.shape and (gh == 1).all()
    y, out = M.ops.gated_recurrence_step(e[:, 0], e[:, 0])
    assert y.shape == (0, 8)


@pytest.mark.gpu
def test_refusals():
    import fairseq_apollo_b200 as M
    x = torch.randn(2, 6, 8, device="cuda")
    for grad in (False, True):
        xg = x.clone().requires_grad_(grad)
        with pytest.raises(TypeError):
            M.gated_recurrence(xg, x.bfloat16())
        with pytest.raises(TypeError):
            M.gated_recurrence(xg.double(), x.double())
        with pytest.raises(ValueError):
            M.gated_recurrence(xg, x[:, :5])
        with pytest.raises(ValueError):
            M.gated_recurrence(xg, x, x[:1])
        with pytest.raises(ValueError):
            M.gated_recurrence(xg[0], x[0])
        with pytest.raises(ValueError):
            M.gated_recurrence(xg, x, padding_mask=torch.zeros(2, 5, device="cuda"))
        with pytest.raises(ValueError):
            M.gated_recurrence(xg, x, reset_mask=torch.zeros(6, 2, device="cuda"))
        with pytest.raises(RuntimeError):
            M.gated_recurrence(xg, x, padding_mask=torch.zeros(2, 6))
        with pytest.raises(ValueError):
            M.gated_recurrence(xg, x, h_in=torch.zeros(2, 9, device="cuda"))
        with pytest.raises(TypeError):
            M.gated_recurrence(xg, x, h_in=torch.zeros(2, 8, device="cuda", dtype=torch.int32))
    with pytest.raises(ValueError):
        M.ops.gated_recurrence_step(x[:, 0], x[:, 0], h=torch.zeros(2, 8, device="cuda"),
                                    h_out=torch.zeros(8, 2, device="cuda").t())
    with pytest.raises(ValueError):
        M.ops.gated_recurrence_step(x, x)
    states = torch.zeros(3, 8, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        M.ops.gated_recurrence_step(x[:, 0], x[:, 0], h=states[:2], h_out=states[1:])
    xg = x.clone().requires_grad_()
    g = M.gated_recurrence(xg, x)
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(g.sum(), xg, create_graph=True)
    y = M.gated_recurrence(xg * 1, x)
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError, match="modified"):   # an operand changed before the backward
        y.sum().backward()


@pytest.mark.gpu
def test_repeats_bit_for_bit_on_streams_and_in_graphs():
    import fairseq_apollo_b200 as M
    r = inputs(2, 700, 96, torch.bfloat16, False, 6, "any", "docs")
    want = run_all(M, r, False)
    x, f, h, dy, pad, cut = (r[k].cuda() for k in ("x", "f", "h_in", "dy", "pad", "reset"))
    leaves = [x.clone().requires_grad_(), f.clone().requires_grad_()]

    def train():
        y = M.gated_recurrence(*leaves, padding_mask=pad, reset_mask=cut, h_in=h)
        # (torch captures no backward pass while an eager graph of the same leaves lives: none is kept)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))

    base = train()
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for s in (side, other, side):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(train())
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(base, o))
    graphs = []
    for _ in range(2):   # two graphs, replayed in turn and at once
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = train()
        graphs.append((g, got))
    for s, (g, _) in zip((side, other), graphs):
        with torch.cuda.stream(s):
            for _ in range(3):
                g.replay()
    torch.cuda.synchronize()
    for _, got in graphs:
        assert all(torch.equal(a, b) for a, b in zip(base, got))
    with torch.no_grad():   # new values in the captured tensors
        leaves[0].copy_(leaves[0].flip(0))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(train(), graphs[0][1]))
    assert torch.equal(want["y"], base[0])


@pytest.mark.gpu
@pytest.mark.parametrize("bidirectional", [False, True])
@pytest.mark.parametrize("gate", [False, True])
def test_module(gate, bidirectional):
    """the layer: its gradients, its state dict, documents that do not see one another"""
    import fairseq_apollo_b200 as M
    torch.manual_seed(0)
    layer = M.GatedRecurrence(48, input_gate=gate, bidirectional=bidirectional).cuda()
    u = torch.randn(2, 61, 48, device="cuda", requires_grad=True)
    pad = torch.zeros(2, 61, dtype=torch.bool, device="cuda")
    pad[1, 40:] = True
    reset = torch.zeros_like(pad)
    reset[:, [0, 17]] = True
    y = layer(u, pad, reset_mask=reset)
    y.square().sum().backward()
    w = {k: v.detach().cpu().to(F64).requires_grad_() for k, v in layer.named_parameters()}
    u64 = u.detach().cpu().to(F64).requires_grad_()

    def walk(name, cut, reverse):
        z = u64 @ w[name + ".weight"].t() + w[name + ".bias"]
        parts = list(z.split(48, -1)) + ([] if gate else [None])
        h = torch.zeros(2, 48, dtype=F64)
        ys = {}
        for t in (range(60, -1, -1) if reverse else range(61)):
            h = torch.where(cut[:, t, None], 0.0, h)
            a = torch.sigmoid(parts[1][:, t])
            new = a * h + (1 - a if parts[2] is None else torch.sigmoid(parts[2][:, t])) * parts[0][:, t]
            dead = pad.cpu()[:, t, None]
            h = torch.where(dead, h, new)
            ys[t] = torch.where(dead, 0.0, h)
        return torch.stack([ys[t] for t in range(61)], 1)

    ref = walk("in_proj", reset.cpu(), False)
    if bidirectional:
        ends = torch.zeros(2, 61, dtype=torch.bool)
        ends[:, 16] = ends[:, 60] = True
        ref = ref + walk("back_proj", ends, True)
    ref.square().sum().backward()
    # (projections in fp32 or TF32-free matmuls: relative 1e-4 leaves room for their order of summation)
    assert float((y.detach().cpu().to(F64) - ref).norm() / ref.norm()) < 1e-5
    assert float((u.grad.cpu().to(F64) - u64.grad).norm() / u64.grad.norm()) < 1e-4
    for k, v in layer.named_parameters():
        assert float((v.grad.cpu().to(F64) - w[k].grad).norm() / w[k].grad.norm()) < 1e-4, k
    with torch.no_grad():
        if not bidirectional:   # prompt, then token by token, reordered on the way
            inc, whole = {}, layer(u)
            a = layer(u[:, :50], incremental_state=inc)
            assert float((a - whole[:, :50]).abs().max()) < 1e-5
            layer.reorder_incremental_state(inc, torch.tensor([1, 0], device="cuda"))
            for t in range(50, 61):
                step = layer(u[:, t:t + 1].flip(0), incremental_state=inc)
                assert float((step.flip(0) - whole[:, t:t + 1]).abs().max()) < 1e-5
        else:
            with pytest.raises(AssertionError):
                layer(u, incremental_state={})
    if not bidirectional:
        with pytest.raises(NotImplementedError):
            layer(u, incremental_state={})
    other = M.GatedRecurrence(48, input_gate=gate, bidirectional=bidirectional)
    other.load_state_dict(layer.state_dict())



@pytest.mark.gpu
def test_training_converts_its_operands_once():
    """channels that are not adjacent, integer masks, a 16-bit state: a training forward allocates what inference does, and the saved states"""
    import fairseq_apollo_b200 as M
    x, f, i = (torch.randn(2, 24, 40, device="cuda").transpose(1, 2) for _ in range(3))
    pad, reset = torch.zeros(2, 40, dtype=torch.int32, device="cuda"), torch.zeros(2, 40, dtype=torch.uint8, device="cuda")
    h = torch.zeros(2, 24, dtype=torch.bfloat16, device="cuda")

    def allocations(x):
        M.gated_recurrence(x, f, i, pad, reset, h, want_state=True)
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        M.gated_recurrence(x, f, i, pad, reset, h, want_state=True)
        return torch.cuda.memory_stats()["allocation.all.allocated"] - before

    with torch.no_grad():
        plain = allocations(x)
    assert allocations(x.detach().requires_grad_()) == plain + 1


@pytest.mark.gpu
def test_a_step_refuses_halves():
    import fairseq_apollo_b200 as M
    f, state = torch.randn(2, 8, device="cuda"), torch.randn(2, 8, device="cuda")
    whole = torch.randn(3, 8, device="cuda")
    for args in ((whole[:2], f, None), (f, whole[:2], None), (f, f, whole[:2]), (whole[1:2].expand(2, 8), f, None),
                 (whole[1:].t().reshape(-1)[:16].view(2, 8).expand(2, 8), f, whole[:2])):
        with pytest.raises(ValueError, match="overlaps"):
            M.ops.gated_recurrence_step(*args, state, h_out=whole[1:])
    half = whole.view(torch.bfloat16)[1:, :8]   # (the same memory in another type)
    with pytest.raises(ValueError, match="overlaps"):
        M.ops.gated_recurrence_step(half, half, None, state, h_out=whole[1:])
    x = torch.randn(2, 8, device="cuda")
    want = M.ops.gated_recurrence_step(x, f, None, state)[1]
    assert torch.equal(M.ops.gated_recurrence_step(x, f, None, state, h_out=x)[1], want)   # x itself, value for value


@pytest.mark.gpu
def test_a_step_in_place_tells_graphs():
    import fairseq_apollo_b200 as M
    f = torch.randn(2, 8, device="cuda")
    p = torch.ones(2, 8, device="cuda", requires_grad=True)
    state = torch.randn(2, 8, device="cuda")
    z = (p * state).sum()   # (keeps the state for p's gradient)
    M.ops.gated_recurrence_step(f, f, None, state, h_out=state)
    with pytest.raises(RuntimeError, match="modified"):
        z.backward()
    with torch.inference_mode():
        s = torch.zeros(2, 8, device="cuda")
        assert M.ops.gated_recurrence_step(f, f, None, s, h_out=s)[1].data_ptr() == s.data_ptr()
    M.ops.gated_recurrence_step(f, f, None, s, h_out=s)


@pytest.mark.gpu
def test_the_split_reckons_with_the_blocks_that_fit():
    """the fp32 backward with an input gate has a multiprocessor for each of its blocks: 100 sequences' tiles by blocks by themselves"""
    import fairseq_apollo_b200 as M
    from fairseq_apollo_b200 import _lib
    r = inputs(20, 1000, 320, torch.float32, True, 1)
    leaves = [cuda(r[k]).requires_grad_() for k in ("x", "f", "i", "h_in")]
    y = M.gated_recurrence(*leaves[:3], h_in=leaves[3])
    dy = cuda(r["dy"])

    def backward(cluster):
        _lib.set_option(8, cluster)
        try:
            return torch.autograd.grad(y, leaves, dy, retain_graph=True)
        finally:
            _lib.set_option(8, 0)

    chosen, one, four = backward(0), backward(1), backward(4)
    assert any(not torch.equal(a, b) for a, b in zip(one, four))   # (maps are joined in another order)
    assert all(torch.equal(a, b) for a, b in zip(chosen, one))
