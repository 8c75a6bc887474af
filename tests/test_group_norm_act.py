"""Group norm with an activation, channels last: forward and gradients against the formulas in 64 bits.

Tolerances.  With u = 2^-24 and a group of n values of size up to X (before the mean is taken off): a mean of tree and lane sums
is off by at most k u X with k = 40 + n / 256 additions in a row (at least 256 lanes walk a run each, runs are joined); xhat by k u X rstd plus
k u relative; z, its sigmoid (relative (8 + |z|) u) and products add a few u each.  A gradient's group sums are off by
k u of the mean of the absolute values.  Each bound below is that sum, with 16-bit outputs half a step, eps / 2, more.
Sums over R sequences and steps (dweight, dbias): (64 + R / 8) u of the sum of absolute values (at least 8 lanes walk a run each),
plus what their terms are off by.
"""
import ctypes

import pytest
import torch

U = 2.0 ** -24
F64 = torch.float64
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference(x, weight, bias, groups, pad=None, eps=1e-5, silu=True, dy=None):
    """outputs as (value, bound); x (B, L, D) of the tested type, weight the scale's offset"""
    half = torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float32 else 0.0
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    B, L, D = x.shape
    gs = D // groups
    K, R = 40 + L * gs / 256, 64 + B * L / 8
    live = torch.ones(B, L, 1, 1, dtype=torch.bool) if pad is None else ~pad.cpu().bool()[..., None, None]
    n = live.sum(1, keepdim=True).to(F64) * gs
    inv = torch.where(n > 0, 1 / n, 0.0)
    x = torch.where(live, x.detach().cpu().to(F64).view(B, L, groups, gs), 0.0)
    w, c = (1 + weight.cpu().to(F64)).view(1, 1, groups, gs), bias.cpu().to(F64).view(1, 1, groups, gs)

    def gmean(t):
        return torch.where(live, t, 0.0).sum((1, 3), keepdim=True) * inv

    mean = gmean(x)
    off = torch.where(live, x - mean, 0.0)
    var = gmean(off.square())
    rstd = 1 / (var + eps).sqrt()
    top = torch.where(live, x.abs(), 0.0).amax((1, 3), keepdim=True)
    em = K * U * top                                         # of the mean
    # of the variance, relative: the sum's k u, and the mean's error squared (its first order vanishes)
    er = K * U + 0.5 * (em * rstd).square() + 4 * U          # of rstd, relative
    xh = off * rstd
    ex = (em + 2 * U * (x.abs() + mean.abs())) * rstd + (er + 2 * U) * xh.abs()
    z = xh * w + c
    ez = w.abs() * ex + 3 * U * (z.abs() + (xh * w).abs() + c.abs())
    s = torch.sigmoid(z) if silu else torch.ones_like(z)
    n_s = torch.sigmoid(-z)
    # sigmoid: its argument's error through its slope s (1 - s), and the exponential's own
    es = s * n_s * ez + (8 + z.abs()) * 2 * U * s + 2.0 ** -125 if silu else torch.zeros_like(z)
    act = z * s
    slope = s * (1 + z * n_s) if silu else torch.ones_like(z)
    curve = s * n_s * (2 + z.abs()) if silu else torch.zeros_like(z)     # |slope'| <= this
    eslope = curve * ez + ((8 + z.abs()) * 2 * U * (s + s * n_s * z.abs() * 2) + 6 * U * (s + (s * z * n_s).abs()) + 4 * U * s * z.abs()
                           + 2.0 ** -120 if silu else 0.0)

    def out(v, err):
        v, err = (torch.where(live, t, 0.0).reshape(B, L, D) for t in (v, err))
        return v, err * 1.01 + half * v.abs() + tiny

    res = {"y": out(act, s * ez + z.abs() * es + 2 * U * act.abs())}
    res["count"] = live.sum((1, 2, 3))
    res["mean"] = (mean.view(B, groups), em.view(B, groups) + tiny)
    res["rstd"] = (rstd.view(B, groups), (er * rstd).view(B, groups))
    if dy is None:
        return res
    dy = torch.where(live, dy.cpu().to(F64).view(B, L, groups, gs), 0.0)
    dz = dy * slope
    edz = dy.abs() * eslope + 2 * U * dz.abs()
    dn, edn = dz * w, edz * w.abs() + 2 * U * (dz * w).abs()
    m1, m2 = gmean(dn), gmean(dn * xh)
    em1 = gmean(edn) + K * U * gmean(dn.abs())
    em2 = gmean(edn * xh.abs() + dn.abs() * ex) + (K + 2) * U * gmean((dn * xh).abs())
    dx = rstd * (dn - m1 - xh * m2)
    size = dn.abs() + m1.abs() + (xh * m2).abs()
    edx = rstd * (edn + em1 + xh.abs() * em2 + ex * m2.abs() + 4 * U * size) + (er + U) * rstd * size
    res["dx"] = out(dx, edx)
    dw, db = (dz * xh).sum((0, 1)).view(D), dz.sum((0, 1)).view(D)
    res["dw"] = (dw, (edz * xh.abs() + dz.abs() * ex + R * U * (dz * xh).abs()).sum((0, 1)).view(D) + tiny)
    res["db"] = (db, (edz + R * U * dz.abs()).sum((0, 1)).view(D) + tiny)
    return res


def close(got, want, what):
    value, bound = want
    got = got.detach().cpu().to(F64).reshape(value.shape)
    bad = ~((got - value).abs() <= bound)
    assert not bad.any(), "%s: %d of %d off, first at %s: %r, not %r +- %r" % (
        what, int(bad.sum()), bad.numel(), tuple(bad.nonzero()[0].tolist()), float(got[bad][0]), float(value[bad][0]), float(bound[bad][0]))


def inputs(B, L, D, dtype, seed, pad=None, shift=0.3):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, L, D, generator=gen) * 1.5 + torch.randn(D, generator=gen) + shift).to(dtype)
    dy = torch.randn(B, L, D, generator=gen).to(dtype)
    w, c = torch.randn(D, generator=gen) * 0.2, torch.randn(D, generator=gen) * 0.2
    n = torch.randint(0, L + 1, (B,), generator=gen)
    mask = {None: None, "right": torch.arange(L)[None] >= n[:, None], "any": torch.rand(B, L, generator=gen) < 0.4,
            "all": torch.ones(B, L, dtype=torch.bool)}[pad]
    if pad == "right" and B > 1:
        mask[-1] = True
    return x, dy, w, c, mask


def run_all(M, x, dy, w, c, mask, groups, activation, shape=lambda t: t):
    D = x.shape[-1]
    norm = M.GroupNorm(D, groups, activation=activation).cuda()
    with torch.no_grad():
        norm.weight.copy_(w)
        norm.bias.copy_(c)
        xs = shape(x.cuda())
        y0 = norm(xs, None if mask is None else mask.cuda())
    xs = xs.detach().requires_grad_()
    y = norm(xs, None if mask is None else mask.cuda())
    assert torch.equal(y.isnan(), y0.isnan()) and torch.equal(y.nan_to_num(), y0.nan_to_num())
    dx, dw, db = torch.autograd.grad(y, [xs, norm.weight, norm.bias], dy.cuda().reshape(y.shape))
    y1, count, mean, rstd = M.ops.group_norm_fwd(xs.detach(), w.cuda() + 1, c.cuda(), groups, None if mask is None else mask.cuda(), 1e-5,
                                                 activation)
    return {"y": y, "dx": dx, "dw": dw, "db": db, "count": count, "mean": mean, "rstd": rstd, "y1": y1}


def check_all(got, x, dy, w, c, mask, groups, activation):
    want = reference(x, w, c, groups, mask, silu=activation == "silu", dy=dy)
    assert torch.equal(got["count"].cpu(), want["count"])
    assert got["y"].dtype == x.dtype and got["dx"].dtype == x.dtype
    for k in ("mean", "rstd", "y", "dx", "dw", "db"):
        close(got[k], want[k], k)
    close(got["y1"], want["y"], "y1")


# --------------------------------------------------------------------------------------- without a GPU
def test_host_refusals():
    import fairseq_apollo_b200 as M
    x = torch.randn(2, 5, 8)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="CUDA"):
            M.GroupNorm(8, 2)(x)
    with pytest.raises(AssertionError):
        M.GroupNorm(8, 3)
    with pytest.raises(ValueError):
        M.GroupNorm(8, 2, activation="tanh")
    with pytest.raises(ValueError):
        M.GroupNorm(10, 2)(x)


def test_abi_refusals():
    import fairseq_apollo_b200 as M
    from fairseq_apollo_b200 import _lib
    lib = _lib.lib()
    one, odd = ctypes.c_void_p(16), ctypes.c_void_p(17)

    def fwd(x=one, dtype=1, B=1, L=2, D=8, G=2, work=one):
        return lib.mega_group_norm_fwd(x, one, dtype, B, L, D, 8, 8, 8, 8, one, one, None, G, 1e-5, 0, one, one, one, work, None)

    def bwd(dy=one, dtype=1, G=2, work=one, dgamma=one):
        return lib.mega_group_norm_bwd(dy, one, one, dtype, 1, 2, 8, 8, 8, 8, 8, 8, 8, one, one, None, G, 0, one, one, one, dgamma, one, work,
                                       None)

    assert fwd(x=None) == 1 and fwd(work=None) == 1 and bwd(dy=None) == 1 and bwd(work=None) == 1 and bwd(dgamma=None) == 1
    assert fwd(dtype=3) == 2 and bwd(dtype=3) == 2
    assert fwd(G=3) == 3 and fwd(G=0) == 3 and fwd(L=0) == 3 and bwd(G=5) == 3
    assert fwd(B=65536) == 7 and fwd(G=70000, D=70000) == 7
    assert fwd(x=odd) == 5 and bwd(dy=odd) == 5
    for backward in (0, 1):
        assert lib.mega_group_norm_work(1, 4, 100, 64, 8, backward) > 0 and lib.mega_group_norm_work(1, 4, 100, 64, 7, backward) == 0


def test_reference_gradients_against_differences():
    x, dy, w, c, mask = inputs(2, 7, 6, torch.float32, 1, "any")
    for silu in (True, False):
        want = reference(x, w, c, 2, mask, silu=silu, dy=dy)

        def value(x, w, c):
            x = x.view(2, 7, 2, 3)
            live = (~mask)[..., None, None]
            n = live.sum(1, keepdim=True) * 3
            m = torch.where(live, x, 0.0).sum((1, 3), keepdim=True) / n
            v = torch.where(live, (x - m) ** 2, 0.0).sum((1, 3), keepdim=True) / n
            z = ((x - m) / (v + 1e-5).sqrt()).view(2, 7, 6) * (1 + w) + c
            y = z * torch.sigmoid(z) if silu else z
            return (torch.where(mask[..., None], 0.0, y) * dy.to(F64)).sum()

        base = [t.to(F64) for t in (x, w, c)]
        for k, name in enumerate(("dx", "dw", "db")):
            v = torch.randn(base[k].shape, generator=torch.Generator().manual_seed(3), dtype=F64)
            up, down = list(base), list(base)
            up[k], down[k] = base[k] + 1e-5 * v, base[k] - 1e-5 * v
            diff = (value(*up) - value(*down)) / 2e-5
            assert abs(float(diff - (want[name][0].reshape(v.shape) * v).sum())) < 1e-6 * (1 + abs(float(diff)))


# ------------------------------------------------------------------------------------------- on the GPU
SHAPES = [(1, 1, 8, 1), (2, 3, 8, 8), (3, 5, 6, 2), (2, 33, 64, 4), (1, 64, 40, 5), (4, 100, 96, 32), (2, 257, 70, 7), (3, 17, 130, 1),
          (2, 65, 512, 2), (1, 300, 256, 1), (2, 1000, 64, 8), (1, 31, 1032, 3), (2, 9, 4100, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_64_bits(shape, dtype, activation):
    import fairseq_apollo_b200 as M
    B, L, D, G = shape
    for pad in (None, "any") if L > 1 else (None,):
        args = inputs(B, L, D, dtype, L + D, pad)
        check_all(run_all(M, *args, G, activation), *args, G, activation)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 40000, 16, 2), (2, 5000, 520, 8), (150, 64, 64, 1), (40, 600, 128, 64), (1, 20000, 130, 1), (3, 4096, 256, 8),
                                   (1, 9000, 64, 2), (1, 30000, 96, 32), (6, 6000, 264, 11)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_and_wide(shape, dtype):
    import fairseq_apollo_b200 as M
    args = inputs(*shape[:3], dtype, 5, "right" if shape[0] == 3 else None)
    check_all(run_all(M, *args, shape[3], "silu"), *args, shape[3], "silu")


@pytest.mark.gpu
def test_forms():
    """small calls in one pass over clusters, larger ones in two: the shapes above reach both"""
    import fairseq_apollo_b200 as M
    from fairseq_apollo_b200 import _lib
    for shape, groups, held in (((3, 4096, 256), 8, True), ((2, 1000, 64), 8, True), ((1, 40000, 16), 2, False), ((6, 6000, 264), 11, False)):
        norm = M.GroupNorm(shape[2], groups, activation="silu").cuda()
        with torch.no_grad():
            norm(torch.randn(shape, device="cuda").bfloat16())
        assert (_lib.last_kernel() == "group_norm_held") == held, shape


@pytest.mark.gpu
@pytest.mark.parametrize("pad", ["right", "any", "all"])
def test_masks(pad):
    import fairseq_apollo_b200 as M
    for dtype in DTYPES:
        for D, G in ((64, 4), (70, 7)):
            x, dy, w, c, mask = inputs(4, 83, D, dtype, 3, pad)
            got = run_all(M, x, dy, w, c, mask, G, "silu")
            check_all(got, x, dy, w, c, mask, G, "silu")
            assert (got["y"].cpu()[mask] == 0).all() and (got["dx"].cpu()[mask] == 0).all()
            xb, db = x.clone(), dy.clone()
            xb[mask], db[mask] = float("nan"), float("inf")
            dirty = run_all(M, xb, db, w, c, mask, G, "silu")
            assert all(torch.equal(got[k], dirty[k]) for k in got)


@pytest.mark.gpu
def test_far_from_zero_and_constant():
    """a mean that is 1000 times the deviation; values that do not deviate at all; large activations"""
    import fairseq_apollo_b200 as M
    args = inputs(2, 500, 64, torch.float32, 2, None, shift=3000.0)
    check_all(run_all(M, *args, 4, "silu"), *args, 4, "silu")
    x, dy, w, c, mask = inputs(2, 100, 64, torch.bfloat16, 2)
    x = torch.full_like(x, 7.0)
    check_all(run_all(M, x, dy, w, c, mask, 4, "silu"), x, dy, w, c, mask, 4, "silu")
    x, dy, w, c, mask = inputs(2, 100, 64, torch.float32, 2)
    for dt in DTYPES:
        a = (x.to(dt), dy.to(dt), w * 300, c * 300, mask)
        check_all(run_all(M, *a, 4, "silu"), *a, 4, "silu")


@pytest.mark.gpu
def test_a_group_that_is_not_finite_stays_by_itself():
    import fairseq_apollo_b200 as M
    x, dy, w, c, mask = inputs(3, 200, 96, torch.bfloat16, 4)
    clean = run_all(M, x, dy, w, c, mask, 3, "silu")
    xb = x.clone()
    xb[1, 100, 40] = float("inf")   # sequence 1, group 1
    bad = run_all(M, xb, dy, w, c, mask, 3, "silu")
    keep = torch.ones(3, 96, dtype=torch.bool)
    keep[1, 32:64] = False
    keep = keep[:, None, :].expand(3, 200, 96)
    for k in ("y", "dx"):
        assert torch.equal(clean[k].cpu()[keep], bad[k].cpu()[keep])
        assert not torch.isfinite(bad[k].cpu()[1, :, 32:64]).any()


@pytest.mark.gpu
def test_axes_memory_orders_and_alignment():
    import fairseq_apollo_b200 as M
    for dtype in DTYPES:
        for D, G in ((64, 4), (36, 6)):
            x, dy, w, c, mask = inputs(2, 60, D, dtype, 8, "any")
            plain = run_all(M, x, dy, w, c, mask, G, "silu")

            def sliced(t):
                wide = torch.full(t.shape[:-1] + (D + 9,), 7.0, dtype=t.dtype, device=t.device)
                wide[..., 5:5 + D] = t
                return wide[..., 5:5 + D]

            for shape in (sliced, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                          lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
                # (not bit for bit: rows that start elsewhere take other vectors, and so another order of the sums)
                got = run_all(M, x, dy, w, c, mask, G, "silu", shape)
                check_all(got, x, dy, w, c, mask, G, "silu")
            norm = M.GroupNorm(D, G, activation="silu").cuda()   # maps of 5 x 12 positions
            with torch.no_grad():
                norm.weight.copy_(w)
                norm.bias.copy_(c)
            x4, m4 = x.cuda().view(2, 5, 12, D), mask.cuda().view(2, 5, 12)
            leaf = x4.clone().requires_grad_()
            y = norm(leaf, m4)
            assert torch.equal(y.view(2, 60, D), plain["y"])
            dx, dw, db = torch.autograd.grad(y, [leaf, norm.weight, norm.bias], dy.cuda().view(2, 5, 12, D))
            assert torch.equal(dx.view(2, 60, D), plain["dx"]) and torch.equal(dw, plain["dw"]) and torch.equal(db, plain["db"])
            nchw = x4.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
            with torch.no_grad():
                assert torch.equal(norm(nchw, m4), y) and torch.equal(norm(x4[:, 0, 0]), norm(x4[:, :1, :1].reshape(2, 1, D))[:, 0])
                out = norm(x4, m4)
                out.mul_(2)
            z = norm(leaf, m4)
            z.mul_(2).sum().backward()   # the result may be changed in place
            wide = x.cuda()[:, :1].expand(2, 60, D).detach().requires_grad_()   # one position for all of them
            assert torch.isfinite(torch.autograd.grad(norm(wide).sum(), wide)[0]).all()


@pytest.mark.gpu
def test_parameter_types():
    import fairseq_apollo_b200 as M
    x, dy, w, c, mask = inputs(2, 50, 64, torch.bfloat16, 6)
    norm = M.GroupNorm(64, 4, activation="silu").cuda()
    with torch.no_grad():
        norm.weight.copy_(w.bfloat16())
        norm.bias.copy_(c.bfloat16())
    xs = x.cuda().requires_grad_()
    want = torch.autograd.grad(norm(xs), [xs, norm.weight, norm.bias], dy.cuda())
    norm = norm.bfloat16()
    got = torch.autograd.grad(norm(xs), [xs, norm.weight, norm.bias], dy.cuda())
    assert torch.equal(got[0], want[0])
    for g, v in zip(got[1:], want[1:]):
        assert g.dtype == torch.bfloat16 and torch.equal(g, v.bfloat16())


@pytest.mark.gpu
def test_empty_and_refused():
    import fairseq_apollo_b200 as M
    norm = M.GroupNorm(8, 2, activation="silu").cuda()
    for shape in ((2, 0, 8), (0, 3, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = norm(x)
        assert y.shape == shape
        assert [tuple(g.shape) for g in torch.autograd.grad(y.sum(), [x, norm.weight, norm.bias])] == [shape, (8,), (8,)]
        with torch.no_grad():
            assert norm(x).shape == shape
    x = torch.randn(2, 5, 8, device="cuda")
    for grad in (True, False):
        with torch.set_grad_enabled(grad):
            with pytest.raises(ValueError):
                norm(x, torch.zeros(2, 4, device="cuda"))
            with pytest.raises(RuntimeError):
                norm(x, torch.zeros(2, 5))
            with pytest.raises(TypeError):
                norm(x.double())
    with pytest.raises(ValueError):
        M.ops.group_norm_fwd(x, torch.ones(8, device="cuda"), torch.ones(8, device="cuda"), 3)
    with pytest.raises(ValueError):
        M.ops.group_norm_fwd(x, torch.ones(7, device="cuda"), torch.ones(8, device="cuda"), 2)
    xg = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(norm(xg).sum(), xg, create_graph=True)


@pytest.mark.gpu
def test_repeats_bit_for_bit_on_streams_and_in_graphs():
    import fairseq_apollo_b200 as M
    for shape, G in (((2, 700, 96), 3), ((1, 30000, 64), 2)):
        x, dy, w, c, mask = inputs(*shape, torch.bfloat16, 6, "any")
        norm = M.GroupNorm(shape[2], G, activation="silu").cuda()
        xs, dy, mask = x.cuda().requires_grad_(), dy.cuda(), mask.cuda()
        leaves = [xs, norm.weight, norm.bias]

        def train():
            y = norm(xs, mask)
            return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))

        base = train()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        outs = []
        for s in streams * 2:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(train())
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                got = train()
            graphs.append(g)
            outs.append(got)
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(base, o))


@pytest.mark.gpu
def test_more_than_31_bits_of_values():
    """offsets past 2^31 values: the last group of a long call against that group by itself"""
    import fairseq_apollo_b200 as M
    L, D, size = 270000, 8192, 16
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    x = torch.randn(1, L, D, device="cuda", dtype=torch.bfloat16, generator=torch.Generator(device="cuda").manual_seed(0))
    x += 1
    norm = M.GroupNorm(D, D // size, activation="silu").cuda()
    x.requires_grad_()
    y = norm(x)
    dx, dw, db = torch.autograd.grad(y, [x, norm.weight, norm.bias], y.detach())
    xl = x.detach()[..., -size:].to(F64).requires_grad_()
    w, c = torch.zeros(size, device="cuda", dtype=F64, requires_grad=True), torch.zeros(size, device="cuda", dtype=F64, requires_grad=True)
    z = (xl - xl.mean()) / (xl.var(unbiased=False) + 1e-5).sqrt() * (1 + w) + c
    want = torch.nn.functional.silu(z)
    grads = torch.autograd.grad(want, [xl, w, c], y.detach()[..., -size:].to(F64))
    assert float((y.detach()[..., -size:].to(F64) - want).norm() / want.norm()) < 2.0 ** -8
    assert float((dx[..., -size:].to(F64) - grads[0]).norm() / grads[0].norm()) < 2.0 ** -8
    for a, b in ((dw, grads[1]), (db, grads[2])):
        assert float((a[-size:].to(F64) - b).norm() / b.norm()) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_then_recurrence(dtype):
    """the two together, as a layer of an encoder takes them: norm and activation, gates, walks in both directions"""
    import fairseq_apollo_b200 as M
    torch.manual_seed(1)
    norm, layer = M.GroupNorm(64, 4, activation="silu").cuda(), M.GatedRecurrence(64, input_gate=True, bidirectional=True).cuda()
    layer = layer.to(dtype)
    x = torch.randn(3, 90, 64, device="cuda").to(dtype)
    pad = torch.arange(90, device="cuda")[None] >= torch.tensor([[90], [31], [0]], device="cuda")
    leaf = x.clone().requires_grad_()
    y = layer(norm(leaf, pad), pad)
    dy = torch.randn(y.shape, device="cuda").to(dtype)
    grads = torch.autograd.grad(y, [leaf, norm.weight, layer.in_proj.weight, layer.back_proj.weight], dy)
    w = {k: v.detach().cpu().to(F64).requires_grad_() for k, v in list(layer.named_parameters()) + [("n." + k, v) for k, v in norm.named_parameters()]}
    u = x.cpu().to(F64).requires_grad_()
    live = ~pad.cpu()[..., None]
    xg = u.view(3, 90, 4, 16)
    n = (live.sum(1, keepdim=True) * 16).clamp(min=1)[..., None]
    mean = torch.where(live[..., None], xg, 0.0).sum((1, 3), keepdim=True) / n
    var = torch.where(live[..., None], (xg - mean) ** 2, 0.0).sum((1, 3), keepdim=True) / n
    z = ((xg - mean) / (var + 1e-5).sqrt()).view(3, 90, 64) * (1 + w["n.weight"]) + w["n.bias"]
    a = torch.where(live, z * torch.sigmoid(z), 0.0)

    def walk(name, reverse):
        v, f, i = (a @ w[name + ".weight"].t() + w[name + ".bias"]).split(64, -1)
        h, ys = torch.zeros(3, 64, dtype=F64), {}
        for t in (range(89, -1, -1) if reverse else range(90)):
            keep = torch.sigmoid(f[:, t])
            h = torch.where(live[:, t], keep * h + torch.sigmoid(i[:, t]) * v[:, t], h)
            ys[t] = torch.where(live[:, t], h, 0.0)
        return torch.stack([ys[t] for t in range(90)], 1)

    ref = walk("in_proj", False) + walk("back_proj", True)
    want = torch.autograd.grad(ref, [u, w["n.weight"], w["in_proj.weight"], w["back_proj.weight"]], dy.cpu().to(F64))
    # (relative L2 over five roundings in a row of intermediate results to the activations' type, each at most eps / 2)
    tol = 5 * torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 2e-5
    assert float((y.detach().cpu().to(F64) - ref).norm() / ref.norm()) < tol
    for g, v in zip(grads, want):
        assert float((g.cpu().to(F64) - v).norm() / v.norm()) < 2 * tol


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2, 700, 514, 2), (3, 1100, 771, 3), (1, 600, 4104, 1), (2, 530, 2600, 2)])
def test_groups_wider_than_a_block_over_long_sequences(shape, dtype):
    """groups of 257 channels and more, padded: runs of 64 values of a thread are joined many times over"""
    import fairseq_apollo_b200 as M
    for pad, activation in (("any", "silu"), ("right", "silu"), (None, None)):
        args = inputs(*shape[:3], dtype, shape[1], pad)
        check_all(run_all(M, *args, shape[3], activation), *args, shape[3], activation)


@pytest.mark.gpu
def test_wide_groups_off_the_boundaries():
    """300 channels to a group fit a tile on whole vectors, and take the wide form on odd 16-bit addresses"""
    import fairseq_apollo_b200 as M
    for dtype in DTYPES:
        x, dy, w, c, mask = inputs(2, 400, 600, dtype, 3, "any")

        def odd(t):
            wide = torch.full(t.shape[:-1] + (t.shape[-1] + 3,), 7.0, dtype=t.dtype, device=t.device)
            wide[..., 1:601] = t
            return wide[..., 1:601]

        for shape in (lambda t: t, odd):
            check_all(run_all(M, x, dy, w, c, mask, 2, "silu", shape), x, dy, w, c, mask, 2, "silu")
