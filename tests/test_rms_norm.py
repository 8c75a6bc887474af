"""Root-mean-square norm with a residual against its formula in 64 bits.

Tolerances: one rounding to the activations' type on each output (half a step, u), sums of n terms in fp32.
"""
import pytest
import torch

import fairseq_apollo_b200 as M
from fairseq_apollo_b200 import _lib

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


def reference(x, weight, res, groups, dy=None, dr=None):
    """r, y[, dx, dweight] and what the terms of dx and dweight add up to by their absolute values"""
    r = (x.float() + res.float()).to(x.dtype) if res is not None else x
    p = r.detach().double().requires_grad_()
    w = weight.detach().double().requires_grad_()
    g = p.unflatten(-1, (groups, -1))
    rstd = 1 / torch.sqrt((g * g).mean(-1, keepdim=True) + EPS)
    y = (g * rstd).flatten(-2) * (1 + w)
    if dy is None:
        return r, y.detach()
    dx, dw = torch.autograd.grad(y, [p, w], dy.double())
    a = (dy.double() * (1 + w)).abs().unflatten(-1, (groups, -1)).detach()
    n = (g * rstd).abs().detach()
    size = (rstd * (a + n * (a * n).mean(-1, keepdim=True))).flatten(-2).detach()
    if dr is not None:
        dx = dx + dr.double()
        size = size + dr.double().abs()
    dims = tuple(range(x.dim() - 1))
    return r, y.detach(), dx, dw, size, (dy.double() * n.flatten(-2)).abs().sum(dims)


def check(dtype, shape, groups, residual=True, dr=True, arrange=lambda t: t):
    dt = DT[dtype]
    gen = torch.Generator().manual_seed(sum(shape) + groups)
    x, res, dy, dsum = (arrange(torch.randn(*shape, generator=gen).to(dt).cuda()) for _ in range(4))
    weight = (torch.randn(shape[-1], generator=gen) * 0.2).cuda()
    leaves = [x.detach().requires_grad_(), weight.clone().requires_grad_()] + ([res.detach().requires_grad_()] if residual else [])
    out = M.rms_norm(leaves[0], leaves[1], leaves[2] if residual else None, groups, EPS)
    with torch.no_grad():
        plain = M.rms_norm(x, weight, res if residual else None, groups, EPS)
    if residual:
        assert torch.equal(plain[0], out[0]) and torch.equal(plain[1], out[1])
        with_dr = dr
        grads = torch.autograd.grad(list(out) if with_dr else out[0], leaves, [dy, dsum] if with_dr else dy)
        assert torch.equal(grads[0], grads[2])
        y = out[0]
    else:
        assert torch.equal(plain, out)
        with_dr = False
        grads = torch.autograd.grad(out, leaves, dy)
        y = out
    r, ry, rdx, rdw, size, wsize = reference(x, weight, res if residual else None, groups, dy, dsum if with_dr else None)
    if residual:
        assert torch.equal(out[1], r)
    n = shape[-1] // groups
    rows = x.numel() // shape[-1]
    # (a warp's sum of n squares: at most n / 32 + 5 additions in a row, then half of it counts under the root)
    u, f = torch.finfo(dt).eps / 2, (n / 32 + 16) * 2.0 ** -24
    tiny = torch.finfo(dt).tiny if dt == torch.float16 else 1e-30
    assert y.shape == x.shape and y.dtype == dt
    assert float(((y.double() - ry).abs() - (u + f) * ry.abs()).max()) <= tiny
    assert float(((grads[0].double() - rdx).abs() - u * rdx.abs() - 4 * f * size).max()) <= tiny
    assert float(((grads[1].double() - rdw).abs() - (f + (rows / 8 + 64) * 2.0 ** -24) * wsize).max()) <= 1e-30


SHAPES = [((1, 1, 1), 1), ((2, 3, 8), 1), ((1, 5, 7), 1), ((2, 33, 64), 8), ((2, 300, 512), 8), ((3, 17, 96), 32), ((2, 40, 2048), 1), ((1, 9, 2048), 2),
          ((1, 7, 4096), 1), ((2, 5, 8192), 1), ((1, 3, 8192), 4), ((1, 2, 20000), 1), ((2, 31, 1000), 1), ((2, 31, 1001), 7), ((1, 64, 1024), 16), ((5, 12), 3),
          ((2, 3, 4, 5, 48), 2), ((1, 1500, 256), 1), ((700, 3, 40), 1), ((1, 4, 4608), 1), ((2, 9, 768), 3), ((1, 6, 384), 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_outputs_and_gradients(dtype, shape, groups):
    check(dtype, shape, groups, residual=True)
    check(dtype, shape, groups, residual=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("width", [256, 250])
def test_strides_and_missing_gradients(dtype, width):
    check(dtype, (3, 20, width), 2, dr=False)
    check(dtype, (3, 20, width), 2, arrange=lambda t: t.transpose(0, 1).contiguous().transpose(0, 1))
    check(dtype, (3, 20, width), 2, arrange=lambda t: torch.cat([t, t], -1)[..., :width])
    check(dtype, (3, 20, width), 2, arrange=lambda t: torch.cat([t[..., :1], t], -1)[..., 1:])     # (rows that start off 16 bytes)
    check(dtype, (3, 20, width), 2, arrange=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2))
    check(dtype, (3, 20, width), 2, arrange=lambda t: t[:, :1].expand_as(t))


@pytest.mark.gpu
def test_gradient_of_the_sum_alone_and_parameter_types():
    x, res = (torch.randn(2, 5, 64, device="cuda", requires_grad=True) for _ in range(2))
    w = torch.zeros(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y, r = M.rms_norm(x, w, res)
    g = torch.autograd.grad(r.sum(), [x, res, w])
    assert torch.equal(g[0], torch.ones_like(x)) and torch.equal(g[1], g[0]) and float(g[2].float().abs().max()) == 0 and g[2].dtype == torch.bfloat16


@pytest.mark.gpu
def test_rows_of_zeros_and_values_that_are_not_finite():
    x = torch.randn(1, 6, 128, device="cuda")
    x[0, 1] = 0
    x[0, 2, 5] = float("inf")
    x[0, 3, 5] = float("nan")
    x[0, 4] *= 1e-20
    w = torch.zeros(128, device="cuda")
    y = M.rms_norm(x, w)
    assert float(y[0, 1].abs().max()) == 0 and torch.isnan(y[0, 2, 5]) and float(y[0, 2, :5].abs().max()) == 0 and torch.isnan(y[0, 3]).all()
    assert torch.isfinite(y[0, [0, 1, 4, 5]]).all()     # (rows know nothing of one another)
    assert torch.allclose(y[0, 4], x[0, 4] / EPS ** 0.5, rtol=1e-5, atol=0)


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    x, res, dy, dr = (torch.randn(4, 50, 512, device="cuda").to(torch.bfloat16) for _ in range(4))
    w = (torch.randn(512, device="cuda") * 0.1).requires_grad_()
    a, b = x.clone().requires_grad_(), res.clone().requires_grad_()

    def go():
        out = M.rms_norm(a, w, b)
        return list(out) + list(torch.autograd.grad(list(out), [a, b, w], [dy, dr]))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = go()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = go()
    g.replay()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    with torch.no_grad():
        a.copy_(res)
    g.replay()
    assert all(torch.equal(p, q) for p, q in zip(got, go()))


@pytest.mark.gpu
def test_module_and_empty_calls():
    m = M.RMSNorm(96, num_groups=4, eps=1e-3).cuda()
    x, res = (torch.randn(2, 5, 96, device="cuda") for _ in range(2))
    y, r = m(x, res)
    assert torch.equal(y.detach(), M.ops.rms_norm_fwd(x, m.weight, res, 4, 1e-3)[0]) and torch.equal(r.detach(), x + res)
    for shape in ((0, 5, 96), (2, 0, 96)):
        x = torch.randn(*shape, device="cuda", requires_grad=True)
        y, r = m(x, x)
        assert y.shape == shape and r.shape == shape
        assert torch.autograd.grad(y.sum() + r.sum(), [x])[0].shape == shape
        with torch.no_grad():
            assert m(x).shape == shape
    with pytest.raises(ValueError):
        m(torch.zeros(2, 5, 95, device="cuda"))


@pytest.mark.gpu
def test_refusals():
    x, w = torch.zeros(2, 3, 12, device="cuda"), torch.zeros(12, device="cuda")
    for bad in (lambda: M.rms_norm(x, w[:11]), lambda: M.rms_norm(x, w, num_groups=5), lambda: M.rms_norm(x, w, num_groups=0), lambda: M.rms_norm(x, w, x[:1]),
                lambda: M.rms_norm(x, w.cpu()), lambda: M.rms_norm(x[0, 0], w), lambda: M.rms_norm(x, w, x.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    for bad in (lambda: M.rms_norm(x.double(), w), lambda: M.rms_norm(x, w, x.half()), lambda: M.rms_norm(x, w.long())):
        with pytest.raises(TypeError):
            bad()


def test_refusals_on_the_host():
    with pytest.raises(RuntimeError):
        M.rms_norm(torch.zeros(2, 3, 4), torch.zeros(4))
    with pytest.raises(AssertionError):
        M.RMSNorm(10, num_groups=3)
    lib = _lib.lib()
    s = [12, 12] * 4
    assert lib.mega_rms_norm_fwd(None, None, 16, None, 0, 1, 1, 12, *s, 16, 1, 1e-5, None) == 1
    assert lib.mega_rms_norm_fwd(16, 16, 16, None, 0, 1, 1, 12, *s, 16, 1, 1e-5, None) == 1     # a residual without a place for the sum
    assert lib.mega_rms_norm_fwd(16, None, 16, None, 9, 1, 1, 12, *s, 16, 1, 1e-5, None) == 2
    assert lib.mega_rms_norm_fwd(16, None, 16, None, 0, 1, 1, 12, *s, 16, 5, 1e-5, None) == 3
    assert lib.mega_rms_norm_fwd(16, None, 16, None, 0, 1, 1, (1 << 20) + 4, *s, 16, 1, 1e-5, None) == 7
    assert lib.mega_rms_norm_bwd(16, None, 16, 16, 0, 1, 1, 12, *s, 16, 1, 1e-5, 16, None, None) == 1
    assert lib.mega_rms_norm_work(0, 1, 1, 12, 1) > 0 and lib.mega_rms_norm_work(0, 1, 1, 12, 5) == 0
