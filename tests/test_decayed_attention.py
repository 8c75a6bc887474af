"""Linear attention with a decay for each head against its recurrence in 64 bits.

Tolerances.  With u half a step of the activations' type, every share of an output is rounded once on its way (a pair's weight, or
the state that is read) and the output once more, so |error| <= u (sum of the shares' absolute values) + u |output|: 2 u times the
same walk over absolute values, which the reference computes along with each output.  fp32 operands are two 11-bit pieces in
products (2^-21 of a product left out or cut off, two products in a row), sums of n terms are cut off n times at 2^-23.
fp16's pieces of weighted keys are multiples of 2^-24 below its normal range: a term of a state is off by up to 2^-25 of its other
factor's value, however small the keys' (or dy's) is, and a segment, or a sequence, has as many terms as steps.
"""
import ctypes

import pytest
import torch

import fairseq_apollo_b200 as M
from fairseq_apollo_b200 import _lib

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _unit(dtype, keys, values):
    """relative error of one rounding on the way (16-bit), or of the products and sums (fp32)"""
    if dtype == torch.float32:
        return 2 * 2.0 ** -21 + (keys + values + 128) * 2.0 ** -23
    return torch.finfo(dtype).eps / 2 + (keys + values + 128) * 2.0 ** -23


def _inputs(dtype, b, n, h, kd, vd, seed=0, gate_dtype=None, spread=2.0, shift=2.0):
    g = torch.Generator().manual_seed(seed)
    dt = DT[dtype]

    def rnd(*s):
        return torch.randn(*s, generator=g)
    q, k, v = rnd(b, n, h, kd).to(dt), rnd(b, n, h, kd).to(dt), rnd(b, n, h, vd).to(dt)
    f = (rnd(b, n, h) * spread + shift).to(gate_dtype or dt)
    hin, dy, dh = rnd(b, h, kd, vd), rnd(b, n, h, vd).to(dt), rnd(b, h, kd, vd)
    return [t.cuda() for t in (q, k, v, f, hin, dy, dh)]


def _walk(q, k, v, a, s, order):
    y = [None] * q.shape[1]
    for t in order:
        s = a[:, t, :, None, None] * s + k[:, t, :, :, None] * v[:, t, :, None, :]
        y[t] = torch.einsum("bhk,bhkv->bhv", q[:, t], s)
    return torch.stack(y, 1), s


def reference(q, k, v, f, hin=None, pad=None, reset=None, scale=1.0, reverse=False, dy=None, dh=None):
    """(outputs, the same over absolute values): y, h[, dq, dk, dv, df, dh_in] in 64 bits by autograd of the recurrence"""
    b, n, h, kd = q.shape
    vd = v.shape[-1]
    found = []
    for absolute in (False, True):
        x = [t.detach().double() for t in (q, k, v, f)]
        x = [torch.where(pad[(...,) + (None,) * (t.dim() - 2)], torch.zeros_like(t), t) if pad is not None else t for t in x]
        if absolute:
            x[:3] = [t.abs() for t in x[:3]]
        s0 = torch.zeros(b, h, kd, vd, dtype=torch.float64, device=q.device) if hin is None else hin.detach().double()
        s0 = s0.abs() if absolute else s0.clone()
        x = [t.clone().requires_grad_() for t in x]
        s0.requires_grad_()
        a = torch.sigmoid(x[3])
        if pad is not None:
            a = torch.where(pad[..., None], torch.ones_like(a), a)
        if reset is not None:
            a = torch.where(reset[..., None], torch.zeros_like(a), a)
        order = list(range(n))
        if reverse:
            order.reverse()
        with torch.enable_grad():
            y, s = _walk(x[0] * scale, x[1], x[2], a, s0, order)
            if pad is not None:
                y = torch.where(pad[..., None, None], torch.zeros_like(y), y)
        out = [y.detach(), s.detach()]
        if dy is not None:
            gy, gh = dy.double(), dh.double()
            if pad is not None:
                gy = torch.where(pad[..., None, None], torch.zeros_like(gy), gy)
            if absolute:
                gy, gh = gy.abs(), gh.abs()
            out += list(torch.autograd.grad([y, s], x + [s0], [gy, gh]))
        found.append(out)
    return found


def check(got, ref, bound, dtype, kd, vd, values=None):
    """every value of y, h and the gradients within the derived bound; df (index 5) by its norm"""
    u = _unit(dtype, kd, vd)
    state = (kd + vd + 128) * 2.0 ** -23 + (2.0 ** -16 if dtype != torch.float32 else 2.0 ** -21)   # (weighted keys are two pieces)
    for i, (x, y, m) in enumerate(zip(got, ref, bound)):
        assert x.shape == y.shape, i
        err = (x.detach().double() - y).abs()
        if i == 5:
            # shares of d log a are rounded once each, the sum once more, independently of one another: rms u / sqrt(3) each
            assert float(err.norm()) <= 1.5 * u * float(y.norm()) + 1e-30, (i, float(err.norm() / y.norm()))
        else:
            tol = (state if i in (1, 6) else 2 * u) * m + 1e-30
            tiny = torch.finfo(torch.float16).tiny if x.dtype == torch.float16 else 0.0   # (fp16: steps below the normal range)
            if dtype == torch.float16 and i in (1, 6):
                tiny = 2.0 ** -25 * values[i]
            worst = float((err - tol - tiny).max()) if err.numel() else 0.0
            assert worst <= 0, (i, float((err / tol).max()))


def run(q, k, v, f, hin=None, pad=None, reset=None, scale=1.0, reverse=False, dy=None, dh=None):
    if dy is None:
        with torch.no_grad():
            return list(M.decayed_attention(q, k, v, f, pad, reset, hin, scale, True, reverse))
    leaves = [t.detach().requires_grad_() for t in (q, k, v, f)] + ([] if hin is None else [hin.detach().requires_grad_()])
    y, h = M.decayed_attention(*leaves[:4], pad, reset, leaves[4] if hin is not None else None, scale, True, reverse)
    return [y, h] + list(torch.autograd.grad([y, h], leaves, [dy, dh]))


def both(dtype, b, n, h, kd, vd, pad=None, reset=None, state=True, reverse=False, seed=0, gate_dtype=None, change=None, shift=2.0, spread=2.0):
    q, k, v, f, hin, dy, dh = _inputs(dtype, b, n, h, kd, vd, seed, gate_dtype, spread, shift)
    if change is not None:
        q, k, v, f, hin, dy, dh = change(q, k, v, f, hin, dy, dh)
    hin = hin if state else None
    kw = dict(hin=hin, pad=pad, reset=reset, scale=kd ** -0.5, reverse=reverse, dy=dy, dh=dh)
    ref, bound = reference(q, k, v, f, **kw)
    got = run(q, k, v, f, **kw)
    # sums over the steps of the factor beside the weighted one: v of the state, q of its gradient
    values = {1: float(v.detach().double().abs().sum(1).max()), 6: float(q.detach().double().abs().sum(1).max())} if dtype == "fp16" else None
    check(got, ref, bound, DT[dtype], kd, vd, values)
    return got, ref


SIZES = [(1, 1, 1, 1, 1), (2, 3, 2, 5, 7), (1, 63, 3, 16, 24), (2, 64, 1, 64, 64), (1, 65, 2, 32, 40), (2, 130, 3, 64, 128), (1, 127, 2, 128, 64),
         (1, 129, 1, 128, 128), (1, 100, 1, 200, 130), (1, 70, 2, 256, 256), (1, 81, 2, 33, 65), (3, 257, 2, 48, 96), (1, 300, 2, 100, 20)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("size", SIZES)
def test_outputs_and_gradients(dtype, size):
    both(dtype, *size, reverse=size[1] % 2 == 0, state=size[1] != 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kd,vd", [("bf16", 64, 64), ("bf16", 128, 128), ("fp16", 64, 128), ("bf16", 40, 24), ("fp32", 64, 32)])
@pytest.mark.parametrize("reverse", [False, True])
def test_padding_and_resets(dtype, kd, vd, reverse):
    b, n, h = 4, 330, 2
    g = torch.Generator().manual_seed(5)
    pad = torch.rand(b, n, generator=g) < 0.3
    pad[1] = True                       # a sequence of padding alone
    pad[2, 100:] = True                 # right padding
    pad[3, :90] = True                  # left padding
    reset = torch.rand(b, n, generator=g) < 0.05
    reset[2, 40:45] = True              # documents of one step
    reset[0, 0] = reset[3, 89] = reset[3, n - 1] = True
    both(dtype, b, n, h, kd, vd, pad.cuda(), reset.cuda(), reverse=reverse)
    both(dtype, b, n, h, kd, vd, None, torch.ones(b, n, dtype=torch.bool).cuda(), reverse=reverse)
    both(dtype, b, n, h, kd, vd, pad.cuda(), None, state=False, reverse=reverse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("reverse", [False, True])
def test_what_lies_at_padded_steps_is_not_used(dtype, reverse):
    b, n, h, kd, vd = 3, 200, 2, 64, 64
    pad = torch.zeros(b, n, dtype=torch.bool)
    pad[0, 150:] = True
    pad[1, 10:90] = True
    pad[2] = True
    pad = pad.cuda()
    q, k, v, f, hin, dy, dh = _inputs(dtype, b, n, h, kd, vd)
    clean = run(q, k, v, f, hin, pad, None, 0.1, reverse, dy, dh)
    for junk in (float("nan"), float("inf"), -float("inf"), torch.finfo(DT[dtype]).min):
        q2, k2, v2, f2, dy2 = (t.masked_fill(pad[(...,) + (None,) * (t.dim() - 2)], junk) for t in (q, k, v, f, dy))
        got = run(q2, k2, v2, f2, hin, pad, None, 0.1, reverse, dy2, dh)
        for x, y in zip(got, clean):
            assert torch.equal(x, y)
    for i in (0, 2, 3, 4):
        assert float(clean[i][pad].abs().max()) == 0
    assert torch.equal(clean[1][2], hin[2]) and torch.equal(clean[6][2], dh[2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_gates_from_closed_to_open(dtype):
    """-inf and far negative gates forget all, +inf ones nothing; the decay keeps its last places next to both ends"""
    def change(q, k, v, f, hin, dy, dh):
        f = f.clone()
        f[:, 20:24] = -float("inf")
        f[:, 70] = -200.0
        f[:, 90:130] = 30.0
        f[:, 131:140] = -40.0
        f[:, 150:] = float("inf")
        return q, k, v, f, hin, dy, dh
    got, ref = both(dtype, 2, 200, 2, 64, 64, change=change)
    assert torch.isfinite(got[5]).all() and float(got[5][:, 20:24].abs().max()) == 0 and float(got[5][:, 150:].abs().max()) == 0
    for shift, spread in ((-6.0, 0.5), (9.0, 1.0), (0.0, 8.0)):
        both(dtype, 2, 150, 2, 64, 64, shift=shift, spread=spread)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("layout", ["sliced", "odd_slices", "time", "shared", "columns", "broadcast"])
def test_strides(dtype, layout):
    b, n, h, kd, vd = 2, 150, 2, 64, 32

    def change(q, k, v, f, hin, dy, dh):
        if layout in ("sliced", "odd_slices"):
            extra = 8 if layout == "sliced" else 3
            z = torch.zeros(b, n, h * (2 * kd + vd + 1) + extra, dtype=q.dtype, device="cuda")
            at, out = (0 if layout == "sliced" else 1), []
            for t in (q, k, v, f):
                w = t[0, 0].numel()
                z[..., at:at + w] = t.flatten(2)
                out.append(z[..., at:at + w].view(b, n, *t.shape[2:]))
                at += w
            return (*out, hin, dy, dh)
        if layout == "time":
            q, k, v, f, dy = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, f, dy))
        elif layout == "shared":      # heads that share keys and values, one decay for all of them
            k, v, f = k[:, :, :1].expand_as(k), v[:, :, :1].expand_as(v), f[:, :, :1].expand_as(f)
        elif layout == "columns":     # the last axis is not contiguous
            q, k, v, dy = (t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v, dy))
        else:                         # the same step over and over
            q, f = q[:, :1].expand_as(q), f[:, :1].expand_as(f)
        return q, k, v, f, hin, dy, dh
    both(dtype, b, n, h, kd, vd, change=change)


@pytest.mark.gpu
def test_shared_heads_and_broadcast_gates_gather_gradients():
    b, n, h, kd, vd = 2, 90, 4, 32, 32
    q, k, v, f, _, dy, dh = _inputs("fp32", b, n, h, kd, vd)
    k1, f1 = k[:, :, :1].clone().requires_grad_(), f[0, 0].clone().requires_grad_()
    y, s = M.decayed_attention(q, k1.expand_as(q), v, f1, scale=0.2, want_state=True)
    got = torch.autograd.grad([y, s], [k1, f1], [dy, dh])
    ref, _ = reference(q, k1.expand_as(q), v, f1.expand(b, n, h), scale=0.2, dy=dy, dh=dh)
    assert torch.allclose(got[0].double(), ref[3].sum(2, keepdim=True), rtol=0, atol=1e-5 * float(ref[3].abs().max()) * h)
    assert torch.allclose(got[1].double(), ref[5].sum((0, 1)), rtol=0, atol=1e-5 * float(ref[5].abs().sum((0, 1)).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,b,n,h,kd,vd", [("bf16", 1, 2500, 1, 64, 64), ("bf16", 2, 2111, 2, 128, 128), ("fp32", 1, 1800, 1, 40, 70),
                                              ("fp16", 1, 1500, 3, 64, 128), ("bf16", 1, 900, 1, 256, 100)])
@pytest.mark.parametrize("reverse", [False, True])
def test_long_sequences_in_segments(dtype, b, n, h, kd, vd, reverse):
    g = torch.Generator().manual_seed(2)
    pad = torch.zeros(b, n, dtype=torch.bool)
    pad[-1, n // 2:n // 2 + 400] = True
    reset = (torch.rand(b, n, generator=g) < 0.002).cuda()
    both(dtype, b, n, h, kd, vd, pad.cuda(), reset, reverse=reverse, shift=4.0)


@pytest.mark.gpu
@pytest.mark.parametrize("kd,vd", [(64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("b,n,h", [(1, 2100, 16), (8, 1200, 16), (3, 640, 60)])
def test_many_heads(kd, vd, b, n, h):
    """enough heads to fill the device, or segments of several chunks: calls one after another, each head as if by itself, no wait given up"""
    q, k, v, f, hin, dy, dh = _inputs("bf16", b, n, h, kd, vd, shift=4.0)
    pad = torch.arange(n, device="cuda")[None] >= torch.randint(n // 3, n + 1, (b, 1), device="cuda")
    outs = [run(q, k, v, f, hin, pad, None, 0.1, False, dy, dh) for _ in range(4)]
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    for other in outs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(outs[0], other))
    part = slice(h - 2, h)
    cut = [t[:1, :, part] for t in (q, k, v, f)]
    ref, bound = reference(*cut, hin[:1, part], pad[:1], None, 0.1, False, dy[:1, :, part], dh[:1, part])
    got = [outs[0][i][:1, part] if i in (1, 6) else outs[0][i][:1, :, part] for i in range(7)]
    check(got, ref, bound, torch.bfloat16, kd, vd)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_parts_of_a_sequence_and_single_steps(dtype):
    """a sequence in two calls and in steps is the sequence in one, and the running state may be written in place"""
    b, n, h, kd, vd = 2, 140, 3, 64, 48
    q, k, v, f, hin, _, _ = _inputs(dtype, b, n, h, kd, vd)
    ref, bound = reference(q, k, v, f, hin, scale=0.3)
    with torch.no_grad():
        y1, s = M.decayed_attention(q[:, :77], k[:, :77], v[:, :77], f[:, :77], h_in=hin, scale=0.3, want_state=True)
        ys = [y1]
        y2, s = M.decayed_attention(q[:, 77:100], k[:, 77:100], v[:, 77:100], f[:, 77:100], h_in=s, scale=0.3, want_state=True)
        ys.append(y2)
        for t in range(100, n):
            y, s2 = M.ops.decayed_attention_step(q[:, t], k[:, t], v[:, t], f[:, t], s, 0.3, h_out=s if t % 2 else None)
            assert (s2.data_ptr() == s.data_ptr()) == bool(t % 2)
            s = s2
            ys.append(y[:, None])
    check([torch.cat(ys, 1), s], ref, bound, DT[dtype], kd, vd)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("size", [(1, 1, 1, 1), (4, 8, 64, 64), (3, 5, 128, 128), (2, 3, 17, 30), (2, 1, 256, 256), (1, 2, 256, 100), (2, 2, 33, 31), (70, 3, 8, 8)])
def test_step(dtype, size):
    b, h, kd, vd = size
    q, k, v, f, hin, _, _ = _inputs(dtype, b, 1, h, kd, vd)
    u = torch.finfo(DT[dtype]).eps / 2
    for state in (hin, None, hin.to(torch.bfloat16), hin.transpose(2, 3).contiguous().transpose(2, 3)):
        ref, bound = reference(q, k, v, f, state, scale=0.5)
        y, s = M.ops.decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], f[:, 0], state, 0.5)
        # sums of kd terms in fp32 and the output's rounding
        assert float(((y.double() - ref[0][:, 0]).abs() - (u + (kd + 8) * 2.0 ** -24) * bound[0][:, 0]).max()) <= 1e-30
        assert float(((s.double() - ref[1]).abs() - 6 * 2.0 ** -24 * bound[1]).max()) <= 1e-30


@pytest.mark.gpu
def test_step_beside_sliced_operands_and_gates():
    b, h, kd, vd = 5, 4, 64, 32
    z = torch.randn(b, h * (2 * kd + vd + 1) + 1, device="cuda").to(torch.bfloat16)[:, 1:]
    q, k, v, f = z.split((h * kd, h * kd, h * vd, h), dim=-1)
    q, k, v = (t.unflatten(-1, (h, -1)) for t in (q, k, v))
    s = torch.randn(b, h, kd, vd, device="cuda")
    want = M.ops.decayed_attention_step(q.contiguous(), k.contiguous(), v.contiguous(), f.contiguous(), s, 0.1)
    got = M.ops.decayed_attention_step(q, k, v, f, s, 0.1)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    per_head = torch.randn(h, device="cuda")
    y1, s1 = M.ops.decayed_attention_step(q, k, v, per_head, s)
    y2, s2 = M.ops.decayed_attention_step(q, k, v, per_head.expand(b, h).contiguous(), s)
    assert torch.equal(y1, y2) and torch.equal(s1, s2)
    # a state that starts off a 16-byte boundary
    odd = torch.empty(s.numel() + 1, device="cuda")[1:].view_as(s).copy_(s)
    y3, s3 = M.ops.decayed_attention_step(q, k, v, f, odd, 0.1, h_out=odd)
    assert s3.data_ptr() == odd.data_ptr()
    # other instructions, the same sums: a state's two terms are below 32 (2^5 2^-23), an output 64 such terms times 0.1 |q|, then bf16
    assert torch.allclose(s3, want[1], rtol=0, atol=2.0 ** -18) and torch.allclose(y3.float(), want[0].float(), rtol=2.0 ** -7, atol=2.0 ** -13)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [torch.float32, None])
def test_gates_in_fp32_beside_16_bit_activations(gate):
    got, _ = both("bf16", 2, 100, 2, 64, 64, gate_dtype=gate)
    assert got[5].dtype == (gate or torch.bfloat16)


@pytest.mark.gpu
def test_state_types_and_states_left_alone():
    q, k, v, f, hin, dy, dh = _inputs("bf16", 2, 70, 2, 64, 64)
    half = hin.to(torch.bfloat16).requires_grad_()
    y, s = M.decayed_attention(q, k, v, f, h_in=half, want_state=True, scale=0.1)
    g, = torch.autograd.grad([y, s], [half], [dy, dh])
    assert g.dtype == torch.bfloat16
    y2, s2 = M.decayed_attention(q, k, v, f, h_in=half.detach().float(), want_state=True, scale=0.1)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    # without the state that leaves; without a gradient of it
    qr = q.clone().requires_grad_()
    a, = torch.autograd.grad(M.decayed_attention(qr, k, v, f, h_in=hin, scale=0.1), [qr], dy)
    y, s = M.decayed_attention(qr, k, v, f, h_in=hin, scale=0.1, want_state=True)
    b, = torch.autograd.grad(y, [qr], dy)
    assert torch.equal(a, b)
    c, = torch.autograd.grad(M.decayed_attention(qr, k, v, f, want_state=True)[1].sum(), [qr])
    assert float(c.abs().max()) == 0


@pytest.mark.gpu
def test_gradients_against_differences():
    """the outputs are linear in each of q, k, v and the state; gates by central differences"""
    b, n, h, kd, vd = 1, 100, 2, 24, 40
    q, k, v, f, hin, dy, dh = _inputs("fp32", b, n, h, kd, vd)
    got = run(q, k, v, f, hin, None, None, 0.2, False, dy, dh)
    g = torch.Generator().manual_seed(9)

    def loss(*x):
        y, s = run(*x, None, None, 0.2)
        return float((y.double() * dy.double()).sum() + (s.double() * dh.double()).sum())
    x = [q, k, v, f, hin]
    for i, grad in enumerate(got[2:]):
        way = torch.randn(x[i].shape, generator=g).cuda()
        step = 1e-2 if i == 3 else 0.5
        up, down = [t.clone() for t in x], [t.clone() for t in x]
        up[i], down[i] = x[i] + step * way, x[i] - step * way
        slope = (loss(*up) - loss(*down)) / (2 * step)
        want = float((grad.double() * way.double()).sum())
        # differences of sums of ~10^4 terms in fp32, and step^2 of the third derivative for the gates
        size = float((grad.double() * way.double()).norm())
        assert abs(slope - want) < 5e-3 * size, (i, slope, want)


@pytest.mark.gpu
def test_the_same_call_twice_gives_the_same_bits():
    q, k, v, f, hin, dy, dh = _inputs("bf16", 2, 1000, 2, 64, 64)
    a = run(q, k, v, f, hin, None, None, 0.1, False, dy, dh)
    for _ in range(3):
        for x, y in zip(run(q, k, v, f, hin, None, None, 0.1, False, dy, dh), a):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_other_streams_and_two_calls_at_once():
    q, k, v, f, hin, dy, dh = _inputs("bf16", 1, 3000, 1, 64, 64)
    a = run(q, k, v, f, hin, None, None, 0.1, False, dy, dh)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run(q, k, v, f, hin, None, None, 0.1, False, dy, dh))
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(x, y) for x, y in zip(r, a))


@pytest.mark.gpu
def test_captured_calls():
    q, k, v, f, hin, dy, dh = _inputs("bf16", 1, 2000, 2, 64, 64)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, f, hin)]
    state = hin.clone()

    def train():
        y, s = M.decayed_attention(*leaves[:4], h_in=leaves[4], scale=0.1, want_state=True)
        return [y, s] + list(torch.autograd.grad([y, s], leaves, [dy, dh]))

    def serve():
        with torch.no_grad():
            y, s = M.decayed_attention(q, k, v, f, h_in=hin, scale=0.1, want_state=True)
            y1, _ = M.ops.decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], f[:, 0], state, 0.1, h_out=state)
        return [y, s, y1]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        train()
        serve()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for fn in (train, serve, serve):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = fn()
        graphs.append((g, out))
    for seed in (1, 2):
        new = _inputs("bf16", 1, 2000, 2, 64, 64, seed=seed)
        with torch.no_grad():
            for to, t in zip((q, k, v, f, hin, dy, dh), new):
                to.copy_(t)
            for to, t in zip(leaves, new):
                to.copy_(t)
            state.copy_(new[4])
        graphs[0][0].replay()
        want = run(*new[:5], None, None, 0.1, False, *new[5:])
        assert all(torch.equal(x, y) for x, y in zip(graphs[0][1], want))
        st = new[4].clone()
        for g, out in graphs[1:]:
            g.replay()
            y1, st = M.ops.decayed_attention_step(new[0][:, 0], new[1][:, 0], new[2][:, 0], new[3][:, 0], st, 0.1)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]) and torch.equal(out[2], y1)
        assert torch.equal(state, st)


@pytest.mark.gpu
def test_empty_calls():
    for b, n, h in ((0, 5, 2), (2, 0, 2), (2, 5, 0)):
        q, v = [torch.randn(b, n, h, w, device="cuda", requires_grad=True) for w in (8, 4)]
        f = torch.randn(b, n, h, device="cuda", requires_grad=True)
        s = torch.randn(b, h, 8, 4, device="cuda", requires_grad=True)
        y, out = M.decayed_attention(q, q, v, f, h_in=s, want_state=True)
        assert y.shape == (b, n, h, 4) and torch.equal(out, s)
        grads = torch.autograd.grad(y.sum() + out.sum(), [q, v, f, s])
        assert [g.shape for g in grads] == [t.shape for t in (q, v, f, s)] and torch.equal(grads[3], torch.ones_like(s))
        with torch.no_grad():
            y, out = M.decayed_attention(q, q, v, f, h_in=s, want_state=True)
            assert torch.equal(out, s) and float(M.decayed_attention(q, q, v, f, want_state=True)[1].abs().sum()) == 0
    y, s = M.ops.decayed_attention_step(torch.zeros(0, 2, 8, device="cuda"), torch.zeros(0, 2, 8, device="cuda"), torch.zeros(0, 2, 4, device="cuda"),
                                        torch.zeros(0, 2, device="cuda"))
    assert y.shape == (0, 2, 4) and s.shape == (0, 2, 8, 4)


@pytest.mark.gpu
def test_refusals():
    q, k, v, f, hin, _, _ = _inputs("bf16", 2, 9, 3, 8, 4)
    call = M.decayed_attention
    pad = torch.zeros(2, 9, dtype=torch.bool, device="cuda")
    for bad in (lambda: call(q, k[:, :8], v, f), lambda: call(q, k, v[:, :8], f), lambda: call(q, k, v, f[:, :8]), lambda: call(q[0], k[0], v[0], f[0]),
                lambda: call(q, k, v, f, pad[:, :8]), lambda: call(q, k, v, f, None, pad[0]), lambda: call(q, k, v, f, pad.cpu()),
                lambda: call(q, k, v, f, h_in=hin[:, :, :7]), lambda: call(q, k, v, f, h_in=hin[0]), lambda: call(q, k, v, f[0, 0, :2]),
                lambda: call(torch.zeros(1, 2, 1, 257, device="cuda"), torch.zeros(1, 2, 1, 257, device="cuda"), torch.zeros(1, 2, 1, 4, device="cuda"),
                             torch.zeros(1, 2, 1, device="cuda")),
                lambda: call(torch.zeros(1, 2, 1, 4, device="cuda"), torch.zeros(1, 2, 1, 4, device="cuda"), torch.zeros(1, 2, 1, 0, device="cuda"),
                             torch.zeros(1, 2, 1, device="cuda"))):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    for bad in (lambda: call(q.double(), k.double(), v.double(), f.double()), lambda: call(q, k.float(), v, f), lambda: call(q, k, v.half(), f),
                lambda: call(q, k, v, f.half()), lambda: call(q, k, v, f, h_in=hin.long())):
        with pytest.raises(TypeError):
            bad()
    step = M.ops.decayed_attention_step
    one = [t[:, 0] for t in (q, k, v, f)]
    flat = torch.zeros(hin.numel() + 64, device="cuda")
    for bad in (lambda: step(q, k, v, f, hin), lambda: step(*one, hin[0]), lambda: step(*one, hin, h_out=hin.double()),
                lambda: step(*one, hin, h_out=hin.transpose(2, 3).contiguous().transpose(2, 3)),
                lambda: step(*one, flat[:hin.numel()].view_as(hin), h_out=flat[8:8 + hin.numel()].view_as(hin)),
                lambda: step(hin[:, :, 0, :4].float().repeat(1, 1, 2)[..., :8], hin[:, :, 0, :4].repeat(1, 1, 2), hin[:, :, 0, :4], hin[:, :, 0, 0], None, h_out=hin)):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            bad()
    x = [t.detach().requires_grad_() for t in (q, k, v, f)]
    y = call(*x)
    g, = torch.autograd.grad(y.float().sum(), [x[0]], create_graph=False)
    with pytest.raises(RuntimeError):
        y = call(*x)
        torch.autograd.grad(y.float().sum(), [x[0]], create_graph=True)
    s = hin.clone().requires_grad_()
    y = call(*x, h_in=s.detach().requires_grad_())
    t = hin.clone()
    y = call(*x, h_in=t)
    step(*one, t, h_out=t)
    with pytest.raises(RuntimeError):   # (the state that the graph needs has been written over)
        y.float().sum().backward()


def test_refusals_on_the_host():
    x = torch.zeros(1, 2, 1, 4)
    with pytest.raises(RuntimeError):
        M.decayed_attention(x, x, x, x[..., 0])
    with pytest.raises(RuntimeError):
        M.ops.decayed_attention_step(x[0], x[0], x[0], x[0, ..., 0])
    lib = _lib.lib()
    a = _lib.DecayedAttentionArgs()
    good = dict(dtype=1, gate_dtype=1, B=2, L=100, H=3, K=64, V=64, q=16, k=16, v=16, f=16, y=16)
    for key, value in good.items():
        setattr(a, key, value)
    assert lib.mega_decayed_attention_fwd(None, None) == 1
    assert lib.mega_decayed_attention_work(ctypes.byref(a), 0) >= 0 and lib.mega_decayed_attention_work(ctypes.byref(a), 1) > 0
    for key, value, status in (("dtype", 7, 2), ("gate_dtype", 2, 2), ("B", 0, 3), ("L", 0, 3), ("K", 0, 3), ("V", -1, 3), ("K", 257, 7), ("V", 300, 7), ("q", 0, 1),
                               ("f", 0, 1), ("y", 0, 1), ("k", 17, 5), ("f", 15, 5)):
        setattr(a, key, value)
        assert lib.mega_decayed_attention_fwd(ctypes.byref(a), None) == status, key
        setattr(a, key, good[key])
    assert lib.mega_decayed_attention_bwd(ctypes.byref(a), None) == 1
    a.h_in = a.h_out = 64       # states that overlap: another segment may still read what one has written
    assert lib.mega_decayed_attention_fwd(ctypes.byref(a), None) == 7
    a.h_out = 66
    assert lib.mega_decayed_attention_fwd(ctypes.byref(a), None) == 5
    a.h_in = a.h_out = None
    assert lib.mega_decayed_attention_step(ctypes.byref(a), None) == 3
    a.L = 1
    assert lib.mega_decayed_attention_step(ctypes.byref(a), None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_module(dtype):
    torch.manual_seed(0)
    m = M.DecayedAttention(48, 3, zdim=48, hdim=96).cuda().to(DT[dtype])
    u = torch.randn(2, 130, 48, device="cuda").to(DT[dtype])
    pad = torch.zeros(2, 130, dtype=torch.bool, device="cuda")
    pad[1, 100:] = True
    with torch.no_grad():
        whole = m(u, pad)
        assert whole.shape == (2, 130, 96)
        q, k, v, f = m._parts(m.in_proj(u))
        assert torch.equal(whole.unflatten(-1, (3, 32)), M.decayed_attention(q, k, v, f, pad, scale=m.scale))
    # the packed gradient is the parts'
    z = m.in_proj(u).detach().requires_grad_()
    dy = torch.randn(2, 130, 3, 32, device="cuda").to(DT[dtype])
    a, = torch.autograd.grad(M.functions.decayed_attention_packed(z, 3, 16, pad, scale=m.scale), [z], dy)
    b, = torch.autograd.grad(M.functions.decayed_attention(*m._parts(z), pad, scale=m.scale), [z], dy)
    assert torch.equal(a, b)
    m(u, pad).float().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())


@pytest.mark.gpu
def test_module_states_and_beams():
    torch.manual_seed(1)
    m = M.DecayedAttention(32, 2).cuda().eval()
    u = torch.randn(3, 90, 32, device="cuda")
    with torch.no_grad():
        whole = m(u)
        state = {}
        parts = [m(u[:, :64], None, state)] + [m(u[:, t:t + 1], None, state) for t in range(64, 70)]
        order = torch.tensor([2, 0, 1], device="cuda")
        m.reorder_incremental_state(state, order)
        parts2 = [m(u[order][:, t:t + 1], None, state) for t in range(70, 90)]
    size = float(whole.abs().max())
    assert torch.allclose(torch.cat(parts, 1), whole[:, :70], atol=1e-5 * size, rtol=0)
    assert torch.allclose(torch.cat(parts2, 1), whole[order][:, 70:], atol=1e-5 * size, rtol=0)
    with pytest.raises(NotImplementedError):
        m(u, None, {})
    both_ways = M.DecayedAttention(32, 2, bidirectional=True).cuda().eval()
    reset = torch.zeros(3, 90, dtype=torch.bool, device="cuda")
    reset[:, 40] = True
    with torch.no_grad():
        y = both_ways(u, None, None, reset)
        for part in (slice(0, 40), slice(40, 90)):   # documents do not see one another
            assert torch.allclose(both_ways(u[:, part]), y[:, part], atol=1e-5 * float(y.abs().max()), rtol=0)


@pytest.mark.gpu
def test_a_block_of_the_operators_together():
    """residual stream -> norm -> attention -> norm of each head -> back to the stream, against 64 bits; gradients of everything"""
    torch.manual_seed(3)
    b, n, d, heads = 2, 100, 64, 4
    norm, attn, out = M.RMSNorm(d).cuda(), M.DecayedAttention(d, heads).cuda(), M.RMSNorm(d, num_groups=heads).cuda()
    with torch.no_grad():
        for p in (norm.weight, out.weight):
            p.normal_(std=0.2)
    x, res = torch.randn(b, n, d, device="cuda", requires_grad=True), torch.randn(b, n, d, device="cuda", requires_grad=True)
    pad = torch.zeros(b, n, dtype=torch.bool, device="cuda")
    pad[1, 80:] = True
    dy = torch.randn(b, n, d, device="cuda")
    params = [x, res] + [p for mod in (norm, attn, out) for p in mod.parameters()]

    y, stream = norm(x, res)
    final = stream + out(attn(y, pad))
    got = [final] + list(torch.autograd.grad(final, params, dy))

    x64 = [p.detach().double().requires_grad_() for p in params]
    wn, (w, c), wo = x64[2], x64[3:5], x64[5]
    r = x64[0] + x64[1]
    t = r / torch.sqrt((r * r).mean(-1, keepdim=True) + norm.eps) * (1 + wn)
    z = t @ w.T + c
    q, k, v, f = z.split((d, d, d, heads), -1)
    q, k, v = (a.unflatten(-1, (heads, -1)) for a in (q, k, v))
    live = (~pad).double()[..., None, None]
    a = torch.where(pad[..., None], 1.0, torch.sigmoid(f))
    o, _ = _walk(q * attn.scale, k * live, v * live, a, torch.zeros(b, heads, d // heads, d // heads, dtype=torch.float64, device="cuda"), range(n))
    o = o * live
    o = (o / torch.sqrt((o * o).mean(-1, keepdim=True) + out.eps)).flatten(-2) * (1 + wo)
    ref64 = r + o
    ref = [ref64] + list(torch.autograd.grad(ref64, x64, dy.double()))
    # fp32 all through but the projection (a library product in fp32): 2^-20 of each value's size; the norm of a head's output divides by
    # what may be as small as a tenth of the usual size, which its gradient does twice
    for i, (p, s) in enumerate(zip(got, ref)):
        err = float((p.double() - s).norm() / s.norm())
        assert err < 1e-4, (i, err)
