"""Linear attention with a decay for each head where states, gradients or gates leave their usual range, and which form takes a call.

A test that takes `form` runs both forms of whole sequences (tcgen05, and mma.sync by way of the option that leaves the first one out).
The reference is the recurrence in 64 bits.  Tolerances are on norms: an elementwise bound adds up every share's largest error, under which a lost piece of
an operand would not show.

Outputs and gradients in 16-bit types have three roundings on their way (a pair's weight, the state that is read, the result), of which
each is at most u = half a step of the value and together, independently of one another, sqrt(3) u / sqrt(3) = u in the mean square.
fp16 below its normal range: half a step is 2^-25 whatever the value, for the result alone.

States are fp32 sums: the products of a chunk cut their sum off up to 24 times (three pieces of eight groups of 16 steps) by at most
2^-23 of a partial sum, half of that on average, of partial sums half as large on average: 24 * 2^-25 = 7e-7; a weight is a product of
two powers of two and a sum of logarithms (8 * 2^-24 ln 2 + 2 * 2^-23 = 6e-7).  Together below 1.5e-6 (two pieces of bf16 keys, where
there is room for no more: 2^-17 of a key besides).
"""
import ctypes
import threading
import time

import pytest
import torch

import fairseq_apollo_b200 as M
from fairseq_apollo_b200 import _lib
from test_decayed_attention import DT, _inputs, both, reference, run

STATE = 1.5e-6
HEADS = [(64, 64), (64, 128), (128, 64), (128, 128), (40, 24)]


@pytest.fixture(params=["tcgen05", "mma"])
def form(request):
    _lib.set_option(1, int(request.param == "mma"))
    yield request.param
    _lib.set_option(1, 0)


def near(got, ref, rel, step=0.0, size=None):
    """|error| <= rel |ref| (or another size) + step for every value, in the mean square"""
    assert torch.isfinite(got).all()
    err, allowed = float((got.detach().double() - ref).norm()), rel * float((ref if size is None else size).norm()) + step * ref.numel() ** 0.5
    assert err <= allowed, (err / allowed, err / (float(ref.norm()) + 1e-300))


@pytest.mark.gpu
def test_a_thread_that_is_new_to_cuda_takes_the_same_form():
    """a thread's first call, with all its memory from the allocator's cache (as an autograd thread's first backward may have it)"""
    q, k, v, f, hin, _, _ = _inputs("bf16", 2, 300, 2, 64, 64)
    _lib.set_option(1, 0)
    with torch.no_grad():
        want = M.decayed_attention(q, k, v, f, h_in=hin)
        assert _lib.last_kernel() == "decayed_attention_tc"
        M.decayed_attention(q, k, v, f, h_in=hin)   # (all sizes are in the cache then)
    got = []

    def first():
        with torch.no_grad():
            got.append(M.decayed_attention(q, k, v, f, h_in=hin))
        got.append(_lib.last_kernel())
    thread = threading.Thread(target=first)
    thread.start()
    thread.join()
    assert got[1] == "decayed_attention_tc" and torch.equal(got[0], want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kd,vd", [("bf16", 64, 64), ("fp16", 64, 128), ("fp16", 128, 128), ("bf16", 128, 128), ("fp32", 64, 40)])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_states_that_are_not_finite_reach_what_reads_them_alone(form, dtype, kd, vd, reverse, value):
    """a state that comes in reaches no step behind a reset and no padded step, the gradient of the one that leaves none before it"""
    b, n, h = 2, 300, 2
    q, k, v, f, hin, dy, dh = _inputs(dtype, b, n, h, kd, vd)
    at = torch.arange(n, device="cuda")
    at = (n - 1 - at if reverse else at)[None].expand(b, n)   # steps in the order of the walk
    reset, pad = at == 30, ((at >= 5) & (at < 10)) | ((at >= 40) & (at < 60)) | ((at >= 130) & (at < 150))
    before, behind = at < 30, at >= 30

    def call(hin, dh):
        return run(q, k, v, f, hin, pad, reset, 0.1, reverse, dy, dh)
    odd = torch.full_like(hin, value)
    want, got = call(torch.zeros_like(hin), dh), call(odd, dh)
    assert torch.equal(got[0][behind], want[0][behind]) and float(got[0][pad].detach().abs().max()) == 0 and torch.equal(got[1], want[1])
    for i in (2, 3, 4, 5):
        assert torch.equal(got[i][behind], want[i][behind]), i
        assert float(got[i][pad].abs().max()) == 0, i
    assert torch.equal(got[6], want[6])
    want, got = call(hin, torch.zeros_like(dh)), call(hin, odd)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2]) and torch.equal(got[6], want[6])
    for i in (3, 4, 5):
        assert torch.equal(got[i][before], want[i][before]), i
        assert float(got[i][pad].abs().max()) == 0, i


@pytest.mark.gpu
@pytest.mark.parametrize("kd,vd", HEADS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4, 1e-5])
def test_states_and_their_gradients_keep_fp32_places(form, dtype, kd, vd, size):
    """weighted keys are held in pieces whose places suffice however small the gradients are"""
    q, k, v, f, hin, dy, dh = _inputs(dtype, 2, 300, 2, kd, vd)
    dy, dh = (dy.float() * size).to(DT[dtype]), dh * size
    kw = dict(hin=hin, scale=kd ** -0.5, dy=dy, dh=dh)
    ref, _ = reference(q, k, v, f, **kw)
    got = run(q, k, v, f, **kw)
    near(got[1], ref[1], STATE)
    two = dtype == "bf16" and form == "tcgen05" and kd > 64 and vd > 64
    near(got[6], ref[6], STATE + (2.0 ** -17 if two else 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("b,n,h", [(5, 700, 16), (1, 2100, 16)])
@pytest.mark.parametrize("kd,vd", HEADS[:4])
def test_fp16_over_many_chunks(form, kd, vd, b, n, h):
    """blocks that walk several chunks, with and without segments; gradients of 1e-4"""
    q, k, v, f, hin, dy, dh = _inputs("fp16", b, n, h, kd, vd, shift=4.0, gate_dtype=torch.float32)
    dy, dh = (dy.float() * 1e-4).half(), dh * 1e-4
    pad = torch.arange(n, device="cuda")[None].expand(b, n) >= n - 150
    got = run(q, k, v, f, hin, pad, None, 0.1, False, dy, dh)
    again = run(q, k, v, f, hin, pad, None, 0.1, False, dy, dh)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0 and all(torch.equal(x, y) for x, y in zip(got, again))
    part = slice(h - 2, h)
    ref, _ = reference(*(t[:1, :, part] for t in (q, k, v, f)), hin[:1, part], pad[:1], None, 0.1, False, dy[:1, :, part], dh[:1, part])
    got = [got[i][:1, part] if i in (1, 6) else got[i][:1, :, part] for i in range(7)]
    near(got[1], ref[1], STATE)
    near(got[6], ref[6], STATE)
    near(got[0], ref[0], 2.0 ** -11)


def gate_sizes(q, k, v, f, hin, scale, dy, dh):
    """d log a_t = a_t <R_t, S_{t-1}> adds up one product for every key and value, with roundings of their own: off by at most u in the
    mean square (three of them) of the products' norm, which may be larger than their sum.  Those norms, times the gates' slope."""
    q, k, v, f, s, dy, r = (t.double() for t in (q, k, v, f, hin, dy, dh))
    a, states, out = torch.sigmoid(f)[..., None, None], [], [None] * q.shape[1]
    for t in range(q.shape[1]):
        states.append(s)
        s = a[:, t] * s + k[:, t, :, :, None] * v[:, t, :, None, :]
    for t in reversed(range(q.shape[1])):
        r = r + scale * q[:, t, :, :, None] * dy[:, t, :, None, :]
        out[t] = (a[:, t] * r * states[t]).square().sum((-1, -2)).sqrt()
        r = a[:, t] * r
    return torch.stack(out, 1) * torch.sigmoid(-f)


@pytest.mark.gpu
@pytest.mark.parametrize("kd,vd", HEADS)
@pytest.mark.parametrize("size", [5e5, 1.0, 1e-4])
def test_fp16_reads_states_of_any_size(form, kd, vd, size):
    """states beyond fp16's range, and below its normal one, beside outputs inside it: keys and values that add next to nothing, and
    queries that bring the outputs back to their usual size"""
    q, k, v, f, hin, dy, dh = _inputs("fp16", 2, 300, 2, kd, vd, gate_dtype=torch.float32, shift=5.0)
    unit = 2.0 ** -10 if size > 1 else 1.0
    q, dy = (t * (unit if size > 1 else 16.0) for t in (q, dy))
    k, v = ((t.float() * (unit if size > 1 else size ** 0.5)).half() for t in (k, v))
    hin, dh = hin * size, dh * size
    kw = dict(hin=hin, scale=kd ** -0.5, dy=dy, dh=dh)
    ref, _ = reference(q, k, v, f, **kw)
    assert all(float(ref[i].abs().max()) < 65504 for i in (0, 2, 3, 4))
    got = run(q, k, v, f, **kw)
    u = 2.0 ** -11
    for i in (0, 2, 3, 4):
        near(got[i], ref[i], u, 2.0 ** -25)
    near(got[5], ref[5], u, size=gate_sizes(q, k, v, f, **kw))
    near(got[1], ref[1], STATE)
    near(got[6], ref[6], STATE)


@pytest.mark.gpu
@pytest.mark.parametrize("kd,vd", HEADS)
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4, 1e-5])
def test_fp16_gradients_of_any_size(form, kd, vd, size):
    q, k, v, f, hin, dy, dh = _inputs("fp16", 2, 300, 2, kd, vd, gate_dtype=torch.float32)
    dy, dh = (dy.float() * size).half(), dh * size
    kw = dict(hin=hin, scale=kd ** -0.5, dy=dy, dh=dh)
    ref, _ = reference(q, k, v, f, **kw)
    got = run(q, k, v, f, **kw)
    u = 2.0 ** -11
    for i in (2, 3, 4):
        near(got[i], ref[i], u, 2.0 ** -25)
    near(got[5], ref[5], u, size=gate_sizes(q, k, v, f, **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("kd,vd", HEADS)
def test_fp16_pairs_of_any_size(form, kd, vd):
    """products of queries and keys beyond fp16's range, beside values so small that the outputs are not"""
    q, k, v, f, hin, dy, dh = _inputs("fp16", 2, 300, 2, kd, vd, gate_dtype=torch.float32)
    q, k, v, dy = q * 256, k * 256, v * 2.0 ** -10, dy * 2.0 ** -10
    kw = dict(hin=hin * 0.1, scale=1.0, dy=dy, dh=dh)
    ref, _ = reference(q, k, v, f, **kw)
    assert float(torch.einsum("blhk,blhk->blh", q.double(), k.double()).abs().max()) > 1e5
    assert all(float(ref[i].abs().max()) < 65504 for i in (0, 2, 3, 4))
    got = run(q, k, v, f, **kw)
    u = 2.0 ** -11
    for i in (0, 2, 3, 4):
        near(got[i], ref[i], u, 2.0 ** -25)
    near(got[5], ref[5], u, size=gate_sizes(q, k, v, f, **kw))


@pytest.mark.gpu
def test_weights_behind_gates_that_are_nearly_closed(form):
    """sums of logarithms of some thousands in front of the pairs that count: the weight between two steps is that of the steps
    between them all the same.  All sequences and heads have the same gates, so a weight's error is common to them and roundings
    are not: the mean over 64 of them, of outputs' components along their reference, is off by sqrt(3 / 16) u / 8 = 3e-5 at most."""
    n, shut, to = (128, 64, 96) if form == "tcgen05" else (64, 30, 48)   # closed gates, then steps with values, then those that read them
    b, h, kd, vd = 8, 8, 64, 128
    q, k, v, f, _, _, _ = _inputs("fp16", b, n, h, kd, vd)
    f = f[:1, :, :1] * 0.25 + 4.0
    f[:, :shut] = -100.0
    f = f.expand(b, n, h)
    v[:, :shut] = 0
    v[:, to:] = 0
    ref, _ = reference(q, k, v, f, scale=kd ** -0.5)
    y = run(q, k, v, f, scale=kd ** -0.5)[0][:, to:].double()
    r = ref[0][:, to:]
    off = ((y * r).sum(-1) / (r * r).sum(-1) - 1).mean((0, 2))
    assert float(off.square().mean().sqrt()) < 4e-5, off


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kd,vd", [(64, 64), (64, 128), (128, 128)])
@pytest.mark.parametrize("pattern", ["half", "some", "documents"])
def test_gradients_of_closed_gates_beside_open_ones(form, dtype, kd, vd, pattern):
    """nothing passes a closed gate: its gradient is next to nothing however much the steps on either side of it have to do with one
    another, and open gates, whose slope is 3e-4, have a small one"""
    q, k, v, f, hin, dy, dh = _inputs(dtype, 2, 300, 2, kd, vd, gate_dtype=torch.float32, shift=8.0, spread=0.5)
    reset = None
    if pattern == "half":
        f[:, 40:100] = -70.0
        f[:, 200:290] = -25.0
    elif pattern == "some":
        f[:, ::23] = -40.0
        f[:, 7::31] = -20.0
    else:
        reset = torch.zeros(2, 300, dtype=torch.bool, device="cuda")
        reset[:, 5::40] = True
        f[:, ::29] = -90.0
    kw = dict(hin=hin, scale=kd ** -0.5, dy=dy, dh=dh)
    ref, _ = reference(q, k, v, f, reset=reset, **kw)
    got = run(q, k, v, f, reset=reset, **kw)
    u = torch.finfo(DT[dtype]).eps / 2 if dtype != "fp32" else 2.0 ** -19
    # (shares of pairs, of both states and of what passes a chunk, each rounded once: 4 u / sqrt(3) / 2, with room for pairs that one walk
    # rounds up and the other down)
    near(got[5], ref[5], 1.5 * u, size=gate_sizes(q, k, v, f if reset is None else f.masked_fill(reset[..., None], -float("inf")), **kw))
    shut = (f < -19)
    # (a decay of e^-20 times products of states of 10 by 10, 128 x 128 of them, is below 1e-4)
    assert float(got[5][shut].abs().max()) < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("mean,shut", [(-2.0, False), (-2.0, True), (2.0, True)])
def test_gates_that_go_from_next_to_closed_to_open(form, mean, shut):
    """the gradient's walks weigh a pair alike, to the last bit where each pair has a power of two of its own"""
    q, k, v, f, hin, dy, dh = _inputs("fp16", 2, 260, 4, 128, 128, gate_dtype=torch.float32, shift=mean, spread=6.0)
    if shut:
        f[:, :130] = -70.0
    kw = dict(hin=hin, scale=128 ** -0.5, dy=dy, dh=dh)
    ref, _ = reference(q, k, v, f, **kw)
    got = run(q, k, v, f, **kw)
    near(got[5], ref[5], 1.2 * 2.0 ** -11)   # (four shares, each rounded once: 2 u / sqrt(3))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_which_form_takes_a_call(dtype):
    """tcgen05 takes 16-bit heads of at most 128 keys and values, more than 64 steps and rows on 16 bytes; mma.sync the rest"""
    _lib.set_option(1, 0)

    def name(change, b=2, n=200, h=4, kd=64, vd=64, backward=True):
        q, k, v, f, hin, dy, dh = _inputs(dtype, b, n, h, kd, vd)
        q, k, v, f, dy = change(q, k, v, f, dy)
        with torch.no_grad():
            M.decayed_attention(q, k, v, f)
        forward = _lib.last_kernel()
        if backward:
            run(q, k, v, f, hin, dy=dy, dh=dh)
            assert _lib.last_kernel() == forward
        return forward

    def same(*x):
        return x

    def columns(extra):   # of one projection, `extra` values off
        def change(q, k, v, f, dy):
            z = torch.zeros(*q.shape[:2], extra + 8 + sum(t[0, 0].numel() for t in (q, k, v, f)), dtype=q.dtype, device="cuda")
            out, at = [], extra
            for t in (q, k, v, f):
                w = t[0, 0].numel()
                z[..., at:at + w] = t.flatten(2)
                out.append(z[..., at:at + w].view(t.shape))
                at += w
            return (*out, dy)
        return change

    def time_major(*x):
        return tuple(t.transpose(0, 1).contiguous().transpose(0, 1) for t in x)

    def shared(q, k, v, f, dy):
        return q, k[:, :, :1].expand_as(k), v[:, :, :1].expand_as(v), f, dy

    def thrice(q, k, v, f, dy):   # the same sequence for all
        return (*(t[:1].expand_as(t) for t in (q, k, v, f)), dy)
    taken = "decayed_attention_tc" if dtype != "fp32" else "other"
    for kd, vd in HEADS + [(8, 8), (72, 16), (16, 120)]:
        assert name(same, kd=kd, vd=vd) == taken, (kd, vd)
    assert name(same, n=65) == taken and name(time_major) == taken and name(shared) == taken and name(thrice) == taken
    assert name(same, b=1, h=1) == taken
    assert name(columns(0), h=8) == taken   # (8 heads: rows of 1544 + 8 values)
    assert name(same, n=64) == "other" and name(same, kd=136) == "other" and name(same, vd=144) == "other" and name(same, kd=36) == "other"
    assert name(columns(1), h=8) == "other" and name(columns(0), h=12) == "other"   # (rows of 2324 + 8 values)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("size", [(2, 130, 3, 64, 128), (1, 129, 1, 128, 128), (3, 257, 2, 48, 96), (1, 65, 2, 32, 40), (2, 300, 2, 64, 64)])
@pytest.mark.parametrize("reverse", [False, True])
def test_both_forms_at_the_same_sizes(form, dtype, size, reverse):
    b, n, h, kd, vd = size
    g = torch.Generator().manual_seed(6)
    pad, reset = (torch.rand(b, n, generator=g) < 0.3).cuda(), (torch.rand(b, n, generator=g) < 0.05).cuda()
    both(dtype, *size, reverse=reverse)
    assert _lib.last_kernel() == ("decayed_attention_tc" if form == "tcgen05" else "other")
    both(dtype, *size, pad, reset, reverse=reverse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads", [8, 12])
@pytest.mark.parametrize("b,n", [(2, 200), (10, 300)])
def test_one_projection(dtype, heads, b, n):
    """the module's layout: z's gradient, written in place of its parts, on tcgen05 (8 heads) and mma.sync (12)"""
    _lib.set_option(1, 0)
    q, k, v, f, hin, dy, dh = _inputs(dtype, b, n, heads, 64, 64, shift=3.0)
    pad = torch.arange(n, device="cuda")[None].expand(b, n) >= torch.arange(n - 10 * b, n, 10, device="cuda")[:, None]
    z = torch.cat([t.flatten(2) for t in (q, k, v, f)], -1).requires_grad_()
    y, h = M.functions.decayed_attention_packed(z, heads, 64, pad, None, hin, 0.125, True)
    form = "decayed_attention_tc" if heads == 8 else "other"
    assert _lib.last_kernel() == form
    dz, = torch.autograd.grad([y, h], [z], [dy, dh])
    assert _lib.last_kernel() == form
    kw = dict(hin=hin, pad=pad, scale=0.125, dy=dy, dh=dh)
    ref, _ = reference(q, k, v, f, **kw)
    u = torch.finfo(DT[dtype]).eps / 2
    want = torch.cat([t.flatten(2) for t in ref[2:6]], -1)
    step = 2.0 ** -25 if dtype == "fp16" else 0.0
    near(y, ref[0], u, step)
    near(h, ref[1], STATE)
    for part, (a, c) in enumerate(zip(dz.split([64 * heads] * 3 + [heads], -1), want.split([64 * heads] * 3 + [heads], -1))):
        # (the gates' gradient: one rounding more, and that of products which may be larger than their sum)
        near(a, c, u * (1.5 if part == 3 else 1.0), step)
    assert float(dz.detach()[pad].abs().max()) == 0
    parts = run(*(t for t in (q, k, v, f)), **kw)
    assert torch.equal(dz, torch.cat([t.flatten(2) for t in parts[2:6]], -1)) or heads == 12   # (rows of 12 heads by themselves: tcgen05)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_the_module_on_tcgen05(dtype):
    torch.manual_seed(0)
    _lib.set_option(1, 0)
    m = M.DecayedAttention(96, 8, zdim=256, hdim=512, bidirectional=True).cuda().to(DT[dtype])
    u = torch.randn(3, 260, 96, device="cuda").to(DT[dtype])
    pad = torch.arange(260, device="cuda")[None] >= torch.tensor([[260], [100], [201]], device="cuda")
    with torch.no_grad():
        y = m(u, pad)
        z, r = m.in_proj(u), m.back_proj(u)
        a = M.decayed_attention(*m._parts(z), pad, scale=m.scale)
        assert _lib.last_kernel() == "decayed_attention_tc"
        c = M.decayed_attention(*m._parts(r), pad, scale=m.scale, reverse=True)
        assert torch.equal(y, (a + c).flatten(-2))
    m(u, pad).float().square().sum().backward()
    assert _lib.last_kernel() == "decayed_attention_tc"
    assert all(torch.isfinite(p.grad).all() and float(p.grad.abs().max()) > 0 for p in m.parameters())


@pytest.mark.gpu
def test_more_than_2_to_the_31_values():
    """the last heads of a call whose offsets pass 32 bits, forward and backward, against a call of their own"""
    b, n, h, kd, vd = 1, 34000, 512, 128, 128
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    _lib.set_option(1, 0)
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v, dy = (torch.randn(b, n, h, kd, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(4))
    f = torch.randn(b, n, h, device="cuda", dtype=torch.float32, generator=g) + 3.0
    assert v.numel() > 2 ** 31
    last = slice(h - 2, h)
    part = run(*(t[:, :, last].contiguous() for t in (q, k, v, f)), None, None, None, 0.1, False, dy[:, :, last].contiguous(),
               torch.zeros(b, 2, kd, vd, device="cuda"))
    whole = run(q, k, v, f, None, None, None, 0.1, False, dy, torch.zeros(b, h, kd, vd, device="cuda"))
    for i in range(6):
        x, y = (whole[i][:, last] if i == 1 else whole[i][:, :, last]).detach().double(), part[i].detach().double()
        # (few heads have segments, whose states are joined in another order: last bits, and a rounding that goes the other way)
        assert float((x - y).norm()) < 2.0 ** -8 * float(y.norm()), i


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("scale", [-0.5, 0.0, 30.0, 1e-6])
@pytest.mark.parametrize("kd,vd", [(64, 64), (64, 128), (128, 128)])
def test_scales_of_any_sign_and_size(form, dtype, scale, kd, vd):
    q, k, v, f, hin, dy, dh = _inputs(dtype, 2, 200, 2, kd, vd, gate_dtype=torch.float32)
    kw = dict(hin=hin, scale=scale, dy=dy, dh=dh)
    ref, _ = reference(q, k, v, f, **kw)
    got = run(q, k, v, f, **kw)
    # (fp32: two products in a row leave out 2^-22 each; queries times keys and pairs times values are cut off at each group of 8 places, at
    # 128 keys 16 + 8 times by 2^-25 on average; weights as above: 5e-7 + 7e-7 + 6e-7 = 1.8e-6)
    u, step = torch.finfo(DT[dtype]).eps / 2 if dtype != "fp32" else 2.0 ** -19, 2.0 ** -25 if dtype == "fp16" else 0.0
    for i in (0, 2, 3, 4):
        near(got[i], ref[i], u, step)
    near(got[5], ref[5], u, size=gate_sizes(q, k, v, f, **kw))
    near(got[1], ref[1], STATE)
    # (with a scale of 0 the state's gradient is dh times the whole sequence's decay 2^-G, a weight far below the 2^-8 that STATE reckons with:
    # its logarithm, 2^-24 of itself off in its terms and once more as a float, is G 2^-23 ln 2 off)
    whole = 0.0 if scale else float(torch.nn.functional.logsigmoid(f.double()).sum(1).abs().max()) * 2.0 ** -23
    near(got[6], ref[6], STATE + whole + (2.0 ** -17 if dtype == "bf16" and form == "tcgen05" and kd > 64 and vd > 64 else 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("kd,vd", [(64, 64), (128, 128)])
def test_fp16_calls_at_once_and_captured(form, kd, vd):
    q, k, v, f, hin, dy, dh = _inputs("fp16", 2, 900, 2, kd, vd)

    def call():
        return run(q, k, v, f, hin, None, None, 0.1, False, dy, dh)
    want = call()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for r in got for x, y in zip(r, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for t in out:
        t.detach().zero_()
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(out, want))
    assert _lib.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_a_prompt_on_tcgen05_and_single_steps_behind_it(dtype):
    torch.manual_seed(2)
    _lib.set_option(1, 0)
    m = M.DecayedAttention(128, 8, zdim=512, hdim=512).cuda().to(DT[dtype]).eval()
    u = torch.randn(3, 210, 128, device="cuda").to(DT[dtype])
    with torch.no_grad():
        q, k, v, f = m._parts(m.in_proj(u))
        ref, _ = reference(q, k, v, f, scale=m.scale)
        state = {}
        parts = [m(u[:, :200], None, state)]
        assert _lib.last_kernel() == "decayed_attention_tc"
        parts += [m(u[:, t:t + 1], None, state) for t in range(200, 210)]
    # (single steps' projections are other library products: a rounding of each operand more)
    near(torch.cat(parts, 1).unflatten(-1, (8, 64)), ref[0], 2 * torch.finfo(DT[dtype]).eps / 2, 2.0 ** -25 if dtype == "fp16" else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kd,vd", HEADS[:4])
@pytest.mark.parametrize("b,n,h", [(5, 700, 16), (1, 2100, 16)])
@pytest.mark.parametrize("padded", [False, True])
def test_a_wait_that_runs_out(dtype, kd, vd, b, n, h, padded):
    """keys of a chunk that never arrive (a test aid; the limit of waits is then a millisecond): every walk of the call ends by itself
    and raises the error word, and the next call is as if nothing had been"""
    q, k, v, f, hin, dy, dh = _inputs(dtype, b, n, h, kd, vd, shift=4.0)
    pad = (torch.arange(n, device="cuda")[None].expand(b, n) % 200 >= 150) if padded else None
    _lib.set_option(1, 0)

    def call():
        return run(q, k, v, f, hin, pad, None, 0.1, False, dy, dh)
    want = call()
    assert _lib.last_kernel() == "decayed_attention_tc" and _lib.device_error(reset=True) == 0
    _lib.set_option(3, 2_000_000)
    _lib.set_option(4, 1)
    try:
        begun = time.time()
        call()
        torch.cuda.synchronize()
        assert time.time() - begun < 5.0
        assert _lib.device_error(reset=True) != 0
    finally:
        _lib.set_option(3, 0)
        _lib.set_option(4, 0)
    for x, y in zip(call(), want):
        assert torch.equal(x, y)
    assert _lib.device_error() == 0


def test_the_longest_sequences_have_their_chunks_counted():
    lib, a = _lib.lib(), _lib.DecayedAttentionArgs()
    for key, value in dict(dtype=1, gate_dtype=1, B=1, H=1, K=8, V=8).items():
        setattr(a, key, value)
    for backward in (0, 1):
        sizes = []
        for length in (2 ** 31 - 256, 2 ** 31 - 1):
            a.L = length
            sizes.append(lib.mega_decayed_attention_work(ctypes.byref(a), backward))
        # (a forward call has the gates of 2^24 chunks of 128 steps, 1216 bytes each)
        assert 2 ** 24 * 1024 < sizes[0] <= sizes[1] < 1.01 * sizes[0], sizes
