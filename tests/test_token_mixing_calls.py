"""Calls of the token-mixing operators (ops.rope, ops.qk_norm_rope, ops.linear_attention, ops.linear_attention_step and their C
entries) at the borders of what is allowed."""
import ctypes

import pytest
import torch

DEV = "cuda:0"


def test_linear_attention_refuses_rows_that_run_backwards():
    """A lane's place in a chunk is an unsigned offset: a negative stride would be 4 GB off."""
    from ironcortex_amd import hip
    lib, EINVAL = hip.lib(), hip.ENUMS["IC_EINVAL"]
    good = dict(B=1, H=2, Hk=1, T=5, Dk=8, Dv=8, dtype=0, q=16, k=16, v=16, rate=16, out=16, ws=16)
    for name, who in (("q_st", "q has"), ("k_st", "k has"), ("v_st", "v has"), ("o_st", "out has")):
        for stride in (-8, -1, -(1 << 22) + 1):
            a = hip.new("ic_lattn_args", **{**good, name: stride})
            assert lib.ic_lattn_fwd(ctypes.byref(a), None) == EINVAL and who in lib.ic_last_error().decode(), (name, stride)
    for name, who in (("do_st", "dout has"), ("dq_st", "dq has"), ("dk_st", "dk has"), ("dv_st", "dv has")):
        b = hip.new("ic_lattn_bwd_args", f=hip.new("ic_lattn_args", **good), dout=16, dq=16, dk=16, dv=16, **{name: -8})
        assert lib.ic_lattn_bwd(ctypes.byref(b), None) == EINVAL and who in lib.ic_last_error().decode(), name
    b = hip.new("ic_lattn_bwd_args", f=hip.new("ic_lattn_args", **{**good, "v_st": -8}), dout=16, dq=16, dk=16, dv=16)
    assert lib.ic_lattn_bwd(ctypes.byref(b), None) == EINVAL and b"v has" in lib.ic_last_error()


@pytest.fixture
def launches(monkeypatch):
    """The names of the C entries called, in place of the calls (CPU tensors in place of the device's)."""
    from ironcortex_amd.hip import ops
    got = []
    monkeypatch.setattr(ops, "_launch", lambda name, blob, device: got.append(name))
    monkeypatch.setattr(ops, "_same_device", lambda *a, **kw: None)
    return got


def test_rope_of_one_side_without_heads_still_launches(launches):
    from ironcortex_amd.hip import ops
    x, none = torch.randn(2, 3, 5, 8), torch.randn(2, 0, 5, 8)
    f, w = torch.ones(4), torch.ones(8)
    for q, k in ((x, none), (none, x)):
        for n, call in enumerate((lambda: ops.rope(q, k, freqs=f), lambda: ops.qk_norm_rope(q, k, w, w, freqs=f))):
            a, b = call()
            assert launches == ["ic_rope_fwd"], n
            assert a.shape == q.shape and b.shape == k.shape
            launches.clear()
    for shape in ((0, 3, 5, 8), (2, 3, 0, 8)):
        e = torch.randn(shape)
        ops.rope(e, e, freqs=f)
        ops.qk_norm_rope(e, e, w, w, freqs=f)
        ops.rope(none, freqs=f)
    assert launches == []


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
def test_rope_of_one_side_without_heads(norm):
    """The same rows and gradients as beside rows of the other side; the absent side's weight gets a zero gradient."""
    from ironcortex_amd.hip import ops
    g = torch.Generator(device=DEV).manual_seed(3)
    f = 10000.0 ** (-torch.arange(8, device=DEV, dtype=torch.float64) / 8)
    x, other = (torch.randn(2, h, 37, 24, generator=g, device=DEV, requires_grad=True) for h in (3, 2))
    none = torch.randn(2, 0, 37, 24, device=DEV, requires_grad=True)
    w = [torch.rand(24, generator=g, device=DEV).requires_grad_(True) for _ in (0, 1)]
    go = torch.randn(2, 3, 37, 24, generator=g, device=DEV)
    call = (lambda q, k: ops.qk_norm_rope(q, k, *w, freqs=f, layout="half", scale=1.5)) if norm else (lambda q, k: ops.rope(q, k, freqs=f, layout="half", scale=1.5))
    for at in (0, 1):
        place = lambda side: (x, side) if at == 0 else (side, x)  # noqa: E731
        want, got = call(*place(other)), call(*place(none))
        leaves = [x] + ([w[at]] if norm else [])
        assert torch.equal(want[at].detach(), got[at].detach()) and got[1 - at].shape == none.shape
        a, b = (torch.autograd.grad(y[at], leaves, go) for y in (want, got))
        assert torch.equal(a[0], b[0])
        if norm:  # other partial sums of the same 222 terms h xhat: either is off by 222 roundings of the terms' sizes at most
            xhat = x.detach() / x.detach().square().mean(-1, keepdim=True).sqrt()
            turned = 1.5 * (go[..., :8].abs() + go[..., 8:16].abs())
            size = (torch.cat((turned, turned, go[..., 16:].abs()), -1) * xhat.abs()).sum((0, 1, 2))
            assert bool(((a[1] - b[1]).abs() <= 2 * 222 * 2.0 ** -24 * size).all())
        if norm:
            gw, = torch.autograd.grad(call(*place(none))[1 - at].sum(), w[1 - at])
            assert float(gw.abs().max()) == 0.0
        with torch.no_grad():
            assert torch.equal(call(*place(none))[at], got[at].detach())


def far_apart(device, which):
    """Inputs whose outputs or gradients would lie 2^22 elements and more from position to position in their usual order."""
    g = torch.Generator(device=device).manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    if which == "many heads":  # H * Dv = 2^22
        return r(1, 3, 1 << 16, 2).transpose(1, 2), r(1, 3, 1 << 16, 2).transpose(1, 2), r(1, 3, 1, 64).transpose(1, 2).expand(1, 1 << 16, 3, 64)
    if which == "one position":  # H * Dk = 2^22, a view whose only position has that stride
        return r(1, 1, 1 << 16, 64).transpose(1, 2), r(1, 1, 1, 64).transpose(1, 2), r(1, 1, 1, 2).transpose(1, 2)
    # keys of one sequence shown to all: their gradient's dense order has the sequences inside the positions
    k = r(1, 3, 64, 128).transpose(1, 2).expand(512, 64, 3, 128)
    return r(512, 3, 64, 128).transpose(1, 2), k, r(512, 3, 64, 1).transpose(1, 2)


FAR = ["many heads", "one position", "shared keys"]


@pytest.mark.parametrize("which", FAR)
def test_linear_attention_lays_out_what_it_makes_within_its_own_limits(which, monkeypatch):
    from ironcortex_amd import hip
    from ironcortex_amd.hip import ops
    got = []

    def launch(name, blob, device):
        a = hip.CLASSES["ic_lattn_args" if name == "ic_lattn_fwd" else "ic_lattn_bwd_args"].from_buffer_copy(blob)
        f = a.f if name == "ic_lattn_bwd" else a
        got.extend([f.q_st, f.k_st, f.v_st] + ([f.o_st] if f is a else [a.do_st, a.dq_st, a.dk_st, a.dv_st]))

    monkeypatch.setattr(ops, "_launch", launch)
    monkeypatch.setattr(ops, "_same_device", lambda *a, **kw: None)
    q, k, v = (x.detach().requires_grad_(True) for x in far_apart("cpu", which))
    H = q.shape[1]
    o, _ = ops.linear_attention(q, k, v, torch.ones(H))
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), torch.ones(o.shape))
    assert len(got) == 11 and all(0 <= s < ops.LATTN_MAX_STRIDE for s in got), got
    assert all(x.numel() == 1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride())) for x in (o, dq, dk, dv))  # dense


@pytest.mark.gpu
@pytest.mark.parametrize("which", FAR)
def test_linear_attention_of_rows_far_apart_equals_a_piece_of_them(which):
    """A few heads (sequences) of such a call give the same rows and gradients as in a call of their own."""
    from ironcortex_amd.hip import ops
    q, k, v = (x.detach().requires_grad_(True) for x in far_apart(DEV, which))
    B, H, T, _ = q.shape
    rate = torch.rand(H, device=DEV) * 0.5
    o, s = ops.linear_attention(q, k, v, rate)
    go = torch.randn(o.shape, device=DEV)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), go)
    nb, nh = (2, H) if B > 1 else (1, 5)
    qs = q.detach()[:nb, H - nh:].clone().requires_grad_(True)
    ks, vs = (x.detach()[:nb, -min(nh, x.shape[1]):].clone().requires_grad_(True) for x in (k, v))
    o2, s2 = ops.linear_attention(qs, ks, vs, rate[H - nh:])
    assert torch.equal(o[:nb, H - nh:].detach(), o2.detach()) and torch.equal(s[:nb, H - nh:].detach(), s2.detach())
    dq2, dk2, dv2 = torch.autograd.grad(o2, (qs, ks, vs), go[:nb, H - nh:])
    assert torch.equal(dq[:nb, H - nh:], dq2)
    if k.shape[1] == H:
        assert torch.equal(dk[:nb, H - nh:], dk2) and torch.equal(dv[:nb, H - nh:], dv2)
    else:  # gradients of a head shared by all: every query head adds to them
        want = (q.detach().double() * (go.double() * v.detach().double()).sum(-1, keepdim=True)).sum(1, keepdim=True)  # (one position)
        size = (q.detach().double() * (go.double() * v.detach().double()).sum(-1, keepdim=True)).abs().sum(1, keepdim=True)
        # a sum over H heads, one rounding each, grows like its root: 4 sqrt(H) u of the sizes
        assert bool(((dk.double() - want).abs() <= 4 * H ** 0.5 * 2.0 ** -24 * size).all())


def masked_mixer(seed=0):
    """A mixer whose context mask takes the plain [T,T] attention behind the rotation; x [2,9,32]; the mask."""
    from ironcortex_amd.mixer import IronRoPESelfAttention
    torch.manual_seed(seed)
    m = IronRoPESelfAttention(32, 2, 64, rope_m=6, fb_m=4).to(DEV)
    x = torch.randn(2, 9, 32, device=DEV)
    mask = torch.ones(2, 9, dtype=torch.bool, device=DEV)
    mask[:, 7:] = False
    return m, x, mask


def plain_rotation(monkeypatch):
    from ironcortex_amd.hip import ops
    monkeypatch.setattr(ops, "ROPE_MAX_D", 0)  # (no row is narrow enough for the kernel)


@pytest.mark.gpu
def test_mixer_hands_tangents_on(monkeypatch):
    import torch.autograd.forward_ad as fw
    m, x, mask = masked_mixer()
    t = torch.randn_like(x)

    def jvp():
        with torch.no_grad(), fw.dual_level():
            return fw.unpack_dual(m(fw.make_dual(x, t), context_mask=mask)).tangent

    got = jvp()
    plain_rotation(monkeypatch)
    assert torch.equal(got, jvp())


@pytest.mark.gpu
def test_mixer_under_torch_func_equals_the_plain_rotation(monkeypatch):
    from ironcortex_amd.mixer import rotate_qk
    g = torch.Generator(device=DEV).manual_seed(2)
    q, k, dq = (torch.randn(3, 2, 5, 8, generator=g, device=DEV) for _ in range(3))
    th = torch.rand(3, 5, 4, generator=g, device=DEV)
    c, s = torch.cos(th), torch.sin(th)
    turn = lambda a: rotate_qk(a, k, c, s)[0]  # noqa: E731
    one = lambda a, b: rotate_qk(a.unsqueeze(0), b.unsqueeze(0), c[:1], s[:1])[0][0]  # noqa: E731
    calls = (lambda: torch.func.grad(lambda a: turn(a).sin().sum())(q), lambda: torch.func.jvp(turn, (q,), (dq,)),
             lambda: torch.func.vmap(one)(q, k), lambda: torch.func.hessian(lambda a: turn(a)[0, 0, 0].sin().sum())(q))
    got = [f() for f in calls]
    plain_rotation(monkeypatch)
    for a, f in zip(got, calls):
        assert all(torch.equal(x, y) for x, y in zip(a, f()))


@pytest.mark.gpu
def test_mixer_traces_record_the_rotation():
    from torch.fx.experimental.proxy_tensor import make_fx
    from ironcortex_amd.mixer import rotate_qk
    g = torch.Generator(device=DEV).manual_seed(2)
    q, k, q2 = (torch.randn(3, 2, 5, 8, generator=g, device=DEV) for _ in range(3))
    th = torch.rand(3, 5, 4, generator=g, device=DEV)
    f = lambda a, b: rotate_qk(a, b, torch.cos(th), torch.sin(th))  # noqa: E731
    want = f(q2, k)
    fake = torch._subclasses.FakeTensorMode(allow_non_fake_inputs=True)
    for h in (torch.jit.trace(f, (q, k), check_trace=False), make_fx(f)(q, k), make_fx(f, tracing_mode="fake", _allow_non_fake_inputs=True)(q, k),
              make_fx(f, pre_dispatch=True)(q, k), torch.compile(f, backend="eager", fullgraph=True)):
        got = h(q2, k)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with fake:
        y, _ = f(fake.from_tensor(q), fake.from_tensor(k))
    assert y.shape == q.shape and y.device == q.device
    m, x, mask = masked_mixer()
    with torch.no_grad():
        m.requires_grad_(False)
        h = torch.jit.trace(lambda a: m(a, context_mask=mask), x, check_trace=False)
        x2 = torch.randn_like(x)
        assert torch.equal(h(x2), m(x2, context_mask=mask))


def test_operators_refuse_traces_transforms_and_dual_numbers(launches):
    import torch.autograd.forward_ad as fw
    from torch.fx.experimental.proxy_tensor import make_fx
    from ironcortex_amd.hip import ops
    x, w, r, st, f = torch.randn(2, 3, 5, 8), torch.ones(8), torch.ones(3), torch.zeros(2, 3, 8, 8), torch.ones(4)
    table = torch.ones(5, 4)
    calls = [lambda a: ops.rope(a, freqs=f), lambda a: ops.rope(x, a, freqs=f)[1], lambda a: ops.qk_norm_rope(a, x, w, w, freqs=f)[0],
             lambda a: ops.linear_attention(a, x, x, r)[0], lambda a: ops.linear_attention_step(a[:, :, 0], x[:, :, 0], x[:, :, 0], r, st)]
    with torch.no_grad():
        for i, f_ in enumerate(calls):
            for go in (lambda: torch.jit.trace(f_, x, check_trace=False), lambda: make_fx(f_)(x), lambda: make_fx(f_, pre_dispatch=True)(x),
                       lambda: torch.func.vmap(f_)(torch.stack((x, x))), lambda: torch.func.jvp(f_, (x,), (x,)), lambda: torch.func.grad(lambda a: f_(a).sum())(x)):
                with pytest.raises(RuntimeError, match="cannot be used|no gradients"):
                    go()
        with fw.dual_level():
            dual = fw.make_dual
            for f_ in calls + [lambda a: ops.qk_norm_rope(x, x, w, a[0, 0, 0], freqs=f)[0], lambda a: ops.linear_attention(x, x, x, a[0, :, 0, 0])[0],
                               lambda a: ops.linear_attention(x, x, x, r, state=a[:, :, :1].expand(2, 3, 8, 8))[0], lambda a: ops.rope(x, cos=a[0, 0, :, :4], sin=table),
                               lambda a: ops.rope(x, freqs=a[0, 0, 0, :4])]:
                with pytest.raises(RuntimeError, match="cannot be used"):
                    f_(dual(x, x))
            assert launches == []
            ops.rope(x, freqs=f)  # (a level without a tangent)
    assert launches == ["ic_rope_fwd"]


@pytest.mark.gpu
@pytest.mark.parametrize("tables", [False, True])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_derivatives_of_second_and_third_order(layout, tables):
    """y = R x: the gradient of sum(y^3) is 3 R^T y^2, along u its derivative is 6 R^T (y R u), and so on."""
    from ironcortex_amd.hip import ops
    g = torch.Generator(device=DEV).manual_seed(6)
    q, k = (torch.randn(2, 21, h, 16, generator=g, device=DEV).transpose(1, 2).requires_grad_(True) for h in (3, 1))
    u = torch.randn(2, 3, 21, 16, generator=g, device=DEV)
    pos, f = torch.randint(0, 1000, (2, 21), generator=g, device=DEV), torch.rand(6, generator=g, device=DEV)
    th = pos.unsqueeze(-1).double() * f.double()
    c, s = torch.cos(th).float(), torch.sin(th).float()
    kw = dict(cos=c, sin=s) if tables else dict(positions=pos, freqs=f)

    def R(x, sign):
        cc, ss = (c.double().unsqueeze(1) * 1.25, s.double().unsqueeze(1) * 1.25 * sign) if tables else (torch.cos(th).unsqueeze(1) * 1.25, torch.sin(th).unsqueeze(1) * 1.25 * sign)
        a, b = (x[..., :6], x[..., 6:12]) if layout == "half" else (x[..., 0:12:2], x[..., 1:12:2])
        ra, rb = a * cc - b * ss, a * ss + b * cc
        return torch.cat((torch.cat((ra, rb), -1) if layout == "half" else torch.stack((ra, rb), -1).flatten(-2), x[..., 12:]), -1)

    y, yk = ops.rope(q, k, layout=layout, scale=1.25, **kw)
    g1, gk = torch.autograd.grad(y.pow(3).sum() + yk.pow(3).sum(), (q, k), create_graph=True)
    g2, = torch.autograd.grad((g1 * u).sum(), q, create_graph=True)
    g3, = torch.autograd.grad((g2 * u).sum(), q)
    yd, ud = R(q.detach().double(), 1), R(u.double(), 1)
    # chains of at most five rotations and four products, 6u of |a| + |b| each: 64 u of the largest value there
    for got, want in ((g1, 3 * R(yd.square(), -1)), (g2, 6 * R(yd * ud, -1)), (g3, 6 * R(ud * ud, -1)), (gk, 3 * R(R(k.detach().double(), 1).square(), -1))):
        assert got.shape == want.shape and float((got.detach().double() - want).abs().max()) <= 64 * 2.0 ** -24 * float(want.abs().max())
    assert g2.stride() == q.stride()  # (laid out like its input)


@pytest.mark.gpu
def test_mixer_second_derivative_equals_the_plain_rotations(monkeypatch):
    m, x, mask = masked_mixer()
    x.requires_grad_(True)

    def twice():
        g, = torch.autograd.grad(m(x, context_mask=mask).sin().sum(), x, create_graph=True)
        return torch.autograd.grad(g.square().sum(), [x, *m.parameters()], allow_unused=True)

    got = twice()
    plain_rotation(monkeypatch)
    for a, b in zip(got, twice()):  # the same products, some sums in another order
        assert (a is None) == (b is None) and (a is None or float((a - b).abs().max()) <= 64 * 2.0 ** -24 * float(b.abs().max().clamp_min(1.0)))


@pytest.mark.gpu
@pytest.mark.parametrize("tables", [False, True])
def test_rope_backward_of_batched_and_dual_gradients(tables):
    """Gradients under vmap (a vectorised Jacobian) and with tangents: those of the gradients one by one."""
    import torch.autograd.forward_ad as fw
    from ironcortex_amd.hip import ops
    g = torch.Generator(device=DEV).manual_seed(8)
    q, k = (torch.randn(2, h, 7, 16, generator=g, device=DEV, requires_grad=True) for h in (2, 1))
    f = torch.rand(4, generator=g, device=DEV)
    th = torch.arange(7, device=DEV).unsqueeze(-1) * f
    kw = dict(cos=torch.cos(th), sin=torch.sin(th)) if tables else dict(freqs=f)
    y = ops.rope(q, k, **kw)
    gos = [torch.randn(3, *t.shape, generator=g, device=DEV) for t in y]
    one = [torch.autograd.grad(y, (q, k), [t[i] for t in gos], retain_graph=True) for i in range(3)]
    many = torch.autograd.grad(y, (q, k), gos, is_grads_batched=True, retain_graph=True)
    close = lambda a, b: float((a - b).abs().max()) <= 16 * 2.0 ** -24 * float(b.abs().max())  # noqa: E731  (two evaluations, 6u of |a| + |b| each)
    for i in range(3):
        assert close(many[0][i], one[i][0]) and close(many[1][i], one[i][1])
    with fw.dual_level():
        d = torch.autograd.grad(y, (q, k), [fw.make_dual(t[0], t[1]) for t in gos])
        assert all(close(fw.unpack_dual(a).primal, p) and close(fw.unpack_dual(a).tangent, t) for a, p, t in zip(d, one[0], one[1]))


def test_backward_refuses_dual_gradients(launches):
    """Norms and linear attention hand no tangent on in their backward either."""
    import torch.autograd.forward_ad as fw
    from ironcortex_amd.hip import ops
    x, w = torch.randn(2, 3, 5, 8, requires_grad=True), torch.ones(8)
    go = torch.randn(2, 3, 5, 8)
    for call in (lambda: ops.qk_norm_rope(x, x, w, w, freqs=torch.ones(4))[0], lambda: ops.linear_attention(x, x, x, torch.ones(3))[0]):
        y = call()
        with fw.dual_level():
            dual = fw.make_dual(go, go)
            with pytest.raises(RuntimeError, match="cannot be used on dual numbers"):
                torch.autograd.grad(y, x, dual, retain_graph=True)
        torch.autograd.grad(y, x, go)
    assert len(launches) == 4


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["rope tables", "rope", "norm", "linear"])
def test_saved_tensors_may_come_back_in_another_layout(which):
    """Hooks for saved tensors keep values and shapes; the memory's order is theirs (here: the dimensions reversed)."""
    from ironcortex_amd.hip import ops
    g = torch.Generator(device=DEV).manual_seed(9)
    q, k, v = (torch.randn(2, h, 70, 16, generator=g, device=DEV, requires_grad=True) for h in (4, 2, 2))
    w = [torch.rand(16, generator=g, device=DEV).requires_grad_(True) for _ in (0, 1)]
    rate, st = torch.rand(4, generator=g, device=DEV).requires_grad_(True), torch.randn(2, 4, 16, 16, generator=g, device=DEV, requires_grad=True)
    pos, f = torch.randint(0, 500, (2, 70), generator=g, device=DEV), torch.rand(6, generator=g, device=DEV)
    th = pos.unsqueeze(-1) * f
    kw = dict(cos=torch.cos(th), sin=torch.sin(th)) if which == "rope tables" else dict(positions=pos, freqs=f)
    run = {"norm": lambda: (ops.qk_norm_rope(q, k, *w, **kw), [q, k, *w]),
           "linear": lambda: (ops.linear_attention(q, k, v, rate, state=st, valid_len=torch.tensor([70, 33], device=DEV)), [q, k, v, rate, st])}.get(
               which, lambda: (ops.rope(q, k, **kw), [q, k]))

    def grads():
        y, leaves = run()
        return torch.autograd.grad([t.sin().sum() for t in y], leaves)

    want = grads()
    turned = lambda t: t.detach().permute(*reversed(range(t.dim()))).contiguous().permute(*reversed(range(t.dim())))  # noqa: E731
    with torch.autograd.graph.saved_tensors_hooks(turned, lambda t: t):
        got = grads()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_attention_of_no_positions_passes_gradients_on(dtype, launches):
    """The state as it came, its gradient with it, and zeros for everything else, as from a call with positions."""
    from ironcortex_amd.hip import ops
    for B, H, T in ((2, 3, 0), (0, 3, 5), (2, 0, 5)):
        q, k, v = (torch.randn(B, H, T, 8, dtype=dtype).requires_grad_(True) for _ in range(3))
        rate, st = torch.full((H,), float("inf"), requires_grad=True), torch.randn(B, H, 8, 8, requires_grad=True)
        for state in (st, None):
            o, s = ops.linear_attention(q, k, v, rate, state=state)
            assert o.shape == (B, H, T, 8) and o.dtype == dtype and s.dtype == torch.float32
            assert torch.equal(s, torch.zeros_like(st) if state is None else st) and (state is None or s.data_ptr() != st.data_ptr() or not s.numel())
            leaves = [q, k, v, rate] + ([] if state is None else [st])
            for y in (o, s):
                got = torch.autograd.grad(y.float().sum(), leaves, retain_graph=True, allow_unused=True)
                for x, gx in zip(leaves, got):
                    assert torch.equal(torch.zeros_like(x) if gx is None else gx, torch.ones_like(st) if x is st and y is s else torch.zeros_like(x))
                assert got[3] is not None
    assert launches == []


def compiled_calls(device):
    from ironcortex_amd.hip import ops
    f, w, r, st = torch.ones(4, device=device), torch.ones(8, device=device), torch.ones(3, device=device), torch.zeros(2, 3, 8, 8, device=device)

    def step(q):
        with torch.no_grad():
            return ops.linear_attention_step(q[:, :, 0], q[:, :, 1], q[:, :, 2], r, st.clone()) * 2

    return {"rope": lambda q: ops.rope(q, freqs=f) * 2, "norm": lambda q: ops.qk_norm_rope(q, q, w, w, freqs=f)[0] * 2,
            "linear": lambda q: ops.linear_attention(q, q, q, r)[0] * 2, "step": step}


@pytest.mark.parametrize("which", ["rope", "norm", "linear", "step"])
@pytest.mark.parametrize("grad", [False, True])
def test_compiled_programs_leave_their_graph_for_a_launch(which, grad, launches):
    x = torch.randn(2, 3, 5, 8, requires_grad=grad)
    torch._dynamo.reset()
    y = torch.compile(compiled_calls("cpu")[which], backend="eager")(x)
    if y.requires_grad:
        y.sum().backward()
    assert len(launches) == (2 if grad and which != "step" else 1)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["rope", "norm", "linear", "step"])
def test_compiled_programs_give_the_same(which):
    x = torch.randn(2, 3, 5, 8, device=DEV, requires_grad=True)
    f = compiled_calls(DEV)[which]
    want = f(x)
    torch._dynamo.reset()
    got = torch.compile(f, backend="eager")(x)
    assert torch.equal(got, want) and got.requires_grad == want.requires_grad == (which != "step")
    if which != "step":
        assert torch.equal(*(torch.autograd.grad(y.sin().sum(), x)[0] for y in (got, want)))
