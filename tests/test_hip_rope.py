"""Rotary positions and per-head norms of queries and keys (ops.rope, ops.qk_norm_rope; csrc/rope.hip) against the formulas in
64 bits.  Every bound is elementwise and counts roundings, u = 2^-24 each in fp32 arithmetic:
  an angle's cos / sin: reduced exactly in 64 bits, one rounding of the reduced angle (<= u), the function itself (<= 2u: one
  unit in the last place), the factor `scale` (u): 4u of `scale`;
  y = a c - b s: 4u from c (s), u per product, u for the difference: 6u (|a| + |b|) scale;
  u_ = w x / sqrt(mean x^2 + eps): a sum of D squares (<= D u, half of it under the root), the division by D, + eps, the
  root, the reciprocal and two products: (D/2 + 6) u relative;
then one rounding to the rows' type (finfo.eps / 2 relative; below the smallest normal number of the type half its spacing)."""
import ctypes
import math

import pytest
import torch

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def ref_angles(B, T, cos=None, sin=None, positions=None, freqs=None, scale=1.0):
    if cos is not None:
        c, s = cos.double(), sin.double()
        c, s = (x.expand(B, *x.shape[-2:]) if x.dim() == 3 else x.unsqueeze(0).expand(B, -1, -1) for x in (c, s))
    else:
        p = torch.arange(T, device=freqs.device) if positions is None else positions
        p = (p if p.dim() == 2 else p.unsqueeze(0)).expand(B, T).double()
        ang = p.unsqueeze(-1) * freqs.double()
        c, s = torch.cos(ang), torch.sin(ang)
    return (c * scale).unsqueeze(1), (s * scale).unsqueeze(1)


def pairs(x, m, layout):
    return (x[..., 0:2 * m:2], x[..., 1:2 * m:2]) if layout == "interleaved" else (x[..., :m], x[..., m:2 * m])


def ref_rotate(x, c, s, layout):
    m = c.shape[-1]
    a, b = pairs(x, m, layout)
    y = x.clone()
    ya, yb = pairs(y, m, layout)
    ya.copy_(a * c - b * s)
    yb.copy_(a * s + b * c)
    return y


def ref_size(x, c, layout, scale):
    """|a| + |b| times scale on the rotated channels, |x| on the others: what the rotation's errors are relative to."""
    m = c.shape[-1]
    y = x.abs()
    a, b = pairs(x.abs(), m, layout)
    t = (a + b) * scale
    ya, yb = pairs(y, m, layout)
    ya.copy_(t)
    yb.copy_(t)
    return y


def within(got, want, bound, what):
    got = got.double()
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), what
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float(((got - want).abs() / bound.clamp_min(1e-300)).max()):.2f} of its bound"


def half_step(y, dt):
    f = torch.finfo(dt)
    return y.abs() * (f.eps / 2) + f.tiny * f.eps / 2


def rows(g, dt, B, H, T, D, how):
    """[B,H,T,D] rows lying in memory as callers have them."""
    if how == "fused":  # a view into a fused projection [B,T,3,H,D]
        return torch.randn(B, T, 3, H, D, generator=g, device=DEV).to(dt)[:, :, 1].transpose(1, 2)
    if how == "tokens":  # [B,T,H,D]
        return torch.randn(B, T, H, D, generator=g, device=DEV).to(dt).transpose(1, 2)
    if how == "odd":  # rows that start one element off
        return torch.randn(B, H, T, D + 1, generator=g, device=DEV).to(dt)[..., 1:]
    if how == "channels":  # channels not side by side
        return torch.randn(B, H, D, T, generator=g, device=DEV).to(dt).transpose(2, 3)
    if how == "shared":  # one head's rows shown to all heads
        return torch.randn(B, 1, T, D, generator=g, device=DEV).to(dt).expand(B, H, T, D)
    return torch.randn(B, H, T, D, generator=g, device=DEV).to(dt)


SIZES = [  # B, T, H, Hk, D, m, how the rows lie
    (1, 1, 1, 1, 64, 32, "dense"), (2, 5, 3, 1, 64, 32, "fused"), (1, 130, 4, 2, 80, 40, "tokens"), (2, 7, 2, 2, 33, 10, "dense"),
    (1, 3, 1, 1, 512, 256, "tokens"), (3, 17, 5, 1, 128, 32, "fused"), (1, 2, 1, 1, 1, 0, "dense"), (2, 9, 20, 4, 96, 20, "tokens"),
    (2, 33, 4, 4, 64, 32, "odd"), (2, 6, 3, 3, 64, 16, "channels"), (2, 11, 4, 2, 32, 8, "shared"), (64, 1, 16, 4, 128, 64, "tokens"),
    (1, 700, 2, 1, 8, 4, "tokens"), (2, 40, 3, 2, 200, 96, "fused"), (1, 5, 2, 1, 510, 255, "dense"), (1, 4, 1, 1, 7, 3, "fused"),
]
ANGLES = ["arange", "int32", "each", "far", "table", "tables"]


def angles(g, kind, B, T, m):
    f = 10000.0 ** (-torch.arange(m, device=DEV, dtype=torch.float64) / max(m, 1))
    if kind == "arange":
        return dict(freqs=f.float())
    if kind == "int32":
        return dict(freqs=f, positions=torch.randint(-50, 5000, (T,), generator=g, device=DEV, dtype=torch.int32))
    if kind == "each":
        return dict(freqs=f.float(), positions=torch.randint(0, 100000, (B, T), generator=g, device=DEV))
    if kind == "far":  # positions beyond what 32 bits hold; angles up to 2^23 (64 bits keep them to 2^-30, far below u)
        return dict(freqs=f.float() / 1024, positions=(1 << 33) + torch.randint(0, 1 << 20, (B, T), generator=g, device=DEV))
    shape = (T, m) if kind == "table" else (B, T, m)
    a = torch.rand(*shape, generator=g, device=DEV) * 6.3
    return dict(cos=torch.cos(a), sin=torch.sin(a))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_rope_and_norm_forward_backward(i, dtype):
    from ironcortex_amd.hip import ops
    B, T, H, Hk, D, m, how = SIZES[i]
    dt = TYPES[dtype]
    for layout, norm in (("interleaved", False), ("half", True), ("interleaved", True), ("half", False)):
        kind = ANGLES[(i + 2 * norm + 3 * (layout == "half")) % len(ANGLES)]
        g = torch.Generator(device=DEV).manual_seed(1000 * i + 10 * norm + (layout == "half"))
        q, k = rows(g, dt, B, H, T, D, how).requires_grad_(True), rows(g, dt, B, Hk, T, D, how).requires_grad_(True)
        kw = angles(g, kind, B, T, m)
        scale = 1.0 if i % 2 else 1.2079441541679836  # (the kernel takes it in fp32)
        scale = float(torch.tensor(scale))
        gq, gk = torch.randn(B, H, T, D, generator=g, device=DEV).to(dt), rows(g, dt, B, Hk, T, D, "tokens")
        wdt = torch.float32 if i % 3 else dt
        w = [(1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(wdt).requires_grad_(True) for _ in (0, 1)]
        eps = float(torch.tensor(1e-5))
        if norm:
            got = ops.qk_norm_rope(q, k, *w, eps=eps, layout=layout, scale=scale, **kw)
            grads = torch.autograd.grad(got, (q, k, *w), (gq, gk))
        else:
            got = ops.rope(q, k, layout=layout, scale=scale, **kw)
            grads = torch.autograd.grad(got, (q, k), (gq, gk))
        c, s = ref_angles(B, T, scale=scale, **kw)
        for j, (x, y, go) in enumerate(((q, got[0], gq), (k, got[1], gk))):
            what = f"{SIZES[i]} {dtype} {layout} norm={norm} {kind} {'qk'[j]}"
            assert y.is_contiguous() and y.dtype == dt
            xd, god = x.detach().double(), go.double()
            h = ref_rotate(god, c, -s, layout)  # the transposed rotation
            hsize = ref_size(god, c, layout, scale)
            if norm:
                wd = w[j].detach().double()
                inv = 1.0 / torch.sqrt(xd.square().mean(-1, keepdim=True) + eps)
                u = xd * inv * wd
                rel = (D / 2 + 6) * U
                xhat = xd * inv
                # gw: every term h xhat is off by 6u of hsize and (D/2 + 6)u of xhat, a sum of n terms by n u of their sizes
                gw, n = (h * xhat).sum((0, 1, 2)), B * x.shape[1] * T
                gb = (hsize * xhat.abs()).sum((0, 1, 2)) * (n + 6 + D / 2 + 6) * U
                within(grads[2 + j], gw, gb + half_step(gw.abs() + gb, wdt), what + " gw")
                mean = (wd * h * xhat).mean(-1, keepdim=True)
                msize = (wd.abs() * hsize * xhat.abs()).mean(-1, keepdim=True)
                gx = inv * (wd * h - xhat * mean)
                # w h: 6u + u; xhat mean: a sum of D terms (D u), its terms' own errors and two roots' worth of inv
                gxb = inv * (wd.abs() * hsize * 8 + xhat.abs() * msize * (2 * D + 24)) * U + gx.abs() * (D / 2 + 8) * U
            else:
                u, rel, gx, gxb = xd, 0.0, h, hsize * 6 * U
            want = ref_rotate(u, c, s, layout)
            b = ref_size(u, c, layout, scale) * (6 * U + rel)
            within(y, want, b + half_step(want.abs() + b, dt), what + " y")
            within(grads[j], gx, gxb + half_step(gx.abs() + gxb, dt), what + " gx")


@pytest.mark.gpu
def test_rope_gradient_equals_differences():
    """The gradients of a random projection of the outputs against central differences of the formulas in 64 bits."""
    from ironcortex_amd.hip import ops
    g = torch.Generator(device=DEV).manual_seed(5)
    B, H, T, D, m = 2, 3, 5, 16, 6
    q, k = (torch.randn(B, H, T, D, generator=g, device=DEV, requires_grad=True) for _ in (0, 1))
    w = [(1 + 0.3 * torch.randn(D, generator=g, device=DEV)).requires_grad_(True) for _ in (0, 1)]
    p = [torch.randn(B, H, T, D, generator=g, device=DEV) for _ in (0, 1)]
    f = 10000.0 ** (-torch.arange(m, device=DEV, dtype=torch.float64) / m)
    grads = torch.autograd.grad(ops.qk_norm_rope(q, k, *w, freqs=f, layout="half"), (q, k, *w), p)
    c, s = ref_angles(B, T, freqs=f)

    def loss(q_, k_, wq, wk):
        tot = 0.0
        for x, ww, pp in ((q_, wq, p[0]), (k_, wk, p[1])):
            tot = tot + (ref_rotate(x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5) * ww, c, s, "half") * pp.double()).sum()
        return tot

    base = [t.detach().double() for t in (q, k, *w)]
    for n in range(4):
        d = torch.randn(base[n].shape, generator=g, device=DEV).double()
        e = 1e-5
        hi, lo = list(base), list(base)
        hi[n], lo[n] = base[n] + e * d, base[n] - e * d
        num = float((loss(*hi) - loss(*lo)) / (2 * e))
        ana = float((grads[n].double() * d).sum())
        size = float((grads[n].double() * d).abs().sum())
        # 64-bit differences: e^2 times third derivatives (order 1e-9) plus cancellation 1e-16/1e-5; fp32 gradients: ~20 u of the sum
        assert abs(num - ana) <= 1e-6 * size + 1e-7, (n, num, ana)


@pytest.mark.gpu
def test_rope_rotates_like_the_mixers_plain_formulation_bit_for_bit():
    from ironcortex_amd.mixer import rope_rotate_pairs, rotate_qk
    g = torch.Generator(device=DEV).manual_seed(6)
    B, T, H, D, m = 3, 70, 4, 64, 32
    qkv = torch.randn(B, T, 3 * H * D, generator=g, device=DEV)
    th = torch.rand(B, T, m, generator=g, device=DEV) * 300
    c, s = torch.cos(th), torch.sin(th)
    res = []
    for own in (True, False):
        q, k, _ = (t.view(B, T, H, D).transpose(1, 2) for t in qkv.clone().requires_grad_(True).split(H * D, dim=2))
        out = rotate_qk(q, k, c, s) if own else tuple(rope_rotate_pairs(x, c.unsqueeze(1), s.unsqueeze(1), m) for x in (q, k))
        gr = torch.autograd.grad(out, (q, k), [torch.cos(o.detach() * 3) for o in out])
        res.append((*[o.detach() for o in out], *gr))
    assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("tables", [False, True])
def test_rope_backward_takes_the_saved_tensors_it_is_given(norm, tables):
    """Tensors saved for the backward may come back as others (hooks, recomputation): the forward's angles are gone by then."""
    from ironcortex_amd.hip import ops
    g = torch.Generator(device=DEV).manual_seed(21)
    B, H, T, D, m = 2, 3, 50, 32, 16
    q, k = (torch.randn(B, n, T, D, generator=g, device=DEV).requires_grad_(True) for n in (H, 1))
    w = [torch.rand(D, generator=g, device=DEV).requires_grad_(True) for _ in range(2)]
    go = [torch.randn(B, n, T, D, generator=g, device=DEV) for n in (H, 1)]
    leaves = [q, k] + (w if norm else [])

    def angles():
        if tables:
            a = torch.arange(T, device=DEV).view(1, T, 1) * torch.linspace(0.1, 1.0, m, device=DEV) + torch.arange(B, device=DEV).view(B, 1, 1)
            return dict(cos=torch.cos(a), sin=torch.sin(a))
        return dict(positions=torch.arange(B * T, device=DEV).view(B, T), freqs=torch.linspace(0.1, 1.0, m, device=DEV, dtype=torch.float64))

    def run():
        y = ops.qk_norm_rope(q, k, *w, **angles()) if norm else ops.rope(q, k, **angles())
        spoil = [torch.full((n,), float("nan"), device=DEV) for n in (B * T * m, B * T * m, 2 * B * T, 2 * m) for _ in range(4)]  # the angles' memory, reused
        return torch.autograd.grad(y, leaves, go), spoil

    want, _ = run()
    with torch.autograd.graph.save_on_cpu():
        got, _ = run()
    assert all(bool(torch.isfinite(a).all()) and torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_mixer_rotates_other_types_as_before():
    """Rows that promote with fp32 angles, fp64 rows, angles with a gradient: the plain formulation."""
    from ironcortex_amd.mixer import rope_rotate_pairs, rotate_qk
    th = torch.rand(2, 5, 4, device=DEV)
    for q, c in ((torch.randn(2, 3, 5, 8, device=DEV).bfloat16(), torch.cos(th)), (torch.randn(2, 3, 5, 8, device=DEV).double(), torch.cos(th).double()),
                 (torch.randn(2, 3, 5, 8, device=DEV), torch.cos(th).requires_grad_(True))):
        a, b = rotate_qk(q, q, c, c)
        w = rope_rotate_pairs(q, c.unsqueeze(1), c.unsqueeze(1), 4)
        assert a.dtype == w.dtype and torch.equal(a, w) and torch.equal(b, w) and a.requires_grad == w.requires_grad


@pytest.mark.gpu
def test_rope_other_stream_empty_rows_and_not_finite_rows():
    from ironcortex_amd.hip import ops
    f = torch.ones(4, device=DEV)
    q = torch.randn(2, 3, 5, 8, device=DEV)
    want = ops.rope(q, freqs=f)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = ops.rope(q, freqs=f)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want)
    for shape in ((0, 3, 5, 8), (2, 0, 5, 8), (2, 3, 0, 8)):
        e = torch.randn(shape, device=DEV, requires_grad=True)
        w = torch.ones(8, device=DEV, requires_grad=True)
        assert ops.rope(e, freqs=f).shape == shape
        a, b = ops.qk_norm_rope(e, e, w, w, freqs=f)
        (a.sum() + b.sum()).backward()
        assert a.shape == shape and float(w.grad.abs().sum()) == 0.0
    # a row of infinities or NaN stays one row's matter; channels that are not rotated keep them as they are
    x = torch.randn(1, 1, 3, 8, device=DEV)
    x[0, 0, 1, 7] = float("inf")
    x[0, 0, 2, 6] = float("nan")
    y = ops.rope(x, freqs=f[:2])
    assert torch.equal(torch.isfinite(y), torch.isfinite(x)) and float(y[0, 0, 1, 7]) == float("inf")
    w = torch.ones(8, device=DEV)
    y, _ = ops.qk_norm_rope(x, x, w, w, freqs=f[:2])
    assert bool(torch.isfinite(y[0, 0, 0]).all()) and bool(torch.isnan(y[0, 0, 2]).all())
    # rows of zeros: eps keeps the norm finite, forward and backward
    z = torch.zeros(1, 2, 3, 8, device=DEV, requires_grad=True)
    a, b = ops.qk_norm_rope(z, z, w, w, freqs=f)
    gz, = torch.autograd.grad(a.sum(), z)
    assert float(a.detach().abs().max()) == 0.0 and bool(torch.isfinite(gz).all())


@pytest.mark.gpu
def test_rope_only_one_output_used_and_gradients_from_a_sum():
    """The other output's gradient is zero; a gradient of all ones comes as an expanded tensor (strides 0)."""
    from ironcortex_amd.hip import ops
    f = torch.tensor([1.0, 0.1], device=DEV)
    q, k = (torch.randn(2, 2, 5, 8, device=DEV, requires_grad=True) for _ in (0, 1))
    w = torch.ones(8, device=DEV, requires_grad=True)
    yq, yk = ops.qk_norm_rope(q, k, w, w, freqs=f)
    yk.sum().backward()
    assert float(q.grad.abs().max()) == 0.0 and float(k.grad.abs().max()) > 0.0
    y = ops.rope(q, freqs=f)
    gq, = torch.autograd.grad(y.sum(), q)
    g1, = torch.autograd.grad(ops.rope(q, freqs=f), q, torch.ones_like(q))
    assert torch.equal(gq, g1)


@pytest.mark.gpu
def test_rope_in_a_captured_graph():
    from ironcortex_amd.hip import ops
    f = 10000.0 ** (-torch.arange(16, device=DEV, dtype=torch.float64) / 16)
    q, k = (torch.randn(2, 37, 3, 32, device=DEV).transpose(1, 2).requires_grad_(True) for _ in (0, 1))
    w = [torch.ones(32, device=DEV, requires_grad=True) for _ in (0, 1)]
    gq = torch.randn(2, 3, 37, 32, device=DEV)
    pos = torch.arange(37, device=DEV)

    def once():
        y = ops.qk_norm_rope(q, k, *w, freqs=f, positions=pos)
        return (*y, *torch.autograd.grad(y, (q, k, *w), (gq, gq)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for n in range(3):
        with torch.no_grad():
            q.copy_(torch.randn_like(q))
            pos.add_(11 * n)
        want = [t.clone() for t in once()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), n


@pytest.mark.gpu
def test_rope_refusals():
    from ironcortex_amd.hip import ops
    q = torch.randn(2, 3, 5, 8, device=DEV)
    f, w = torch.ones(4, device=DEV), torch.ones(8, device=DEV)
    t = torch.ones(5, 4, device=DEV)
    bad = [dict(), dict(freqs=f, cos=t, sin=t), dict(cos=t), dict(freqs=f, layout="pairs"), dict(freqs=torch.ones(5, device=DEV)),
           dict(freqs=f.half()), dict(freqs=f, positions=torch.zeros(5, device=DEV)), dict(freqs=f, positions=torch.zeros(3, 5, device=DEV, dtype=torch.int64)),
           dict(cos=t.half(), sin=t.half()), dict(cos=t, sin=t[:, :3]), dict(cos=t[:4], sin=t[:4]), dict(cos=t, sin=t, positions=torch.arange(5, device=DEV))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.rope(q, **kw)
    for a in ((q[0],), (q.double(),), (q, q.half()), (q, q[:, :, :4]), (torch.randn(1, 1, 2, 513, device=DEV),)):
        with pytest.raises(ValueError):
            ops.rope(*a, freqs=f)
    for ww in (w[:7], w.half(), w.view(1, 8)):
        with pytest.raises(ValueError):
            ops.qk_norm_rope(q, q, w, ww, freqs=f)
    with pytest.raises(RuntimeError):
        ops.rope(q, freqs=f.clone().requires_grad_(True))
    with pytest.raises(RuntimeError):
        ops.rope(q, freqs=f.cpu())
    # angles changed between forward and backward are noticed
    x = q.clone().requires_grad_(True)
    y = ops.rope(x, cos=t, sin=t)
    t.mul_(2.0)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_rope_refuses_cpu_tensors_and_bad_arguments_of_the_c_entry():
    from ironcortex_amd import hip
    from ironcortex_amd.hip import ops
    assert ops.ROPE_PARTS == hip.lib().ic_rope_parts()
    with pytest.raises(RuntimeError):
        ops.rope(torch.randn(1, 1, 2, 4), freqs=torch.ones(2))
    lib = hip.lib()
    good = dict(B=1, T=2, D=8, m=2, dtype=0, layout=0, freqs=8)

    def rc(fn="ic_rope_fwd", q=(1, 8, 8), **kw):
        a = hip.new("ic_rope_args", **{**good, **kw})
        a.q.H, a.q.x, a.q.y = q
        if fn == "ic_rope_bwd":
            a = hip.new("ic_rope_bwd_args", f=a)
        return getattr(lib, fn)(ctypes.byref(a), None), lib.ic_last_error().decode()

    for kw, text in ((dict(B=0), "B=0"), (dict(T=-1), "T=-1"), (dict(D=513), "D=513"), (dict(m=5), "m=5"), (dict(m=-1), "m=-1"), (dict(dtype=3), "dtype=3"),
                     (dict(layout=2), "layout=2"), (dict(freqs=None), "freqs"), (dict(cos=8), "cos"), (dict(cos=8, sin=8), "both"), (dict(q=(0, 8, 8)), "H=0"),
                     (dict(q=(1, None, 8)), "NULL"), (dict(q=(1, 8, None)), "NULL"), (dict(B=1 << 16, T=1 << 16), "B=65536"), (dict(fn="ic_rope_bwd"), "weight")):
        got, msg = rc(**kw)
        assert got == hip.ENUMS["IC_EINVAL"] and text in msg, (kw, msg)
    assert lib.ic_rope_fwd(None, None) == hip.ENUMS["IC_EINVAL"] and lib.ic_rope_bwd(None, None) == hip.ENUMS["IC_EINVAL"]


def test_rope_freqs():
    from ironcortex_amd.mixer import rope_freqs
    f, s = rope_freqs(8)
    assert f.dtype == torch.float64 and s == 1.0 and torch.allclose(f, 10000.0 ** (-torch.arange(8).double() / 8), rtol=1e-14)
    assert torch.equal(rope_freqs(8, scaling="linear", factor=4.0)[0], f / 4)
    b, _ = rope_freqs(8, scaling="base", factor=4.0)
    assert float(b[0]) == 1.0 and abs(float(b[-1] / f[-1]) - 0.25) < 1e-12 and bool((b <= f).all())
    r, s = rope_freqs(64, scaling="ramp", factor=4.0, trained_len=4096)
    n = rope_freqs(64)[0]
    assert torch.equal(r[0], n[0]) and abs(float(r[-1] / n[-1]) - 0.25) < 1e-12 and abs(s - 1 - 0.1 * math.log(4.0)) < 1e-12
    assert bool(((r <= n * (1 + 1e-12)) & (r >= n / 4 * (1 - 1e-12))).all()) and bool((r[1:] < r[:-1]).all())
    assert rope_freqs(1, scaling="base", factor=2.0)[0].shape == (1,)
    for kw in (dict(m=0), dict(m=4, factor=0.5), dict(m=4, scaling="ntk"), dict(m=4, scaling="ramp"), dict(m=4, scaling="ramp", trained_len=10, turns=(3.0, 2.0))):
        with pytest.raises(ValueError):
            rope_freqs(**kw)
