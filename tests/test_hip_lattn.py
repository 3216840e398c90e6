"""Linear attention with a decay for each head (ops.linear_attention, ops.linear_attention_step; csrc/lattn.hip) against the
recurrence in 64 bits, run position by position, and its gradients by autograd through that recurrence.

Bounds.  Every output is a sum of products; with A = the same computation on absolute values (64 bits), an fp32 evaluation is
off by at most A times the number of roundings along a term's path, u = 2^-24 each:
  q . k: Dk roundings, its decay factor (exp2 of a rounded exponent: the exponent's error |r lag| u is met by its own factor
  e^{-r lag}, at most u / e, plus one unit in the last place each for the factor and log2 e: 4u), the sum over a chunk (64),
  the sum over key channels of the state's part (Dk), the states' sums over chunks and segments (one fma each: T/64 + 64),
  the scale: N = Dk + Dv + 160 + T/64 roundings bound every path, forward and backward.
Rounding errors of sums grow like the root of their number (the terms' signs are random): 4 sqrt(N) u A is asserted, which
four standard deviations of N roundings of at most u each do not reach.  bf16 rows run through matrix instructions on operands split
into two bf16 parts (16 bits of each computed operand: 2^-17 of a term, two such operands on a path): 2^-16 A more.
Then one rounding to the rows' type."""
import ctypes
import math

import pytest
import torch

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def recurrence(q, k, v, rate, scale, state, valid):
    """Position by position, in the inputs' type (64 bits); padding rows give zeros and leave the state."""
    B, H, T, Dk = q.shape
    G = H // k.shape[1]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    S = torch.zeros(B, H, Dk, v.shape[-1], dtype=q.dtype, device=q.device) if state is None else state
    lam = torch.exp(-rate).view(1, H, 1, 1)
    outs = []
    for t in range(T):
        live = (valid > t).view(B, 1, 1, 1)
        kt, vt, qt = (torch.where(live[..., 0], x[:, :, t], torch.zeros((), dtype=x.dtype, device=x.device)) for x in (k, v, q))
        S = torch.where(live, lam * S + kt.unsqueeze(-1) * vt.unsqueeze(-2), S)
        outs.append(scale * (qt.unsqueeze(-2) @ S).squeeze(-2))
    return torch.stack(outs, 2), S


def bound(A, N, dt, y):
    f = torch.finfo(dt)
    mixed = 2.0 ** -16 * A if dt != torch.float32 else 0.0
    b = 4 * math.sqrt(N) * U * A + mixed
    return b + (y.abs() + b) * (f.eps / 2) + f.tiny * f.eps / 2


def within(got, want, b, what):
    assert got.shape == want.shape, what
    got = got.double()
    assert bool(torch.isfinite(got).all()), what + ": not finite"
    worst = float(((got - want).abs() / b.clamp_min(1e-300)).max()) if got.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of its bound, error {float((got - want).abs().max()):.2e}"


def inputs(g, dt, B, T, H, Hk, Dk, Dv, how):
    def rows(heads, D):
        if how == "heads":
            return torch.randn(B, heads, T, D, generator=g, device=DEV).to(dt)
        if how == "odd":
            return torch.randn(B, T, heads, D + 1, generator=g, device=DEV).to(dt)[..., 1:].transpose(1, 2)
        if how == "channels":
            return torch.randn(B, heads, D, T, generator=g, device=DEV).to(dt).transpose(2, 3)
        if how == "backwards":  # head-major in memory, the longest stride on t
            return torch.randn(T, heads, B, D, generator=g, device=DEV).to(dt).permute(2, 1, 0, 3)
        return torch.randn(B, T, heads, D, generator=g, device=DEV).to(dt).transpose(1, 2)
    return rows(H, Dk), rows(Hk, Dk), rows(Hk, Dv)


CASES = [  # B, T, H, Hk, Dk, Dv, how, state, valid
    (1, 1, 1, 1, 32, 32, "tokens", False, None), (2, 33, 4, 4, 32, 32, "tokens", True, None), (3, 64, 2, 1, 64, 64, "heads", True, [64, 0, 1]),
    (2, 65, 3, 3, 64, 64, "odd", False, [65, 64]), (1, 200, 4, 2, 128, 128, "tokens", True, None), (2, 130, 2, 2, 8, 128, "channels", True, [130, 77]),
    (2, 131, 2, 1, 80, 24, "tokens", False, [3, 131]), (1, 700, 2, 2, 64, 64, "backwards", True, None), (2, 300, 6, 2, 16, 100, "odd", True, [299, 128]),
    (1, 129, 1, 1, 1, 1, "tokens", True, None), (40, 70, 16, 16, 32, 32, "tokens", False, None), (4, 257, 128, 128, 8, 8, "tokens", True, [257, 256, 0, 200]),
    (1, 513, 3, 1, 33, 65, "heads", False, None), (1, 64, 8, 8, 128, 64, "tokens", True, None),
]
RATES = {"mixed": lambda g, H: torch.exp(torch.rand(H, generator=g, device=DEV) * math.log(5e4) + math.log(1e-4)),  # 1e-4 .. 5
         "none": lambda g, H: torch.zeros(H, device=DEV), "hard": lambda g, H: torch.full((H,), 60.0, device=DEV)}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("i", range(len(CASES)))
def test_linear_attention_forward_backward(i, dtype):
    from ironcortex_amd.hip import ops
    B, T, H, Hk, Dk, Dv, how, has_state, valid = CASES[i]
    dt = TYPES[dtype]
    g = torch.Generator(device=DEV).manual_seed(40 + i)
    q, k, v = (x.requires_grad_(True) for x in inputs(g, dt, B, T, H, Hk, Dk, Dv, how))
    rate = RATES[list(RATES)[0 if i % 4 else (1 + (i // 4) % 2)]](g, H).requires_grad_(True)
    state = torch.randn(B, H, Dk, Dv, generator=g, device=DEV).requires_grad_(True) if has_state else None
    scale = float(torch.tensor(Dk ** -0.5))
    vl = None if valid is None else torch.tensor(valid, device=DEV)
    n = torch.full((B,), T, device=DEV) if valid is None else vl
    go = torch.randn(B, H, T, Dv, generator=g, device=DEV).to(dt)
    gs = torch.randn(B, H, Dk, Dv, generator=g, device=DEV)
    with torch.no_grad():  # what lies in padded rows does not matter
        for x in (q, k, v, go):
            if valid is not None and how != "channels":
                x.masked_fill_((torch.arange(T, device=DEV) >= n.view(B, 1)).view(B, 1, T, 1), float("nan"))
    leaves = [x for x in (q, k, v, rate, state) if x is not None]
    got = ops.linear_attention(q, k, v, rate, scale=scale, state=state, valid_len=vl)
    grads = torch.autograd.grad(got, leaves, (go, gs))
    clean = lambda x: torch.nan_to_num(x.detach().double(), nan=0.0)  # noqa: E731
    ref = [clean(x).requires_grad_(True) for x in leaves]
    mag = [clean(x).abs().requires_grad_(True) for x in leaves]
    with torch.no_grad():
        mag[3].copy_(ref[3])
    st = lambda r: r[4] if has_state else None  # noqa: E731
    want = recurrence(*ref[:4], scale, st(ref), n)
    size = recurrence(*mag[:4], scale, st(mag), n)
    wg = torch.autograd.grad(want, ref, (clean(go), gs.double()), allow_unused=True)
    ag = torch.autograd.grad(size, mag, (clean(go).abs(), gs.double().abs()), allow_unused=True)
    N = Dk + Dv + 160 + T / 64
    what = f"{CASES[i]} {dtype}"
    within(got[0], want[0].detach(), bound(size[0].detach(), N, dt, want[0].detach()), what + " out")
    within(got[1], want[1].detach(), bound(size[1].detach(), N, torch.float32, want[1].detach()) + (2.0 ** -16 * size[1].detach() if dt != torch.float32 else 0), what + " state")
    assert got[0].dtype == dt and got[0].transpose(1, 2).is_contiguous()
    pad = (torch.arange(T, device=DEV) >= n.view(B, 1)).view(B, 1, T, 1)
    assert not bool((got[0] != 0).logical_and(pad).any()), what + " padded rows"
    for j, nm in enumerate(("q", "k", "v", "rate", "state")[:len(leaves)]):
        w = torch.zeros_like(ref[j].detach()) if wg[j] is None else wg[j]
        A = torch.zeros_like(ref[j].detach()) if ag[j] is None else ag[j].abs()
        # d rate sums B T (i, j) pairs: its partial sums are 64-bit, a chunk's are of at most 64 * 128 products
        M = N + 64 if nm == "rate" else N + 8 * (H // Hk)
        e = torch.float32 if nm in ("rate", "state") else dt
        b = bound(A, M, e, w) + (2.0 ** -16 * A if dt != torch.float32 else 0)
        within(grads[j], w, b, f"{what} d{nm}")
    # run-to-run identical
    again = ops.linear_attention(q, k, v, rate, scale=scale, state=state, valid_len=vl)
    ga = torch.autograd.grad(again, leaves, (go, gs))
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1]) and all(torch.equal(a, b) for a, b in zip(ga, grads))


@pytest.mark.gpu
def test_linear_attention_gradient_equals_differences():
    from ironcortex_amd.hip import ops
    g = torch.Generator(device=DEV).manual_seed(7)
    B, T, H, D = 2, 70, 2, 16
    q, k, v = (x.requires_grad_(True) for x in inputs(g, torch.float32, B, T, H, H, D, D, "tokens"))
    rate = torch.tensor([0.02, 0.4], device=DEV, requires_grad=True)
    state = torch.randn(B, H, D, D, generator=g, device=DEV, requires_grad=True)
    go, gs = torch.randn(B, H, T, D, generator=g, device=DEV), torch.randn(B, H, D, D, generator=g, device=DEV)
    leaves = [q, k, v, rate, state]
    grads = torch.autograd.grad(ops.linear_attention(q, k, v, rate, state=state), leaves, (go, gs))
    n = torch.full((B,), T, device=DEV)
    base = [x.detach().double() for x in leaves]

    def loss(x):
        o, s = recurrence(*x[:4], 1.0, x[4], n)
        return float((o * go.double()).sum() + (s * gs.double()).sum())

    for j in range(5):
        d = torch.randn(base[j].shape, generator=g, device=DEV).double()
        e = 1e-5
        hi, lo = list(base), list(base)
        hi[j], lo[j] = base[j] + e * d, base[j] - e * d
        num, ana = (loss(hi) - loss(lo)) / (2 * e), float((grads[j].double() * d).sum())
        size = float((grads[j].double() * d).abs().sum())
        # differences: 1e-10 times third derivatives (rate: up to T^3 of the loss's 1e4 terms), cancellation 1e-16 * 1e6 / 1e-5;
        # fp32 gradients: far below 1e-5 of the terms' sizes
        assert abs(num - ana) <= 1e-5 * size + 1e-4, (j, num, ana)


@pytest.mark.gpu
def test_linear_attention_long_rows_in_pieces_and_steps():
    """A prompt read in one call, in pieces of odd lengths with the state handed on, and its tail position by position."""
    from ironcortex_amd.hip import ops
    g = torch.Generator(device=DEV).manual_seed(8)
    B, T, H, Hk, D = 2, 4133, 4, 2, 64
    for dt in (torch.float32, torch.bfloat16):
        q, k, v = inputs(g, dt, B, T, H, Hk, D, D, "tokens")
        rate = torch.tensor([0.001, 0.01, 0.1, 1.0], device=DEV)
        whole, S = ops.linear_attention(q, k, v, rate, scale=0.125)
        st, parts, t = None, [], 0
        for n in (1, 63, 64, 65, 1000, 2923):
            o, st = ops.linear_attention(q[:, :, t:t + n], k[:, :, t:t + n], v[:, :, t:t + n], rate, scale=0.125, state=st)
            parts.append(o)
            t += n
        while t < T:
            parts.append(ops.linear_attention_step(q[:, :, t], k[:, :, t], v[:, :, t], rate, st, scale=0.125).unsqueeze(2))
            t += 1
        pieces = torch.cat(parts, 2)
        assert pieces.shape == whole.shape
        # two fp32 evaluations of the same sums (sizes: sqrt(1 / (2 rate)) * sqrt(D) ~ 180, u sqrt(N) of them each way), then the type's rounding
        rms = float(whole.float().square().mean().sqrt())
        eps = torch.finfo(dt).eps
        assert float((pieces.float() - whole.float()).abs().max()) <= 64 * (2.0 ** -20) * rms + 8 * rms * eps
        assert float((st - S).abs().max()) <= 2.0 ** -13 * float(S.square().mean().sqrt()) * (1 if dt == torch.float32 else 4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("B,H,Hk,Dk,Dv", [(1, 4, 4, 64, 64), (3, 6, 2, 80, 100), (65, 3, 1, 128, 128), (2, 2, 2, 1, 1), (1, 1, 1, 200, 33), (7, 16, 4, 32, 1024)])
def test_linear_attention_step(B, H, Hk, Dk, Dv, dtype):
    from ironcortex_amd.hip import ops
    dt = TYPES[dtype]
    g = torch.Generator(device=DEV).manual_seed(9)
    fused = torch.randn(B, H * Dk + Hk * (Dk + Dv), generator=g, device=DEV).to(dt)  # one projection's row for each sequence
    q, k, v = (x.view(B, -1, D) for x, D in zip(fused.split([H * Dk, Hk * Dk, Hk * Dv], dim=1), (Dk, Dk, Dv)))
    rate = torch.rand(H, generator=g, device=DEV)
    pool = torch.randn(B + 2, H, Dk, Dv, generator=g, device=DEV)
    before = pool.clone()
    active = torch.rand(B, generator=g, device=DEV) < 0.7 if B > 1 else None
    version = pool._version
    o = ops.linear_attention_step(q, k, v, rate, pool[1:B + 1], scale=0.5, active=active)
    assert pool._version > version
    on = torch.ones(B, dtype=torch.bool, device=DEV) if active is None else active
    kd, vd = (x.double().repeat_interleave(H // Hk, 1) for x in (k, v))
    S = before[1:B + 1].double()
    lam = torch.exp(-rate.double()).view(1, H, 1, 1)
    W = torch.where(on.view(B, 1, 1, 1), lam * S + kd.unsqueeze(-1) * vd.unsqueeze(-2), S)
    A = lam * S.abs() + (kd.unsqueeze(-1) * vd.unsqueeze(-2)).abs()
    # the decay factor (one unit in the last place and its rounded argument, at most u each), its product, the fma: 4u of the sizes
    within(pool[1:B + 1], W, 4 * U * A + 1e-300, "state")
    assert torch.equal(pool[0], before[0]) and torch.equal(pool[B + 1], before[B + 1])
    wo = torch.where(on.view(B, 1, 1), 0.5 * (q.double().unsqueeze(-2) @ W).squeeze(-2), torch.zeros((), device=DEV, dtype=torch.float64))
    so = 0.5 * (q.double().abs().unsqueeze(-2) @ A).squeeze(-2)
    f = torch.finfo(dt)
    b = (Dk + 6) * U * so  # a sum of Dk products
    within(o, wo, b + (wo.abs() + b) * f.eps / 2 + f.tiny * f.eps / 2, "out")


@pytest.mark.gpu
def test_linear_attention_other_stream_empty_and_extreme_rates():
    from ironcortex_amd.hip import ops
    g = torch.Generator(device=DEV).manual_seed(10)
    q, k, v = inputs(g, torch.float32, 2, 150, 3, 3, 32, 32, "tokens")
    rate = torch.tensor([0.0, 0.5, float("inf")], device=DEV)
    want = ops.linear_attention(q, k, v, rate)
    # an infinite rate forgets at once: only the position's own pair is left
    own = (q[:, 2] * k[:, 2]).sum(-1, keepdim=True) * v[:, 2]
    assert torch.allclose(want[0][:, 2], own, rtol=1e-4, atol=1e-4) and bool(torch.isfinite(want[0]).all()) and bool(torch.isfinite(want[1]).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.linear_attention(q, k, v, rate)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    s = torch.randn(2, 3, 32, 32, device=DEV)
    e = q[:, :, :0].detach().requires_grad_(True)
    o, st = ops.linear_attention(e, k[:, :, :0], v[:, :, :0], rate, state=s)
    o.sum().backward()
    assert o.shape == (2, 3, 0, 32) and torch.equal(st, s) and st.data_ptr() != s.data_ptr()
    o, st = ops.linear_attention(q[:0], k[:0], v[:0], rate)
    assert o.shape == (0, 3, 150, 32) and st.shape == (0, 3, 32, 32)
    assert ops.linear_attention_step(q[:0, :, 0], k[:0, :, 0], v[:0, :, 0], rate, st).shape == (0, 3, 32)
    # no valid position at all: zeros, the state as it came, its gradient passed on
    s.requires_grad_(True)
    o, st = ops.linear_attention(q, k, v, rate, state=s, valid_len=torch.zeros(2, dtype=torch.int32, device=DEV))
    gs, = torch.autograd.grad(st, s, torch.ones_like(s))
    assert float(o.abs().max()) == 0.0 and torch.equal(st, s) and torch.equal(gs, torch.ones_like(s))
    # lengths beyond T and below 0 count as T and 0
    o2, _ = ops.linear_attention(q, k, v, rate, valid_len=torch.tensor([1 << 20, -5], device=DEV))
    assert torch.equal(o2[0], want[0][0]) and float(o2[1].abs().max()) == 0.0


@pytest.mark.gpu
def test_linear_attention_only_some_gradients():
    from ironcortex_amd.hip import ops
    g = torch.Generator(device=DEV).manual_seed(11)
    q, k, v = inputs(g, torch.float32, 2, 100, 2, 2, 16, 16, "tokens")
    rate = torch.tensor([0.1, 0.3], device=DEV)
    s = torch.randn(2, 2, 16, 16, device=DEV)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v, rate, s)]
    full_o = torch.autograd.grad(ops.linear_attention(*leaves[:4], state=leaves[4])[0].sum(), leaves)
    full_s = torch.autograd.grad(ops.linear_attention(*leaves[:4], state=leaves[4])[1].sum(), leaves)
    for j in range(5):  # one leaf at a time gives the same as all of them
        xs = [x.clone() for x in (q, k, v, rate, s)]
        xs[j].requires_grad_(True)
        o, st = ops.linear_attention(*xs[:4], state=xs[4])
        for y, full in ((o, full_o), (st, full_s)):
            got, = torch.autograd.grad(y.sum(), xs[j], retain_graph=True)
            assert torch.equal(got, full[j]), j
    assert float(full_s[0].abs().max()) == 0.0


@pytest.mark.gpu
def test_linear_attention_in_captured_graphs():
    """Two captured graphs (a training pass and single steps) replayed in turn with eager calls between them."""
    from ironcortex_amd.hip import ops
    g = torch.Generator(device=DEV).manual_seed(12)
    q, k, v = (x.contiguous().requires_grad_(True) for x in inputs(g, torch.float32, 2, 900, 2, 1, 64, 64, "tokens"))
    rate = torch.tensor([0.01, 0.2], device=DEV, requires_grad=True)
    go = torch.randn(2, 2, 900, 64, generator=g, device=DEV)
    S = torch.zeros(2, 2, 64, 64, device=DEV)

    def train():
        o, st = ops.linear_attention(q, k, v, rate)
        return (o, st, *torch.autograd.grad(o, (q, k, v, rate), go))

    def step():
        with torch.no_grad():
            return ops.linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], rate, S)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
        step()
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        h1 = train()
    with torch.cuda.graph(g2):
        h2 = step()
    for n in range(3):
        with torch.no_grad():
            for x in (q, k, v):
                x.copy_(torch.randn(x.shape, generator=g, device=DEV))
        S.normal_(generator=g)
        keep = S.clone()
        want = [t.detach().clone() for t in train()]
        ws = step().clone()
        wS = S.clone()
        S.copy_(keep)
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.detach(), b) for a, b in zip(h1, want)), n
        assert torch.equal(h2, ws) and torch.equal(S, wS), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("Dk,Dv", [(32, 24), (64, 64), (128, 128), (33, 65)])
def test_linear_attention_not_finite_rows_reach_only_what_follows(Dk, Dv, dtype):
    """A value that is not finite, at a position t: the outputs in front of t are those of finite rows; where it is one of v's,
    the other columns are, too."""
    from ironcortex_amd.hip import ops
    dt, B, T, H = TYPES[dtype], 4, 200, 2
    g = torch.Generator(device=DEV).manual_seed(14)
    rows = inputs(g, dt, B, T, H, 1, Dk, Dv, "tokens")
    rate, scale = torch.tensor([0.0, 0.3], device=DEV), 0.25
    n = torch.full((B,), T, device=DEV)
    want, _ = recurrence(*(x.double() for x in rows), rate.double(), scale, None, n)
    A, _ = recurrence(*(x.double().abs() for x in rows), rate.double(), scale, None, n)
    b = bound(A, Dk + Dv + 160 + T / 64, dt, want)
    for which in range(3):
        for bad in (float("inf"), float("-inf"), float("nan")):
            x = [r.clone() for r in rows]
            at = (5, 70, 100, 191)
            for i, t in enumerate(at):
                x[which][i, -1, t, 3] = bad
            got = ops.linear_attention(*x, rate, scale=scale)[0]
            for i, t in enumerate(at):
                within(got[i, :, :t], want[i, :, :t], b[i, :, :t], f"in front of {t}")
                hit = got[i, -1, t, 3 if which == 2 else slice(None)]
                assert not bool(torch.isfinite(hit).any())
                if which == 0:  # a query is its own position's only
                    within(got[i, :, t + 1:], want[i, :, t + 1:], b[i, :, t + 1:], "behind a query")
                if which == 2:
                    keep = [c for c in range(Dv) if c != 3]
                    within(got[i][:, :, keep], want[i][:, :, keep], b[i][:, :, keep], "other columns")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 65])
def test_linear_attention_many_sequences(T):
    """More sequences and heads than a grid's second dimension holds; a piece of them gives the same rows."""
    from ironcortex_amd.hip import ops
    B, H, D = 17500, 4, 8
    g = torch.Generator(device=DEV).manual_seed(15)
    q, k, v = (torch.randn(B, T, H, D, generator=g, device=DEV).transpose(1, 2) for _ in range(3))
    rate, st = torch.rand(H, generator=g, device=DEV), torch.randn(B, H, D, D, generator=g, device=DEV)
    lo = B - 11

    def run(*x):
        x = [t.detach().requires_grad_(True) for t in x]
        y, s = ops.linear_attention(x[0], x[1], x[2], rate, state=x[3])
        return (y.detach(), s.detach(), *torch.autograd.grad((y.square().sum() + s.square().sum()), x))

    for a, b in zip(run(q, k, v, st), run(q[lo:], k[lo:], v[lo:], st[lo:])):
        # other segments: sums of 65 + 8 terms in another order, twice 73 * 2^-24 = 8.7e-6 of the terms' magnitudes
        assert float((a[lo:] - b).abs().max()) <= 2e-5 * float(b.abs().max())
    s2 = st.clone()
    y = ops.linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], rate, s2)
    y1, s1 = ops.linear_attention(q[:, :, :1], k[:, :, :1], v[:, :, :1], rate, state=st)
    for a, b in ((y, y1[:, :, 0]), (s2, s1)):
        assert float((a - b).abs().max()) <= 2e-5 * float(b.abs().max())


@pytest.mark.gpu
def test_linear_attention_far_apart_positions_inference_mode_and_second_derivatives():
    from ironcortex_amd.hip import ops
    g = torch.Generator(device=DEV).manual_seed(13)
    T, D = 70, 16
    far = torch.randn(T, ops.LATTN_MAX_STRIDE + 16, generator=g, device=DEV)[:, :D].view(1, 1, T, D)  # 16 MB from position to position
    near = far.contiguous()
    assert far.stride(2) > ops.LATTN_MAX_STRIDE
    rate = torch.tensor([0.1], device=DEV)
    res = []
    for x in (far, near):
        x = [x.detach().requires_grad_(True) for _ in range(3)]
        o, st = ops.linear_attention(*x, rate)
        res.append((o.detach(), st.detach(), *torch.autograd.grad(o, x, far)))
    assert all(torch.equal(a, b) for a, b in zip(*res))
    with torch.inference_mode():  # tensors of the mode keep no version
        o, st = ops.linear_attention(near, near, near, rate)
        y = ops.linear_attention_step(near[:, :, 0], near[:, :, 0], near[:, :, 0], rate, st)
        ops.rope(near, freqs=rate)
    assert bool(torch.isfinite(y).all()) and torch.equal(o, res[0][0])
    x = near.clone().requires_grad_(True)
    gx, = torch.autograd.grad(ops.linear_attention(x, x, x, rate)[0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()
    gx, = torch.autograd.grad(ops.rope(x, freqs=rate).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


@pytest.mark.gpu
def test_linear_attention_refusals():
    from ironcortex_amd.hip import ops
    q, k, v = (torch.randn(2, 4, 5, 8, device=DEV) for _ in range(3))
    r = torch.ones(4, device=DEV)
    s = torch.zeros(2, 4, 8, 8, device=DEV)
    for a, kw in (((q[0], k, v, r), {}), ((q, k.half(), v, r), {}), ((q.double(), k.double(), v.double(), r), {}), ((q, k[:, :3], v[:, :3], r), {}),
                  ((q, k[:, :, :4], v, r), {}), ((q, k, v[:, :2], r), {}), ((q, k[..., :4], v, r), {}), ((q, k, v, r[:3]), {}), ((q, k, v, r.half()), {}),
                  ((q, k, v, r), dict(state=s[:1])), ((q, k, v, r), dict(state=s.half())), ((q, k, v, r), dict(valid_len=torch.ones(3, device=DEV, dtype=torch.int32))),
                  ((q, k, v, r), dict(valid_len=torch.ones(2, device=DEV))), ((torch.randn(1, 1, 2, 129, device=DEV),) * 3 + (r[:1],), {})):
        with pytest.raises(ValueError):
            ops.linear_attention(*a, **kw)
    with pytest.raises(RuntimeError):
        ops.linear_attention(q, k, v, r.cpu())
    t = lambda x: x[:, :, 0]  # noqa: E731
    for a, kw in (((q, t(k), t(v), r, s), {}), ((t(q), t(k), t(v), r, s[:, :, :, :4]), {}), ((t(q), t(k), t(v), r, s.transpose(2, 3)), {}),
                  ((t(q), t(k), t(v), r, s[:1].expand(2, 4, 8, 8)), {}), ((t(q), t(k), t(v), r, s), dict(active=torch.ones(2, device=DEV)))):
        with pytest.raises(ValueError):
            ops.linear_attention_step(*a, **kw)
    with pytest.raises(RuntimeError):
        ops.linear_attention_step(t(q).clone().requires_grad_(True), t(k), t(v), r, s)


def test_lattn_refuses_cpu_tensors_and_bad_arguments_of_the_c_entries():
    from ironcortex_amd import hip
    from ironcortex_amd.hip import ops
    lib = hip.lib()
    x = torch.randn(1, 1, 2, 4)
    with pytest.raises(RuntimeError):
        ops.linear_attention(x, x, x, torch.ones(1))
    with pytest.raises(RuntimeError):
        ops.linear_attention_step(x[:, :, 0], x[:, :, 0], x[:, :, 0], torch.ones(1), torch.zeros(1, 1, 4, 4))
    good = dict(B=1, H=2, Hk=1, T=5, Dk=8, Dv=8, dtype=0, q=8, k=8, v=8, rate=8, out=8)
    EINVAL = hip.ENUMS["IC_EINVAL"]
    for kw, text in ((dict(B=0), "B=0"), (dict(T=0), "T=0"), (dict(H=3, Hk=2), "Hk=2"), (dict(Hk=0), "Hk=0"), (dict(Dk=129), "Dk=129"), (dict(Dv=0), "Dv=0"),
                     (dict(dtype=7), "dtype=7"), (dict(B=1 << 21, H=4), "B*H"), (dict(q=None), "NULL"), (dict(rate=None), "NULL"), (dict(out=None), "NULL"),
                     (dict(state=16, state_out=16), "state_out"), (dict(T=1000), "workspace"), (dict(k_st=1 << 22), "k has"), (dict(o_st=-(1 << 40)), "out has")):
        a = hip.new("ic_lattn_args", **{**good, **kw})
        assert lib.ic_lattn_fwd(ctypes.byref(a), None) == EINVAL and text in lib.ic_last_error().decode(), (kw, lib.ic_last_error())
    a = hip.new("ic_lattn_args", **good)
    n = ctypes.c_int64(-1)
    assert lib.ic_lattn_ws(ctypes.byref(a), 0, ctypes.byref(n)) == 0 and n.value == 0  # one chunk needs none
    assert lib.ic_lattn_ws(ctypes.byref(a), 0, None) == EINVAL
    a.T = 100000
    assert lib.ic_lattn_ws(ctypes.byref(a), 1, ctypes.byref(n)) == 0 and n.value > 100000 * 16  # rows of dk and dv in fp32
    b = hip.new("ic_lattn_bwd_args", f=hip.new("ic_lattn_args", **good))
    assert lib.ic_lattn_bwd(ctypes.byref(b), None) == EINVAL and b"NULL" in lib.ic_last_error()
    for n_ in ("dout", "dq", "dk", "dv"):
        setattr(b, n_, 8)
    assert lib.ic_lattn_bwd(ctypes.byref(b), None) == EINVAL and b"workspace" in lib.ic_last_error()
    for fn in ("ic_lattn_fwd", "ic_lattn_bwd", "ic_lattn_step"):
        assert getattr(lib, fn)(None, None) == EINVAL
    sg = dict(B=1, H=2, Hk=1, Dk=8, Dv=8, q=8, k=8, v=8, rate=8, out=8, state=8)
    for kw in (dict(B=0), dict(Hk=3), dict(Dk=1025), dict(dtype=-1), dict(state=None), dict(out=None)):
        a = hip.new("ic_lattn_step_args", **{**sg, **kw})
        assert lib.ic_lattn_step(ctypes.byref(a), None) == EINVAL
