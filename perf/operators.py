"""Timing cases for the token-mixing operators of ironcortex_amd.hip.ops: `rope`, `qk_norm_rope`, `linear_attention` and
`linear_attention_step`.

`run` computes a case in plain torch operations, or, where `own` is set, through the library's entry points; `exact` gives
the same outputs from the operators' definitions in 64 bits.  Notation: B sequences, H query heads, Hk key / value heads
(head h of the queries uses head h // (H / Hk) of the keys), T positions, m rotated channel pairs of a row of D channels."""
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5
CHUNK = 64


# ------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the token mixer of the 10M-parameter configuration in a training step: 16 sequences of 256 positions and their
        # anchors, 4 heads of 64 channels, angles from two-dimensional coordinates given as tables
        dict(name="rope mixer train", op="rope", dtype="fp32", B=16, T=266, H=4, Hk=4, D=64, m=32, layout="interleaved",
             tables=True, start=0, spread=0, factor=1.0, train=True),
        # one very long document, far beyond the trained length: half of each head rotated, frequencies scaled
        dict(name="rope long document", op="rope", dtype="bf16", B=1, T=131072, H=8, Hk=2, D=128, m=32, layout="half",
             tables=False, start=900001, spread=0, factor=8.0, train=False),
        # serving: one token for each of 64 running sequences, every one at a position of its own
        dict(name="qk norm decode", op="norm", dtype="bf16", B=64, T=1, H=16, Hk=4, D=128, m=64, layout="half",
             tables=False, start=5, spread=30000, factor=1.0, train=False),
        # a training step at the mixer's sizes, anchors included
        dict(name="qk norm mixer train", op="norm", dtype="fp32", B=16, T=520, H=4, Hk=4, D=64, m=32, layout="interleaved",
             tables=False, start=0, spread=0, factor=1.0, train=True),
        # a training step over the longest sequences the configuration allows (8192 positions), shared key heads
        dict(name="qk norm long train", op="norm", dtype="bf16", B=4, T=8192, H=16, Hk=4, D=128, m=64, layout="half",
             tables=False, start=0, spread=0, factor=1.0, train=True),
        # a few short prompts at the default width (heads of 32 channels): latency counts
        dict(name="linear short prompts", op="linear", dtype="fp32", B=2, T=33, H=4, Hk=4, Dk=32, Dv=32, ragged=False,
             state=False, train=False),
        # a batch of prompts of different lengths that continue earlier text (a state comes in)
        dict(name="linear ragged prompts", op="linear", dtype="fp32", B=16, T=1064, H=4, Hk=4, Dk=64, Dv=64, ragged=True,
             state=True, train=False),
        # a training step at the width of the 10M-parameter configuration
        dict(name="linear mixer train", op="linear", dtype="fp32", B=16, T=1024, H=4, Hk=4, Dk=64, Dv=64, ragged=False,
             state=False, train=True),
        # one long document read in one call
        dict(name="linear long document", op="linear", dtype="bf16", B=1, T=65536, H=8, Hk=8, Dk=128, Dv=128, ragged=False,
             state=False, train=False),
        # a training step of a wider mixer with shared key / value heads
        dict(name="linear wide train", op="linear", dtype="bf16", B=8, T=4096, H=8, Hk=4, Dk=128, Dv=128, ragged=False,
             state=False, train=True),
        # serving one conversation: one token, the mixer's 4 heads
        dict(name="step one sequence", op="step", dtype="fp32", B=1, T=1, H=4, Hk=4, Dk=64, Dv=64),
        # serving 256 conversations at once
        dict(name="step many sequences", op="step", dtype="bf16", B=256, T=1, H=16, Hk=4, Dk=128, Dv=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "norm", "linear", "linear", "step"])
    dtype = rng.choice(["fp32", "fp32", "bf16", "bf16", "fp16"])
    Hk = rng.choice([1, 2, 3, 4, 8])
    H = Hk * rng.choice([1, 1, 2, 4])
    if op == "step":
        Dk, Dv = rng.choice([16, 32, 64, 64, 96, 128]), rng.choice([32, 64, 64, 100, 128])
        return dict(op=op, dtype=dtype, B=_log(rng, 1, 256), T=1, H=min(H, 16), Hk=min(Hk, 16), Dk=Dk, Dv=Dv)
    if op == "linear":
        train = rng.random() < 0.5
        Dk = rng.choice([8, 32, 64, 64, 80, 128])
        Dv = Dk if rng.random() < 0.6 else rng.choice([24, 32, 64, 128])
        B = _log(rng, 1, 16)
        most = (8 * 4096 * 8 * 128 if train else 65536 * 8 * 128) // (B * H * max(Dk, Dv, 64))
        return dict(op=op, dtype=dtype, B=B, T=min(_log(rng, 1, 32768), max(1, most)), H=H, Hk=Hk, Dk=Dk, Dv=Dv,
                    ragged=rng.random() < 0.4, state=rng.random() < 0.4, train=train)
    D = rng.choice([32, 64, 64, 80, 96, 128, 128, 192, 256])
    B = _log(rng, 1, 64)
    train = rng.random() < 0.5
    most = (4 * 8192 * 20 * 128 if train or op == "norm" else 131072 * 10 * 128) // (B * (H + Hk) * D)
    tables = rng.random() < 0.3
    return dict(op=op, dtype=dtype, B=B, T=min(_log(rng, 1, 65536), max(1, most)), H=H, Hk=Hk, D=D,
                m=rng.choice([D // 2, D // 2, D // 4, D // 8]), layout=rng.choice(["interleaved", "half"]), tables=tables,
                start=0 if tables else rng.choice([0, 0, 1000, 1000003]), spread=0 if tables else rng.choice([0, 0, 5000]),
                factor=rng.choice([1.0, 1.0, 4.0, 8.0]), train=train)


# ----------------------------------------------------------------------------------------------------------- the inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)


def _rows(g, dtype, *shape):
    """Projected rows as a linear layer leaves them: [B,T,heads,width], normal values."""
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    c = dict(case)
    B, T, H, Hk = c["B"], c["T"], c["H"], c["Hk"]
    st = {"c": c}
    if c["op"] in ("rope", "norm"):
        D, m = c["D"], c["m"]
        # token-major rows [B,T,heads,D], handed over as [B,heads,T,D] views
        st["q"], st["k"] = _rows(g, dt, B, T, H, D), _rows(g, dt, B, T, Hk, D)
        if c["tables"]:
            pos = torch.arange(T, device=DEV, dtype=torch.float64)
            w = torch.exp(torch.linspace(math.log(1e-4), 0.0, m, device=DEV, dtype=torch.float64))
            shift = torch.rand(B, 1, 1, generator=g, device=DEV).double()
            ang = (pos.view(1, T, 1) * (1.0 + 1.0 / T) + shift) * w  # (position, relative position) coordinates
            st["cos"], st["sin"] = torch.cos(ang).float(), torch.sin(ang).float()  # [B,T,m]
        else:
            first = torch.randint(0, c["spread"] + 1, (B, 1), generator=g, device=DEV) + c["start"]
            st["positions"] = first + torch.arange(T, device=DEV)  # [B,T] int64
            # log-spaced frequencies, divided by the factor by which the context outgrew the trained one
            st["freqs"] = (10000.0 ** (-torch.arange(m, device=DEV, dtype=torch.float64) / m) / c["factor"]).float()
        st["scale"] = 1.0 + 0.1 * math.log(c["factor"])
        if c["op"] == "norm":
            st["wq"] = (1.0 + 0.2 * torch.randn(D, generator=g, device=DEV))
            st["wk"] = (1.0 + 0.2 * torch.randn(D, generator=g, device=DEV))
        if c["train"]:
            st["gq"], st["gk"] = _rows(g, dt, B, H, T, D), _rows(g, dt, B, Hk, T, D)
            for n in ("q", "k", "wq", "wk"):
                if n in st:
                    st[n].requires_grad_(True)
        return st
    Dk, Dv = c["Dk"], c["Dv"]
    st["rate"] = torch.exp(torch.rand(H, generator=g, device=DEV) * math.log(5000.0) + math.log(2e-4))  # 2e-4 .. 1
    st["scale"] = Dk ** -0.5
    if c["op"] == "step":
        st["q"], st["k"], st["v"] = _rows(g, dt, B, H, Dk), _rows(g, dt, B, Hk, Dk), _rows(g, dt, B, Hk, Dv)
        st["state"] = torch.randn(B, H, Dk, Dv, generator=g, device=DEV)
        return st
    st["q"], st["k"], st["v"] = _rows(g, dt, B, T, H, Dk), _rows(g, dt, B, T, Hk, Dk), _rows(g, dt, B, T, Hk, Dv)
    st["state"] = torch.randn(B, H, Dk, Dv, generator=g, device=DEV) if c["state"] else None
    st["valid"] = torch.randint(T // 2, T + 1, (B,), generator=g, device=DEV).to(torch.int32) if c["ragged"] else None
    if c["train"]:
        st["go"] = _rows(g, dt, B, H, T, Dv)
        st["gs"] = torch.randn(B, H, Dk, Dv, generator=g, device=DEV)
        for n in ("q", "k", "v", "rate", "state"):
            if st[n] is not None:
                st[n].requires_grad_(True)
    return st


# ------------------------------------------------------------------------------------------------------- the plain forms
def _tables(st, c):
    """(cos, sin) [B,T,m] fp32; angles formed in 64 bits, since a far position's angle loses its fraction in 32."""
    if c["tables"]:
        return st["cos"] * st["scale"], st["sin"] * st["scale"]
    ang = st["positions"].double().unsqueeze(-1) * st["freqs"].double()
    return (torch.cos(ang) * st["scale"]).float(), (torch.sin(ang) * st["scale"]).float()


def _rotate(x, cos, sin, layout):
    """x [B,H,T,D] -> rotated, in x's precision; cos / sin [B,T,m]."""
    m = cos.shape[-1]
    cos, sin = cos.unsqueeze(1), sin.unsqueeze(1)
    a, b = (x[..., 0:2 * m:2], x[..., 1:2 * m:2]) if layout == "interleaved" else (x[..., :m], x[..., m:2 * m])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    rot = torch.stack((ra, rb), dim=-1).flatten(-2) if layout == "interleaved" else torch.cat((ra, rb), dim=-1)
    return torch.cat((rot, x[..., 2 * m:]), dim=-1) if 2 * m < x.shape[-1] else rot


def _norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _plain_rope(st, c):
    cos, sin = _tables(st, c)
    out = []
    for n, w in (("q", "wq"), ("k", "wk")):
        x = st[n].transpose(1, 2).float()
        out.append(_rotate(_norm(x, st[w]) if w in st else x, cos, sin, c["layout"]).to(st[n].dtype))
    return tuple(out)


def _plain_linear(st, c):
    """Chunks of 64 positions: the products inside a chunk as a masked [64,64] matrix, the states at the chunks' borders as
    one product with the matrix of decays from border to border."""
    q, k, v, rate = st["q"].transpose(1, 2).float(), st["k"].transpose(1, 2).float(), st["v"].transpose(1, 2).float(), st["rate"]
    B, H, T, Dk = q.shape
    Dv, G, dev = v.shape[-1], H // k.shape[1], q.device
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    N = -(-T // CHUNK)
    pad = N * CHUNK - T
    n = torch.full((B,), T, device=dev) if st["valid"] is None else st["valid"].long()
    t = torch.arange(N * CHUNK, device=dev)
    live = (t < n.view(B, 1)).view(B, 1, N * CHUNK, 1)
    cut = lambda x: torch.where(live, torch.nn.functional.pad(x, (0, 0, 0, pad)), torch.zeros((), device=dev)).view(B, H, N, CHUNK, -1)  # noqa: E731
    q, k, v = cut(q), cut(k), cut(v)
    r = rate.view(1, H, 1, 1, 1)
    i = torch.arange(CHUNK, device=dev)
    lag = (i.view(-1, 1) - i).float()
    inside = torch.where(lag >= 0, torch.exp(-r * lag.clamp_min(0)), torch.zeros((), device=dev))
    # positions counted up to a border, which no padding passes: [B, N+1]
    border = torch.minimum((torch.arange(N + 1, device=dev) * CHUNK).view(1, -1), n.view(B, 1))
    left = (border[:, 1:, None] - 1 - t.view(1, N, CHUNK)).clamp_min(0).float().view(B, 1, N, CHUNK, 1)
    local = (k * torch.exp(-r * left)).transpose(-2, -1) @ v  # [B,H,N,Dk,Dv]
    gap = (border[:, :, None] - border[:, None, 1:]).float().view(B, 1, N + 1, N)
    hops = torch.where(torch.arange(N + 1, device=dev).view(-1, 1) > torch.arange(N, device=dev),
                       torch.exp(-rate.view(1, H, 1, 1) * gap.clamp_min(0)), torch.zeros((), device=dev))
    states = (hops @ local.reshape(B, H, N, Dk * Dv)).view(B, H, N + 1, Dk, Dv)
    if st["state"] is not None:
        states = states + torch.exp(-r * border.float().view(B, 1, N + 1, 1, 1)) * st["state"].unsqueeze(2)
    out = ((q @ k.transpose(-2, -1).contiguous()) * inside) @ v + torch.exp(-r * (i + 1).float().view(-1, 1)) * (q @ states[:, :, :N])
    out = (out * st["scale"]).reshape(B, H, N * CHUNK, Dv)[:, :, :T]
    return out.to(st["q"].dtype), states[:, :, N]


def _plain_step(st, c):
    G = c["H"] // c["Hk"]
    k, v = st["k"].float().repeat_interleave(G, 1), st["v"].float().repeat_interleave(G, 1)
    st["state"].mul_(torch.exp(-st["rate"]).view(1, -1, 1, 1)).add_(k.unsqueeze(-1) * v.unsqueeze(-2))
    out = (st["q"].float().unsqueeze(-1) * st["state"]).sum(-2) * st["scale"]
    return out.to(st["q"].dtype), st["state"]


# ------------------------------------------------------------------------------------------------ the library's operators
def _own(st, c):
    from ironcortex_amd.hip import ops

    if c["op"] in ("rope", "norm"):
        q, k = st["q"].transpose(1, 2), st["k"].transpose(1, 2)
        kw = dict(cos=st["cos"], sin=st["sin"]) if c["tables"] else dict(positions=st["positions"], freqs=st["freqs"])
        kw.update(layout=c["layout"], scale=st["scale"])
        return ops.qk_norm_rope(q, k, st["wq"], st["wk"], eps=EPS, **kw) if c["op"] == "norm" else ops.rope(q, k, **kw)
    if c["op"] == "step":
        return ops.linear_attention_step(st["q"], st["k"], st["v"], st["rate"], st["state"], scale=st["scale"]), st["state"]
    return ops.linear_attention(st["q"].transpose(1, 2), st["k"].transpose(1, 2), st["v"].transpose(1, 2), st["rate"],
                                scale=st["scale"], state=st["state"], valid_len=st["valid"])


def run(state):
    c = state["c"]
    if own:
        out = _own(state, c)
    else:
        out = {"rope": _plain_rope, "norm": _plain_rope, "linear": _plain_linear, "step": _plain_step}[c["op"]](state, c)
    if not c.get("train"):
        return tuple(out)
    if c["op"] == "linear":
        leaves = [state[n] for n in ("q", "k", "v", "rate", "state") if state[n] is not None]
        return tuple(out) + torch.autograd.grad(out, leaves, (state["go"], state["gs"]))
    leaves = [state[n] for n in ("q", "k", "wq", "wk") if n in state]
    return tuple(out) + torch.autograd.grad(out, leaves, (state["gq"], state["gk"]))


# --------------------------------------------------------------------------------------------------- what a case has to do
def work(case):
    c, e = case, {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    rows = c["B"] * c["T"]
    if c["op"] in ("rope", "norm"):
        x = rows * (c["H"] + c["Hk"]) * c["D"]
        angles = rows * c["m"] * 8 if c["tables"] else rows * 8 + c["m"] * 4
        w = 2 * c["D"] * 4 if c["op"] == "norm" else 0
        passes = 2 + (0 if not c["train"] else 3 if c["op"] == "norm" else 2)  # x, y; then gy, gx (and x again)
        return {"bytes": x * e * passes + angles + w * (2 if c["train"] else 1),
                "flops": x * (3 if c["op"] == "rope" else 7) * (3 if c["train"] else 1)}
    qo, kv = c["H"] * (c["Dk"] + c["Dv"]), c["Hk"] * (c["Dk"] + c["Dv"])
    s = c["B"] * c["H"] * c["Dk"] * c["Dv"]
    if c["op"] == "step":
        return {"bytes": rows * (qo + kv) * e + 8 * s, "flops": 5 * s}
    states = s * 4 * (2 if c["state"] else 1)
    if not c["train"]:  # the recurrence's own products: k v^T into the state, q out of it
        return {"bytes": rows * (qo + kv) * e + states, "flops": 4 * c["T"] * s}
    # training: q, k, v, d out in; out, dq, dk, dv out; the state's and its gradient's recurrences and five products with them
    return {"bytes": rows * (2 * qo + 2 * kv) * e + 2 * states, "flops": 14 * c["T"] * s}


# ------------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_rotation(x, st, c, back):
    """Pairs rotated by complex numbers; `back`: by the conjugate (the transposed rotation)."""
    m, D = c["m"], c["D"]
    if c["tables"]:
        z = torch.complex(st["cos"].detach().double(), st["sin"].detach().double()) * st["scale"]
    else:
        ang = st["positions"].double().unsqueeze(-1) * st["freqs"].double()
        z = torch.polar(torch.full_like(ang, st["scale"]), ang)
    z = z.conj().unsqueeze(1) if back else z.unsqueeze(1)
    first = torch.arange(m, device=x.device) * (2 if c["layout"] == "interleaved" else 1)
    second = first + (1 if c["layout"] == "interleaved" else m)
    r = torch.complex(x[..., first], x[..., second]) * z
    y = x.clone()
    y[..., first], y[..., second] = r.real, r.imag
    return y


def _exact_rope(st, c):
    outs, grads, wgrads = [], [], []
    for n, w, gn in (("q", "wq", "gq"), ("k", "wk", "gk")):
        x = st[n].detach().transpose(1, 2).double()
        if w in st:
            inv = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
            outs.append(_exact_rotation(x * inv * st[w].detach().double(), st, c, False))
        else:
            outs.append(_exact_rotation(x, st, c, False))
        if c["train"]:
            h = _exact_rotation(st[gn].double(), st, c, True)
            if w in st:
                wgrads.append((h * x * inv).sum((0, 1, 2)))
                h = h * st[w].detach().double()
                h = h * inv - x * inv.pow(3) * (h * x).mean(-1, keepdim=True)
            grads.append(h.transpose(1, 2))
    return tuple(outs + grads + wgrads)


def _exact_linear(st, c):
    """Every pair of positions, one (sequence, head) and a block of queries at a time."""
    B, T, H, Dk, Dv = c["B"], c["T"], c["H"], c["Dk"], c["Dv"]
    G, dev, f64 = H // c["Hk"], DEV, torch.float64
    z = lambda *s: torch.zeros(*s, device=dev, dtype=f64)  # noqa: E731
    out, last = z(B, H, T, Dv), z(B, H, Dk, Dv)
    dq, dk, dv, dr, ds = z(B, T, H, Dk), z(B, T, c["Hk"], Dk), z(B, T, c["Hk"], Dv), z(H), z(B, H, Dk, Dv)
    valid = [T] * B if st["valid"] is None else st["valid"].tolist()
    sc = st["scale"]
    for b in range(B):
        n = valid[b]
        t = torch.arange(n, device=dev, dtype=f64)
        for h in range(H):
            q, k, v = (st[a].detach()[b, :n, j].double() for a, j in (("q", h), ("k", h // G), ("v", h // G)))
            r = st["rate"].detach()[h].double()
            s0 = z(Dk, Dv) if st["state"] is None else st["state"].detach()[b, h].double()
            tail = torch.exp(-r * (n - 1 - t)).unsqueeze(1)
            last[b, h] = torch.exp(-r * n) * s0 + (k * tail).T @ v
            if c["train"]:
                gs = st["gs"][b, h].double()
                ds[b, h] += torch.exp(-r * n) * gs
                dr[h] -= n * torch.exp(-r * n) * (gs * s0).sum()
                dk[b, :n, h // G] += tail * (v @ gs.T)
                dv[b, :n, h // G] += tail * (k @ gs)
                dr[h] -= ((n - 1 - t).unsqueeze(1) * tail * k * (v @ gs.T)).sum()
            for lo in range(0, n, 4096):
                hi = min(n, lo + 4096)
                lag = t[lo:hi].unsqueeze(1) - t[:hi]
                w = torch.where(lag >= 0, torch.exp(-r * lag.clamp_min(0.0)), z(1)) * sc
                a = (q[lo:hi] @ k[:hi].T) * w
                enter = sc * torch.exp(-r * (t[lo:hi] + 1)).unsqueeze(1)
                out[b, h, lo:hi] = a @ v[:hi] + enter * (q[lo:hi] @ s0)
                if c["train"]:
                    go = st["go"][b, h, lo:hi].double()
                    da = (go @ v[:hi].T) * w
                    dq[b, lo:hi, h] += da @ k[:hi] + enter * (go @ s0.T)
                    dk[b, :hi, h // G] += da.T @ q[lo:hi]
                    dv[b, :hi, h // G] += a.T @ go
                    dr[h] -= (lag * a * (go @ v[:hi].T)).sum() + ((t[lo:hi] + 1).unsqueeze(1) * enter * go * (q[lo:hi] @ s0)).sum()
                    ds[b, h] += (enter * q[lo:hi]).T @ go
    if not c["train"]:
        return out, last
    return (out, last, dq, dk, dv, dr) + ((ds,) if c["state"] else ())


def exact(case, seed):
    st = prepare(case, seed)
    c = st["c"]
    with torch.no_grad():
        if c["op"] in ("rope", "norm"):
            return _exact_rope(st, c)
        if c["op"] == "linear":
            return _exact_linear(st, c)
        G = c["H"] // c["Hk"]
        k, v = (st[n].double().repeat_interleave(G, 1) for n in ("k", "v"))
        s = torch.exp(-st["rate"].double()).view(1, -1, 1, 1) * st["state"].double() + torch.einsum("bhk,bhv->bhkv", k, v)
        return torch.einsum("bhk,bhkv->bhv", st["q"].double(), s) * st["scale"], s
