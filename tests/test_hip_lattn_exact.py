"""How exact linear attention is (ops.linear_attention; csrc/lattn.hip), against the sums over pairs of positions in 64 bits.

Mean square errors, relative to the mean square of the result.  A rounding to fp32 is off by 0.42 * 2^-24 = 2.5e-8 of its value in
the mean square (uniform within half a unit in the last place, over a binade).  A sum of n terms of both signs grows like the root
of their number and is rounded n times (a matrix instruction on fp32 rounds after each product): 2.5e-8 sqrt(n / 2) of the result.
Sixteen chunks, one segment, slow decays:
  state: sums of 32 positions (1e-7), two additions at the state's size for every chunk (1e-7), the decayed values (3.5e-8):
  1.5e-7.  2e-7 is asserted; 64 additions at the state's size for every chunk would leave 5.7e-7.
  rows: the state (1.5e-7), its product with a query (D terms: 2.5e-8 sqrt(D / 2)), the chunk's own part, a quarter of the row at
  most (q . k, the sum over a chunk, four factors: 8e-8): 2.2e-7 for 64 channels, 2.6e-7 for 128.  1.2 times that is asserted of
  fp32 rows.
  16-bit rows: the roundings that fall to the other side.  A result y off by e does so with the chance e / step, steps between
  eps |y| / 2 and eps |y|; over normally distributed y, cut off where the step reaches e: E(1 / |y|) = 0.8 ln(1e5) = 9.2.  With
  E|e| = 0.8 * 2.6e-7 that is 9.2 * 2.1e-7 * 1.41 / eps: 3.5e-4 of bf16 rows, 2.8e-3 of fp16 rows.  Three times that is asserted;
  operands of 16 bits (e = 2^-18.5 in the mean) would leave 4e-3 of bf16 rows.
  d rate: a sum of terms of both signs -- one for every pair of positions and for every row's share of the first and last state --
  each of them as exact as a row.  Its error goes with the root of the sum of their squares, R, and not with the value, which
  may come out small: of the heads' values here the ones expected at 5e6 lie between 3e5 and 1e7.  8e-7 R is asserted, four
  times a row's error."""
import math

import pytest
import torch

from tests.test_hip_lattn import DEV, TYPES


def pairs64(q, k, v, r, scale, s0):
    """One sequence: q [H,T,Dk], k [H,T,Dk], v [H,T,Dv], r [H], s0 [H,Dk,Dv] or None, in 64 bits, as sums over pairs of positions."""
    T = q.shape[1]
    t = torch.arange(T, device=q.device, dtype=torch.float64)
    lag = t.view(-1, 1) - t
    r = r.view(-1, 1, 1)
    W = torch.where(lag >= 0, torch.exp(-r * lag.clamp_min(0.0)), torch.zeros((), device=q.device, dtype=torch.float64))
    out = ((q @ k.transpose(1, 2)) * W) @ v
    state = (k * torch.exp(-r * (T - 1 - t).view(1, -1, 1))).transpose(1, 2) @ v
    if s0 is not None:
        out = out + torch.exp(-r * (t + 1).view(1, -1, 1)) * (q @ s0)
        state = state + torch.exp(-r * T) * s0
    return scale * out, state


def rate_terms(q, k, v, r, scale, s0, go, gs):
    """[H] sums of the squares of the terms of d rate (one sequence, as in pairs64)."""
    T = q.shape[1]
    t = torch.arange(T, device=q.device, dtype=torch.float64)
    lag = (t.view(-1, 1) - t).clamp_min(0.0)  # (no lag, no term)
    r = r.view(-1, 1, 1)
    pairs = (scale * lag * torch.exp(-r * lag) * (q @ k.transpose(1, 2)) * (go @ v.transpose(1, 2))).square().sum((1, 2))
    enter = (scale * (t + 1).view(1, -1, 1) * torch.exp(-r * (t + 1).view(1, -1, 1)) * (q @ s0) * go).square().sum((1, 2))
    last = ((T - 1 - t).view(1, -1, 1) * torch.exp(-r * (T - 1 - t).view(1, -1, 1)) * (k @ gs) * v).square().sum((1, 2))
    return pairs + enter + last + (T * torch.exp(-r * T) * s0 * gs).square().sum((1, 2))


def rms(x):
    return float(x.double().square().mean().sqrt())


def check_exactness(dtype, B, H, Hk, T, D):
    from ironcortex_amd.hip import ops
    dt, some, scale = TYPES[dtype], 3, 0.125
    g = torch.Generator(device=DEV).manual_seed(60 + D)
    q, k, v = (torch.randn(B, T, h, D, generator=g, device=DEV).to(dt).transpose(1, 2).requires_grad_(True) for h in (H, Hk, Hk))
    rate = torch.exp(torch.linspace(math.log(2e-4), math.log(2e-2), H, device=DEV)).requires_grad_(True)
    state = torch.randn(B, H, D, D, generator=g, device=DEV).requires_grad_(True)
    go = torch.randn(B, H, T, D, generator=g, device=DEV).to(dt)
    gs = torch.randn(B, H, D, D, generator=g, device=DEV)
    go[some:], gs[some:] = 0, 0  # (d rate sums over all sequences: the others add nothing)
    leaves = (q, k, v, rate, state)
    y = ops.linear_attention(q, k, v, rate, scale=scale, state=state)
    got = [x.detach() for x in (*y, *torch.autograd.grad(y, leaves, (go, gs)))]
    want, drate, terms = [[] for _ in range(6)], torch.zeros(H, device=DEV, dtype=torch.float64), 0.0
    for b in range(some):
        x = [t.detach()[b].double().requires_grad_(True) for t in (q, k, v)] + [rate.detach().double().requires_grad_(True), state.detach()[b].double().requires_grad_(True)]
        kh, vh = (t.repeat_interleave(H // Hk, 0) for t in x[1:3])
        o, s = pairs64(x[0], kh, vh, x[3], scale, x[4])
        dq, dk, dv, dr, ds = torch.autograd.grad((o, s), x, (go[b].double(), gs[b].double()))
        drate += dr
        with torch.no_grad():
            terms = terms + rate_terms(x[0], kh, vh, x[3], scale, x[4], go[b].double(), gs[b].double())
        for w, e in zip(want, (o, s, dq, dk, dv, ds)):
            w.append(e.detach())
    o, s, dq, dk, dv, ds = (torch.stack(w) for w in want)
    what = f"{dtype} {(B, H, Hk, T, D)}"
    for n, a, b in (("state", got[1][:some], s), ("d state", got[6][:some], ds)):
        assert rms(a - b) <= 2e-7 * rms(b), f"{what} {n}: {rms(a - b) / rms(b):.2e}"
    for n, a, b in (("out", got[0], o), ("dq", got[2], dq), ("dk", got[3], dk), ("dv", got[4], dv)):
        a = a[:some]
        if dt == torch.float32:
            most = 1.2 * math.sqrt(1.5e-7 ** 2 + 2.5e-8 ** 2 * D / 2 + 8e-8 ** 2)
            assert rms(a - b) <= most * rms(b), f"{what} {n}: {rms(a - b) / rms(b):.2e}"
        else:
            other = float((a != b.to(dt)).float().mean())
            assert other <= 3 * 9.2 * 2.1e-7 * 1.41 / torch.finfo(dt).eps, f"{what} {n}: {other:.2e} of the rows' values rounded otherwise"
    e = float(((got[5].double() - drate).abs() / terms.sqrt()).max())
    assert e <= 8e-7, f"{what} d rate: {e:.2e}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("B,H,Hk,T,D", [(96, 8, 8, 1024, 64), (48, 8, 4, 1024, 128)])
def test_rows_on_fp32_products_are_as_exact_as_fp32_allows(dtype, B, H, Hk, T, D):
    check_exactness(dtype, B, H, Hk, T, D)


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,T,D", [(96, 8, 8, 1024, 64), (48, 8, 4, 1024, 128), (96, 8, 4, 1024, 32)])
def test_bf16_rows_are_as_exact_as_fp32_products(B, H, Hk, T, D):
    """Three bf16 parts of an fp32 operand hold all of its 24 bits, two of them 16."""
    check_exactness("bf16", B, H, Hk, T, D)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_slow_decays_over_many_chunks(dtype):
    """256 chunks of one segment, rates down to 1e-6: a factor rounded next to 1 (off by 2^-26 of it in the mean) and applied 256
    times would leave a state off by 256 * 1.5e-8 / 2 = 2e-6.  Rounded additions: 2.5e-8 sqrt(512 / 2) = 4e-7, and 1.1e-7 inside the
    chunks; 6e-7 is asserted of every head."""
    from ironcortex_amd.hip import ops
    dt, B, H, T, D = TYPES[dtype], 128, 8, 16384, 16
    g = torch.Generator(device=DEV).manual_seed(70)
    k, v = (torch.randn(B, T, H, D, generator=g, device=DEV).to(dt).transpose(1, 2) for _ in (0, 1))
    rate = torch.exp(torch.linspace(math.log(1e-6), math.log(2e-4), H, device=DEV))
    s0 = torch.randn(B, H, D, D, generator=g, device=DEV)
    got = ops.linear_attention(k, k, v, rate, state=s0)[1][:4]
    t, r = torch.arange(T, device=DEV, dtype=torch.float64), rate.double().view(1, H, 1, 1)
    want = torch.exp(-r * T) * s0[:4].double()
    want += (k[:4].double() * torch.exp(-r * (T - 1 - t).view(1, 1, T, 1))).transpose(2, 3) @ v[:4].double()
    for h in range(H):
        e = rms(got[:, h] - want[:, h]) / rms(want[:, h])
        assert e <= 6e-7, f"{dtype} rate {float(rate[h]):.1e}: {e:.2e}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T", [50, 700])
def test_an_infinite_state_stays_infinite(T, dtype):
    """Entries that are not finite stay what they are, whatever the decay; the others are those of a finite state."""
    from ironcortex_amd.hip import ops
    dt, B, H, D = TYPES[dtype], 3, 4, 16
    g = torch.Generator(device=DEV).manual_seed(71)
    q, k, v = (torch.randn(B, T, H, D, generator=g, device=DEV).to(dt).transpose(1, 2) for _ in range(3))
    rate = torch.tensor([0.0, 1e-4, 1e-2, 0.05], device=DEV)
    n = torch.tensor([T, 0, T // 2], device=DEV)
    s = torch.randn(B, H, D, D, generator=g, device=DEV)
    bad = s.clone()
    bad[..., 3, 5], bad[..., 4, 6], bad[..., 7, 7] = float("inf"), float("-inf"), float("nan")
    o, want = ops.linear_attention(q, k, v, rate, state=s, valid_len=n)
    o2, got = ops.linear_attention(q, k, v, rate, state=bad, valid_len=n)
    odd = ~torch.isfinite(bad)
    assert torch.equal(got[~odd], want[~odd]) and torch.equal(torch.nan_to_num(got[odd], nan=7.0), torch.nan_to_num(bad[odd], nan=7.0))
    keep = [c for c in range(D) if c not in (5, 6, 7)]
    assert torch.equal(o2[..., keep], o[..., keep])
    live = torch.arange(T, device=DEV) < n.view(B, 1)
    assert not bool(torch.isfinite(o2.transpose(1, 2)[live][..., [5, 6, 7]]).any())


@pytest.mark.gpu
def test_steps_outputs_are_as_exact_as_sums_in_pairs():
    """64 key channels: the state's two roundings and its factor's (4.6e-8), two channels a thread and five levels of pairs (6.1e-8),
    the scale (2.5e-8): 8e-8 in the mean square; 9.5e-8 is asserted.  Adding 32 partial sums one after the other leaves 1.2e-7."""
    from ironcortex_amd.hip import ops
    B, H, D = 256, 8, 64
    g = torch.Generator(device=DEV).manual_seed(72)
    q, k, v = (torch.randn(B, H, D, generator=g, device=DEV) for _ in range(3))
    rate, s = torch.rand(H, generator=g, device=DEV), torch.randn(B, H, D, D, generator=g, device=DEV)
    want = torch.exp(-rate.double()).view(1, H, 1, 1) * s.double() + k.double().unsqueeze(-1) * v.double().unsqueeze(-2)
    want = 0.3 * (q.double().unsqueeze(-2) @ want).squeeze(-2)
    got = ops.linear_attention_step(q, k, v, rate, s, scale=float(torch.tensor(0.3)))
    want *= float(torch.tensor(0.3)) / 0.3
    assert rms(got - want) <= 9.5e-8 * rms(want), f"{rms(got - want) / rms(want):.2e}"
