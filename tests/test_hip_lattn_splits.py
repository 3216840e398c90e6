"""Linear attention cut into segments of several chunks (ops.linear_attention; csrc/lattn.hip): the segments' sums with weights from
their ends, the scan over them, the pass from each start state, forward and backward, with lengths that end in the first, a middle
and the last segment.  Against sums over pairs of positions in 64 bits, elementwise: 4 sqrt(N) u A with A the same sums of absolute
values, N = Dk + Dv + 160 + T / 64 roundings along a term's path and u = 2^-24, whatever the rows' type (bf16 operands are held in
three parts, 24 bits), then one rounding to it.  Gradients of shared heads: 8 for every query head more; d rate: 64 more."""
import ctypes
import math

import pytest
import torch

from tests.test_hip_lattn import DEV, TYPES, U, inputs, within
from tests.test_hip_lattn_exact import pairs64

CASES = [  # B, T, H, Hk, Dk, Dv, how the rows lie
    (16, 1064, 4, 2, 64, 64, "tokens"), (16, 1064, 4, 4, 64, 48, "heads"), (8, 1300, 8, 4, 128, 128, "tokens"), (7, 1300, 8, 8, 128, 96, "tokens"),
    (12, 1300, 8, 4, 100, 100, "odd"), (24, 1100, 8, 4, 32, 32, "tokens"),
]


def spans(B, T, H, Hk, Dk, Dv, bf16):
    """(segments, chunks of one) of the forward, of dq with and without d rate, of dk and dv: the library's rule, restated."""
    d, up = max(Dk, Dv), lambda a, b: -(-a // b)
    NC = up(T, 64)

    def slots(lag):
        return 256 * (4 if d <= 32 else (2 if lag else 3) if d <= 64 else 2 if bf16 and not lag else 1)

    def span(have, n):
        found, best, ns, cps = (1, NC), None, 1, NC
        while ns <= (2 * n + have - 1) // have:
            cps = up(NC, ns)
            rounds = (have * ns + n - 1) // n
            cost = rounds * (cps + 1.0) + (0.4 * rounds * cps + 2.0 if ns > 1 else 0.0)
            if best is None or cost < best:
                best, found = cost, (ns, cps)
            if cps == 1:
                break
            cps -= 1
            ns = up(NC, cps)
        return found

    return span(B * H, slots(False)), span(B * H, slots(True)), span(B * H, slots(False)), span(2 * B * Hk, slots(False))


def check_split(B, T, H, Hk, Dk, Dv, dt):
    """The rule above is the library's: the workspaces it asks for are those of these segments."""
    from ironcortex_amd import hip
    from ironcortex_amd.hip import ops
    fwd, q, q0, kv = spans(B, T, H, Hk, Dk, Dv, dt == torch.bfloat16)
    a, n, dd, bh = hip.new("ic_lattn_args", B=B, H=H, Hk=Hk, T=T, Dk=Dk, Dv=Dv, dtype=ops.DTYPES[dt]), ctypes.c_int64(0), Dk * Dv, B * H
    assert hip.lib().ic_lattn_ws(ctypes.byref(a), 0, ctypes.byref(n)) == 0 and n.value == (bh * fwd[0] * dd if fwd[0] > 1 else 0)
    want = max(bh * s[0] * (2 * lag + (dd * (1 + lag) if s[0] > 1 else 0)) for lag, s in ((1, q), (0, q0)))
    want += (bh * kv[0] * dd if kv[0] > 1 else 0) + 2 + (B * Hk * T * (Dk + Dv) + 8 if H != Hk else 0)
    assert hip.lib().ic_lattn_ws(ctypes.byref(a), 1, ctypes.byref(n)) == 0 and n.value == want
    return fwd, q, kv


@pytest.mark.parametrize("dtype", list(TYPES))
def test_the_cases_are_cut_into_segments_of_several_chunks(dtype):
    for c in CASES:
        for s in check_split(*c[:6], TYPES[dtype]):
            assert s[0] > 1 and s[1] > 1, (c, s)


def lengths(B, T, cps):
    """Ends in the first, in middle and in the last segment, at their borders and next to them; none and all."""
    seg = 64 * cps
    at = [T, 1, seg, seg + 1, seg - 1, 2 * seg - 70, T - 1, 0, 2 * seg, seg + seg // 2, T - 64, 63, 64, 65, T // 2, 2 * seg + 1]
    return [max(0, min(T, at[i % len(at)])) for i in range(B)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("i", range(len(CASES)))
def test_segments_of_several_chunks_forward_and_backward(i, dtype):
    from ironcortex_amd.hip import ops
    B, T, H, Hk, Dk, Dv, how = CASES[i]
    dt = TYPES[dtype]
    fwd, _, _ = check_split(B, T, H, Hk, Dk, Dv, dt)
    g = torch.Generator(device=DEV).manual_seed(80 + i)
    q, k, v = (x.requires_grad_(True) for x in inputs(g, dt, B, T, H, Hk, Dk, Dv, how))
    rate = torch.exp(torch.linspace(math.log(1e-4), math.log(2.0), H, device=DEV)).requires_grad_(True)
    state = torch.randn(B, H, Dk, Dv, generator=g, device=DEV).requires_grad_(True)
    scale, n = float(torch.tensor(Dk ** -0.5)), lengths(B, T, fwd[1])
    go, gs = torch.randn(B, H, T, Dv, generator=g, device=DEV).to(dt), torch.randn(B, H, Dk, Dv, generator=g, device=DEV)
    with torch.no_grad():  # what lies in padded rows does not matter
        for b in range(B):
            for x in (q, k, v, go):
                x[b, :, n[b]:] = float("nan")
    leaves = (q, k, v, rate, state)
    y = ops.linear_attention(q, k, v, rate, scale=scale, state=state, valid_len=torch.tensor(n, device=DEV))
    got = [x.detach() for x in (*y, *torch.autograd.grad(y, leaves, (go, gs)))]
    N, f = Dk + Dv + 160 + T / 64, torch.finfo(dt)

    def one(b, size):
        """Outputs and gradients of one sequence's valid rows; of the absolute values: their sizes."""
        x = [t.detach()[b, :, :n[b]].double() for t in (q, k, v)] + [state.detach()[b].double()]
        gob, gsb = go[b, :, :n[b]].double(), gs[b].double()
        if size:
            x, gob, gsb = [t.abs() for t in x], gob.abs(), gsb.abs()
        x = [t.requires_grad_(True) for t in (*x[:3], rate.detach().double(), x[3])]
        o, s = pairs64(x[0], x[1].repeat_interleave(H // Hk, 0), x[2].repeat_interleave(H // Hk, 0), x[3], scale, x[4])
        return [t.detach() for t in (o, s, *torch.autograd.grad((o, s), x, (gob, gsb)))]

    names = ("out", "state", "dq", "dk", "dv", "d rate", "d state")
    drate, asize = torch.zeros(H, device=DEV, dtype=torch.float64), torch.zeros(H, device=DEV, dtype=torch.float64)
    for b in range(B):
        want, size = one(b, False), one(b, True)
        for j, nm in enumerate(names):
            if nm == "d rate":
                drate += want[j]
                asize += size[j].abs()
                continue
            rows = nm in ("out", "dq", "dk", "dv")
            a = got[j][b, :, :n[b]] if rows else got[j][b]
            e = 4 * math.sqrt(N + (8 * (H // Hk) if nm in ("dk", "dv") else 0)) * U * size[j]
            if rows:
                e = e + (want[j].abs() + e) * f.eps / 2 + f.tiny * f.eps / 2
                assert not bool((got[j][b, :, n[b]:] != 0).any()), f"{nm}: padded rows of sequence {b}"
            within(a, want[j], e + 1e-300, f"{CASES[i]} {dtype} sequence {b} of {n[b]}: {nm}")
    within(got[5], drate, 4 * math.sqrt(N + 64) * U * asize, f"{CASES[i]} {dtype} d rate")
