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
