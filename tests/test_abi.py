"""CPU checks of the C-ABI boundary: the library loads, exports every symbol declared in
include/ironcortex_hip.h, and the ctypes struct layouts equal the C compiler's."""
import ctypes
import os
import subprocess
import sys

import pytest

from ironcortex_amd import hip


def test_library_exports_every_declared_symbol():
    lib = hip.lib()
    assert len(hip.FUNCTIONS) >= 19
    for fn in hip.FUNCTIONS:
        assert hasattr(lib, fn), fn
    assert lib.ic_version() >= 1
    assert lib.ic_bwd_nslab(256) == 8 and lib.ic_bwd_nslab(512) == 64


def test_struct_layouts_match_c(tmp_path):
    names = sorted(hip.CLASSES)
    src = tmp_path / "sz.c"
    body = "".join(f'printf("{n} %zu\\n", sizeof({n}));' for n in names)
    src.write_text('#include <stdio.h>\n#include "ironcortex_hip.h"\nint main(){' + body + "return 0;}")
    exe = tmp_path / "sz"
    inc = os.path.dirname(hip.HEADER_PATH)
    subprocess.check_call(["gcc", "-I", inc, str(src), "-o", str(exe)])
    out = dict(line.split() for line in subprocess.check_output([str(exe)], text=True).splitlines())
    for n in names:
        assert int(out[n]) == ctypes.sizeof(hip.CLASSES[n]), n


def test_errors_are_reported_not_thrown():
    lib = hip.lib()
    rc = lib.ic_kwta_fwd(None, None, None, 1, 256, 4, 0, ctypes.c_float(1.0), None)
    assert rc == hip.ENUMS["IC_EINVAL"]
    assert b"NULL" in lib.ic_last_error()
    a = hip.new("ic_region_args", S=1, R=1, d=6)
    assert lib.ic_region_phase_fwd(ctypes.byref(a), None) == hip.ENUMS["IC_EINVAL"]
    assert b"d=6" in lib.ic_last_error()


def test_ops_refuse_cpu_tensors():
    import torch
    from ironcortex_amd.utils import KWTA
    with pytest.raises(RuntimeError):
        KWTA(torch.randn(2, 8), 2)


def _flat(obj, prefix=""):
    for name, ct in obj._fields_:
        v = getattr(obj, name)
        if isinstance(v, ctypes.Structure):
            yield from _flat(v, prefix + name + "_")
        else:
            yield prefix + name, v or 0


def test_packed_structs_equal_the_assigned_ones():
    """hip.packer: the same bytes as setting every field of the ctypes structure."""
    def fill(obj, kw, n):
        for name, ct in obj._fields_:
            if isinstance(ct, type) and issubclass(ct, ctypes.Structure):
                n = fill(getattr(obj, name), kw, n)
            else:
                n += 1
                setattr(obj, name, n)
                kw.append(n)
        return n

    for s in ("ic_rope_args", "ic_rope_bwd_args", "ic_lattn_args", "ic_lattn_bwd_args", "ic_lattn_step_args"):
        obj, kw = hip.CLASSES[s](), []
        fill(obj, kw, 0)
        pack, names = hip.packer(s)
        assert pack(*kw) == bytes(obj) and names == [n for n, _ in _flat(obj)], s


def test_token_mixing_ops_pack_every_value_under_its_name(monkeypatch):
    """What the ops of the rotation and of linear attention hand to the C entries, decoded by the header's field names."""
    import torch
    from ironcortex_amd.hip import ops
    got = []
    monkeypatch.setattr(ops, "_launch", lambda name, blob, device: got.append((name, blob)))
    B, H, Hk, T, D, m = 2, 6, 3, 5, 16, 4

    def last(struct):
        return dict(_flat(hip.CLASSES[struct].from_buffer_copy(got[-1][1])))

    def strides(f, n, t):
        return (f[n + "_sb"], f[n + "_sh"], f[n + "_st"]) == t.stride()[:3]

    q, k = torch.randn(B, T, H, D).transpose(1, 2), torch.randn(B, T, Hk, D).transpose(1, 2)
    w, wk = torch.randn(D), torch.randn(D).bfloat16()
    pos, fr = torch.arange(B * T).view(B, T), torch.rand(m, dtype=torch.float64)
    cos, sin = torch.rand(B, T, m), torch.rand(B, T, m)
    monkeypatch.setattr(ops, "_same_device", lambda *a, **kw: None)
    yq, yk = ops.qk_norm_rope(q, k, w, w, eps=0.25, positions=pos, freqs=fr, layout="half", scale=1.5)
    f = last("ic_rope_args")
    assert got[-1][0] == "ic_rope_fwd"
    assert [f[n] for n in ("B", "T", "D", "m", "dtype", "layout", "inverse", "pos64", "freq64", "scale", "eps", "cos", "sin", "cs_sb", "pos_sb")] == [
        B, T, D, m, 0, 1, 0, 1, 1, 1.5, 0.25, 0, 0, 0, T]
    assert f["positions"] == pos.data_ptr() and f["freqs"] == fr.data_ptr() and f["q_w"] == f["k_w"] == w.data_ptr()
    assert (f["q_x"], f["q_y"], f["q_H"], f["k_x"], f["k_y"], f["k_H"]) == (q.data_ptr(), yq.data_ptr(), H, k.data_ptr(), yk.data_ptr(), Hk)
    assert strides(f, "q_x", q) and strides(f, "q_y", yq) and strides(f, "k_x", k) and strides(f, "k_y", yk)
    y = ops.rope(q.bfloat16(), cos=cos, sin=sin)
    f = last("ic_rope_args")
    assert (f["cos"], f["sin"], f["cs_sb"], f["freqs"], f["positions"], f["k_H"], f["dtype"], f["q_y"]) == (cos.data_ptr(), sin.data_ptr(), T * m, 0, 0, 0, 1, y.data_ptr())
    qg, wg = q.clone().requires_grad_(True), w.clone().requires_grad_(True)
    out = ops.qk_norm_rope(qg, k, wg, w, freqs=fr)
    gq, gk = torch.randn(B, H, T, D), torch.randn(B, Hk, T, D)
    dq, dw = torch.autograd.grad(out, (qg, wg), (gq, gk))
    f = last("ic_rope_bwd_args")
    assert got[-1][0] == "ic_rope_bwd" and (f["q_g"], f["k_g"], f["f_q_x"], f["f_k_x"], f["f_q_w"]) == (gq.data_ptr(), gk.data_ptr(), qg.data_ptr(), k.data_ptr(), wg.data_ptr())
    assert (f["q_gx"], f["q_gw"]) == (dq.data_ptr(), dw.data_ptr()) and strides(f, "q_g", gq) and strides(f, "q_gx", dq) and strides(f, "k_g", gk) and f["part"]

    v = torch.randn(B, T, Hk, 8).transpose(1, 2)
    rate, st, vl = torch.rand(H, requires_grad=True), torch.randn(B, H, D, 8, requires_grad=True), torch.ones(B, dtype=torch.int32)
    o, so = ops.linear_attention(q, k, v, rate, scale=0.5, state=st, valid_len=vl)
    f = last("ic_lattn_args")
    assert [f[n] for n in ("B", "H", "Hk", "T", "Dk", "Dv", "dtype", "scale")] == [B, H, Hk, T, D, 8, 0, 0.5]
    assert [f[n] for n in ("q", "k", "v", "rate", "valid_len", "state", "out", "state_out")] == [
        t.data_ptr() for t in (q, k, v, rate, vl, st, o, so)]
    assert strides(f, "q", q) and strides(f, "k", k) and strides(f, "v", v) and strides(f, "o", o)
    go, gs = torch.randn(B, T, H, 8).transpose(1, 2), torch.randn(B, H, D, 8)
    dr, ds = torch.autograd.grad((o, so), (rate, st), (go, gs))
    f = last("ic_lattn_bwd_args")
    assert got[-1][0] == "ic_lattn_bwd" and [f[n] for n in ("dout", "dstate_out", "drate", "dstate", "f_q", "f_state")] == [
        t.data_ptr() for t in (go, gs, dr, ds, q, st)]
    assert strides(f, "do", go) and all((f[n + "_sb"], f[n + "_sh"], f[n + "_st"]) == t.stride()[:3] and f[n] for n, t in (("dq", q), ("dk", k), ("dv", v)))
    s = st.detach()
    act = torch.ones(B, dtype=torch.bool)
    qt, kt, vt = q[:, :, 0], k[:, :, 1], v[:, :, 2]
    with torch.no_grad():
        o = ops.linear_attention_step(qt, kt, vt, rate, s, scale=0.25, active=act)
    f = last("ic_lattn_step_args")
    assert [f[n] for n in ("B", "H", "Hk", "Dk", "Dv", "dtype", "scale")] == [B, H, Hk, D, 8, 0, 0.25]
    assert [f[n] for n in ("q", "k", "v", "rate", "active", "state", "out")] == [t.data_ptr() for t in (qt, kt, vt, rate, act, s, o)]
    assert all((f[n + "_sb"], f[n + "_sh"]) == t.stride()[:2] for n, t in (("q", qt), ("k", kt), ("v", vt), ("o", o)))
