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
