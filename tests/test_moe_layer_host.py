"""Refusals of fni8_moe_layer_w8a8 and moe.layer on the host (no GPU)."""
import pytest
import torch


def test_c_abi_refusals():
    from fni8 import _native as n

    L = n.lib()
    p = 1 << 20

    def call(x=p, dt=n.F16, T=2, H=64, logits=p, k=2, scoring=0, ng=0, tg=0, w=p, E=4, I=32, act=0, out=p, ws=p,
             wsb=1 << 30):
        return L.fni8_moe_layer_w8a8(x, dt, T, H, logits, k, scoring, None, ng, tg, 1, 1.0, w, p, p, p, E, I, act, out,
                                     ws, wsb, None)

    assert call(dt=n.F32) == n.ERR_INVALID and call(T=-1) == n.ERR_INVALID and call(H=0) == n.ERR_INVALID
    assert call(k=0) == n.ERR_INVALID and call(k=5) == n.ERR_INVALID and call(k=33, E=64) == n.ERR_INVALID
    assert call(scoring=2) == n.ERR_INVALID and call(act=2) == n.ERR_INVALID
    assert call(ng=3, tg=1) == n.ERR_INVALID and call(ng=2, tg=3) == n.ERR_INVALID and call(ng=2, tg=0) == n.ERR_INVALID
    assert call(E=513) == n.ERR_UNSUPPORTED and call(E=2000) == n.ERR_INVALID
    assert call(H=72) == n.ERR_UNSUPPORTED and call(I=40) == n.ERR_UNSUPPORTED
    for name in ("x", "logits", "w", "out"):
        assert call(**{name: None}) == n.ERR_INVALID, name
    assert call(ws=None) == n.ERR_WORKSPACE and call(wsb=64) == n.ERR_WORKSPACE and call(ws=p + 128) == n.ERR_ALIGN
    assert call(T=0, x=None) == n.OK
    assert L.fni8_moe_layer_workspace_bytes(0, 64, 2, 4, 32) == 0
    assert L.fni8_moe_layer_workspace_bytes(2, 64, 2, 4, 32) > L.fni8_moe_experts_workspace_bytes(2, 64, 2, 4, 32)


def test_python_refuses_cpu_tensors():
    from fni8 import moe

    stack = moe.ExpertStack(torch.zeros(4, 64, 64, dtype=torch.int8), torch.ones(4, 64),
                            torch.zeros(4, 64, 32, dtype=torch.int8), torch.ones(4, 64))
    with pytest.raises(RuntimeError):
        moe.layer(torch.zeros(2, 64, dtype=torch.float16), torch.zeros(2, 4), stack, 2)
