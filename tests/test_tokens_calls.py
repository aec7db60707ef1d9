"""What the token operators refuse or take before any launch, without a GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwd


def test_tangents_are_noticed():
    from sqd import nnops
    x = torch.ones(3)
    nnops._refuse_tangents("op", x, None)
    with fwd.dual_level():
        nnops._refuse_tangents("op", x, None)
        with pytest.raises(RuntimeError, match="sqd: op: forward-mode"):
            nnops._refuse_tangents("op", None, x, fwd.make_dual(x, x))

    def f(t):
        nnops._refuse_tangents("op", t)
        return t
    with pytest.raises(RuntimeError, match="sqd: op: forward-mode"):
        torch.func.jvp(f, (x,), (x,))


def test_c_sizes_past_a_launch_are_refused():
    """counters of a kernel and threads of a launch are 32-bit: what does not fit is refused before any launch"""
    import ctypes
    from sqd import lib
    from test_tokens_host import _attn
    L, p = lib.lib(), 4096
    for C in (2 ** 31 - 8, 2 ** 27 + 1):
        assert L.sqd_rms_norm_fwd(p, None, p, p, None, None, 1, C, 1e-6, 0, 0, None) == -1
        assert L.sqd_rms_norm_bwd(p, None, p, p, p, p, p, p, 1, C, 0, 0, None) == -1
    assert L.sqd_rms_norm_bwd(p, None, p, p, p, p, p, p, 1 << 24, 9000, 0, 0, None) == -1
    from sqd import tokens
    a = tokens.RotaryArgs()
    a.q = a.pos = a.freq = p
    a.q_out = 8192
    a.B, a.S, a.Hq, a.Hk, a.D, a.axes, a.pos_bytes = 1, 1, 1 << 27, 0, 128, 1, 4
    a.pairs[0] = 64
    assert L.sqd_rotary_axes(ctypes.byref(a)) == -1
    big = dict(B=65535, Hkv=256, Hq=256, D=8, q_stride=[0, 8, 8], k_stride=[0, 8, 8], v_stride=[0, 8, 8], go_stride=[0, 8, 8])
    a = _attn(Sq=129, Sk=1, **big)                      # 2 x 65535 x 256 workgroups
    assert L.sqd_attn_fwd(ctypes.byref(a)) == -1 and L.sqd_attn_bwd(ctypes.byref(a)) == -1
    a = _attn(Sq=1, Sk=1100, **dict(big, B=8192))       # the keys' side of the backward: 9 x 8192 x 256
    assert L.sqd_attn_bwd(ctypes.byref(a)) == -1
