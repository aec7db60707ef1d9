"""Token operators without a GPU: host tensors are refused, the C entry points refuse bad arguments before they touch the device, the argument
blocks have the C layout, and the 64-bit references that the GPU tests use agree with autograd."""
import ctypes
import math
import re
import os

import pytest
import torch

from isa_waits import LLVM, functions, short_waits
from token_refs import attention_ref, norm_ref, rotary_ref

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_host_tensors_are_refused():
    from sqd import nnops
    x, q = torch.zeros(4, 8), torch.zeros(1, 2, 1, 8)
    for call in (lambda: nnops.rms_norm_residual(x, torch.ones(8)), lambda: nnops.rotary_axes(q, q, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(4).double(), (4,)),
                 lambda: nnops.attention(q, q, q)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_argument_blocks_have_the_c_layout(tmp_path):
    """sizes and offsets of the ctypes structures against a C compiler's"""
    import subprocess
    from sqd import tokens
    src, lines = tmp_path / "layout.c", []
    for cls, name in ((tokens.RotaryArgs, "sqd_rotary_args"), (tokens.AttnArgs, "sqd_attn_args")):
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (name, f[0]) for f in cls._fields_]
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "%s"\nint main(void) { %s return 0; }\n' % (os.path.join(REPO, "include", "sqd.h"), " ".join(lines)))
    exe = str(tmp_path / "layout")
    subprocess.check_call(["gcc", str(src), "-o", exe])
    got = [int(t) for t in subprocess.check_output([exe], text=True).split()]
    want = []
    for cls in (tokens.RotaryArgs, tokens.AttnArgs):
        want.append(ctypes.sizeof(cls))
        want += [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want


def _attn(**kw):
    from sqd import tokens
    a = tokens.AttnArgs()
    for n in ("q", "k", "v", "o", "go", "gq", "gk", "gv", "lse", "scratch"):
        setattr(a, n, 4096)                                     # never read: the checks come first
    a.B, a.Sq, a.Sk, a.Hq, a.Hkv, a.D, a.scale, a.dtype = 1, 4, 4, 2, 1, 16, 0.25, 1
    for s in (a.q_stride, a.k_stride, a.v_stride, a.go_stride):
        s[:] = [128, 32, 16]
    for n, v in kw.items():
        if n.endswith("_stride"):
            getattr(a, n)[:] = v
        else:
            setattr(a, n, v)
    return a


@pytest.mark.parametrize("bad", [dict(D=12), dict(D=136), dict(D=0), dict(Hq=3, Hkv=2), dict(Hkv=0), dict(B=-1), dict(scale=0.0), dict(scale=math.nan),
                                 dict(softcap=-1.0), dict(dtype=3), dict(prefix=4096), dict(q_docs=4096), dict(q=None), dict(k=None), dict(q=4097),
                                 dict(v_stride=[128, 33, 16]), dict(o=None), dict(Sk=1 << 24)])
def test_c_attention_refuses(bad):
    from sqd import lib
    L = lib.lib()
    a = _attn(**bad)
    assert L.sqd_attn_fwd(ctypes.byref(a)) == -1 and L.sqd_last_error()
    if "o" not in bad:
        assert L.sqd_attn_bwd(ctypes.byref(a)) == -1
    assert L.sqd_attn_fwd(None) == -1 and L.sqd_attn_bwd(None) == -1 and L.sqd_attn_fwd_scratch(None) == -1


def test_c_empty_calls_do_nothing():
    from sqd import lib
    L = lib.lib()
    a = _attn(B=0, q=None, k=None, v=None, o=None)
    assert L.sqd_attn_fwd(ctypes.byref(a)) == 0 and L.sqd_attn_bwd(ctypes.byref(a)) == 0 and L.sqd_attn_fwd_scratch(ctypes.byref(a)) == 0
    assert L.sqd_rms_norm_fwd(None, None, None, None, None, None, 0, 8, 1e-6, 0, 0, None) == 0


def test_c_norm_and_rotary_refuse():
    from sqd import lib, tokens
    L = lib.lib()
    p = 4096
    for args in ((p, None, p, p, None, None, 2, 0, 1e-6, 0, 0), (p, None, p, p, None, None, -1, 8, 1e-6, 0, 0), (p, p, p, p, None, None, 2, 8, 1e-6, 0, 0),
                 (p, None, p, p, None, None, 2, 8, 1e-6, 7, 0), (p, None, p, p, None, None, 2, 8, 1e-6, 1, 2), (None, None, p, p, None, None, 2, 8, 1e-6, 0, 0),
                 (p, None, p, p, None, None, 2, 8, -1.0, 0, 0)):
        assert L.sqd_rms_norm_fwd(*args, None) == -1
    assert L.sqd_rms_norm_bwd(p, None, p, p, None, p, p, p, 2, 8, 0, 0, None) == -1

    def rot(**kw):
        a = tokens.RotaryArgs()
        a.q = a.k = p
        a.q_out = a.k_out = 8192
        a.pos = a.freq = p
        a.B, a.S, a.Hq, a.Hk, a.D, a.axes, a.pos_bytes = 1, 2, 1, 1, 8, 1, 4
        a.pairs[0] = 4
        a.q_stride[:] = a.k_stride[:] = [16, 8, 8]
        for n, v in kw.items():
            setattr(a, n, v)
        return L.sqd_rotary_axes(ctypes.byref(a))
    for bad in (dict(axes=0), dict(axes=5), dict(D=6), dict(D=7), dict(pos_bytes=2), dict(q=None), dict(q_out=p), dict(freq=None), dict(dtype=9), dict(D=2048),
                dict(q=p + 2, interleaved=1), dict(B=-1)):
        assert rot(**bad) == -1, bad
    assert rot(B=0) == 0 and L.sqd_rotary_axes(None) == -1


def test_references_agree_with_autograd():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float32)                                             # noqa: E731
    x, res, w, gy, gs = r(5, 12), r(5, 12), r(12), r(5, 12), r(5, 12)
    e = [t.double().requires_grad_(True) for t in (x, res, w)]
    s = (e[0] + e[1])
    y = s * torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + 1e-6) * e[2]
    want = torch.autograd.grad((y, s), e, (gy.double(), gs.double()))
    ref = norm_ref(x, w, res, 1e-6, gy, gs)
    # (the reference rounds the stream to fp32)
    assert torch.allclose(ref["y"], y, rtol=1e-6, atol=1e-6) and torch.allclose(ref["gx"], want[0], rtol=1e-5, atol=1e-6) and torch.allclose(ref["gw"], want[2], atol=1e-5)

    q, k, v, go = r(2, 6, 4, 8), r(2, 9, 2, 8), r(2, 9, 2, 8), r(2, 6, 4, 8)
    kw = dict(softcap=2.0, slopes=torch.tensor([0.5, 0.1, 0.2, 0.0]), causal=True, prefix=torch.tensor([2, 0], dtype=torch.int32),
              k_len=torch.tensor([9, 4], dtype=torch.int32))
    ref = attention_ref(q, k, v, go=go, **kw)
    e = [t.double().requires_grad_(True) for t in (q, k, v)]
    k2, v2 = e[1].repeat_interleave(2, 2), e[2].repeat_interleave(2, 2)
    z = 2 * torch.tanh(torch.einsum("bihd,bjhd->bhij", e[0], k2) / math.sqrt(8) / 2)
    rows = []
    for b, n in enumerate((9, 4)):
        pos = torch.arange(6)[:, None] + n - 6
        j = torch.arange(9)[None]
        see = (j < n) & ((j <= pos) | (j < int(kw["prefix"][b])))
        zz = z[b] - kw["slopes"].double().view(4, 1, 1) * (pos - j).abs()
        p = torch.softmax(zz.masked_fill(~see, -1e30), -1) * see
        rows.append(torch.einsum("hij,jhd->ihd", p, v2[b]))
    o = torch.stack(rows)
    assert torch.allclose(o, ref["o"], atol=1e-12)
    for name, want in zip(("gq", "gk", "gv"), torch.autograd.grad(o, e, go.double())):
        assert torch.allclose(ref[name], want, atol=1e-12), name

    pos = torch.tensor([[0, 3], [1, -2]])
    out, _ = rotary_ref(q[:, :2], pos, torch.tensor([1.0, 0.5, 0.25]).double(), (1, 2))
    a = 3 * 0.5
    assert abs(float(out[0, 0, 0, 1]) - (float(q[0, 0, 0, 1]) * math.cos(a) - float(q[0, 0, 0, 4]) * math.sin(a))) < 1e-12


def test_frequency_tables():
    from sqd import nnops
    f = nnops.rotary_frequencies((2, 4), 16.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.25, 1.0, 0.5, 0.25, 0.125]).double())
    assert torch.allclose(nnops.rotary_frequencies((1, 3), 16.0, shared=True, device="cpu"), torch.tensor([1.0, 0.5, 0.25, 0.125]).double())


def test_wait_counter():
    """the way through the branch is the short one; an accumulation chain needs no wait; a filled wait is none too short"""
    mfma = "v_mfma_f32_32x32x16_bf16 a[0:15], v[0:3], v[4:7], a[0:15]"
    use = "v_accvgpr_read_b32 v9, a15"
    long_way = ["v_mov_b32_e32 v20, v21"] * 8
    (n, want, _, _), = short_waits([mfma, "s_cbranch_vccnz L1"] + long_way + ["L1:", "s_nop 3", use])
    assert (n, want) == (5, 12)
    assert not short_waits([mfma, "s_nop 11", "s_cbranch_vccnz L1"] + long_way + ["L1:", use])
    assert not short_waits([mfma, mfma, "s_nop 7", "s_nop 3", use]) and short_waits([mfma, mfma, "s_nop 7", "s_nop 2", use])
    assert short_waits(["L0:", use, mfma, "s_cbranch_scc1 L0", "s_endpgm"])
    assert short_waits([mfma, "s_nop 2", "v_mfma_f32_32x32x16_bf16 a[16:31], a[0:3], v[4:7], a[16:31]"])


@pytest.mark.parametrize("source", ["attention", "attention_bwd"])
def test_results_of_matrix_instructions_are_waited_for(source, tmp_path):
    """every way from a product to its use in the built kernels (the values cannot show it: which elements come early depends on the neighbours)"""
    from sqd import lib
    obj = os.path.join(lib.OBJ_DIR, source + ".o")
    if not (os.path.exists(obj) and os.path.exists(LLVM)):
        pytest.skip("no object file of this source, or no disassembler")
    code = functions(obj, str(tmp_path))
    assert sum(any(line.lstrip().startswith("v_mfma") for line in c) for c in code.values()) > 20
    bad = {name: short_waits(c) for name, c in code.items()}
    assert not any(bad.values()), {name: b[:2] for name, b in bad.items() if b}
