"""Autograd nodes of the token operators of image / video encoders (csrc/token_norm.hip, rotary.hip, attention*.hip): residual RMS norm,
rotary positions over several axes, attention with capped scores, distance bias, document and prefix masks.  nnops holds the public
functions; here: the argument blocks, output and scratch memory, the launches.

float32, bfloat16 and float16 tensors.  Every call runs on the current stream of its tensors' device."""
import contextlib
import ctypes

import torch

from . import lib as _l
from .ops import _ptr, _stream

DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}          # SQD_F32 | SQD_BF16 | SQD_F16
_SAME = contextlib.nullcontext()
_current = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def on_device(t):
    """the launches of a call go to the device its tensors live on, whichever device is current"""
    return _SAME if t.get_device() == _current() else torch.cuda.device(t.device)


def _rows16(t):
    """t [B,S,H,D] with features dense, every other stride and the address in whole 16-byte pieces, the tokens' stride below 2^22 elements and
    the heads' times their number below 2^28: itself, or a copy"""
    n = 16 // t.element_size()
    if t.numel() == 0:
        return t
    (b, s, h, e), (B, S, H, _) = t.stride(), t.shape
    if (e == 1 and t.data_ptr() % 16 == 0 and (B == 1 or b % n == 0) and (S == 1 or (s % n == 0 and 0 <= s < 1 << 22))
            and (H == 1 or (h % n == 0 and 0 <= h * H < 1 << 28))):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    """element strides of batch, token and head; 0 where there is one only"""
    (b, s, h, _), (B, S, H, _) = t.stride(), t.shape
    return (b if B > 1 else 0, s if S > 1 else 0, h if H > 1 else 0)


# ------------------------------------------------------------------------------------------------------------------ residual RMS norm
def _norm_fwd(x, w, res, eps, want_rstd):
    C = x.shape[-1]
    rows = x.numel() // C
    x = x.contiguous()
    y = torch.empty_like(x)
    s = torch.empty_like(x) if res is not None else x
    rstd = torch.empty(rows, device=x.device, dtype=torch.float32) if want_rstd else None
    if res is not None:
        res = res.contiguous()
    _l.check(_l.lib().sqd_rms_norm_fwd(x.data_ptr(), _ptr(res), w.data_ptr(), y.data_ptr(), s.data_ptr() if res is not None else None, _ptr(rstd), rows, C,
                                       eps, DTYPE[x.dtype], DTYPE[w.dtype], _stream()), "rms_norm_fwd")
    return y, s, rstd


class RmsNormResidual(torch.autograd.Function):
    """forward(x, w, res or None, eps) -> y, stream (res None: y alone)"""

    @staticmethod
    def forward(ctx, x, w, res, eps):
        with on_device(x):
            w = w.contiguous()
            y, s, rstd = _norm_fwd(x, w, res, eps, True)
        ctx.save_for_backward(s, w, rstd)
        ctx.set_materialize_grads(False)
        ctx.residual = res is not None
        return (y, s) if res is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, gs=None):
        s, w, rstd = ctx.saved_tensors
        if gy is None:                                     # only the stream was used
            return gs, None, gs if ctx.residual else None, None
        C = s.shape[-1]
        rows = s.numel() // C
        L = _l.lib()
        with on_device(s):
            gy = gy.contiguous()
            gs = gs.contiguous() if gs is not None else None
            gx, gw = torch.empty_like(s), torch.empty_like(w)
            part = torch.empty(L.sqd_rms_norm_nblk(rows) * C, device=s.device, dtype=torch.float32)
            _l.check(L.sqd_rms_norm_bwd(gy.data_ptr(), _ptr(gs), s.data_ptr(), w.data_ptr(), rstd.data_ptr(), gx.data_ptr(), gw.data_ptr(), part.data_ptr(),
                                        rows, C, DTYPE[s.dtype], DTYPE[w.dtype], _stream()), "rms_norm_bwd")
        return gx, gw, gx if ctx.residual else None, None


# ------------------------------------------------------------------------------------------------------------------------------ rotary
class RotaryArgs(ctypes.Structure):
    """struct sqd_rotary_args (include/sqd.h)."""
    _P, _L, _I = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
    _fields_ = [("q", _P), ("k", _P), ("q_out", _P), ("k_out", _P), ("pos", _P), ("freq", _P), ("stream", _P),
                ("q_stride", _L * 3), ("k_stride", _L * 3), ("pos_batch_stride", _L), ("pairs", _I * 4),
                ("B", _I), ("S", _I), ("Hq", _I), ("Hk", _I), ("D", _I), ("axes", _I), ("pos_bytes", _I), ("interleaved", _I),
                ("inverse", _I), ("dtype", _I)]


def _rotate(q, k, pos, freq, pairs, interleaved, inverse):
    B, S, Hq, D = q.shape
    with on_device(q):
        q, k = _rows16(q), _rows16(k) if k is not None else None
        qo = torch.empty((B, S, Hq, D), device=q.device, dtype=q.dtype)
        ko = torch.empty(k.shape, device=q.device, dtype=q.dtype) if k is not None else None
        a = RotaryArgs(q.data_ptr(), _ptr(k), qo.data_ptr(), _ptr(ko), pos.data_ptr(), freq.data_ptr(), _stream(), _strides(q),
                       _strides(k) if k is not None else (0, 0, 0), pos.stride(0) if pos.dim() == 3 else 0, pairs, B, S, Hq,
                       k.shape[2] if k is not None else 0, D, len(pairs), pos.element_size(), interleaved, inverse, DTYPE[q.dtype])
        _l.check(_l.lib().sqd_rotary_axes(ctypes.byref(a)), "rotary_axes")
    return qo, ko


class RotaryAxes(torch.autograd.Function):
    """forward(q, k or None, pos, freq, pairs, interleaved) -> q', k' (k None: q' alone)"""

    @staticmethod
    def forward(ctx, q, k, pos, freq, pairs, interleaved):
        ctx.save_for_backward(pos, freq)
        ctx.cfg = (pairs, interleaved, q.shape, None if k is None else k.shape)
        ctx.set_materialize_grads(False)
        qo, ko = _rotate(q, k, pos, freq, pairs, interleaved, 0)
        return qo if k is None else (qo, ko)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk=None):
        pos, freq = ctx.saved_tensors
        pairs, interleaved = ctx.cfg[:2]
        if gq is None and gk is None:
            return None, None, None, None, None, None
        if gq is None:
            return None, _rotate(gk, None, pos, freq, pairs, interleaved, 1)[0], None, None, None, None
        gq, gk = _rotate(gq, gk, pos, freq, pairs, interleaved, 1)
        return gq, gk, None, None, None, None


# --------------------------------------------------------------------------------------------------------------------------- attention
class AttnArgs(ctypes.Structure):
    """struct sqd_attn_args (include/sqd.h)."""
    _P, _L, _I, _F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float
    _fields_ = [("q", _P), ("k", _P), ("v", _P), ("go", _P), ("o", _P), ("o_low", _P), ("gq", _P), ("gk", _P), ("gv", _P), ("lse", _P), ("scratch", _P),
                ("slopes", _P), ("prefix", _P), ("q_docs", _P), ("k_docs", _P), ("k_len", _P), ("stream", _P),
                ("q_stride", _L * 3), ("k_stride", _L * 3), ("v_stride", _L * 3), ("go_stride", _L * 3), ("scale", _F), ("softcap", _F),
                ("B", _I), ("Sq", _I), ("Sk", _I), ("Hq", _I), ("Hkv", _I), ("D", _I), ("causal", _I), ("dtype", _I)]


def _attn_args(q, k, v, cfg, masks, out, go=None):
    """the argument block; out = (o, o_low, gq, gk, gv, lse, scratch), masks = (slopes, prefix, q_docs, k_docs, k_len)"""
    B, Sq, Hq, D = q.shape
    o, o_low, gq, gk, gv, lse, scratch = [_ptr(t) for t in out]
    return AttnArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(go), o, o_low, gq, gk, gv, lse, scratch, *[_ptr(m) for m in masks], _stream(),
                    _strides(q), _strides(k), _strides(v), _strides(go) if go is not None else (0, 0, 0), cfg[0], cfg[1], B, Sq, k.shape[1], Hq,
                    k.shape[2], D, cfg[2], DTYPE[q.dtype])


def attn_fwd(q, k, v, cfg, masks, want_lse):
    """-> o [B,Sq,Hq,D]; for the backward (want_lse): what its rounding left (16-bit types) and lse [B,Hkv,Sq*G], else None.
    cfg = (scale, softcap, causal), masks = (slopes, prefix, q_docs, k_docs, k_len)"""
    L = _l.lib()
    o = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    low = lse = None
    if want_lse:
        lse = torch.empty((q.shape[0], k.shape[2], q.shape[1] * (q.shape[2] // k.shape[2])), device=q.device, dtype=torch.float32)
        if o.dtype != torch.float32:
            low = torch.empty_like(o)
    a = _attn_args(q, k, v, cfg, masks, (o, low, None, None, None, lse, None))
    n = L.sqd_attn_fwd_scratch(ctypes.byref(a))
    if n > 0:
        scratch = torch.empty(n, device=q.device, dtype=torch.float32)
        a.scratch = scratch.data_ptr()
    _l.check(L.sqd_attn_fwd(ctypes.byref(a)), "attn_fwd")
    return o, low, lse


class Attention(torch.autograd.Function):
    """forward(q, k, v, cfg, slopes, prefix, q_docs, k_docs, k_len) -> o"""

    @staticmethod
    def forward(ctx, q, k, v, cfg, *masks):
        with on_device(q):
            q, k, v = _rows16(q), _rows16(k), _rows16(v)
            o, low, lse = attn_fwd(q, k, v, cfg, masks, True)
        ctx.save_for_backward(q, k, v, o, low, lse, *masks)
        ctx.cfg = cfg
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, go):
        q, k, v, o, low, lse, *masks = ctx.saved_tensors
        L = _l.lib()
        with on_device(q):
            go = _rows16(go)
            want_q, want_kv = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
            gq = torch.empty(q.shape, device=q.device, dtype=q.dtype) if want_q else None
            gk, gv = (torch.empty(t.shape, device=q.device, dtype=q.dtype) if want_kv else None for t in (k, v))
            a = _attn_args(q, k, v, ctx.cfg, masks, (o, low, gq, gk, gv, lse, None), go)
            scratch = torch.empty(max(4, L.sqd_attn_bwd_scratch(ctypes.byref(a))), device=q.device, dtype=torch.float32)
            a.scratch = scratch.data_ptr()
            _l.check(L.sqd_attn_bwd(ctypes.byref(a)), "attn_bwd")
        return (gq, gk, gv) + (None,) * 6
