"""What the 16-bit forward leaves for the backward: o and o_low together are the output to more bits than o has, and delta = (o + o_low) . go needs them.
Equal scores make every packed probability exactly representable, so that the output's rounding is the only one."""
import ctypes
import math

import pytest
import torch

from token_refs import F32 as EPS32
from token_refs import HALF, check

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
GRID = {BF16: 2.0 ** -134, F16: 2.0 ** -25}
# many rows; few rows; few rows and many rows whose keys are split over workgroups
SHAPES = [(2, 140, 300, 4, 2, 64), (64, 3, 200, 8, 8, 128), (1, 1, 3000, 4, 1, 128), (1, 200, 2000, 1, 1, 40)]


def _uniform(B, Sq, Sk, Hq, Hkv, D, dtype):
    """equal scores: every key of a head is the same vector"""
    g = torch.Generator().manual_seed(Sq + Sk)
    q = torch.randn(B, Sq, Hq, D, generator=g).to(dtype)
    k = torch.full((B, Sk, Hkv, D), 0.25).to(dtype)
    v = (2.0 + 0.1 * torch.randn(B, Sk, Hkv, D, generator=g)).to(dtype)
    go = torch.randn(B, Sq, Hq, D, generator=g).to(dtype)
    return q, k, v, go


def _forward(q, k, v):
    from sqd import tokens
    cfg, masks = (q.shape[-1] ** -0.5, 0.0, 0), (None,) * 5
    return cfg, masks, tokens.attn_fwd(q, k, v, cfg, masks, True)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_output_and_what_its_rounding_left(shape, dtype):
    """o: half a step.  o + o_low: sums of Sk fp32 terms in any order and their quotient, and half a step of o_low, which is half a step of o at most"""
    q, k, v, _ = _uniform(*shape, dtype)
    _, _, (o, low, lse) = _forward(q.cuda(), k.cuda(), v.cuda())
    B, Sq, Sk, Hq, Hkv, D = shape
    want = v.double().mean(1, keepdim=True).repeat_interleave(Hq // Hkv, 2).expand(B, Sq, Hq, D)
    fine = want.abs() * (EPS32 * (Sk + 32) + 2 * HALF[dtype] ** 2) + GRID[dtype]
    check(o, want, fine + want.abs() * HALF[dtype], "o")
    check(o.double() + low.double(), want, fine, "o + o_low")
    assert float(low.float().abs().max()) > 0
    z = torch.einsum("bihd,bhd->bhi", q.double(), k.double()[:, 0].repeat_interleave(Hq // Hkv, 1)) / math.sqrt(D)
    want_lse = (z / math.log(2.0) + math.log2(Sk)).view(B, Hkv, Hq // Hkv, Sq).transpose(2, 3).reshape(B, Hkv, -1)
    check(lse, want_lse, EPS32 * ((D + 16) * float(z.abs().max() + 16) + Sk + 64) * torch.ones_like(want_lse), "lse")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[1] > 1])
def test_gradients_take_what_the_rounding_left(shape, dtype):
    """the score gradients of a row add up to nothing, and with equal keys so does the queries' gradient: what is left are half steps of dS and fp32 sums.
    An error of delta comes Sk times instead, and it is half a step of o where o_low is missing: 2^8 or 2^11 times half a step of o_low, 16 times
    what fp32 adds (a backward that took no notice of o_low would be off by as much either way)"""
    from sqd import lib, tokens
    q, k, v, go = _uniform(*shape, dtype)
    B, Sq, Sk, Hq, Hkv, D = shape
    d = [t.cuda() for t in (q, k, v)]
    cfg, masks, (o, low, lse) = _forward(*d)
    L, dgo = lib.lib(), go.cuda()
    v64, g64 = v.double().repeat_interleave(Hq // Hkv, 2), go.double()
    dp = torch.einsum("bihd,bjhd->bhij", g64, v64)
    ds = (dp - dp.mean(-1, keepdim=True)).abs() / Sk
    mag = torch.einsum("bihd,bjhd->bhij", g64.abs(), v64.abs()).sum(-1) / Sk                       # what meets in the fp32 sums of a row
    # half a step of each dS (fp16: lifted clear of its grid); dP, delta and the probabilities in fp32; delta: half a step of o_low
    row = HALF[dtype] * ds.sum(-1) + EPS32 * (2 * D + Sk + 64) * 2 * mag + 2 * HALF[dtype] ** 2 * mag + GRID[dtype] * g64.abs().sum(-1).transpose(1, 2)
    tol = D ** -0.5 * 0.25 * row.transpose(1, 2)[..., None].expand(B, Sq, Hq, D) + GRID[dtype]
    worst = []
    for left in (low, None):
        gq, gk, gv = (torch.empty_like(t) for t in d)
        a = tokens._attn_args(*d, cfg, masks, (o, left, gq, gk, gv, lse, None), dgo)
        scratch = torch.empty(max(4, L.sqd_attn_bwd_scratch(ctypes.byref(a))), device="cuda")
        a.scratch = scratch.data_ptr()
        lib.check(L.sqd_attn_bwd(ctypes.byref(a)), "attn_bwd")
        worst.append(float((gq.double().cpu().abs() / tol).max()))
    assert worst[0] <= 1 and worst[1] > 16 * worst[0], worst


@pytest.mark.parametrize("dtype", [torch.float32, BF16, F16])
@pytest.mark.parametrize("std", [0.5, 60.0])
def test_rows_of_one_key_at_any_score(std, dtype):
    """single-token documents inside longer rows: no gradient of the score while it is below 8 in base 2; beyond, P is off by half a unit of the score
    (2^-24 of it, 2^-15 for the scores here) and dP - delta by the roundings of two sums of D products, of o and its quotient"""
    from sqd import nnops
    g = torch.Generator().manual_seed(9)
    B, S, H, D = 2, 150, 2, 128
    q, k, v, go = (torch.randn(B, S, H, D, generator=g) for _ in range(4))
    q, k, v, go = (q * std).to(dtype), k.to(dtype), v.to(dtype), go.to(dtype)
    docs = torch.arange(S, dtype=torch.int32).expand(B, S).contiguous()
    docs[:, 100:] = 1000                                          # ... and one document of fifty
    d = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    gq, gk, gv = torch.autograd.grad(nnops.attention(*d, q_docs=docs.cuda()), d, go.cuda())
    noise = D ** -0.5 * EPS32 * (2 * D + 64) * (go.double() * v.double()).abs().sum(-1, keepdim=True) + GRID.get(dtype, 0.0)
    score = (q.double() * k.double()).sum(-1, keepdim=True).abs() * D ** -0.5 / math.log(2.0)
    near = score < 7.9
    assert bool(near[:, :100].any()) and (std < 1 or bool((~near[:, :100]).any()))
    for got, other in ((gq, k), (gk, q)):
        got = got.double().cpu()[:, :100]
        assert not bool(got[near[:, :100].expand_as(got)].any())
        assert bool((got.abs() <= (noise * other.double().abs())[:, :100] + GRID.get(dtype, 0.0)).all())
    assert float(score.max()) < 1024 and bool(gq[:, 100:].any())  # (half a unit of a score up to 1024: 2^-15)
    check(gv[:, :100], go[:, :100].double(), (go.double().abs() * (HALF[dtype] + 2.0 ** -15))[:, :100], "gv")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kw", [{}, {"causal": True}, {"softcap": 20.0, "causal": True}])
@pytest.mark.parametrize("B,S,Hq,Hkv,D", [(2, 300, 4, 2, 64), (8, 300, 16, 16, 128), (4, 260, 64, 64, 32)])
def test_score_gradients_carry_more_than_one_rounding(B, S, Hq, Hkv, D, kw, dtype):
    """each gradient kernel.  The results' own rounding is one error of relative size r; a second of that size, independent of it, would make 1.41 r (that of dS
    in one term; the values' gradient has it from P), rounding noise of delta at some hundred keys less than 0.3 r: 1.05 r together"""
    from sqd import nnops
    from token_refs import attention_ref
    g = torch.Generator().manual_seed(S + D)
    q, k, v, go = (torch.randn(B, S, h, D, generator=g).to(dtype) for h in (Hq, Hkv, Hkv, Hq))
    d = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(nnops.attention(*d, **kw), d, go.cuda())
    ref = attention_ref(q, k, v, go=go, **kw)
    for name, t, most in (("gq", got[0], 1.2), ("gk", got[1], 1.2), ("gv", got[2], 1.5)):
        once = float((ref[name].to(dtype).double() - ref[name]).norm())
        err = float((t.double().cpu() - ref[name]).norm())
        assert err < most * once, (name, err / once)
