"""Token operators (residual RMS norm, multi-axis rotary positions, attention) against plain 64-bit implementations."""
import math

import pytest
import torch

from token_refs import HALF, attention_ref, check, norm_ref, rotary_ref

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _ops():
    from sqd import nnops
    return nnops


def _rand(gen, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(dtype)


# ------------------------------------------------------------------------------------------------------------------ residual RMS norm
NORM = [(1, 1), (3, 7), (5, 64), (12, 1024), (70, 480), (4, 1001), (9, 2048), (2, 4099), (3, 9000), (2100, 56), (0, 64)]


@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)])
@pytest.mark.parametrize("rows,C", NORM)
def test_norm(rows, C, dtype, wdtype):
    g = torch.Generator().manual_seed(rows * 7919 + C)
    x, res = _rand(g, rows, C, dtype=dtype), _rand(g, rows, C, dtype=dtype, std=3.0)
    w = (1 + _rand(g, C, std=0.2)).to(wdtype)
    gy, gs = _rand(g, rows, C, dtype=dtype), _rand(g, rows, C, dtype=dtype)
    if rows > 2:
        x[1], res[1] = 0, 0                                      # a row of zeros
    ref = norm_ref(x, w, res, 1e-6, gy, gs)
    d = [t.cuda().requires_grad_(True) for t in (x, w, res)]
    y, s = _ops().rms_norm_residual(d[0], d[1], d[2], eps=1e-6)
    gx, gw, gr = torch.autograd.grad((y, s), d, (gy.cuda(), gs.cuda()))
    assert y.dtype == s.dtype == gx.dtype == gr.dtype == dtype and gw.dtype == wdtype
    assert torch.equal(s.detach().cpu().double(), ref["s"])
    check(y, ref["y"], ref["y_tol"], "y")
    check(gx, ref["gx"], ref["gx_tol"], "gx")
    check(gr, ref["gx"], ref["gx_tol"], "gres")
    check(gw, ref["gw"], ref["gw_tol"], "gw")
    with torch.no_grad():                                        # the serving form: the same bits
        y2, s2 = _ops().rms_norm_residual(d[0], d[1], d[2], eps=1e-6)
    assert torch.equal(y, y2) and torch.equal(s, s2)


def test_norm_without_residual_strided_and_partial_gradients():
    g = torch.Generator().manual_seed(1)
    base = _rand(g, 3, 5, 2, 72, dtype=BF16).cuda()
    x = base[:, :, 1].detach().requires_grad_(True)              # rows with a stride
    w = (1 + _rand(g, 72, std=0.1)).cuda().requires_grad_(True)
    y, s = _ops().rms_norm_residual(x, w)
    assert s is x
    gy = _rand(g, 3, 5, 72, dtype=BF16)
    ref = norm_ref(x.detach().cpu(), w.detach().cpu(), None, 1e-6, gy)
    gx, gw = torch.autograd.grad(y, (x, w), gy.cuda())
    check(y, ref["y"], ref["y_tol"], "y")
    check(gx, ref["gx"], ref["gx_tol"], "gx")
    check(gw, ref["gw"], ref["gw_tol"], "gw")
    r = torch.zeros_like(x).requires_grad_(True)
    y, s = _ops().rms_norm_residual(x, w, r)
    gx, gr = torch.autograd.grad(s, (x, r), gy.cuda())           # the stream alone: its gradient passes through
    assert torch.equal(gx, gy.cuda()) and torch.equal(gr, gy.cuda())
    y, s = _ops().rms_norm_residual(x, w, r)
    gx, = torch.autograd.grad(y, x, gy.cuda())
    check(gx, ref["gx"], ref["gx_tol"], "gx of y alone")


# ------------------------------------------------------------------------------------------------------------------------------ rotary
ROT = [  # B, S, Hq, Hk, D, pairs, interleaved
    (1, 1, 1, 1, 2, (1,), False), (2, 7, 3, 1, 16, (8,), False), (2, 7, 3, 1, 16, (3, 5), True), (3, 5, 4, 2, 64, (16, 16), False),
    (1, 33, 8, 2, 128, (16, 24, 24), False), (2, 9, 2, 2, 40, (4, 8, 8), False), (2, 9, 2, 1, 40, (2, 2, 2, 2), False),
    (1, 6, 2, 2, 24, (0, 5), False), (1, 6, 2, 2, 24, (0, 5), True), (1, 4500, 2, 1, 32, (8, 8), False), (0, 4, 2, 2, 16, (8,), False)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,S,Hq,Hk,D,pairs,inter", ROT)
def test_rotary(B, S, Hq, Hk, D, pairs, inter, dtype):
    g = torch.Generator().manual_seed(S * 31 + D)
    q, k = _rand(g, B, S, Hq, D, dtype=dtype), _rand(g, B, S, Hk, D, dtype=dtype)
    gq, gk = _rand(g, B, S, Hq, D, dtype=dtype), _rand(g, B, S, Hk, D, dtype=dtype)
    big = 1000000 if S % 2 else 50
    pos = torch.randint(-big, big, (S, len(pairs)) if S % 3 else (B, S, len(pairs)), generator=g, dtype=torch.int32 if D % 16 else torch.int64)
    freq = _ops().rotary_frequencies(pairs, 100.0, shared=inter, device="cpu")
    qd, kd = q.cuda().requires_grad_(True), k.cuda().requires_grad_(True)
    qo, ko = _ops().rotary_axes(qd, kd, pos.cuda(), freq.cuda(), pairs, interleaved=inter)
    dq, dk = torch.autograd.grad((qo, ko), (qd, kd), (gq.cuda(), gk.cuda()))
    if B == 0:
        assert qo.shape == q.shape and dk.shape == k.shape
        return
    for got, src, inv in ((qo, q, False), (ko, k, False), (dq, gq, True), (dk, gk, True)):
        assert got.dtype == dtype
        check(got, *rotary_ref(src, pos, freq, pairs, inter, inv), "rotary")


def test_rotary_far_positions_slices_and_queries_alone():
    g = torch.Generator().manual_seed(3)
    qkv = _rand(g, 2, 11, 6, 64, dtype=F32)                      # packed projections: 4 query heads, 1 key head, 1 value head
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, 10 ** 6, 1, 0, 123456789, 7, 8, 9, 10, 11], dtype=torch.int32)[:, None]
    freq = _ops().rotary_frequencies((32,), 10000.0, device="cpu")
    d = qkv.cuda()
    qo, ko = _ops().rotary_axes(d[:, :, :4], d[:, :, 4:5], pos.cuda(), freq.cuda(), (32,))
    check(qo, *rotary_ref(qkv[:, :, :4], pos, freq, (32,)), "q")
    check(ko, *rotary_ref(qkv[:, :, 4:5], pos, freq, (32,)), "k")
    alone, none = _ops().rotary_axes(d[:, :, :4].requires_grad_(True), None, pos.cuda(), freq.cuda(), (32,))
    assert none is None and torch.equal(alone, qo)
    odd = d[..., 1:63]                                           # features that do not start on 16 bytes
    check(_ops().rotary_axes(odd, None, pos.cuda(), freq.cuda()[:31], (31,))[0], *rotary_ref(qkv[..., 1:63], pos, freq[:31], (31,)), "odd")


# --------------------------------------------------------------------------------------------------------------------------- attention
def _case(B, Sq, Sk, Hq, Hkv, D, **kw):
    return dict(B=B, Sq=Sq, Sk=Sk, Hq=Hq, Hkv=Hkv, D=D, **kw)


def _docs(B, S, n, pad):
    """n documents in a row, of different lengths in every row of the batch; the last `pad` tokens padding"""
    return torch.stack([torch.tensor([min(n - 1, (j * n + b) // max(1, S - pad)) if j < S - pad else -1 - b for j in range(S)], dtype=torch.int32)
                        for b in range(B)])


ATTN = [
    _case(1, 1, 1, 1, 1, 8), _case(2, 1, 1, 4, 2, 64, causal=True), _case(2, 2, 2, 2, 1, 16), _case(1, 33, 33, 2, 2, 32),
    _case(2, 65, 65, 4, 2, 64, causal=True), _case(1, 200, 200, 3, 1, 40, causal=True, prefix=[77]), _case(2, 130, 130, 4, 4, 96, slopes=True),
    _case(1, 257, 257, 2, 1, 128, softcap=5.0), _case(2, 150, 150, 4, 1, 128, softcap=20.0, slopes=True, causal=True, prefix=[0, 151]),
    _case(2, 190, 190, 2, 1, 64, docs=(4, 21)), _case(2, 100, 100, 4, 2, 24, docs=(3, 0), causal=True), _case(1, 70, 70, 2, 2, 16, docs=(1, 70)),
    _case(3, 5, 300, 6, 2, 64, causal=True, k_len=[300, 3, 0]), _case(3, 1, 700, 8, 2, 128, causal=True, k_len=[700, 1, 64], softcap=30.0),
    _case(2, 40, 170, 2, 2, 64, k_len=[170, 33]), _case(1, 300, 20, 2, 1, 32), _case(1, 300, 20, 2, 1, 32, causal=True),
    _case(2, 3, 1500, 2, 1, 80, slopes=True, causal=True), _case(1, 4, 0, 2, 2, 16), _case(2, 0, 5, 2, 2, 16), _case(0, 4, 4, 2, 2, 16),
    _case(1, 7, 1, 12, 4, 64), _case(2, 17, 600, 8, 8, 128, docs_random=True), _case(1, 129, 129, 5, 1, 64, causal=True, scale=0.3),
]


def _build(c, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + c["Sq"] * 1000 + c["Sk"] + c["D"])
    B, Sq, Sk, Hq, Hkv, D = (c[k] for k in ("B", "Sq", "Sk", "Hq", "Hkv", "D"))
    q, k, v = _rand(g, B, Sq, Hq, D, dtype=dtype, std=1.5), _rand(g, B, Sk, Hkv, D, dtype=dtype), _rand(g, B, Sk, Hkv, D, dtype=dtype)
    go = _rand(g, B, Sq, Hq, D, dtype=dtype)
    kw = {n: c[n] for n in ("softcap", "causal", "scale") if n in c}
    if c.get("slopes"):
        kw["slopes"] = 2.0 ** (-8.0 * torch.arange(1, Hq + 1).float() / Hq)
    for n in ("prefix", "k_len"):
        if n in c:
            kw[n] = torch.tensor(c[n], dtype=torch.int32)
    if "docs" in c:
        kw["q_docs"] = kw["k_docs"] = _docs(B, Sq, *c["docs"])
    if c.get("docs_random"):
        kw["q_docs"], kw["k_docs"] = (torch.randint(-2, 5, (B, n), generator=g, dtype=torch.int32) for n in (Sq, Sk))
    return q, k, v, go, kw


def _cuda(kw):
    return {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in kw.items()}


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n", range(len(ATTN)))
def test_attention(n, dtype):
    q, k, v, go, kw = _build(ATTN[n], dtype)
    ref = attention_ref(q, k, v, go=go, **kw)
    d = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = _ops().attention(*d, **_cuda(kw))
    assert o.dtype == dtype
    check(o, ref["o"], ref["o_tol"], "o")
    for name, got in zip(("gq", "gk", "gv"), torch.autograd.grad(o, d, go.cuda())):
        assert got.dtype == dtype
        check(got, ref[name], ref[name + "_tol"], name)
    with torch.no_grad():
        assert torch.equal(_ops().attention(*d, **_cuda(kw)), o)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("extra", [{}, {"softcap": 20.0}, {"slopes": True}, {"softcap": 6.0, "slopes": True}])
def test_attention_documents_with_every_score(extra, D, dtype):
    """documents against each kernel (few rows, many) and each form of the scores; whole tiles of one document, so that every key of a tile counts"""
    cases = [_case(2, 32, 32, 1, 1, D, docs=(1, 0), **extra), _case(2, 32, 32, 2, 2, D, docs=(5, 4), **extra), _case(1, 8, 8, 12, 3, D, docs=(2, 1), **extra),
             _case(2, 5, 330, 4, 2, D, docs_random=True, **extra), _case(2, 96, 96, 2, 1, D, docs=(1, 0), **extra), _case(1, 200, 200, 2, 2, D, docs=(3, 8), causal=True, **extra)]
    for c in cases:
        q, k, v, go, kw = _build(c, dtype)
        ref = attention_ref(q, k, v, go=go, **kw)
        d = [t.cuda().requires_grad_(True) for t in (q, k, v)]
        o = _ops().attention(*d, **_cuda(kw))
        check(o, ref["o"], ref["o_tol"], "o %s" % c)
        for name, got in zip(("gq", "gk", "gv"), torch.autograd.grad(o, d, go.cuda())):
            check(got, ref[name], ref[name + "_tol"], "%s %s" % (name, c))


# the variants a size selects: 128-key workgroups of 8 and of 4 waves, keys or rows split over workgroups (few heads, long sequences), key heads that
# share an XCD unevenly
WIDE = [
    (_case(8, 200, 200, 16, 16, 128, docs=(3, 17), softcap=20.0), BF16), (_case(8, 150, 290, 8, 8, 96, causal=True, k_len=[290, 2, 150, 149, 77, 200, 13, 290]), F16),
    (_case(6, 129, 129, 70, 70, 16, causal=True, prefix=[0, 1, 50, 129, 200, 128]), BF16), (_case(6, 140, 140, 65, 65, 8, slopes=True), F32),
    (_case(1, 1100, 1100, 1, 1, 64, causal=True), BF16), (_case(1, 901, 1203, 3, 1, 40, softcap=9.0, causal=True, prefix=[300]), F32),
    (_case(8, 130, 130, 40, 40, 64, slopes=True, docs=(2, 9)), BF16), (_case(4, 200, 260, 64, 64, 48, causal=True, softcap=8.0), F16),
    (_case(3, 700, 700, 2, 1, 128, docs=(4, 90), slopes=True), F16), (_case(1, 700, 701, 5, 5, 64, causal=True, k_len=[640]), BF16),
]


@pytest.mark.parametrize("n", range(len(WIDE)))
def test_attention_variants(n):
    c, dtype = WIDE[n]
    q, k, v, go, kw = _build(c, dtype)
    ref = attention_ref(q, k, v, go=go, **kw)
    d = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = _ops().attention(*d, **_cuda(kw))
    check(o, ref["o"], ref["o_tol"], "o")
    first = torch.autograd.grad(o, d, go.cuda(), retain_graph=True)
    for name, got in zip(("gq", "gk", "gv"), first):
        check(got, ref[name], ref[name + "_tol"], name)
    for a, b in zip(first, torch.autograd.grad(o, d, go.cuda())):
        assert torch.equal(a, b)


def test_attention_one_key_has_no_score_gradient():
    q, k, v, go, kw = _build(_case(3, 1, 1, 4, 2, 128, causal=True), BF16)
    d = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    gq, gk, gv = torch.autograd.grad(_ops().attention(*d, causal=True, softcap=50.0), d, go.cuda())
    assert not bool(gq.any()) and not bool(gk.any()) and bool(gv.any())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_strides_and_repeatability(dtype):
    """slices of a packed projection, a cache longer than its contents, a gradient with strides; the same bits every run"""
    g = torch.Generator().manual_seed(5)
    B, S, Hq, Hkv, D = 2, 96, 4, 2, 64
    packed = _rand(g, B, S, Hq + 2 * Hkv, D, dtype=dtype)
    p = packed.cuda().requires_grad_(True)
    go = _rand(g, B, Hq, S, D, dtype=dtype)
    ref = attention_ref(packed[:, :, :Hq], packed[:, :, Hq:Hq + Hkv], packed[:, :, Hq + Hkv:], causal=True, go=go.permute(0, 2, 1, 3))
    runs = []
    for _ in range(2):
        o = _ops().attention(p[:, :, :Hq], p[:, :, Hq:Hq + Hkv], p[:, :, Hq + Hkv:], causal=True)
        gp, = torch.autograd.grad(o, p, go.cuda().permute(0, 2, 1, 3))
        runs.append((o.detach(), gp))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    check(runs[0][0], ref["o"], ref["o_tol"], "o")
    check(runs[0][1], torch.cat([ref["gq"], ref["gk"], ref["gv"]], 2), torch.cat([ref["gq_tol"], ref["gk_tol"], ref["gv_tol"]], 2), "packed gradient")
    # features that do not start on 16 bytes
    t = [x[..., 1:1 + 56] for x in (packed[:, :, :Hq], packed[:, :, Hq:Hq + Hkv], packed[:, :, Hq + Hkv:])]
    ref = attention_ref(*t)
    big = packed.cuda()
    check(_ops().attention(*[x[..., 1:1 + 56] for x in (big[:, :, :Hq], big[:, :, Hq:Hq + Hkv], big[:, :, Hq + Hkv:])]), ref["o"], ref["o_tol"], "unaligned")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf])
def test_attention_hidden_places_hold_anything(dtype, junk):
    """keys behind the length and padding tokens hold NaN or infinities: results and gradients as if they held zeros"""
    for c in (_case(2, 6, 210, 4, 2, 64, causal=True, k_len=[170, 3]), _case(2, 140, 140, 2, 1, 48, docs=(3, 31))):
        q, k, v, go, kw = _build(c, dtype)
        see = {"k": torch.ones(c["B"], c["Sk"], dtype=torch.bool), "q": torch.ones(c["B"], c["Sq"], dtype=torch.bool)}
        if "k_len" in kw:
            see["k"] = torch.arange(c["Sk"])[None] < kw["k_len"][:, None]
            pos = torch.arange(c["Sq"])[None] + kw["k_len"][:, None] - c["Sq"]
            see["q"] = pos >= 0
        else:
            see["k"] = see["q"] = kw["k_docs"] >= 0
        ref = attention_ref(q, k, v, go=go, **kw)
        k[~see["k"]], v[~see["k"]], q[~see["q"]], go[~see["q"]] = junk, junk, junk, junk
        d = [t.cuda().requires_grad_(True) for t in (q, k, v)]
        o = _ops().attention(*d, **_cuda(kw))
        check(o, ref["o"], ref["o_tol"], "o")
        assert not bool(o.detach().cpu()[~see["q"]].any())
        for name, got in zip(("gq", "gk", "gv"), torch.autograd.grad(o, d, go.cuda())):
            check(got, ref[name], ref[name + "_tol"], name)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cap", [0.5, 300.0, 30000.0])
def test_attention_small_and_large_caps(cap, dtype):
    """fp32 keeps scores far below the cap; the 16-bit types lose 4 2^-24 of the cap, which the bounds count"""
    q, k, v, go, kw = _build(_case(2, 90, 90, 4, 2, 64, softcap=cap, causal=True), dtype)
    ref = attention_ref(q, k, v, go=go, **kw)
    d = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = _ops().attention(*d, **_cuda(kw))
    check(o, ref["o"], ref["o_tol"], "o")
    if dtype == F32:           # the bound counts the short form's loss; fp32 must not have it: as exact as without a cap (64 roundings of 2^-24)
        assert float((o.detach().cpu().double() - ref["o"]).norm() / ref["o"].norm()) < 64 * 2.0 ** -24
    for name, got in zip(("gq", "gk", "gv"), torch.autograd.grad(o, d, go.cuda())):
        check(got, ref[name], ref[name + "_tol"], name)


def test_attention_frozen_inputs_and_expanded_gradients():
    """only what requires a gradient gets one; keys and values expanded over the batch; the gradient of a sum is an expanded scalar"""
    g = torch.Generator().manual_seed(2)
    q, k, v = _rand(g, 3, 20, 4, 32), _rand(g, 1, 30, 2, 32), _rand(g, 1, 30, 2, 32)
    ref = attention_ref(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1), go=torch.ones_like(q))
    dq, dk, dv = q.cuda().requires_grad_(True), k.cuda().requires_grad_(True), v.cuda().requires_grad_(True)
    gq, gk, gv = torch.autograd.grad(_ops().attention(dq, dk.expand(3, -1, -1, -1), dv.expand(3, -1, -1, -1)).sum(), (dq, dk, dv))
    check(gq, ref["gq"], ref["gq_tol"], "gq")
    check(gk, ref["gk"].sum(0, keepdim=True), ref["gk_tol"].sum(0, keepdim=True) + 3 * 2.0 ** -24 * ref["gk"].abs().sum(0, keepdim=True), "gk")
    check(gv, ref["gv"].sum(0, keepdim=True), ref["gv_tol"].sum(0, keepdim=True) + 3 * 2.0 ** -24 * ref["gv"].abs().sum(0, keepdim=True), "gv")
    only, = torch.autograd.grad(_ops().attention(dq, k.cuda().expand(3, -1, -1, -1), v.cuda().expand(3, -1, -1, -1)).sum(), dq)
    assert torch.equal(only, gq)
    value, = torch.autograd.grad(_ops().attention(q.cuda(), k.cuda().expand(3, -1, -1, -1), dv.expand(3, -1, -1, -1)).sum(), dv)
    assert torch.equal(value, gv)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_queries_of_a_document_without_keys_hold_anything(dtype):
    q, k, v, go, kw = _build(_case(2, 90, 150, 4, 2, 64, docs_random=True), dtype)
    kw["k_docs"] = torch.where(kw["k_docs"] == 3, 4, kw["k_docs"])                    # nobody has document 3
    lost = (kw["q_docs"] == 3) | (kw["q_docs"] < 0)
    ref = attention_ref(q, k, v, go=go, **kw)
    q[lost], go[lost] = math.nan, math.inf
    d = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = _ops().attention(*d, **_cuda(kw))
    check(o, ref["o"], ref["o_tol"], "o")
    for name, got in zip(("gq", "gk", "gv"), torch.autograd.grad(o, d, go.cuda())):
        check(got, ref[name], ref[name + "_tol"], name)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_negative_prefix_is_no_prefix(dtype):
    """down to the type's lowest value"""
    q, k, v, go, _ = _build(_case(3, 70, 90, 4, 2, 64, causal=True), dtype)
    lens = torch.tensor([90, 40, 90], dtype=torch.int32)
    prefix = torch.tensor([-2 ** 31, -2 ** 31, -5], dtype=torch.int32)
    ref = attention_ref(q, k, v, go=go, causal=True, k_len=lens, prefix=torch.zeros_like(prefix))
    d = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = _ops().attention(*d, causal=True, k_len=lens.cuda(), prefix=prefix.cuda())
    check(o, ref["o"], ref["o_tol"], "o")
    for name, got in zip(("gq", "gk", "gv"), torch.autograd.grad(o, d, go.cuda())):
        check(got, ref[name], ref[name + "_tol"], name)
    check(_ops().attention(q[:1, -1:].cuda(), k[:1].cuda(), v[:1].cuda(), causal=True, prefix=prefix[:1].cuda()), ref["o"][:1, -1:], ref["o_tol"][:1, -1:], "token")


def test_attention_gradient_against_differences():
    """the directional derivative of sum(o go) in fp32 against central differences of the 64-bit definition (truncation h^2: 1e-8 relative)"""
    q, k, v, go, kw = _build(_case(1, 37, 37, 4, 2, 32, causal=True, prefix=[9], softcap=3.0, slopes=True), F32)
    d = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(_ops().attention(*d, **_cuda(kw)), d, go.cuda())
    g = torch.Generator().manual_seed(11)
    ref = attention_ref(q, k, v, go=go, **kw)
    for n, name in enumerate(("gq", "gk", "gv")):
        step = _rand(g, *d[n].shape).double()
        h = 1e-4
        at = [[t.double() for t in (q, k, v)] for _ in range(2)]
        at[0][n] += h * step
        at[1][n] -= h * step
        plus, minus = (_value(a, go, kw) for a in at)
        want = (plus - minus) / (2 * h)
        got = float((grads[n].double().cpu() * step).sum())
        tol = float((ref[name + "_tol"] * step.abs()).sum()) + 1e-6 * float((ref[name].abs() * step.abs()).sum()) + 1e-6
        assert abs(got - want) <= tol, (name, got, want, tol)


def _value(t, go, kw):
    q, k, v = t
    B, Sq, Hq, D = q.shape
    G = Hq // k.shape[2]
    z = torch.einsum("bihd,bjhd->bhij", q, k.repeat_interleave(G, 2)) / math.sqrt(D)
    z = kw["softcap"] * torch.tanh(z / kw["softcap"])
    i, j = torch.arange(Sq)[:, None], torch.arange(Sq)[None]
    z = z - kw["slopes"].double().view(1, Hq, 1, 1) * (i - j).abs()
    z = z.masked_fill(~((j <= i) | (j < kw["prefix"].view(-1, 1, 1)))[:, None], -math.inf)
    o = torch.einsum("bhij,bjhd->bihd", torch.softmax(z, -1), v.repeat_interleave(G, 2))
    return float((o * go.double()).sum())


# -------------------------------------------------------------------------------------------- together, other streams, captured graphs
def _block(ops, x, res, w, wqkv, pos, freq, docs, heads, kv):
    """norm -> projection -> rotary -> attention, as an encoder layer runs them"""
    y, s = ops.rms_norm_residual(x, w, res)
    B, S, C = x.shape
    D = wqkv.shape[0] // (heads + 2 * kv)
    p = (y @ wqkv.t()).view(B, S, heads + 2 * kv, D)
    q, k = ops.rotary_axes(p[:, :, :heads], p[:, :, heads:heads + kv], pos, freq, (D // 4, D // 4))
    return s, q, k, p[:, :, heads + kv:], ops.attention(q, k, p[:, :, heads + kv:], softcap=20.0, q_docs=docs)


def _block_inputs(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    B, h, w_, C, heads, kv, D = 2, 6, 10, 96, 4, 2, 32
    S = h * w_
    x, res = _rand(g, B, S, C, dtype=dtype), _rand(g, B, S, C, dtype=dtype)
    w, wqkv = 1 + _rand(g, C, std=0.1), _rand(g, (heads + 2 * kv) * D, C, dtype=dtype, std=C ** -0.5)
    pos = torch.cartesian_prod(torch.arange(h), torch.arange(w_)).to(torch.int32)
    go = _rand(g, B, S, heads, D, dtype=dtype)
    return x, res, w, wqkv, pos, _docs(B, S, 3, 7), go, heads, kv


def test_block_of_the_three_operators():
    """norm, rotary, attention behind each other in fp32: outputs and gradients against autograd of the 64-bit composition"""
    ops = _ops()
    x, res, w, wqkv, pos, docs, go, heads, kv = _block_inputs(F32)
    D = 32
    freq = ops.rotary_frequencies((D // 4, D // 4), 100.0, device="cpu")
    d = [t.cuda().requires_grad_(True) for t in (x, res, w, wqkv)]
    s, q, k, v, o = _block(ops, d[0], d[1], d[2], d[3], pos.cuda(), freq.cuda(), docs.cuda(), heads, kv)
    got = torch.autograd.grad((o, s), d, (go.cuda(), torch.ones_like(s)))
    e = [t.double().requires_grad_(True) for t in (x, res, w, wqkv)]
    s64 = e[0] + e[1]
    y = s64 / torch.sqrt(s64.pow(2).mean(-1, keepdim=True) + 1e-6) * e[2]
    p = (y @ e[3].t()).view(2, 60, heads + 2 * kv, D)
    ang = pos.double()[:, [0] * (D // 4) + [1] * (D // 4)] * freq
    c, sn = ang.cos()[None, :, None], ang.sin()[None, :, None]
    rot = lambda t: torch.cat([t[..., :D // 2] * c - t[..., D // 2:] * sn, t[..., D // 2:] * c + t[..., :D // 2] * sn], -1)       # noqa: E731
    q64, k64 = rot(p[:, :, :heads]), rot(p[:, :, heads:heads + kv]).repeat_interleave(2, 2)
    z = 20 * torch.tanh(torch.einsum("bihd,bjhd->bhij", q64, k64) / math.sqrt(D) / 20)
    see = ((docs[:, :, None] == docs[:, None]) & (docs[:, :, None] >= 0))[:, None]
    pr = torch.softmax(z.masked_fill(~see, -1e30), -1) * see
    o64 = torch.einsum("bhij,bjhd->bihd", pr, p[:, :, heads + kv:].repeat_interleave(2, 2))
    want = torch.autograd.grad((o64, s64), e, (go.double(), torch.ones_like(s64)))
    # sums of at most 96 + 60 + 32 fp32 products and some fifty roundings stand between input and output, each relative 2^-24 to the
    # magnitudes that meet in it; those exceed the results by less than a factor of 30 (norms): 2^-24 * 240 * 30 = 4.3e-4
    for name, a, b in [("o", o, o64)] + list(zip(("gx", "gres", "gw", "gwqkv"), got, want)):
        err = float((a.double().cpu() - b).norm() / b.norm())
        assert err < 4.3e-4, (name, err)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_block_replays(dtype):
    """forward and backward of the block in one captured graph, replayed on new inputs with eager work between the replays"""
    ops = _ops()
    x, res, w, wqkv, pos, docs, go, heads, kv = _block_inputs(dtype)
    freq = ops.rotary_frequencies((8, 8), 100.0)
    static = [t.cuda().requires_grad_(True) for t in (x, res, w, wqkv)]
    sgo, pos, docs = go.cuda(), pos.cuda(), docs.cuda()

    def step(t, g):
        if dtype == F32:
            s, _, _, _, o = _block(ops, *t, pos, freq, docs, heads, kv)
        else:
            s, _, _, _, o = _block(ops, t[0], t[1], t[2], t[3], pos, freq, docs, heads, kv)
        return (o, s) + torch.autograd.grad((o, s), t, (g, torch.ones_like(s)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static, sgo)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static, sgo)
    for seed in range(1, 5):
        new = _block_inputs(dtype, seed)
        with torch.no_grad():
            for t, n in zip(static, new[:4]):
                t.copy_(n.cuda())
            sgo.copy_(new[6].cuda())
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in outs]
        want = step([t.cuda().requires_grad_(True) for t in new[:4]], new[6].cuda())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    ops = _ops()
    cases = [_build(_case(2, 3, 900, 8, 2, 128, causal=True, k_len=[900, 412]), BF16, seed) for seed in range(2)]
    streams = [torch.cuda.Stream() for _ in cases]
    dev = [([t.cuda() for t in c[:3]], _cuda(c[4])) for c in cases]
    want = [ops.attention(*t, **kw) for t, kw in dev]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, (t, kw) in zip(streams, dev):
            with torch.cuda.stream(s):
                got.append(ops.attention(*t, **kw))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])


# ------------------------------------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    ops = _ops()
    z = lambda *s, dtype=F32: torch.zeros(*s, device="cuda", dtype=dtype)                                        # noqa: E731
    i32 = torch.int32
    q, k = z(2, 4, 4, 16), z(2, 4, 2, 16)
    pos, freq = z(4, 1, dtype=i32), z(8, dtype=torch.float64)
    calls = [
        lambda: ops.rms_norm_residual(z(4, 8).half(), z(8).bfloat16()), lambda: ops.rms_norm_residual(z(4, 8), z(7)),
        lambda: ops.rms_norm_residual(z(4, 8), z(8), z(4, 7)), lambda: ops.rms_norm_residual(z(4, 8), z(8), z(4, 8).half()),
        lambda: ops.rms_norm_residual(z(4, 8).double(), z(8).double()), lambda: ops.rms_norm_residual(z(4, 8), z(8), eps=-1.0),
        lambda: ops.rms_norm_residual(z(4, 8), torch.zeros(8)), lambda: ops.rms_norm_residual(z(4, 8), z(8), eps=math.nan),
        lambda: ops.rotary_axes(q, k, pos, freq, (9,)), lambda: ops.rotary_axes(q, k, pos, freq, (4, 4)),
        lambda: ops.rotary_axes(q, k, pos.float(), freq, (8,)), lambda: ops.rotary_axes(q, k, pos, freq.float(), (8,)),
        lambda: ops.rotary_axes(q, k, pos[:3], freq, (8,)), lambda: ops.rotary_axes(q, k.half(), pos, freq, (8,)),
        lambda: ops.rotary_axes(q, k[:1], pos, freq, (8,)), lambda: ops.rotary_axes(q, k, pos, freq[:0], ()),
        lambda: ops.rotary_axes(q, k, pos, freq, (9, -1)), lambda: ops.rotary_axes(q[..., :15], None, pos, freq[:7], (7,)),
        lambda: ops.attention(q, k, k[:, :3]), lambda: ops.attention(q, z(2, 4, 3, 16), z(2, 4, 3, 16)), lambda: ops.attention(q[..., :12], k[..., :12], k[..., :12]),
        lambda: ops.attention(z(1, 2, 1, 136), z(1, 2, 1, 136), z(1, 2, 1, 136)), lambda: ops.attention(q, k.half(), k.half()),
        lambda: ops.attention(q, k, k, scale=0.0), lambda: ops.attention(q, k, k, scale=math.nan), lambda: ops.attention(q, k, k, softcap=-1.0),
        lambda: ops.attention(q, k, k, prefix=z(2, dtype=i32)), lambda: ops.attention(q, k, k, causal=True, prefix=z(2)),
        lambda: ops.attention(q, k, k, causal=True, prefix=z(3, dtype=i32)), lambda: ops.attention(q, k, k, slopes=z(2)),
        lambda: ops.attention(q, k, k, slopes=z(4).requires_grad_(True)), lambda: ops.attention(q, k, k, k_docs=z(2, 4, dtype=i32)),
        lambda: ops.attention(q[:, :2], k, k, q_docs=z(2, 2, dtype=i32)), lambda: ops.attention(q, k, k, k_len=torch.zeros(2, dtype=i32)),
        lambda: ops.attention(q, k, k, q_docs=z(2, 4, dtype=torch.int64)),
    ]
    for n, call in enumerate(calls):
        with pytest.raises(RuntimeError, match="sqd: "):
            call()
            pytest.fail("call %d was not refused" % n)


def test_constants_that_want_a_gradient_are_refused():
    ops = _ops()
    q = torch.zeros(2, 4, 4, 16, device="cuda")
    pos, freq = torch.zeros(4, 1, device="cuda", dtype=torch.int32), torch.zeros(8, device="cuda", dtype=torch.float64, requires_grad=True)
    for call in (lambda: ops.rotary_axes(q, None, pos, freq, (8,)), lambda: ops.rotary_axes(q.clone().requires_grad_(True), q, pos, freq, (8,)),
                 lambda: ops.attention(q, q, q, slopes=[0.5] * 4), lambda: ops.attention(q, q, q, slopes=torch.zeros(4, device="cuda", requires_grad=True))):
        with pytest.raises(RuntimeError, match="sqd: "):
            call()


def test_sizes_past_32_bits_are_refused():
    """expanded tensors (no memory behind the sizes): they must not be taken modulo 2^32"""
    ops = _ops()
    n = 2 ** 32 + 4
    row = torch.zeros(1, device="cuda", dtype=F16)
    q, few = torch.zeros(1, 1, 1, 16, device="cuda", dtype=F16), torch.zeros(1, 4, 1, 16, device="cuda", dtype=F16)
    pos, freq = torch.zeros(1, 1, device="cuda", dtype=torch.int32), torch.zeros(8, device="cuda", dtype=torch.float64)
    long = q.expand(1, n, 1, 16)
    for call in (lambda: ops.rms_norm_residual(row.expand(n), row.expand(n)), lambda: ops.rotary_axes(long, None, pos.expand(n, 1), freq, (8,)),
                 lambda: ops.attention(long, few, few), lambda: ops.attention(few, long, long), lambda: ops.attention(q.expand(n, 1, 1, 16), q, q)):
        with pytest.raises(RuntimeError, match="sqd: "):
            call()


def test_second_derivatives_are_refused():
    ops = _ops()
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    y, _ = ops.rms_norm_residual(x, w)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
