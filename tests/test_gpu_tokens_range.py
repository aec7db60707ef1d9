"""Token operators at the ends of their number ranges and call forms.  References: the 64-bit definitions of token_refs.py."""
import math

import pytest
import torch

import token_refs
from token_refs import HALF, attention_ref, check
from test_gpu_tokens import _build, _case, _cuda, _ops, _rand

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# ------------------------------------------------------------------------------------------------------------ caps far above the scores
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cap", [2e3, 3e4, 1e6, 1e8, 1e20])
def test_attention_far_caps(cap, dtype):
    """the bounds are those of the scores without a cap: tanh is off by two units of its result and its argument and product by half a unit each,
    4 2^-24 of the score together, and the uncapped bound counts 8 2^-24 of the largest score behind the product"""
    for c in (_case(2, 90, 90, 4, 2, 64, causal=True), _case(2, 3, 400, 4, 2, 128, causal=True), _case(1, 70, 70, 2, 1, 40, slopes=True)):
        q, k, v, go, kw = _build(c, dtype)
        ref, tol = attention_ref(q, k, v, go=go, softcap=cap, **kw), attention_ref(q, k, v, go=go, **kw)
        d = [t.cuda().requires_grad_(True) for t in (q, k, v)]
        o = _ops().attention(*d, softcap=cap, **_cuda(kw))
        check(o, ref["o"], tol["o_tol"], "o %s" % c)
        for name, got in zip(("gq", "gk", "gv"), torch.autograd.grad(o, d, go.cuda())):
            check(got, ref[name], tol[name + "_tol"], "%s %s" % (name, c))


# -------------------------------------------------------------------------------------------------------------------------- hidden places
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("extra", [{}, {"softcap": 5.0}, {"softcap": 5.0, "slopes": True}, {"softcap": 1e6}])
def test_attention_lost_queries_hold_anything_under_every_score(extra, dtype):
    """queries of a document without keys hold NaN: zeros and zero gradients, for them and from them, in every form of the scores"""
    q, k, v, go, kw = _build(_case(2, 90, 150, 4, 2, 64, docs_random=True, **extra), dtype)
    kw["k_docs"] = torch.where(kw["k_docs"] == 3, 4, kw["k_docs"])
    lost = (kw["q_docs"] == 3) | (kw["q_docs"] < 0)
    ref = attention_ref(q, k, v, go=go, **kw)
    q[lost], go[lost] = math.nan, math.nan
    d = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = _ops().attention(*d, **_cuda(kw))
    assert not bool(o.detach().cpu()[lost].any())
    grads = torch.autograd.grad(o, d, go.cuda())
    assert not bool(grads[0].cpu()[lost].any())
    for name, got in zip(("gq", "gk", "gv"), grads):
        check(got, ref[name], ref[name + "_tol"], name)


# ---------------------------------------------------------------------------------------------- fp16 numbers far below and far above one
# sizes that reach each gradient kernel: 64 keys by 64 rows (split and whole), 128 keys by 64 rows in 8 waves, 128 keys by 32 rows
F16_RANGE = [_case(1, 1500, 1500, 1, 1, 64), _case(2, 130, 150, 4, 2, 32, causal=True, softcap=20.0), _case(8, 130, 130, 16, 16, 128, docs=(2, 9)),
             _case(4, 130, 200, 64, 64, 48, slopes=True)]


@pytest.mark.parametrize("size", [3e-5, 1e-4, 1e-3, 1.0, 6e3])
@pytest.mark.parametrize("n", range(len(F16_RANGE)))
def test_attention_fp16_gradients_of_any_size(n, size, monkeypatch):
    """incoming gradients of 3e-5 to 6e3: score gradients keep their 11 bits, however small, and none overflows.  Bounds: those of token_refs.py without
    the fixed grid of small fp16 numbers inside the sums.  In its place: P has 2^14 of room below that grid (2^-25 - 14 a pair), dS is lifted to
    within a factor of two of 2^15 / b, b <= 2 max|go| max|v| (2^-25 b / 2^14 a pair); the results' own grid is 2^-25"""
    c = F16_RANGE[n]
    # large keys, large gradients of the queries, and the other way round; results have to fit the type
    for a, b in ((4.0, 0.1), (0.1, 4.0)) if size <= 1 else ((0.1, 0.1),):
        q, k, v, go, kw = _build(c, F16)
        q, k, go = (q.float() / 1.5 * a).half(), (k.float() * b).half(), (go.float() * size).half()
        monkeypatch.setitem(token_refs.HALF_MIN, F16, 0.0)
        ref = attention_ref(q, k, v, go=go, scale=1.0, **kw)
        monkeypatch.undo()
        assert max(float(ref[g].abs().max()) for g in ("gq", "gk", "gv")) < 6e4
        ds = 2.0 ** -38 * float(go.double().norm(dim=-1).max() * v.double().norm(dim=-1).max())
        G, over = c["Hq"] // c["Hkv"], lambda t: t.double().abs().sum(1, keepdim=True)                           # noqa: E731
        heads = lambda t: over(t).view(t.shape[0], 1, c["Hkv"], G, -1).sum(3)                                    # noqa: E731
        grid = {"gq": ds * over(k).repeat_interleave(G, 2), "gk": ds * heads(q), "gv": 2.0 ** -39 * heads(go)}
        d = [t.cuda().requires_grad_(True) for t in (q, k, v)]
        o = _ops().attention(*d, scale=1.0, **_cuda(kw))
        for name, got in zip(("gq", "gk", "gv"), torch.autograd.grad(o, d, go.cuda())):
            check(got, ref[name], ref[name + "_tol"] + grid[name] + 2.0 ** -25, "%s, %s, %s" % (name, a, b))


@pytest.mark.parametrize("Sq", [1, 40])
def test_attention_fp16_probabilities_far_below_the_largest(Sq):
    """one key holds nearly all of a row's weight and a value of zero; the output is what 6000 keys of 2^-27 each leave, summed in fp32.  Bound: half a
    step of the output (2^-11 relative, 2^-25 absolute), half a step of each probability, and the fp32 sums"""
    S, D = 6000, 16
    q, k, v = torch.zeros(1, Sq, 1, D), torch.zeros(1, S, 1, D), torch.ones(1, S, 1, D)
    q[..., 0], k[:, 4321, :, 0], v[:, 4321] = 1.0, 27.0 * math.log(2.0), 0.0
    q, k, v = q.half(), k.half(), v.half() * 16
    z = torch.einsum("bihd,bjhd->bij", q.double(), k.double())
    p = torch.softmax(z, -1)
    want = torch.einsum("bij,bjhd->bihd", p, v.double())
    got = _ops().attention(q.cuda(), k.cuda(), v.cuda(), scale=1.0)
    check(got, want, want.abs() * (2 * HALF[F16] + 2.0 ** -24 * (S + 64)) + 2.0 ** -25, "o")


# -------------------------------------------------------------------------------------------------------------- forward-mode derivatives
def test_forward_mode_derivatives_are_refused():
    """no tangent is computed, so none may be dropped: with and without other inputs that require a gradient, and in constants"""
    import torch.autograd.forward_ad as fwd
    ops = _ops()
    x, w = torch.randn(4, 8, device="cuda"), torch.ones(8, device="cuda")
    q = torch.randn(1, 4, 2, 16, device="cuda")
    pos, freq, slopes = torch.zeros(4, 1, device="cuda", dtype=torch.int32), torch.zeros(8, device="cuda", dtype=torch.float64), torch.ones(2, device="cuda")
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))                                                    # noqa: E731
        calls = [lambda: ops.rms_norm_residual(dual(x), w), lambda: ops.rms_norm_residual(x, dual(w)), lambda: ops.rms_norm_residual(x, w, dual(x)),
                 lambda: ops.rotary_axes(dual(q), q, pos, freq, (8,)), lambda: ops.rotary_axes(q, dual(q), pos, freq, (8,)), lambda: ops.rotary_axes(q, None, pos, dual(freq), (8,)),
                 lambda: ops.attention(dual(q), q, q), lambda: ops.attention(q, dual(q), q), lambda: ops.attention(q, q, dual(q)), lambda: ops.attention(q, q, q, slopes=dual(slopes)),
                 lambda: ops.attention(dual(q), q.clone().requires_grad_(True), q), lambda: ops.rms_norm_residual(dual(x), w.clone().requires_grad_(True))]
        for n, call in enumerate(calls):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="sqd: "):
                    call()
                    pytest.fail("call %d was not refused" % n)
        ops.attention(q, q, q), ops.rms_norm_residual(x, w), ops.rotary_axes(q, q, pos, freq, (8,))     # no tangent: as ever


# --------------------------------------------------------------------------------------------------------------------- empty sides
@pytest.mark.parametrize("B,Sq,Sk", [(2, 0, 5), (2, 5, 0), (0, 4, 4), (1, 0, 0)])
def test_attention_empty_sides_with_documents(B, Sq, Sk):
    z = lambda n: torch.zeros(B, n, 2, 16, device="cuda", requires_grad=True)                                    # noqa: E731
    docs = [torch.zeros(B, n, device="cuda", dtype=torch.int32) for n in (Sq, Sk)]
    q, k, v = z(Sq), z(Sk), z(Sk)
    kw = dict(q_docs=docs[0], k_docs=docs[1], causal=True, prefix=torch.zeros(B, device="cuda", dtype=torch.int32), k_len=torch.full((B,), Sk, device="cuda", dtype=torch.int32))
    o = _ops().attention(q, k, v, **kw)
    assert o.shape == q.shape and not bool(o.any())
    for t, g in zip((q, k, v), torch.autograd.grad(o, (q, k, v), torch.ones_like(o))):
        assert g.shape == t.shape and not bool(g.any())


def test_rotary_without_query_heads():
    g = torch.Generator().manual_seed(4)
    k = _rand(g, 2, 5, 3, 16, dtype=BF16).cuda()
    pos, freq = torch.arange(5, device="cuda", dtype=torch.int32)[:, None], _ops().rotary_frequencies((8,))
    qo, ko = _ops().rotary_axes(k[:, :, :0], k, pos, freq, (8,))
    assert qo.shape == (2, 5, 0, 16) and torch.equal(ko, _ops().rotary_axes(k, None, pos, freq, (8,))[0])


# ----------------------------------------------------------------------------------------------- more threads than a launch can count
def test_norm_of_more_rows_than_a_launch_counts():
    """64 threads a row: 2^26 rows are 2^32 threads"""
    n, C = 2 ** 26 + 5, 8
    x = torch.full((n, C), 7.0, device="cuda", dtype=BF16)
    at = torch.tensor([0, 1, 2 ** 20, 2 ** 26 - 5, 2 ** 26 - 4, 2 ** 26 - 1, 2 ** 26, n - 1], device="cuda")
    x[at] = _rand(torch.Generator().manual_seed(0), len(at), C, dtype=BF16).cuda()
    x.requires_grad_(True)
    w = torch.ones(C, device="cuda")
    y, _ = _ops().rms_norm_residual(x, w, torch.zeros_like(x))
    few = x.detach()[at].clone().requires_grad_(True)
    want, _ = _ops().rms_norm_residual(few, w, torch.zeros_like(few))
    assert torch.equal(y[at], want) and bool((y.detach() == 1.0).sum() >= (n - len(at)) * C)
    g, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(g[at], torch.autograd.grad(want, few, torch.ones_like(want))[0])


def test_rotary_of_more_tokens_than_a_launch_counts():
    """256 threads for 8 tokens: 2^27 tokens are 2^32 threads"""
    n = 2 ** 27 + 9
    q = torch.ones(1, n, 1, 2, device="cuda", dtype=BF16)
    pos = torch.zeros(n, 1, device="cuda", dtype=torch.int32)
    pos[-20:] = 1
    out, _ = _ops().rotary_axes(q, None, pos, torch.full((1,), math.pi / 2, device="cuda", dtype=torch.float64), (1,))
    assert bool((out[0, :-20] == 1.0).all()) and torch.equal(out[0, -20:, 0].cpu(), torch.tensor([[-1.0, 1.0]] * 20, dtype=BF16))


# ------------------------------------------------------------------------------------------------------ long caches, fp16 in a captured graph
@pytest.mark.parametrize("Sq", [2, 40])
def test_attention_cache_past_32_bit_offsets(Sq):
    """2.2 million keys of 8 heads of 128: elements past 2^31, bytes past 2^32.  The queries' document is the last hundred keys, whose results and gradients
    are those of a cache of a hundred; the other keys get none"""
    S, n, H, D = 2200000, 100, 8, 128
    c = _case(1, Sq, n, H, H, D, causal=True, slopes=True)
    q, k, v, go, kw = _build(c, BF16)
    ref = attention_ref(q, k, v, go=go, **kw)
    big = []
    for t in (k, v):
        b = torch.zeros(1, S, H, D, device="cuda", dtype=BF16)
        b[:, -n:] = t.cuda()
        big.append(b.requires_grad_(True))
    kd = torch.zeros(1, S, device="cuda", dtype=torch.int32)
    kd[:, -n:] = 7
    dq = q.cuda().requires_grad_(True)
    o = _ops().attention(dq, *big, q_docs=torch.full((1, Sq), 7, device="cuda", dtype=torch.int32), k_docs=kd, **_cuda(kw))
    check(o, ref["o"], ref["o_tol"], "o")
    gq, gk, gv = torch.autograd.grad(o, [dq] + big, go.cuda())
    for name, got in (("gq", gq), ("gk", gk[:, -n:]), ("gv", gv[:, -n:])):
        check(got, ref[name], ref[name + "_tol"], name)
    assert not bool(gk[:, :-n].any()) and not bool(gv[:, :-n].any())


def test_captured_block_replays_in_fp16():
    """the lifts of the backward are computed on the device, anew in every replay"""
    import test_gpu_tokens
    test_gpu_tokens.test_captured_block_replays(F16)
