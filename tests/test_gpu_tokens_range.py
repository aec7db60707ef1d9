"""Token operators at the ends of their number ranges and call forms.  References: the 64-bit definitions of token_refs.py."""
import math

import pytest
import torch

from token_refs import attention_ref, check
from test_gpu_tokens import _build, _case, _cuda, _ops

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
