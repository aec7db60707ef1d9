"""Token operators at the ends of their number ranges and call forms.  References: the 64-bit definitions of token_refs.py."""
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
