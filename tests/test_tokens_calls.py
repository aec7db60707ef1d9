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
