"""What qnn.functional would compute without a word of what is missing, and refuses: before it looks for a device."""
import pytest
import torch
from torch.autograd import forward_ad


@pytest.fixture(scope="module")
def F():
    from qnn import functional
    return functional


def calls(F):
    """Each operator as a function of its first argument: (name, call, that argument)."""
    x, w, i = torch.randn(2, 4), torch.randn(3, 4), torch.zeros(2, 4, dtype=torch.long)
    return (("linear_act", lambda a: F.linear_act(a, w), x), ("layer_norm", lambda a: F.layer_norm(a), x),
            ("topk_distill_loss", lambda a: F.topk_distill_loss(a, x, i), x))


@pytest.mark.parametrize("leaf", [False, True])
def test_tangents_are_refused(F, leaf):
    """A dual tensor came out without its tangent."""
    with forward_ad.dual_level():
        for name, call, x in calls(F):
            dual = forward_ad.make_dual(x.clone().requires_grad_(leaf), torch.ones_like(x))
            with pytest.raises(RuntimeError, match=f"{name} has no forward-mode derivative"):
                call(dual)
            # a primal without its tangent is an ordinary tensor
            with pytest.raises(RuntimeError, match=f"{name}.*ROCm"):
                call(forward_ad.unpack_dual(dual).primal)


def test_tracing_is_refused(F):
    """torch.jit.trace recorded the allocation of an output that nothing fills."""
    for name, call, x in calls(F):
        with pytest.raises(RuntimeError, match=f"{name} cannot be recorded"):
            torch.jit.trace(call, (x,))
