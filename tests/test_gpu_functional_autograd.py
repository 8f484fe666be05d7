"""qnn.functional on the device where autograd hands it more than plain tensors."""
import warnings

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def F(gpu):
    from qnn import functional
    return functional


def calls(F):
    """Each operator with its differentiable arguments: (name, function of them, arguments)."""
    x, w, v, b, r = (torch.randn(*s, device="cuda") for s in ((2, 4), (3, 4), (4,), (3,), (2, 3)))
    i = torch.zeros(2, 4, dtype=torch.long, device="cuda")
    return (("linear_act", lambda *a: F.linear_act(*a), [x, w, b, r]), ("layer_norm", lambda *a: F.layer_norm(*a), [x, v, v.clone()]),
            ("topk_distill_loss", lambda s: F.topk_distill_loss(s, x, i), [x]))


def test_tangents_and_traces_are_refused(F):
    for name, f, args in calls(F):
        want = f(*args)
        with forward_ad.dual_level():
            for at, a in enumerate(args):
                dual = forward_ad.make_dual(a, torch.ones_like(a))
                with pytest.raises(RuntimeError, match=f"{name} has no forward-mode derivative"):
                    f(*args[:at], dual, *args[at + 1:])
            assert torch.equal(f(*args), want)
        with pytest.raises(RuntimeError, match=f"{name} cannot be recorded"):
            torch.jit.trace(f, tuple(args))
        assert torch.equal(f(*args), want)


def test_a_dual_teacher_is_a_constant(F):
    """As one that requires a gradient is."""
    s, t, i = torch.randn(2, 9, device="cuda"), torch.randn(2, 4, device="cuda"), torch.arange(8, device="cuda").view(2, 4)
    want = F.topk_distill_loss(s, t, i)
    with forward_ad.dual_level():
        got = F.topk_distill_loss(s, forward_ad.make_dual(t, torch.ones_like(t)), i)
        assert torch.equal(got, want) and forward_ad.unpack_dual(got).tangent is None


def test_negated_views(F):
    """A view with torch's negative bit (the imaginary part of a conjugate) gives what its values do, forward and backward:
    the kernels took what lies in memory."""
    negated = torch._neg_view
    cases = calls(F) + (("one feature", lambda x, w: F.linear_act(x, w), [torch.randn(3, 1, device="cuda"), torch.randn(2, 1, device="cuda")]),
                        ("rows of losses", lambda s: F.topk_distill_loss(s, s.detach(), torch.zeros_like(s, dtype=torch.int32), reduction="none"),
                         [torch.randn(5, 6, device="cuda")]))
    for name, f, args in cases:
        plain = [(-a).requires_grad_(True) for a in args]
        views = [negated(a.clone()).requires_grad_(True) for a in args]
        assert all(v.is_neg() and torch.equal(v, p) for v, p in zip(views, plain))
        with torch.no_grad():
            assert torch.equal(f(*views), f(*plain)), name
        y, want = f(*views), f(*plain)
        assert torch.equal(y, want), name
        dy = torch.randn_like(want)
        for p, q in zip(torch.autograd.grad(y, views, negated(-dy)), torch.autograd.grad(want, plain, dy)):
            assert torch.equal(p, q), name
    part = torch.randn(4, 6, dtype=torch.cfloat, device="cuda").conj().imag
    assert part.is_neg() and torch.equal(F.layer_norm(part), F.layer_norm(part.resolve_neg()))


def test_constant_gradients_under_create_graph_warn(F):
    """A penalty on such a gradient sends nothing back, which was not said; where the gradient depends on nothing that
    requires one, and without create_graph, there is nothing to say."""
    def grad(y, *leaves, **kw):
        with warnings.catch_warnings(record=True) as seen:
            warnings.simplefilter("always")
            got = torch.autograd.grad(y, leaves, torch.ones_like(y), **kw)
        assert not any(g.requires_grad for g in got)
        return [str(w.message) for w in seen if "create_graph" in str(w.message)]

    for name, f, args in calls(F):
        leaves = [a.clone().requires_grad_(True) for a in args]
        said = grad(f(*leaves), *leaves, create_graph=True)
        assert len(said) == 1 and name in said[0], said
        assert not grad(f(*leaves), *leaves)
    (_, _, (x, w, b, _)), (_, _, (_, v, _)), _ = calls(F)
    leaf = lambda a: a.clone().requires_grad_(True)
    for y, of in ((F.linear_act(leaf(x), w), 0), (F.linear_act(x, leaf(w), activation="relu"), 0), (F.linear_act(x, w, leaf(b)), 0),
                  (F.layer_norm(x, leaf(v)), 0), (F.linear_act(x, leaf(w), activation="gelu"), 1), (F.layer_norm(leaf(x)), 1)):
        node = y.grad_fn.next_functions
        assert len(grad(y, *(n.variable for n, _ in node if n is not None), create_graph=True)) == of
