"""The student's training path over topk_distill_loss (qnn/distill.py) with the package's own models."""
import pytest
import torch

from conftest import load_fixture
from fixtures_util import build_model
from oracle import float_oracle as FO

pytestmark = pytest.mark.gpu


@pytest.fixture()
def pair(gpu):
    from qnn import synthetic
    teacher, x = build_model(load_fixture("model_resnet18_cifar"))
    student, _ = build_model(load_fixture("model_resnet18_cifar"))
    synthetic.init_params(student, 77)
    return teacher.to(gpu), student.to(gpu), x.to(gpu)


def test_top_logits(pair):
    from qnn import distill
    teacher, _, x = pair
    teacher.train()
    values, classes = distill.top_logits(teacher, x, 3)
    assert teacher.training and classes.dtype == torch.int32 and not values.requires_grad
    teacher.eval()
    with torch.no_grad():
        y = teacher(x)
    assert torch.equal(values, y.topk(3).values) and torch.equal(y.gather(1, classes.long()), values)
    with pytest.raises(ValueError, match="at least one"):
        distill.top_logits(teacher, x, 0)


@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_step_gradients_of_the_loss(pair, reduction):
    """The loss and what it sends into the student are the definition's for the student's own logits,
    and every parameter gets a finite gradient, not all zero."""
    from qnn import distill
    teacher, student, x = pair
    values, classes = distill.top_logits(teacher, x, 4)
    student.train()
    seen = []
    hook = student.register_forward_hook(lambda m, a, out: (seen.append(out), out.retain_grad())[0])
    loss = distill.step(student, x, values, classes, temperature=4.0, reduction=reduction)
    hook.remove()
    out = seen[0]
    want = FO.topk_distill(out.detach().cpu(), values.cpu(), classes.cpu(), 4.0, reduction)
    assert abs(loss.item() - want["loss"][0].item()) <= want["loss"][1].item() and not loss.requires_grad
    assert ((out.grad.cpu().double() - want["ds"][0]).abs() <= want["ds"][1]).all()
    grads = [p.grad for p in student.parameters() if p.requires_grad]
    assert all(g is not None and g.isfinite().all() for g in grads) and all(g.any() for g in grads if g.numel() > 64)


def test_step_refuses_rows_of_losses(pair):
    from qnn import distill
    teacher, student, x = pair
    values, classes = distill.top_logits(teacher, x, 2)
    with pytest.raises(ValueError, match="reduction"):
        distill.step(student, x, values, classes, reduction="none")
