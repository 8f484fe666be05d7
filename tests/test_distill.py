"""qnn.distill.top_logits without a device: what it returns and the state in which it leaves the teacher."""
import pytest
import torch

from qnn import distill


class Teacher(torch.nn.Module):
    """A head behind a norm layer whose running statistics move in train mode."""

    def __init__(self):
        super().__init__()
        self.norm, self.drop = torch.nn.BatchNorm1d(6), torch.nn.Dropout(0.5)
        self.body = torch.nn.Sequential(torch.nn.Linear(6, 9), torch.nn.BatchNorm1d(9))
        self.fails = False

    def forward(self, x):
        if self.fails:
            raise ArithmeticError("no logits")
        return self.body(self.drop(self.norm(x)))


def modes(model):
    return {name: m.training for name, m in model.named_modules()}


@pytest.mark.parametrize("training", [True, False])
def test_top_logits_leaves_every_module_in_its_mode(training):
    """Frozen norm layers in a teacher in train mode, and a part in train mode under one in eval mode, stay so,
    also where the forward raises; the logits are those of eval mode."""
    teacher = Teacher().train(training)
    teacher.norm.train(not training)
    teacher.body[1].train(not training)
    before, x = modes(teacher), torch.randn(5, 6)
    stats = [b.clone() for b in teacher.buffers()]
    values, classes = distill.top_logits(teacher, x, 3)
    assert modes(teacher) == before
    assert all(torch.equal(a, b) for a, b in zip(teacher.buffers(), stats))
    with torch.no_grad():
        want = Teacher.forward(teacher.eval(), x).topk(3)
    assert torch.equal(values, want.values) and torch.equal(classes, want.indices.int())
    for name, m in teacher.named_modules():
        m.training = before[name]
    teacher.fails = True
    with pytest.raises(ArithmeticError):
        distill.top_logits(teacher, x, 3)
    assert modes(teacher) == before
