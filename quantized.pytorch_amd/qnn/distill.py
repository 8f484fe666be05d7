"""Training a quantized student from a teacher of whom the top logits are kept (the float trainer of the
reference's distillation, qdistiler_main.py:874-1094, on this package's models).

The teacher runs once over the data, in eval mode through the int8 path (the cached engine where
`qnn.dispatch` builds one), and `top_logits` keeps a few values and classes of each row.  A student
step then runs the int8 forward with its straight-through backward (`qnn.quantize._QLayerTrain`) under
`qnn.functional.topk_distill_loss`, forward and backward HIP kernels:

    values, classes = distill.top_logits(teacher, images, 5)
    loss = distill.step(student, images, values, classes, temperature=4.0)   # .grad of every parameter
    optimizer.step()

Under DistributedDataParallel the student is the wrapped module; the averaging happens in backward.
"""
import torch

from .functional import topk_distill_loss

__all__ = ["top_logits", "step"]


def top_logits(teacher, images, top):
    """The `top` largest logits of each row of teacher(images) and their classes (int32), in eval mode
    and without gradients; the teacher and each of its modules are left in the mode that they were in."""
    if top < 1:
        raise ValueError(f"qnn: top_logits keeps at least one logit, got top={top}")
    training = [(m, m.training) for m in teacher.modules()]
    teacher.eval()
    try:
        with torch.no_grad():
            values, classes = torch.topk(teacher(images), top, dim=-1)
    finally:
        teacher.train(training[0][1])
        for m, mode in training:  # train() gives every module the teacher's own mode, frozen ones too
            m.training = mode
    return values, classes.int()


def step(student, images, teacher_logits, teacher_index, temperature=1.0, reduction="mean"):
    """One backward pass of the student's distillation loss on a batch: accumulates `.grad` as
    loss.backward() does and returns the loss (detached).  reduction "mean" or "sum"."""
    if reduction == "none":
        raise ValueError("qnn: distill.step needs one loss, reduction 'mean' or 'sum'")
    loss = topk_distill_loss(student(images), teacher_logits, teacher_index, temperature, reduction)
    loss.backward()
    return loss.detach()
