"""What topk_distill_loss is where a teacher names a class more than once: the KL divergence of the dense distributions plus a
constant of the teacher, with that KL's gradient."""
import math

import pytest
import torch

from oracle import float_oracle as O


def dense_kl(s, t, i, temp):
    """Per row temp^2 KL(P || q) with P scattered over the vocabulary, and temp^2 sum_e p_e log(p_e / P at e's class)."""
    u = torch.where(i >= 0, t.double() / temp, -math.inf)
    p = torch.softmax(u, -1)
    at = i.clamp(min=0).long()
    big = torch.zeros(s.shape, dtype=torch.float64).scatter_add(-1, at, p)
    logq = torch.log_softmax(s.double() / temp, -1)
    kl = torch.xlogy(big, big).sum(-1) - (big * logq).sum(-1)
    constant = (torch.xlogy(p, p) - torch.xlogy(p, big.gather(-1, at))).sum(-1)
    return temp * temp * kl, temp * temp * constant


def case(rows=40, vocab=7, top=6, seed=0):
    g = torch.Generator().manual_seed(seed)
    s, t = 2 * torch.randn(rows, vocab, generator=g), 2 * torch.randn(rows, top, generator=g)
    i = torch.randint(-1, vocab, (rows, top), generator=g)
    i[0], i[1], i[:, 0] = 3, torch.arange(top), i[:, 0].clamp(min=0)
    return s, t, i


@pytest.mark.parametrize("temp", [1.0, 2.0])
def test_definition(temp):
    s, t, i = case()
    kl, constant = dense_kl(s, t, i, temp)
    got = O.topk_distill(s, t, i, temp, "none", torch.ones(len(s)))
    torch.testing.assert_close(got["loss"][0], kl + constant, rtol=1e-10, atol=1e-10)
    assert constant[1].abs() < 1e-12 and (constant <= 1e-12).all() and constant[0] < -0.1
    leaf = s.double().requires_grad_(True)
    want, = torch.autograd.grad(dense_kl(leaf, t, i, temp)[0].sum(), leaf)
    torch.testing.assert_close(got["ds"][0], want, rtol=1e-10, atol=1e-10)


def test_two_entries_of_one_class():
    """Equal entries of class 0, which has all of q to 1.4e-4 at temperature 2: 4 log 2 under the KL."""
    s, t, i = torch.tensor([[20.0, 0, 0, 0]]), torch.zeros(1, 2), torch.zeros(1, 2, dtype=torch.long)
    kl = 4 * math.log(1 + 3 * math.exp(-10))
    assert abs(O.topk_distill(s, t, i, 2.0, "none")["loss"][0].item() - (kl - 4 * math.log(2))) < 1e-12


@pytest.mark.gpu
@pytest.mark.parametrize("temp", [1.0, 2.0])
def test_on_the_device(gpu, temp):
    from qnn import functional as F
    s, t, i = case(rows=500, seed=1)
    kl, constant = dense_kl(s, t, i, temp)
    leaf = s.cuda().requires_grad_(True)
    loss = F.topk_distill_loss(leaf, t.cuda(), i.cuda(), temp, "none")
    bound = O.topk_distill(s, t, i, temp, "none", torch.ones(len(s)))
    assert ((loss.detach().cpu().double() - (kl + constant)).abs() <= bound["loss"][1]).all()
    ds, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    wide = s.double().requires_grad_(True)
    want, = torch.autograd.grad(dense_kl(wide, t, i, temp)[0].sum(), wide)
    assert ((ds.cpu().double() - want).abs() <= bound["ds"][1]).all()
