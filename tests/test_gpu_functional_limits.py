"""The float operators at sizes where launches, offsets and sums reach their limits: rows in the millions, rows of a few
elements, rows of millions.  The definition is computed in float64 on the device."""
import math

import pytest
import torch

from oracle import float_oracle as O
from test_gpu_functional import IDS, TYPES, gen, near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def F(gpu):
    from qnn import functional
    return functional


def normal(*shape, seed, dt=torch.float32):
    return torch.randn(shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(dt)


# ------------------------------------------------------------------------------------ layer_norm
def norm_check(F, x, w, b, dy, eps=1e-5):
    want = O.layer_norm(x, w, b, eps, dy)
    with torch.no_grad():
        near(F.layer_norm(x, w, b, eps), want["y"], "y (no grad)")
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    y = F.layer_norm(*leaves, eps)
    near(y, want["y"], "y")
    for q, v in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, dy)):
        near(v, want[q], q)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("dim", range(1, 8))
def test_layer_norm_rows_shorter_than_a_group(F, dt, dim):
    """A row a thread: around a wave, a workgroup and a turn of the launch, with weights of either type and strided rows."""
    for n, rows in enumerate((1, 63, 65, 255, 257, 131071, 131073, 600000)):
        x, dy = normal(rows, dim, seed=n, dt=dt), normal(rows, dim, seed=n + 50, dt=dt)
        for wt in {dt, torch.float32}:
            norm_check(F, x.detach(), 1 + normal(dim, seed=7).to(wt) / 4, normal(dim, seed=8).to(wt), dy)
    x, dy = (normal(700, dim + 3, seed=s, dt=dt)[::2, 1:1 + dim] for s in (3, 4))
    norm_check(F, x.detach(), normal(dim, seed=7), normal(dim, seed=8), dy)
    # one gradient alone
    x, w = normal(300, dim, seed=1, dt=dt), normal(dim, seed=7, dt=dt)
    want = O.layer_norm(x, w, w, 1e-5, dy[:300])
    for at, q in enumerate(("dx", "dw", "db")):
        leaves = [x.clone(), w.clone(), w.clone()]
        leaf = leaves[at].requires_grad_(True)
        near(torch.autograd.grad(F.layer_norm(*leaves), leaf, dy[:300])[0], want[q], q)


@pytest.mark.parametrize("dt,dim", [(torch.bfloat16, 4), (torch.float16, 7), (torch.float32, 3)], ids=["bf16-4", "fp16-7", "fp32-3"])
def test_layer_norm_millions_of_short_rows(F, dt, dim):
    rows = 4_200_000
    norm_check(F, normal(rows, dim, seed=1, dt=dt), 1 + normal(dim, seed=2) / 4, normal(dim, seed=3), normal(rows, dim, seed=4, dt=dt))


@pytest.mark.parametrize("rows,dim", [(4_000_000, 3), (1 << 26, 4), (3_000_000, 520), (300_000_000, 4)])
def test_layer_norm_sums_over_many_rows(F, rows, dim):
    """dw and db of equal terms, where a long chain of fp32 additions drifts: the rows are all the same one."""
    x = torch.arange(dim, device="cuda", dtype=torch.float32).expand(rows, dim).contiguous()
    dy = torch.full((rows, dim), 1.1, device="cuda")
    w, b = torch.ones(dim, device="cuda", requires_grad=True), torch.zeros(dim, device="cuda", requires_grad=True)
    want = O.layer_norm(x[:1], w.detach(), b.detach(), 1e-5, dy[:1])
    dw, db = torch.autograd.grad(F.layer_norm(x, w, b), (w, b), dy)
    chain = (O.CHAIN + 2) * O.E
    for q, got in (("dw", dw), ("db", db)):
        value, err = want[q]
        near(got, (rows * value, rows * (err + chain * value.abs())), q)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,dim", [(2, 600_001), (1, (1 << 25) + 3)])
def test_layer_norm_rows_of_millions(F, dt, rows, dim):
    """Equal terms again, in y and dx: a large mean and a constant gradient."""
    x = (3 + normal(rows, dim, seed=1)).to(dt)
    norm_check(F, x, 1 + normal(dim, seed=2, dt=dt) / 4, normal(dim, seed=3, dt=dt), torch.full((rows, dim), 1.1, dtype=dt, device="cuda"))


# ----------------------------------------------------------------------------- topk_distill_loss
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_topk_distill_more_rows_than_a_launch_holds(F, reduction):
    """70 million rows of three classes: the rows around the launches' borders, and the mean."""
    rows, vocab = 70_000_000, 3
    s = normal(rows, vocab, seed=1, dt=torch.float16).requires_grad_(True)
    t = normal(rows, 2, seed=2, dt=torch.bfloat16)
    i = torch.randint(-1, vocab, (rows, 2), generator=torch.Generator("cuda").manual_seed(3), device="cuda", dtype=torch.int32)
    loss = F.topk_distill_loss(s, t, i, 2.0, reduction)
    grad = normal(rows, seed=4) if reduction == "none" else torch.ones((), device="cuda")
    ds, = torch.autograd.grad(loss, s, grad)
    counted = int((i >= 0).any(1).sum())
    border = ((1 << 32) - 1) // 256 * 4
    for at in (0, border - 300, border, rows - 300):
        at = slice(at, at + 300)
        part = grad[at] if reduction == "none" else torch.full((300,), 1 / counted)
        want = O.topk_distill(s[at].detach().cpu(), t[at].cpu(), i[at].cpu(), 2.0, "none", part)
        near(ds[at], (want["ds"][0], want["ds"][1] + 2 * O.E * want["ds"][0].abs()), "ds")
        if reduction == "none":
            near(loss[at], want["loss"], "loss")
    if reduction == "mean":
        with torch.no_grad():
            each = F.topk_distill_loss(s, t, i, 2.0, "none").double()
        assert abs(loss.item() - each.sum().item() / counted) <= 2 * O.E * each.abs().sum().item() / counted


def test_topk_distill_sums_over_a_large_vocabulary(F):
    """Terms 1 and e^-0.1 in turn in each of 64 pieces of a row, where a long chain of additions drifts: q from the definition."""
    vocab = (1 << 31) - 1
    s = torch.zeros(1, vocab, device="cuda")
    s[0, 1::2] = -0.1
    term = math.exp(s[0, 1].item())
    s.requires_grad_(True)
    t, i = torch.zeros(1, 1, device="cuda"), torch.zeros(1, 1, dtype=torch.long, device="cuda")
    loss = F.topk_distill_loss(s, t, i)
    ds, = torch.autograd.grad(loss, s)
    total = (vocab + 1) // 2 + vocab // 2 * term
    eps = (1.5 * 1 + 2 + O.CHAIN) * O.E
    assert abs(loss.item() - math.log(total)) <= eps * (2 + math.log(total))
    for part, value in ((ds[0, 2::2], 1 / total), (ds[0, 1::2], term / total)):
        low, high = part.aminmax()
        assert abs(low.item() / value - 1) <= eps and abs(high.item() / value - 1) <= eps
    assert abs(ds[0, 0].item() + 1 - 1 / total) <= eps


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,vocab", [(1025, 262_144), (1025, 262_147), (1025, 600_001), (1, 20_000_003)])
def test_topk_distill_rows_of_several_sums(F, dt, rows, vocab):
    """A lane's sums join into others at 262144 classes of a row that one workgroup has; largest logits early and late."""
    s = normal(rows, vocab, seed=1, dt=dt)
    s[-1, :9] += 20
    s[0, -9:] += 20
    if rows > 2:
        s[1, vocab // 2:], s[2, :vocab // 2] = -math.inf, -math.inf
    s.requires_grad_(True)
    t, i = normal(rows, 5, seed=2), torch.randint(0, vocab, (rows, 5), generator=gen(3)).cuda()
    if rows > 2:
        i[1] %= vocab // 2
        i[2] = i[2] % (vocab // 2) + vocab // 2
    loss = F.topk_distill_loss(s, t, i, 1.0, "none")
    grad = normal(rows, seed=5)
    ds, = torch.autograd.grad(loss, s, grad)
    for at in (0, 1, 2, rows - 1):
        if at < rows:
            at = slice(at, at + 1)
            want = O.topk_distill(s[at].detach().cpu(), t[at].cpu(), i[at].cpu(), 1.0, "none", grad[at])
            near(loss[at], want["loss"], "loss")
            near(ds[at], want["ds"], "ds")


# ------------------------------------------------------------------------------------ linear_act
@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_linear_act_empty_batch_of_a_large_weight(F, dt):
    """No rows through a weight of over 20 million elements, forward and backward: zeros for the gradients."""
    w, b = normal(4096, 8192, seed=1, dt=dt).requires_grad_(True), normal(4096, seed=2, dt=dt).requires_grad_(True)
    for shape in ((0, 8192), (3, 0, 8192)):
        for act in ("none", "relu", "gelu"):
            x = torch.zeros(*shape, device="cuda", dtype=dt).requires_grad_(True)
            y = F.linear_act(x, w, b, None, act)
            assert y.shape == (*shape[:-1], 4096)
            dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
            assert dx.shape == x.shape and not dw.any() and not db.any()


def test_linear_act_no_rows_and_the_largest_weight(F):
    """The gradient of a weight of over 2^32 elements from no rows: zeros, all of them."""
    n = k = 65544
    x = torch.zeros(0, k, device="cuda", dtype=torch.bfloat16)
    w = torch.empty(n, k, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    y = F.linear_act(x, w)
    torch.full((n, k), math.nan, device="cuda", dtype=torch.bfloat16)  # (what the allocator may hand out again)
    dw, = torch.autograd.grad(y, w, torch.zeros_like(y))
    assert dw.shape == w.shape and not dw.any()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_linear_act_most_rows_of_a_launch(F, dt):
    """Tall matrices of one column: single products, rounded once."""
    m = 2_000_000_001
    x = torch.empty(m, 1, device="cuda", dtype=dt).normal_(generator=torch.Generator("cuda").manual_seed(1)).requires_grad_(True)
    w = torch.tensor([[0.7]], device="cuda", dtype=dt)
    y = F.linear_act(x, w)
    with torch.no_grad():
        assert torch.equal(y, x * w)
    dx, = torch.autograd.grad(y, x, y.detach())
    with torch.no_grad():
        assert torch.equal(dx, y * w)


def test_linear_act_refuses_more(F):
    x = torch.zeros((1 << 31) - 1, 1, device="cuda", dtype=torch.float16)
    before = torch.cuda.memory_allocated()
    with pytest.raises(RuntimeError, match="too many rows"):
        F.linear_act(x, torch.ones(1, 1, device="cuda", dtype=torch.float16))
    assert torch.cuda.memory_allocated() <= before


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n", [(1 << 26, 8), (3_000_000, 600), (70_000, 30_011), (300_000_000, 2), (4097, 65)])
def test_linear_act_bias_gradient_over_many_rows(F, dt, m, n):
    """Equal terms, where a long chain of fp32 additions drifts."""
    x, b = torch.zeros(m, 1, device="cuda", dtype=dt), torch.zeros(n, device="cuda", dtype=dt).requires_grad_(True)
    dy = torch.full((m, n), 1.1e-3, device="cuda", dtype=dt)
    one = dy[0, 0].item()
    for act, slope, err in (("none", 1.0, 0.0), ("relu", 1.0, 0.0)) if m * n > 1 << 27 else (("none", 1.0, 0.0), ("relu", 1.0, 0.0), ("gelu", 0.5, 2.0 ** -14)):
        bias = b if act != "relu" else torch.ones_like(b).requires_grad_(True)
        y = F.linear_act(x, torch.zeros(n, 1, device="cuda", dtype=dt), bias, None, act)
        db, = torch.autograd.grad(y, bias, dy)
        value = torch.full((n,), m * one * slope, dtype=torch.float64)
        value, err = O._out(value, ((O.CHAIN + 2) * O.E + err) * value, dt)
        # (sums past fp16's largest, 65504: 2^26 and 3e8 terms of 1.1e-3 round to infinity)
        near(db, (torch.where(value > torch.finfo(dt).max, float("inf"), value), err), act)
