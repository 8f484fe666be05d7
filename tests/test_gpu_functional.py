"""qnn.functional on the device against its definitions in float64 (oracle/float_oracle.py), at the
sizes, strides and values where such kernels go wrong.  Every tolerance is the oracle's bound."""
import ctypes
import math
import threading

import pytest
import torch

from oracle import float_oracle as O

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]


@pytest.fixture(scope="module")
def F(gpu):
    from qnn import functional
    return functional


def gen(seed):
    return torch.Generator().manual_seed(seed)


def near(got, want, name):
    v, err = want[0].detach().cpu(), want[1].detach().cpu()
    got = got.detach().cpu().double().reshape(v.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(v)), f"{name}: NaN elsewhere"
    inf = torch.isinf(v)
    assert torch.equal(got[inf], v[inf]), f"{name}: infinities"
    ok = ~(torch.isnan(v) | inf)
    over = ((got - v).abs() - err)[ok]
    if over.numel() and over.max() > 0:
        at = int(over.argmax())
        raise AssertionError(f"{name}: {int((over > 0).sum())} of {over.numel()} over the bound, worst at {at}: got "
                             f"{got[ok][at]}, want {v[ok][at]} +- {err[ok][at]}")


def dev(*ts, grad=False):
    return [None if t is None else t.to("cuda").requires_grad_(grad) for t in ts]


# ------------------------------------------------------------------------------------ linear_act
SIZES = [(1, 1, 1), (1, 8, 8), (1, 1000, 513), (1, 1040, 2048), (2, 130, 4100), (3, 5, 7), (7, 72, 1536), (16, 64, 64),
         (17, 130, 72), (31, 24, 264), (33, 1000, 512), (64, 64, 32), (65, 257, 96), (127, 129, 131), (128, 256, 64),
         (200, 1000, 515), (257, 512, 256), (300, 8, 4096), (2050, 40, 24), (520, 776, 328)]


def linear_case(m, n, k, dt, bias, res, seed=0):
    g = gen(seed + m * 7 + n * 3 + k)
    x, w = torch.randn(m, k, generator=g).to(dt), (torch.randn(n, k, generator=g) / math.sqrt(k)).to(dt)
    b = torch.randn(n, generator=g).to(dt) if bias else None
    r = torch.randn(m, n, generator=g).to(dt) if res else None
    return x, w, b, r, torch.randn(m, n, generator=g).to(dt)


def linear_check(F, x, w, b, r, dy, act, label=""):
    dx, dw_, db_, dr_ = dev(x, w, b, r, grad=True)
    want = O.linear_act(x, w, b, r, act, dy)
    with torch.no_grad():
        near(F.linear_act(dx, dw_, db_, dr_, act), want["y"], label + "y (no grad)")
    y = F.linear_act(dx, dw_, db_, dr_, act)
    near(y, want["y"], label + "y")
    leaves = {"dx": dx, "dw": dw_, "db": db_, "dr": dr_}
    leaves = {k: v for k, v in leaves.items() if v is not None}
    for k, v in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy.to("cuda"))):
        assert v.dtype == x.dtype and v.shape == leaves[k].shape
        near(v, want[k], label + k)


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_linear_act(F, dt, m, n, k):
    for j, act in enumerate(("none", "relu", "gelu")):
        print(m, n, k, dt, act, flush=True)
        x, w, b, r, dy = linear_case(m, n, k, dt, (m + j) % 2 == 0, (n + j) % 3 != 0)
        linear_check(F, x, w, b, r, dy, act, f"{act} ")


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(700, 1100, 900), (1024, 768, 512), (1, 4096, 4096), (12, 3000, 1000), (40, 520, 6000)])
def test_linear_act_larger(F, dt, m, n, k):
    x, w, b, r, dy = linear_case(m, n, k, dt, True, True)
    linear_check(F, x, w, b, r, dy, "gelu")


def plan(m, n, k, dt, grads):
    from qnn import _lib
    tm, tn, sp = ctypes.c_int(), ctypes.c_int(), (ctypes.c_int * 2)()
    _lib.call("qnn_linear_act_plan", m, n, k, code_of(dt), int(grads), ctypes.byref(tm), ctypes.byref(tn), sp)
    return (tm.value, tn.value), tuple(sp)


def code_of(dt):
    return TYPES.index(dt) + 1 if dt != torch.float32 else 0  # QNN_BF16, QNN_F16, QNN_F32


# sizes whose products take every tile, split and whole, with ragged edges on each side
TILED = [(300, 200, 4000), (700, 5100, 136), (1500, 1900, 1032), (2100, 3900, 360), (4200, 4100, 520), (4090, 4000, 4072), (30000, 72, 40), (50, 40, 20000),
         (1030, 1020, 999), (510, 4080, 1024)]


@pytest.mark.parametrize("m,n,k", TILED)
@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_linear_act_every_tile(F, dt, m, n, k):
    """Against the definition in float64 on the device."""
    print(m, n, k, dt, plan(m, n, k, dt, False), plan(m, n, k, dt, True), flush=True)
    x, w, b, r, dy = dev(*linear_case(m, n, k, dt, True, (m + n) % 200 != 0))
    act = ("gelu", "relu", "none")[(m + k) // 10 % 3]
    want = O.linear_act(x, w, b, r, act, dy)
    leaves = {"dx": x, "dw": w, "db": b, "dr": r}
    leaves = {q: v.requires_grad_(True) for q, v in leaves.items() if v is not None}
    y = F.linear_act(x, w, b, r, act)
    near(y, want["y"], "y")
    for q, v in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)):
        near(v, want[q], q)


def test_tiled_sizes_take_every_tile(F):
    for dt in TYPES:
        for grads in (False, True):
            seen = {(plan(*z, dt, grads)[0], max(plan(*z, dt, grads)[1]) > 1) for z in TILED}
            tiles = {t for t, _ in seen}
            assert tiles >= ({(64, 64)} if dt == torch.float32 else {(256, 256), (128, 128), (128, 64)}), seen
            assert dt != torch.float32 or {(128, 128), (128, 64)} & tiles, seen
            assert {s for _, s in seen} == {False, True}, seen


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(20, 70, 1), (20, 70, 5), (33, 65, 31), (64, 64, 33), (65, 130, 47), (100, 1001, 95), (203, 500, 129),
                                   (64, 100, 4001), (130, 2001, 515), (1000, 1001, 259), (40, 33, 20001)])
def test_linear_act_rows_that_begin_anywhere(F, dt, m, n, k):
    """Odd lengths around whole stages, short and split reductions, edges on both sides."""
    x, w, b, r, dy = linear_case(m, n, k, dt, True, k % 4 == 1)
    linear_check(F, x, w, b, r, dy, "gelu" if m % 2 else "none")


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(20, 70, 2), (20, 70, 6), (33, 66, 30), (65, 130, 46), (64, 6, 100), (17, 10, 12), (100, 1002, 94), (64, 100, 4002),
                                   (130, 2002, 514), (1000, 1002, 258), (40, 34, 20002), (203, 1006, 1030), (510, 4082, 1026),
                                   (700, 5102, 138), (1, 70, 4098), (18, 1000, 1002), (2002, 1470, 1034)])
def test_linear_act_rows_that_begin_at_words(F, dt, m, n, k):
    """Even lengths that are no whole groups, around whole stages, short and split reductions, edges on both sides."""
    x, w, b, r, dy = linear_case(m, n, k, dt, m % 2 == 0, k % 4 == 2)
    linear_check(F, x, w, b, r, dy, ("none", "gelu", "relu")[m % 3])


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("n,k", [(66, 72), (72, 66), (66, 70), (66, 67), (67, 66)])
@pytest.mark.parametrize("m", [30, 200])
def test_linear_act_infinities_at_the_ends_of_rows(F, dt, m, n, k):
    """An infinity in a row's last element, next to the following row's first, stays in its row and column, and what lies
    between the rows is not read."""
    def matrix(rows, cols, gap, seed, at):
        v = torch.full((rows, cols + gap), math.nan, dtype=dt, device="cuda")
        v[:, :cols] = torch.randn(rows, cols, generator=gen(seed)).to(dt).cuda()
        for i, j in at:
            v[i, j] = math.inf
        return v[:, :cols]
    for gap in (0, 2, 3):
        a, c = matrix(m, k, gap, 60, [(3, k - 1), (4, 0)]), matrix(n, k, gap, 61, [(9, k - 1), (12, 0)])
        d = matrix(m, n, gap, 62, [(5, n - 1), (7, 0), (m - 1, n - 1)])
        want = O.linear_act(a.cpu(), c.cpu(), None, None, "none", d.cpu())
        a.requires_grad_(True), c.requires_grad_(True)
        y = F.linear_act(a, c)
        assert torch.isfinite(want["y"][0]).any() and not torch.isfinite(want["dw"][0]).all()
        near(y, want["y"], f"{gap} y")
        for q, v in zip(("dx", "dw"), torch.autograd.grad(y, (a, c), d)):
            near(v, want[q], f"{gap} {q}")


@pytest.mark.parametrize("dt", TYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("m,n,k", [(1336, 700, 1000), (4090, 3900, 72), (300, 200, 4008), (410, 2720, 1016), (260, 300, 8), (140, 1000, 20024),
                                   (2100, 2050, 1032)])
def test_linear_act_rows_off_64_byte_boundaries(F, dt, m, n, k):
    """Rows that begin at every 16 bytes between two such boundaries, by their stride and by their first one, with NaN
    between them; products whole and split."""
    def matrix(rows, cols, before, after, seed):
        v = torch.full((rows, before + cols + after), math.nan, dtype=dt, device="cuda")
        v[:, before:before + cols] = torch.randn(rows, cols, generator=gen(seed)).to(dt).cuda() / (1 if seed else math.sqrt(cols))
        return v[:, before:before + cols]
    for before, after in ((0, 0), (8, 8), (24, 64 - (24 + k) % 32), (16, 24)):
        print(m, n, k, dt, before, plan(m, n, k, dt, False), plan(m, n, k, dt, True), flush=True)
        x, w, dy = matrix(m, k, before, after, 1), matrix(n, k, after, before, 0), matrix(m, n, 8, 8, 2)
        want = O.linear_act(x, w, None, None, "none", dy)
        x.requires_grad_(True), w.requires_grad_(True)
        y = F.linear_act(x, w)
        near(y, want["y"], "y")
        for q, v in zip(("dx", "dw"), torch.autograd.grad(y, (x, w), dy)):
            near(v, want[q], q)


def test_linear_act_low_tiles_are_taken(F):
    assert {plan(m, n, k, torch.float32, g)[0] for m, n, k in ((18, 1000, 1002), (20, 4096, 1000), (30, 10000, 2000), (510, 500, 512)) for g in (False, True)} >= {(32, 64)}


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_linear_act_around_few_rows(F, dt):
    for m in (2, 4, 8, 15, 16, 17, 18):
        for n, k in ((50, 1000), (33, 77), (16, 2050)):
            x, w, b, r, dy = linear_case(m, n, k, dt, True, m % 2 == 0)
            linear_check(F, x, w, b, r, dy, "gelu" if m % 3 else "relu", f"{m} {n} {k} ")


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_linear_act_strides(F, dt):
    """Sliced, transposed, misaligned, broadcast and three-dimensional operands give what dense ones do."""
    g = gen(5)
    big = torch.randn(90, 300, generator=g).to(dt).cuda()
    wt = (torch.randn(129, 70, generator=g) / 12).to(dt).cuda()
    row = torch.randn(70, generator=g).to(dt).cuda()
    for x in (big[:, 8:137], big[::2, 3:132], big[:, ::2][:, :129], big.t()[:90, :90].t().contiguous()[:, :64].repeat(1, 3)[:, :129],
              big[5:6, 1:130], big.flatten()[1:1 + 129 * 8].view(8, 129), big[:1, :129].expand(6, 129),
              big[:88, :258].reshape(4, 22, 258)[:, 1:5, ::2]):
        w, r = wt.t(), row.expand(*x.shape[:-1], 70)
        linear_check(F, x.cpu().reshape(-1, 129), w.cpu(), None, r.cpu().reshape(-1, 70), torch.ones(x[..., 0].numel(), 70, dtype=dt), "gelu")
        want = O.linear_act(x.cpu(), w.cpu(), row.cpu(), r.cpu(), "relu")
        got = F.linear_act(x, w, row, r, "relu")
        assert got.shape == (*x.shape[:-1], 70) and got.is_contiguous()
        near(got, want["y"], "y")
    # a broadcast residual's gradient, through autograd's own expand
    x, w = big[:, :128].detach().clone().requires_grad_(True), wt[:128].t().contiguous()
    rr = row.clone().requires_grad_(True)
    dy = torch.randn(90, 70, generator=g).to(dt).cuda()
    got, = torch.autograd.grad(F.linear_act(x, w, None, rr.expand(90, 70)), rr, dy)
    want = dy.double().sum(0).cpu()
    assert (got.cpu().double() - want).abs().max() <= 90 * torch.finfo(dt).eps * dy.double().abs().sum(0).max().item()


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_linear_act_rows_with_aligned_stride_and_odd_length(F, dt):
    """A row stride of whole 16-byte groups over rows that are not: what lies between the rows is not read."""
    x = torch.full((40, 80), math.nan, dtype=dt, device="cuda")
    x[:, :67] = torch.randn(40, 67, generator=gen(6)).to(dt).cuda()
    w = torch.full((33, 72), math.inf, dtype=dt, device="cuda")
    w[:, :67] = torch.randn(33, 67, generator=gen(7)).to(dt).cuda()
    dy = torch.full((40, 40), math.nan, dtype=dt, device="cuda")
    dy[:, :33] = torch.randn(40, 33, generator=gen(8)).to(dt).cuda()
    a, b = x[:, :67].detach().requires_grad_(True), w[:, :67].detach().requires_grad_(True)
    want = O.linear_act(a.detach().cpu(), b.detach().cpu(), None, None, "none", dy[:, :33].cpu())
    y = F.linear_act(a, b)
    near(y, want["y"], "y")
    for k, v in zip(("dx", "dw"), torch.autograd.grad(y, (a, b), dy[:, :33])):
        near(v, want[k], k)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_linear_act_special_values(F, dt):
    """Infinities and NaN stay in their rows; the activations' limits."""
    x = torch.zeros(20, 16, dtype=dt)
    x[:, 0] = torch.linspace(-9, 9, 20).to(dt)
    x[3, 0], x[5, 0], x[7, 0] = math.inf, -math.inf, math.nan
    w = torch.zeros(9, 16, dtype=dt)
    w[:, 0] = 1
    for act in ("none", "relu", "gelu"):
        xd = x.cuda().requires_grad_(True)
        y = F.linear_act(xd, w.cuda(), None, None, act)
        z = x[:, :1].double().expand(20, 9)
        want = {"none": z, "relu": torch.where(z <= 0, 0.0, z), "gelu": O.gelu(z)[0]}[act]
        # w's zeros times an infinity are NaN by the definition, for every column but none here: x's other columns are 0
        # the last term: fp16's values below 2^-14 are 2^-24 apart, so off by up to 2^-25 (gelu(-5.2) = -4.9e-7)
        near(y, (want, 64 * torch.finfo(torch.float32).eps * want.abs() + torch.finfo(dt).eps / 2 * want.abs() + 1e-9 + O._tiny(dt)), act)
        dx, = torch.autograd.grad(y, xd, torch.ones(20, 9, dtype=dt).cuda())
        slope = {"none": torch.ones(20, dtype=torch.float64), "relu": torch.where(z[:, 0] <= 0, 0.0, 1.0), "gelu": O.gelu(z[:, 0])[1]}[act]
        if act == "gelu":
            slope[7] = math.nan
        got = dx[:, 0].cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(slope))
        ok = ~torch.isnan(slope)
        assert ((got - 9 * slope)[ok].abs() <= 9 * (torch.finfo(dt).eps * 1.2 + 4e-5)).all()


def test_linear_act_empty_and_partial_needs(F):
    x = torch.zeros(0, 12, device="cuda", requires_grad=True)
    w = torch.randn(5, 12, device="cuda", requires_grad=True)
    b = torch.randn(5, device="cuda", requires_grad=True)
    for act in ("none", "gelu"):
        y = F.linear_act(x, w, b, None, act)
        assert y.shape == (0, 5)
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert gx.shape == (0, 12) and not gw.any() and not gb.any() and gw.shape == w.shape
    assert F.linear_act(torch.zeros(2, 0, 12, device="cuda"), w).shape == (2, 0, 5)
    x = torch.randn(6, 12, device="cuda")
    for leaf in (w, b):
        g, = torch.autograd.grad(F.linear_act(x, w, b, None, "gelu").sum(), leaf)
        near(g, O.linear_act(x.cpu(), w.detach().cpu(), b.detach().cpu(), None, "gelu", torch.ones(6, 5))[
            "dw" if leaf is w else "db"], "partial")


def test_linear_act_refusals(F):
    x, w = torch.zeros(2, 4, device="cuda"), torch.zeros(3, 4, device="cuda")
    for bad, word in ((lambda: F.linear_act(x, w.half()), "weight"), (lambda: F.linear_act(x.double(), w.double()), "x of"),
                      (lambda: F.linear_act(x, w, torch.zeros(3, device="cuda").half()), "bias")):
        with pytest.raises(TypeError, match=word):
            bad()
    for bad, word in ((lambda: F.linear_act(x, w[:, :3]), "in"), (lambda: F.linear_act(x, w, torch.zeros(4, device="cuda")), "bias"),
                      (lambda: F.linear_act(x, w, None, torch.zeros(1, 3, device="cuda")), "residual"),
                      (lambda: F.linear_act(x, w, activation="tanh"), "activation"), (lambda: F.linear_act(x[:, :0], w[:, :0]), "features"),
                      (lambda: F.linear_act(x[:, :1].expand(2, (1 << 21) + 1), w[:, :1].expand(3, (1 << 21) + 1)), "2\\^21"),
                      (lambda: F.linear_act(x, w[0]), "weight")):
        with pytest.raises(ValueError, match=word):
            bad()
    with pytest.raises(RuntimeError, match="bias"):
        F.linear_act(x, w, torch.zeros(3))


# ------------------------------------------------------------------------------------ layer_norm
def norm_check(F, x, w, b, dy, eps=1e-5):
    xd, wd, bd = dev(x, w, b, grad=True)
    want = O.layer_norm(x, w, b, eps, dy)
    with torch.no_grad():
        near(F.layer_norm(xd, wd, bd, eps), want["y"], "y (no grad)")
    y = F.layer_norm(xd, wd, bd, eps)
    near(y, want["y"], "y")
    leaves = {k: v for k, v in {"dx": xd, "dw": wd, "db": bd}.items() if v is not None}
    for k, v in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy.to("cuda"))):
        assert v.dtype == leaves[k].dtype and v.shape == leaves[k].shape
        near(v, want[k], k)


@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 2048), (2, 3), (3, 64), (5, 100), (7, 512), (9, 513), (1000, 24), (64, 1000),
                                      (17, 1024), (33, 1537), (6, 2056), (130, 4096), (4, 5003), (3, 8192), (2, 8200), (2, 16384),
                                      (2, 40000), (1030, 136), (700, 640)])
@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_layer_norm(F, dt, rows, dim):
    g = gen(rows + dim)
    x = (torch.randn(rows, dim, generator=g) * torch.exp(torch.randn(rows, 1, generator=g)) + 3 * torch.randn(rows, 1, generator=g)).to(dt)
    dy = torch.randn(rows, dim, generator=g).to(dt)
    for wt, has_w, has_b in ((dt, True, True), (torch.float32, True, True), (dt, False, False), (dt, True, False), (torch.float32, False, True)):
        w = (1 + 0.3 * torch.randn(dim, generator=g)).to(wt) if has_w else None
        b = torch.randn(dim, generator=g).to(wt) if has_b else None
        norm_check(F, x, w, b, dy)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_layer_norm_at_every_width(F, dt):
    """Both sides of each width at which the kernels change, and rows that are no whole number of groups."""
    g = gen(12)
    group = 4 if dt == torch.float32 else 8
    for groups in (1, 16, 64, 128, 256, 512, 1024, 2048, 4096):
        for dim in (groups * group - 1, groups * group, groups * group + 1):
            if dim < 1:
                continue
            x, dy = torch.randn(3, dim, generator=g).to(dt), torch.randn(3, dim, generator=g).to(dt)
            norm_check(F, x, torch.randn(dim, generator=g).to(dt), torch.randn(dim, generator=g).to(dt), dy)
    for rows, dim in ((3000, 40), (2600, 136), (1700, 264), (1300, 2056)):  # more rows than one turn of the launch
        x, dy = torch.randn(rows, dim, generator=g).to(dt), torch.randn(rows, dim, generator=g).to(dt)
        norm_check(F, x, torch.randn(dim, generator=g), None, dy)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_layer_norm_hard_rows(F, dt):
    """Rows of one value (variance 0), far from 0, very small and very large, infinite and NaN."""
    g = gen(9)
    x = torch.randn(12, 520, generator=g)
    x[0] = 3.0
    x[1] = 0.0
    x[2] += 1000
    x[3] *= 1e-3
    x[4] *= 1e3
    x = x.to(dt)
    w, b = torch.randn(520, generator=g).to(dt), torch.randn(520, generator=g).to(dt)
    norm_check(F, x, w, b, torch.randn(12, 520, generator=g).to(dt))
    x[5, 7], x[6, 519], x[7, 0] = math.inf, math.nan, -math.inf
    y = F.layer_norm(x.cuda(), w.cuda(), b.cuda()).cpu()
    assert y[5:8].isnan().all() and y[:5].isfinite().all() and y[8:].isfinite().all()


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_layer_norm_strides(F, dt):
    g = gen(10)
    big = torch.randn(60, 400, generator=g).to(dt).cuda()
    w = torch.randn(150, generator=g).to(dt).cuda()
    dys = torch.randn(60, 400, generator=g).to(dt).cuda()
    for x, dy in ((big[:, 8:158], dys[:, 16:166]), (big[::3, 1:151], dys[::3, 3:153]), (big[:, ::2][:, :150], dys[:, 1::2][:, :150]),
                  (big.t()[:150, :].t(), dys.t()[:150].t()), (big[:1, :150].expand(5, 150), dys[:1, :150].expand(5, 150)),
                  (big[:, :300].reshape(4, 15, 300)[:, 2:9, :150], dys[:, :300].reshape(4, 15, 300)[:, 2:9, :150])):
        want = O.layer_norm(x.cpu(), w.cpu(), None, 1e-6, dy.cpu())
        a, ww = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = F.layer_norm(a, ww, None, 1e-6)
        assert y.shape == x.shape
        near(y, want["y"], "y")
        for k, v in zip(("dx", "dw"), torch.autograd.grad(y, (a, ww), dy)):
            near(v, want[k], k)


def test_layer_norm_empty_and_refusals(F):
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    y = F.layer_norm(x, w, w)
    gx, gw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == (0, 8) and gx.shape == (0, 8) and not gw.any()
    x = torch.zeros(3, 8, device="cuda")
    for bad in (lambda: F.layer_norm(x[:, :0]), lambda: F.layer_norm(x, w[:4]), lambda: F.layer_norm(x, eps=-1.0),
                lambda: F.layer_norm(x, eps=math.nan), lambda: F.layer_norm(x, None, w.view(1, 8))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: F.layer_norm(x.double()), lambda: F.layer_norm(x, w.half()), lambda: F.layer_norm(x.half(), w.half(), w),
                lambda: F.layer_norm(x.half(), w.bfloat16())):
        with pytest.raises(TypeError):
            bad()


# ----------------------------------------------------------------------------- topk_distill_loss
def distill_case(rows, vocab, top, dt, tdt, seed=0):
    g = gen(seed + rows + vocab + top)
    s = (3 * torch.randn(rows, vocab, generator=g)).to(dt)
    t = (2 * torch.randn(rows, top, generator=g) + 4).to(tdt)
    i = torch.randint(0, vocab, (rows, top), generator=g)  # a class twice where vocab is small
    i = torch.where(torch.rand(rows, top, generator=g) < 0.15, -1 - i, i)
    if rows > 2:
        i[1] = -1
    return s, t, i


def distill_check(F, s, t, i, temp, reduction, grad=None):
    want = O.topk_distill(s.cpu(), t.cpu(), i.cpu(), temp, reduction, grad)
    sd = s.cuda().requires_grad_(True)
    t, i = t.cuda(), i.cuda()
    with torch.no_grad():
        near(F.topk_distill_loss(sd, t, i, temp, reduction), want["loss"], "loss (no grad)")
    loss = F.topk_distill_loss(sd, t, i, temp, reduction)
    assert loss.dtype == torch.float32 and loss.shape == (s.shape[:-1] if reduction == "none" else ())
    near(loss, want["loss"], "loss")
    ds, = torch.autograd.grad(loss, sd, torch.ones_like(loss) if grad is None else grad.cuda())
    assert ds.dtype == s.dtype and ds.shape == s.shape
    near(ds, want["ds"], "ds")


@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 5), (3, 7, 3), (4, 10, 40), (128, 1000, 5), (5, 1001, 20), (2, 8192, 1024),
                                            (1, 131072, 100), (9, 50021, 33), (600, 264, 8), (3, 16384, 256), (17, 33000, 64), (1100, 40, 3)])
@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_topk_distill(F, dt, rows, vocab, top):
    for n, (temp, reduction, tdt, it) in enumerate(((1.0, "mean", dt, torch.int64), (4.0, "sum", torch.float32, torch.int32),
                                                    (0.5, "none", torch.float16, torch.int64))):
        print(rows, vocab, top, dt, reduction, flush=True)
        s, t, i = distill_case(rows, vocab, top, dt, tdt, n)
        grad = torch.randn(rows, generator=gen(n)) if reduction == "none" else torch.tensor(-1.5) if reduction == "sum" else None
        distill_check(F, s, t, i.to(it), temp, reduction, grad)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,vocab,top", [(2, 4095, 3), (2, 4096, 3), (2, 4097, 3), (3, 8191, 3), (3, 8192, 3), (3, 8193, 3), (16, 30000, 9),
                                            (17, 30000, 9), (1, 200001, 1024), (520, 9000, 4), (20000, 11, 2)])
def test_topk_distill_where_the_kernels_change(F, dt, rows, vocab, top):
    s, t, i = distill_case(rows, vocab, top, dt, torch.float32)
    distill_check(F, s, t, i, 2.0, "mean")


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("vocab", [50, 4099, 66000])
def test_topk_distill_hard_rows(F, dt, vocab):
    g = gen(vocab)
    s = torch.randn(12, vocab, generator=g)
    t = torch.randn(12, 6, generator=g)
    i = torch.stack([torch.randperm(vocab, generator=g)[:6] for _ in range(12)])
    i[0] = i[0, 0]                       # one class six times
    i[1] = -1                            # nothing is left
    t[2] = -math.inf                     # nothing is left either
    t[3, :5] = -math.inf                 # one entry with all of the mass
    s[4, i[4, 0]] = -math.inf            # a masked class that the teacher names: loss inf
    s[5, :] = torch.finfo(dt).min / 4    # every class as low as masks go
    s[6, vocab // 2:] = -math.inf        # half of the vocabulary masked
    i[6] = torch.arange(6)
    t[6, 0] = -math.inf                  # and an entry without mass at a masked class
    s[6, 0] = -math.inf
    i[7, 2:] = -7
    s[8] = s[8] * 20
    s[9, 0] = 3e4
    i[10, 5], i[11, 5] = vocab - 1, 0
    s, t = s.to(dt), t.to(dt)
    distill_check(F, s, t, i, 1.0, "none", torch.randn(12, generator=g))
    distill_check(F, s[[0, 1, 2, 3, 6, 7]], t[[0, 1, 2, 3, 6, 7]], i[[0, 1, 2, 3, 6, 7]], 2.0, "mean")
    # rows that are NaN by the definition, alone
    s[0, 3], s[1, 1] = math.nan, math.nan
    s[2], t[2] = -math.inf, 1.0
    i[3, 0], i[4, 1] = vocab, 1 << 40
    s[5, 2] = math.inf
    t[8, 1] = math.nan
    sd = s.cuda().requires_grad_(True)
    loss = F.topk_distill_loss(sd, t.cuda(), i.cuda(), 1.0, "none")
    ds, = torch.autograd.grad(loss, sd, torch.ones_like(loss))
    nans = [True, False, True, True, True, True, False, False, True, False, False, False]
    assert loss.cpu().isnan().tolist() == nans and ds.cpu().isnan().any(1).tolist() == nans
    assert ds[[2, 3, 4, 8]].isnan().all() and not ds[1].any()


def test_topk_distill_nothing_counted(F):
    s = torch.randn(5, 30, device="cuda", requires_grad=True)
    i = torch.full((5, 4), -1, device="cuda")
    for reduction in ("mean", "sum", "none"):
        loss = F.topk_distill_loss(s, torch.randn(5, 4, device="cuda"), i, 1.0, reduction)
        ds, = torch.autograd.grad(loss.sum(), s)
        assert not loss.any() and not ds.any()
    loss = F.topk_distill_loss(s[:0], torch.zeros(0, 4, device="cuda"), i[:0])
    assert loss.item() == 0.0 and torch.autograd.grad(loss, s)[0].shape == s.shape


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_topk_distill_strides(F, dt):
    s, t, i = distill_case(24, 600, 12, dt, dt)
    big = torch.full((24, 616), math.nan, dtype=dt)
    big[:, 8:608] = s
    odd = torch.full((24, 603), math.nan, dtype=dt)
    odd[:, 2:602] = s
    want = O.topk_distill(s, t, i, 1.0, "mean")
    for v in (big.cuda()[:, 8:608], odd.cuda()[:, 2:602], s.t().contiguous().cuda().t(), s.cuda().view(4, 6, 600)):
        lead = v.shape[:-1]
        v = v.detach().requires_grad_(True)
        loss = F.topk_distill_loss(v, t.t().contiguous().cuda().t().reshape(*lead, 12), i.cuda().repeat_interleave(2, 1)[:, ::2].reshape(*lead, 12))
        near(loss, want["loss"], "loss")
        near(torch.autograd.grad(loss, v)[0], want["ds"], "ds")


def test_topk_distill_refusals(F):
    s, t, i = torch.zeros(2, 9, device="cuda"), torch.zeros(2, 3, device="cuda"), torch.zeros(2, 3, dtype=torch.long, device="cuda")
    for bad in (lambda: F.topk_distill_loss(s, t, i[:, :2]), lambda: F.topk_distill_loss(s, t[:1], i[:1]), lambda: F.topk_distill_loss(s, t, i, 0.0),
                lambda: F.topk_distill_loss(s, t, i, math.inf), lambda: F.topk_distill_loss(s, t, i, 1e-30), lambda: F.topk_distill_loss(s, t, i, math.nan), lambda: F.topk_distill_loss(s, t, i, reduction="batchmean"),
                lambda: F.topk_distill_loss(s, t[:, :0], i[:, :0]), lambda: F.topk_distill_loss(s, t.repeat(1, 400), i.repeat(1, 400)),
                lambda: F.topk_distill_loss(s[:, :0], t, i)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: F.topk_distill_loss(s.double(), t, i), lambda: F.topk_distill_loss(s, t, i.float()), lambda: F.topk_distill_loss(s, t.double(), i)):
        with pytest.raises(TypeError):
            bad()


# ------------------------------------------------------------------------------------- together
def mlp(F, dt, seed=0, width=96, hidden=200, vocab=777, rows=50):
    """A residual block and a head of a student, as its training step runs them."""
    g = gen(seed)
    norm, up = F.LayerNorm(width, dtype=dt), F.LinearAct(width, hidden, activation="gelu", dtype=dt)
    down, head = F.LinearAct(hidden, width, dtype=dt), F.LinearAct(width, vocab, bias=False, dtype=dt)
    mods = torch.nn.ModuleList([norm, up, down, head])
    with torch.no_grad():
        for p in mods.parameters():
            p.copy_((torch.randn(p.shape, generator=g) / math.sqrt(p.shape[-1])).to(dt))
    x = torch.randn(2, rows // 2, width, generator=g).to(dt)
    t = (3 * torch.randn(2, rows // 2, 10, generator=g)).to(dt)
    i = torch.randint(0, vocab, (2, rows // 2, 10), generator=g)
    i[0, 3] = -1
    return mods, x, t, i


def mlp_step(F, mods, x, t, i):
    norm, up, down, head = mods
    h = down(up(norm(x)), residual=x)
    return F.topk_distill_loss(head(h), t, i, temperature=2.0)


def mlp_exact(mods, x, t, i):
    norm, up, down, head = mods
    p = [v.detach().cpu().double().requires_grad_(True) for v in mods.parameters()]
    x = x.detach().cpu().double().requires_grad_(True)
    lin = torch.nn.functional.linear
    h = lin(torch.nn.functional.gelu(lin(torch.nn.functional.layer_norm(x, x.shape[-1:], p[0], p[1]), p[2], p[3])), p[4], p[5]) + x
    logq = torch.log_softmax(lin(h, p[6]) / 2, -1)
    there = i >= 0
    counted = there.any(-1)
    pt = torch.softmax(t.double()[counted] / 2, -1)
    rows = 4 * (pt * (pt.log() - logq[counted].gather(-1, i[counted]))).sum(-1)
    loss = rows.sum() / counted.sum()
    return loss.detach(), torch.autograd.grad(loss, [x, *p])


def test_training_step_of_all_three(F):
    """In float32, where each operator is within about 1e-6 of its definition: the chain of five keeps
    its gradients within 1e-4 of the largest one (a condition number of 100 allowed)."""
    mods, x, t, i = mlp(F, torch.float32)
    want_loss, want = mlp_exact(mods, x, t, i)
    mods, x = mods.cuda(), x.cuda().requires_grad_(True)
    loss = mlp_step(F, mods, x, t.cuda(), i.cuda())
    got = torch.autograd.grad(loss, [x, *mods.parameters()])
    assert abs(loss.item() - want_loss.item()) <= 1e-5 * want_loss.item()
    for a, b in zip(got, want):
        assert (a.cpu().double() - b).abs().max() <= 1e-4 * b.abs().max()


@pytest.mark.parametrize("dt", TYPES[:2], ids=IDS[:2])
def test_training_step_16_bits(F, dt):
    """The stored activations and gradients of the chain are each half a step off: ten roundings on the
    longest path from the loss to the first weight, in relation to the gradient's norm."""
    mods, x, t, i = mlp(F, dt)
    want_loss, want = mlp_exact(mods, x, t, i)
    mods, x = mods.cuda(), x.cuda().requires_grad_(True)
    loss = mlp_step(F, mods, x, t.cuda(), i.cuda())
    got = torch.autograd.grad(loss, [x, *mods.parameters()])
    u = torch.finfo(dt).eps / 2
    assert abs(loss.item() - want_loss.item()) <= 10 * u * want_loss.item()
    for a, b in zip(got, want):
        assert (a.cpu().double() - b).norm() <= 10 * u * b.norm()


def test_gradients_against_differences(F):
    """Directional derivatives in float32: a central difference of step h is off by h^2 / 6 of the third
    derivative and by the loss's error (2^-20 of its size) over h."""
    mods, x, t, i = mlp(F, torch.float32, seed=4)
    mods, x, t, i = mods.cuda(), x.cuda().requires_grad_(True), t.cuda(), i.cuda()
    leaves = [x, *mods.parameters()]
    loss = mlp_step(F, mods, x, t, i)
    grads = torch.autograd.grad(loss, leaves)
    h = 2e-2
    for leaf, gr in zip(leaves, grads):
        d = gr / gr.norm()
        with torch.no_grad():
            keep = leaf.clone()
            leaf.copy_(keep + h * d)
            up = mlp_step(F, mods, x, t, i).item()
            leaf.copy_(keep - h * d)
            down = mlp_step(F, mods, x, t, i).item()
            leaf.copy_(keep)
        slope = (up - down) / (2 * h)
        assert abs(slope - gr.norm().item()) <= 2e-2 * gr.norm().item() + 2.0 ** -20 * loss.item() / h


def test_gradients_of_gradients_are_refused(F):
    mods, x, t, i = mlp(F, torch.float32)
    mods, x = mods.cuda(), x.cuda().requires_grad_(True)
    dy = torch.randn(2, 25, 96, device="cuda", requires_grad=True)
    y = F.layer_norm(x, mods[0].weight)
    gx, = torch.autograd.grad(y, x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="layer_norm's gradients"):
        gx.sum().backward()
    up = torch.randn(2, 25, 200, device="cuda", requires_grad=True)
    gx, = torch.autograd.grad(F.linear_act(x, mods[1].weight, activation="gelu"), x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="linear_act's gradients"):
        gx.sum().backward()
    # a gradient made under create_graph is a plain one where nothing asks further
    gx, = torch.autograd.grad(F.layer_norm(x), x, dy.detach(), create_graph=True)
    assert not gx.requires_grad


def test_training_with_backward_and_accumulation(F):
    """loss.backward() into .grad, twice: the sum of two equal gradients."""
    mods, x, t, i = mlp(F, torch.bfloat16, seed=8)
    mods, x, t, i = mods.cuda(), x.cuda(), t.cuda(), i.cuda()
    mlp_step(F, mods, x, t, i).backward()
    once = [p.grad.clone() for p in mods.parameters()]
    mlp_step(F, mods, x, t, i).backward()
    assert all(torch.equal(p.grad, 2 * g) for p, g in zip(mods.parameters(), once))


def test_a_saved_input_that_was_changed_is_refused(F):
    x = torch.randn(4, 8, device="cuda")
    w = torch.randn(8, 8, device="cuda", requires_grad=True)
    y = F.linear_act(x, w)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_same_bits_every_time(F):
    for dt in TYPES:
        mods, x, t, i = mlp(F, dt, seed=2, width=264, hidden=520, rows=300)
        mods, x, t, i = mods.cuda(), x.cuda().requires_grad_(True), t.cuda(), i.cuda()
        runs = []
        for _ in range(3):
            loss = mlp_step(F, mods, x, t, i)
            runs.append([loss.detach(), *torch.autograd.grad(loss, [x, *mods.parameters()])])
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_other_stream(F):
    mods, x, t, i = mlp(F, torch.bfloat16, seed=3)
    mods, x, t, i = mods.cuda(), x.cuda().requires_grad_(True), t.cuda(), i.cuda()
    loss = mlp_step(F, mods, x, t, i)
    want = [loss.detach(), *torch.autograd.grad(loss, [x, *mods.parameters()])]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        loss = mlp_step(F, mods, x, t, i)
        got = [loss.detach(), *torch.autograd.grad(loss, [x, *mods.parameters()])]
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_two_captured_training_steps(F):
    """Two graphs captured one after the other and replayed in turn on new inputs, with eager work
    between, give what eager calls do: neither keeps its workspaces in the other's."""
    sets = [mlp(F, torch.bfloat16, seed=s, width=w, hidden=h, rows=r) for s, w, h, r in ((5, 96, 200, 50), (6, 264, 520, 300))]
    sets = [(m.cuda(), x.cuda().requires_grad_(True), t.cuda(), i.cuda()) for m, x, t, i in sets]

    def step(m, x, t, i):
        loss = mlp_step(F, m, x, t, i)
        return [loss.detach(), *torch.autograd.grad(loss, [x, *m.parameters()])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a in sets:
            step(*a)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*a))
        graphs.append(g)
    for turn in range(4):
        for a in sets:
            with torch.no_grad():
                a[1].copy_(torch.randn(a[1].shape, generator=gen(20 + turn)).to(a[1].dtype))
        for g in graphs if turn % 2 else reversed(graphs):
            g.replay()
        torch.cuda.synchronize()
        for a, out in zip(sets, outs):
            for p, q in zip(step(*a), out):
                assert torch.equal(p, q)


def test_threads_at_once(F):
    """Four threads on streams of their own, two sizes: what one alone gets."""
    cases = []
    for m, n, k in ((300, 500, 1000), (128, 1000, 512)):
        x, w, b, r, dy = dev(*linear_case(m, n, k, torch.bfloat16, True, False))
        t, i = torch.randn(m, 5, generator=gen(m)).cuda(), torch.randint(0, n, (m, 5), generator=gen(n)).cuda()
        cases.append((x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True), t, i))

    def step(x, w, b, t, i):
        y = F.linear_act(F.layer_norm(x), w, b, activation="gelu")
        return torch.autograd.grad(F.topk_distill_loss(y, t, i, 2.0), (x, w, b))

    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    got = [None] * 4

    def run(at):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got[at] = step(*cases[at % 2])
        stream.synchronize()

    threads = [threading.Thread(target=run, args=(at,)) for at in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for at in range(4):
        for p, q in zip(got[at], want[at % 2]):
            assert torch.equal(p, q)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(1, 33, 70), (5, 40, 64), (130, 67, 96), (70, 200, 130), (34, 66, 98), (150, 1002, 514), (20, 6, 10)])
def test_nothing_is_written_past_the_outputs(F, dt, m, n, k):
    """The C entries on buffers with a guard behind each output and behind the workspace."""
    from qnn import _lib
    code = code_of(dt)

    def guarded(count, dtype):
        size = count * torch.empty((), dtype=dtype).element_size()
        b = torch.full((size + 256,), 0x5A, dtype=torch.uint8, device="cuda")
        return b, size

    def work(name, *args):
        n = ctypes.c_int64(0)
        _lib.call(name, *args, ctypes.byref(n))
        return guarded(n.value, torch.uint8)

    def p(t):
        return None if t is None else t.data_ptr()

    x, w, b, r, dy = dev(*linear_case(m, n, k, dt, True, True))
    st = torch.cuda.current_stream().cuda_stream
    for act in (0, 1, 2):
        slope_n, slope_t = ((m * ((n + 7) // 8), torch.uint8), (m * n, torch.float32 if code == 0 else torch.int16))[act == 2]
        outs = {"y": guarded(m * n, dt), "slope": guarded(slope_n, slope_t), "dz": guarded(m * n, dt), "dx": guarded(m * k, dt),
                "dw": guarded(n * k, dt), "db": guarded(n, dt), "wf": work("qnn_linear_act_fwd_work", m, n, k, code),
                "wb": work("qnn_linear_act_bwd_work", m, n, k, code)}
        a = {q: p(v[0]) for q, v in outs.items()}
        _lib.call("qnn_linear_act_fwd", p(x), k, p(w), k, p(b), p(r), n, a["y"], a["slope"] if act else None, m, n, k, code, act, a["wf"],
                  outs["wf"][1], st)
        _lib.call("qnn_linear_act_bwd", p(dy), n, a["slope"], p(x), k, p(w), k, a["dz"], a["dx"], a["dw"], a["db"], m, n, k, code, act,
                  a["wb"], outs["wb"][1], st)
        for q, (buf, size) in outs.items():
            assert (buf[size:] == 0x5A).all(), q
    outs = {"y": guarded(m * k, dt), "mean": guarded(m, torch.float32), "rstd": guarded(m, torch.float32), "dx": guarded(m * k, dt),
            "dw": guarded(k, dt), "db": guarded(k, dt), "wb": work("qnn_layer_norm_bwd_work", m, k, code)}
    a = {q: p(v[0]) for q, v in outs.items()}
    _lib.call("qnn_layer_norm_fwd", p(x), k, p(w), p(w), a["y"], a["mean"], a["rstd"], m, k, 1e-5, code, code, st)
    _lib.call("qnn_layer_norm_bwd", p(x), k, p(x), k, p(w), a["mean"], a["rstd"], a["dx"], a["dw"], a["db"], m, k, code, code, a["wb"],
              outs["wb"][1], st)
    for q, (buf, size) in outs.items():
        assert (buf[size:] == 0x5A).all(), q
    i = torch.randint(-3, k, (m, 5), generator=gen(m)).cuda()
    t = torch.randn(m, 5, device="cuda")
    grad = torch.ones(1, device="cuda")
    outs = {"rl": guarded(m, torch.float32), "stats": guarded(4 * m + 4, torch.float32), "loss": guarded(1, torch.float32),
            "ds": guarded(m * k, dt), "wf": work("qnn_topk_distill_fwd_work", m, k, code)}
    a = {q: p(v[0]) for q, v in outs.items()}
    _lib.call("qnn_topk_distill_fwd", p(x), k, p(t), 5, p(i), 5, m, k, 5, 1.0, 1, code, 0, 8, a["rl"], a["stats"], a["loss"], a["wf"],
              outs["wf"][1], st)
    _lib.call("qnn_topk_distill_bwd", p(x), k, p(t), 5, p(i), 5, a["stats"], p(grad), 0, a["ds"], m, k, 5, 1.0, 1, code, 0, 8, st)
    for q, (buf, size) in outs.items():
        assert (buf[size:] == 0x5A).all(), q


# ------------------------------------------------------------------------------------ past 32 bits
def large(*shape, seed):
    """bf16 on the device, over 2^31 elements."""
    assert math.prod(shape) > 2 ** 31
    return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(seed))


def test_linear_act_long_batch(F):
    m, n, k = 131080, 40, 16392
    x = large(m, k, seed=1).requires_grad_(True)
    w = (torch.randn(n, k, generator=gen(2)) / math.sqrt(k)).bfloat16().cuda().requires_grad_(True)
    dy = torch.randn(m, n, generator=gen(3)).bfloat16().cuda()
    y = F.linear_act(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    with torch.no_grad():
        for at in (slice(0, 40), slice(m - 40, m)):
            want = O.linear_act(x[at].cpu(), w.cpu(), None, None, "none", dy[at].cpu())
            near(y[at], want["y"], "y")
            near(dx[at], want["dx"], "dx")
        value, size = 0.0, 0.0
        for i in range(0, m, 8192):
            a, b = dy[i:i + 8192].t().double(), x[i:i + 8192].double()
            value, size = value + a @ b, size + a.abs() @ b.abs()
        near(dw, O._out(value, (m + 1) * O.E * size, torch.bfloat16), "dw")


@pytest.mark.parametrize("m", [1, 2, 20])
def test_linear_act_large_weight(F, m):
    n, k = 36000, 60000
    x = torch.randn(m, k, generator=gen(4)).bfloat16().cuda().requires_grad_(True)
    w = large(n, k, seed=5).requires_grad_(True)
    dy = torch.randn(m, n, generator=gen(6)).bfloat16().cuda()
    y = F.linear_act(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    with torch.no_grad():
        for at in (slice(0, 40), slice(n - 40, n)):
            want = O.linear_act(x.cpu(), w[at].cpu(), None, None, "none", dy[:, at].cpu())
            near(y[:, at], want["y"], "y")
            near(dw[at], want["dw"], "dw")
        value, size = 0.0, 0.0
        for i in range(0, n, 4096):
            a, b = dy[:, i:i + 4096].double(), w[i:i + 4096].double()
            value, size = value + a @ b, size + a.abs() @ b.abs()
        near(dx, O._out(value, (n + 1) * O.E * size, torch.bfloat16), "dx")


def test_layer_norm_long_batch(F):
    rows, dim = 262200, 8192
    x = large(rows, dim, seed=7).requires_grad_(True)
    w, b = (torch.randn(dim, generator=gen(s)).cuda().requires_grad_(True) for s in (8, 9))
    dy = large(rows, dim, seed=10)
    y = F.layer_norm(x, w, b)
    dx, = torch.autograd.grad(y, x, dy)
    with torch.no_grad():
        for at in (slice(0, 20), slice(rows - 20, rows)):
            want = O.layer_norm(x[at].cpu(), w.cpu(), b.cpu(), 1e-5, dy[at].cpu())
            near(y[at], want["y"], "y")
            near(dx[at], want["dx"], "dx")


def test_topk_distill_long_batch(F):
    rows, vocab, top = 16400, 131072, 16
    s = large(rows, vocab, seed=11).requires_grad_(True)
    g = gen(12)
    t, i = torch.randn(rows, top, generator=g), torch.randint(0, vocab, (rows, top), generator=g)
    loss = F.topk_distill_loss(s, t.cuda(), i.cuda(), 2.0, "none")
    grad = torch.randn(rows, generator=g)
    ds, = torch.autograd.grad(loss, s, grad.cuda())
    with torch.no_grad():
        for at in (slice(0, 4), slice(rows - 4, rows)):
            want = O.topk_distill(s[at].cpu(), t[at], i[at], 2.0, "none", grad[at])
            near(loss[at], want["loss"], "loss")
            near(ds[at], want["ds"], "ds")
