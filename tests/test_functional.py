"""qnn.functional without a device: what it refuses, its modules, the C entries' own checks, and the
oracle's bounds against autograd in float64."""
import ctypes
import math

import pytest
import torch

from oracle import float_oracle as O


@pytest.fixture(scope="module")
def F():
    from qnn import functional
    return functional


def test_cpu_tensors_are_refused(F):
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match="linear_act.*ROCm"):
        F.linear_act(x, w)
    with pytest.raises(RuntimeError, match="layer_norm.*ROCm"):
        F.layer_norm(x)
    with pytest.raises(RuntimeError, match="topk_distill_loss.*ROCm"):
        F.topk_distill_loss(x, x, torch.zeros(2, 4, dtype=torch.long))
    with pytest.raises(TypeError, match="tensor for x"):
        F.linear_act([1.0], w)


def test_modules_keep_torch_parameters(F):
    a, b = F.LinearAct(8, 4, activation="gelu"), torch.nn.Linear(8, 4)
    a.load_state_dict(b.state_dict(), strict=True)
    assert "gelu" in repr(a)
    F.LayerNorm(8).load_state_dict(torch.nn.LayerNorm(8).state_dict(), strict=True)
    assert F.LayerNorm(8, bias=False).bias is None
    with pytest.raises(ValueError, match="activation"):
        F.LinearAct(8, 4, activation="tanh")
    with pytest.raises(ValueError, match="last dimension"):
        F.LayerNorm((4, 8))
    with pytest.raises(ValueError, match="LayerNorm\\(8\\)"):
        F.LayerNorm(8)(torch.zeros(2, 4))


def test_package_offers_it():
    import qnn
    assert qnn.functional.linear_act and "functional" in qnn.__all__


def _call(name, *args):
    from qnn import _lib
    return getattr(_lib.load(), name)(*args), _lib.load().qnn_last_error()


P = ctypes.c_void_p(4096)  # an address that no check reads


@pytest.mark.parametrize("args,word", [
    ((P, 8, P, 8, None, None, 0, P, None, -1, 4, 8, 0, 0, None, 0, None), b"m:"),
    ((P, 8, P, 8, None, None, 0, P, None, 2, 0, 8, 0, 0, None, 0, None), b"n:"),
    ((P, 8, P, 8, None, None, 0, P, None, 2, 4, 0, 0, 0, None, 0, None), b"k:"),
    ((P, 7, P, 8, None, None, 0, P, None, 2, 4, 8, 0, 0, None, 0, None), b"stride"),
    ((P, 8, P, 8, None, P, 3, P, None, 2, 4, 8, 0, 0, None, 0, None), b"stride"),
    ((P, 8, P, 8, None, None, 0, P, None, 2, 4, 8, 7, 0, None, 0, None), b"dtype"),
    ((P, 8, P, 8, None, None, 0, P, None, 2, 4, 8, 0, 3, None, 0, None), b"act:"),
    ((None, 8, P, 8, None, None, 0, P, None, 2, 4, 8, 0, 0, None, 0, None), b"null"),
])
def test_linear_act_fwd_entry_refuses(args, word):
    rc, msg = _call("qnn_linear_act_fwd", *args)
    assert rc == 1 and word in msg


@pytest.mark.parametrize("args,word", [
    ((P, 4, None, P, 8, P, 8, None, P, P, P, 2, 4, 8, 0, 1, P, 1 << 20, None), b"slope"),
    ((P, 3, None, P, 8, P, 8, None, P, P, P, 2, 4, 8, 0, 0, P, 1 << 20, None), b"stride"),
    ((P, 4, None, None, 8, P, 8, None, P, P, P, 2, 4, 8, 0, 0, P, 1 << 20, None), b"null"),
    ((P, 4, None, P, 8, P, 8, None, P, P, P, 2, 4, 8, 9, 0, P, 1 << 20, None), b"dtype"),
])
def test_linear_act_bwd_entry_refuses(args, word):
    rc, msg = _call("qnn_linear_act_bwd", *args)
    assert rc == 1 and word in msg


@pytest.mark.parametrize("args,word", [
    ((P, 8, None, None, P, None, None, -1, 8, 1e-5, 0, 0, None), b"rows"),
    ((P, 8, None, None, P, None, None, 2, 0, 1e-5, 0, 0, None), b"dim"),
    ((P, 7, None, None, P, None, None, 2, 8, 1e-5, 0, 0, None), b"stride"),
    ((P, 8, None, None, P, None, None, 2, 8, -1.0, 0, 0, None), b"eps"),
    ((P, 8, None, None, P, None, None, 2, 8, math.nan, 0, 0, None), b"eps"),
    ((P, 8, None, None, None, None, None, 2, 8, 1e-5, 0, 0, None), b"null"),
    ((P, 8, None, None, P, None, None, 2, 8, 1e-5, 0, 2, None), b"wdtype"),
    ((P, 8, None, None, P, None, None, 2, 8, 1e-5, 5, 0, None), b"dtype"),
])
def test_layer_norm_entry_refuses(args, word):
    rc, msg = _call("qnn_layer_norm_fwd", *args)
    assert rc == 1 and word in msg


@pytest.mark.parametrize("change,word", [
    ({"rows": -1}, b"rows"), ({"vocab": 0}, b"vocab"), ({"top": 0}, b"top"), ({"top": 1025, "ldt": 1025, "ldi": 1025}, b"top"),
    ({"lds": 9}, b"stride"), ({"ldt": 2}, b"stride"), ({"ldi": 2}, b"stride"), ({"temp": 0.0}, b"temp"),
    ({"temp": math.inf}, b"temp"), ({"temp": math.nan}, b"temp"), ({"tdtype": 3}, b"tdtype"), ({"index_bytes": 2}, b"index_bytes"),
    ({"stats": None}, b"null"), ({"s": None}, b"null"), ({"dtype": 4}, b"dtype"),
])
def test_topk_distill_entry_refuses(change, word):
    a = dict(s=P, lds=10, t=P, ldt=3, index=P, ldi=3, rows=2, vocab=10, top=3, temp=1.0, mean=1, dtype=0, tdtype=0,
             index_bytes=8, row_loss=P, stats=P, loss=P, work=P, work_bytes=1 << 20, stream=None)
    a.update(change)
    rc, msg = _call("qnn_topk_distill_fwd", *a.values())
    assert rc == 1 and word in msg


def test_work_entries():
    from qnn import _lib
    n = ctypes.c_int64(-1)
    for name, args in (("qnn_linear_act_fwd_work", (5, 7, 9, 0)), ("qnn_linear_act_bwd_work", (5, 7, 9, 1)),
                       ("qnn_layer_norm_bwd_work", (5, 7, 2)), ("qnn_topk_distill_fwd_work", (5, 7, 2))):
        _lib.call(name, *args, ctypes.byref(n))
        assert n.value >= 0
        assert _call(name, *args, None)[0] == 1
        assert _call(name, -1, *args[1:], ctypes.byref(n))[0] == 1


def test_linear_act_plan():
    from qnn import _lib
    tm, tn, sp = ctypes.c_int(), ctypes.c_int(), (ctypes.c_int * 2)()
    out = (ctypes.byref(tm), ctypes.byref(tn), sp)
    _lib.call("qnn_linear_act_plan", 8192, 8192, 4096, 1, 0, *out)
    assert (tm.value, tn.value, *sp) == (256, 256, 1, 1)
    _lib.call("qnn_linear_act_plan", 64, 4096, 4096, 1, 0, *out)
    assert (tm.value, tn.value) == (64, 64) and sp[0] > 1
    for grads in (0, 1):  # every size has a plan with scratch to match
        for m, n, k in ((1, 1, 1), (17, 1, 1 << 21), (1 << 20, 64, 64), (300, 1 << 21, 8), (2 ** 31 - 1, 8, 8)):
            for code in (0, 1, 2):
                assert _call("qnn_linear_act_plan", m, n, k, code, grads, *out)[0] == 0 and 1 <= sp[0] <= 64 and 1 <= sp[1] <= 64
    assert _call("qnn_linear_act_plan", 0, 8, 8, 0, 0, *out)[0] == 1
    assert _call("qnn_linear_act_plan", 8, 8, (1 << 21) + 1, 0, 0, *out)[0] == 1
    assert _call("qnn_linear_act_plan", 8, 8, 8, 0, 0, None, None, None)[0] == 1


def test_misaligned_rows_and_missing_work_are_refused():
    a = ctypes.c_void_p(4098)
    rc, msg = _call("qnn_linear_act_fwd", a, 64, P, 64, None, None, 0, P, None, 20, 8, 64, 1, 0, P, 1 << 20, None)
    assert rc == 1 and b"boundaries" in msg
    rc, msg = _call("qnn_linear_act_fwd", P, 65, P, 64, None, None, 0, P, None, 20, 8, 64, 1, 0, P, 1 << 20, None)
    assert rc == 1 and b"boundaries" in msg
    rc, msg = _call("qnn_linear_act_fwd", P, 8192, P, 8192, None, None, 0, P, None, 64, 64, 8192, 0, 0, None, 0, None)
    assert rc == 1 and b"work" in msg
    rc, msg = _call("qnn_linear_act_bwd", P, 9, None, P, 64, P, 64, None, P, P, None, 20, 9, 64, 1, 0, None, 0, None)
    assert rc == 1 and b"work" in msg
    rc, msg = _call("qnn_layer_norm_bwd", P, 8, P, 8, P, P, P, P, P, P, 4, 8, 0, 0, None, 0, None)
    assert rc == 1 and b"work" in msg
    rc, msg = _call("qnn_topk_distill_fwd", P, 100000, P, 3, P, 3, 2, 100000, 3, 1.0, 1, 0, 0, 8, P, P, P, None, 0, None)
    assert rc == 1 and b"work" in msg


def test_empty_batches_are_no_ops():
    assert _call("qnn_linear_act_fwd", None, 8, None, 8, None, None, 0, None, None, 0, 4, 8, 0, 0, None, 0, None)[0] == 0
    assert _call("qnn_layer_norm_fwd", None, 8, None, None, None, None, None, 0, 8, 1e-5, 0, 0, None)[0] == 0


@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
def test_oracle_linear_act_is_autograd(act):
    g = torch.Generator().manual_seed(1)
    x, w, b, r, dy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((5, 7), (6, 7), (6,), (5, 6), (5, 6)))
    leaves = [v.clone().requires_grad_(True) for v in (x, w, b, r)]
    z = leaves[0] @ leaves[1].t() + leaves[2] + leaves[3]
    y = {"none": lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu}[act](z)
    want = dict(zip(("dx", "dw", "db", "dr"), torch.autograd.grad(y, leaves, dy)), y=y)
    for k, (v, _) in O.linear_act(x, w, b, r, act, dy).items():
        torch.testing.assert_close(v, want[k].detach(), rtol=1e-12, atol=1e-13)


def test_oracle_layer_norm_is_autograd():
    g = torch.Generator().manual_seed(2)
    x, w, b, dy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((5, 7), (7,), (7,), (5, 7)))
    leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
    y = torch.nn.functional.layer_norm(leaves[0], (7,), leaves[1], leaves[2], 1e-5)
    want = dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, dy)), y=y)
    for k, (v, _) in O.layer_norm(x, w, b, 1e-5, dy).items():
        torch.testing.assert_close(v, want[k].detach(), rtol=1e-12, atol=1e-13)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_oracle_topk_distill_is_autograd(reduction):
    g = torch.Generator().manual_seed(3)
    s = torch.randn(4, 11, generator=g, dtype=torch.float64).requires_grad_(True)
    t = torch.randn(4, 3, generator=g, dtype=torch.float64)
    i = torch.tensor([[1, 5, 9], [0, 0, 3], [2, -1, -1], [-1, -1, -1]])
    rows = []
    for r in range(4):
        on = i[r] >= 0
        if on.any():
            p = torch.softmax(t[r][on] / 2, 0)
            rows.append(4 * (p * (p.log() - torch.log_softmax(s[r] / 2, 0)[i[r][on]])).sum())
    rows = torch.stack(rows + [0 * s[3].sum()])
    loss = {"mean": rows.sum() / 3, "sum": rows.sum(), "none": rows}[reduction]
    grad = torch.tensor([1.0, -2.0, 0.5, 3.0], dtype=torch.float64) if reduction == "none" else torch.tensor(0.7, dtype=torch.float64)
    want, = torch.autograd.grad(loss, s, grad)
    got = O.topk_distill(s.detach(), t, i, 2.0, reduction, grad)
    torch.testing.assert_close(got["loss"][0], loss.detach(), rtol=1e-12, atol=1e-13)
    torch.testing.assert_close(got["ds"][0], want, rtol=1e-12, atol=1e-13)
