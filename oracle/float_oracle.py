"""The float operators of qnn.functional from their definitions, in float64 on the CPU, with bounds on
what a computation with fp32 sums and one rounding to `dtype` may differ by.

Each function takes CPU tensors of the operator's type and returns {name: (value, bound)}, both float64.
u is half a step of the type relative to the value (torch.finfo(dtype).eps / 2), e = 2^-24 that of
fp32.  A sum of n fp32 terms, in whatever order, is within n e of the sum of the terms' sizes; where
the kernels add in chains far shorter than n (a tree over lanes and waves), CHAIN bounds their length.
"""
import math

import torch

E = 2.0 ** -24
# No kernel adds more than this many terms one after another, beside the products' chains: lanes stop at 512, and the sums of
# those are added in a few levels (rows of a layer norm up to 2^29 elements, everything else at any size).
CHAIN = 1024


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    """Half the step among the type's subnormal numbers (fp32's may be flushed)."""
    f = torch.finfo(dtype)
    return f.smallest_normal if dtype == torch.float32 else f.smallest_normal * f.eps / 2


def _out(v, err, dtype):
    return v, err * (1 + 2 * _u(dtype)) + _u(dtype) * v.abs() + _tiny(dtype)


def gelu(z):
    # the lower tail through erfc, so that it keeps its digits; 0 at -inf
    cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    pdf = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    y = torch.where(z == -math.inf, -0.0, z * cdf)
    return y, torch.where(z.isinf(), cdf, cdf + z * pdf)


def slope_code(d, off, dtype):
    """What GELU's derivative d, computed within `off`, loses between the passes of a 16-bit type: bf16 keeps it as fp16 of
    d 2^15, fp16 keeps sign(d) |d|^(1/4) in fixed point of 1 / 40192 (two square roots in fp32 and a sum of up to 65536
    before it: 0.5 + 2^-7 of a step, and 4 e on the way back)."""
    if dtype == torch.float32:
        return torch.zeros_like(d)
    size = d.abs() + off
    if dtype == torch.bfloat16:
        return 2.0 ** -11 * size + 2.0 ** -40
    root, step = size ** 0.25, (0.5 + 2.0 ** -7 + 4 * 40192 * E) / 40192
    return (root + step) ** 4 - size + 4 * E * size


def linear_act(x, w, b=None, r=None, act="none", dy=None):
    dt = x.dtype
    u = _u(dt)
    n, k = w.shape
    x, w = x.double().reshape(-1, k), w.double()
    m = x.shape[0]
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    for v in (b, r):
        if v is not None:
            v = v.double() if v is b else v.double().reshape(m, n)
            z, size = z + v, size + v.abs()
    ez = (k + 2) * E * size
    if act == "relu":
        y, slope, es, ey = torch.where(z <= 0, 0.0, z), torch.where(z <= 0, 0.0, 1.0), 0.0, ez
        # where z may be on either side of the border the slope may be either
        es = torch.where((z.abs() <= ez) & (ez > 0), 1.0, 0.0)
    elif act == "gelu":
        y, slope = gelu(z)
        # |gelu'| <= 1.13, |gelu''| <= 0.8; the exponential's and the fit's own error: 2^-17 z^2 e of what
        # they multiply, under 40 e of |z| and of 1
        ey = 1.13 * ez + 40 * E * z.abs()
        es = 0.8 * ez + 40 * E
        es = es + slope_code(slope, es, dt)
    else:
        y, slope, es, ey = z, torch.ones_like(z), 0.0, ez
    out = {"y": _out(y, ey, dt)}
    if dy is None:
        return out
    dy = dy.double().reshape(m, n)
    dz = dy * slope
    edz = dy.abs() * es
    if act != "none":
        edz = edz + u * (dz.abs() + edz) + _tiny(dt)  # rounded once before the products
        out["dr"] = (dz, edz)
    else:
        out["dr"] = (dz, torch.zeros_like(dz))
    out["dx"] = _out(dz @ w, edz @ w.abs() + (n + 1) * E * ((dz.abs() + edz) @ w.abs()), dt)
    out["dw"] = _out(dz.t() @ x, edz.t() @ x.abs() + (m + 1) * E * ((dz.abs() + edz).t() @ x.abs()), dt)
    out["db"] = _out(dz.sum(0), edz.sum(0) + min(m, CHAIN) * E * (dz.abs() + edz).sum(0), dt)
    return out


def layer_norm(x, w=None, b=None, eps=1e-5, dy=None):
    dt = x.dtype
    dim = x.shape[-1]
    x = x.double().reshape(-1, dim)
    wt = w.dtype if w is not None else b.dtype if b is not None else dt
    w64 = torch.ones(dim, dtype=torch.float64) if w is None else w.double()
    b64 = torch.zeros(dim, dtype=torch.float64) if b is None else b.double()
    g = (min(dim, CHAIN) + 4) * E
    mean = x.mean(1, keepdim=True)
    d = x - mean
    var = (d * d).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = d * rstd
    # the mean is off by g mean|x|, a deviation by that and a rounding, the variance by twice that in
    # relation to the root mean square (and g of itself), rstd by half of the variance's
    emean = g * x.abs().mean(1, keepdim=True)
    ed = emean + 2 * E * (d.abs() + emean)
    erstd = rstd * ((emean * emean + 2 * emean * E * d.abs().mean(1, keepdim=True)) * rstd * rstd + g + 8 * E)
    exh = ed * rstd + (d.abs() + ed) * erstd + E * xh.abs()
    y = xh * w64 + b64
    out = {"y": _out(y, exh * w64.abs() + 2 * E * (xh.abs() * w64.abs() + b64.abs()), dt)}
    if dy is None:
        return out
    dy = dy.double().reshape(-1, dim)
    gg = dy * w64
    sg, sx = gg.mean(1, keepdim=True), (gg * xh).mean(1, keepdim=True)
    esg = g * gg.abs().mean(1, keepdim=True)
    esx = (gg.abs() * exh).mean(1, keepdim=True) + g * (gg * xh).abs().mean(1, keepdim=True)
    inner = gg - sg - xh * sx
    einner = (esg + exh * sx.abs() + (xh.abs() + exh) * esx
              + 4 * E * (gg.abs() + sg.abs() + xh.abs() * sx.abs()))
    out["dx"] = _out(rstd * inner, rstd * einner + (inner.abs() + einner) * erstd, dt)
    rows = x.shape[0]
    gr = (min(rows, CHAIN) + 2) * E
    out["dw"] = _out((dy * xh).sum(0), (dy.abs() * exh).sum(0) + gr * (dy.abs() * (xh.abs() + exh)).sum(0), wt)
    out["db"] = _out(dy.sum(0), gr * dy.abs().sum(0), wt)
    return out


def topk_distill(s, t, i, temp=1.0, reduction="mean", grad=None):
    """loss and ds; grad: the loss's gradient (a tensor of the loss's shape), 1 if None."""
    dt = s.dtype
    vocab, top = s.shape[-1], t.shape[-1]
    s, t, i = s.double().reshape(-1, vocab) / temp, t.double().reshape(-1, top) / temp, i.reshape(-1, top).long()
    rows = s.shape[0]
    # an exponential of an argument of size a is within (1.5 a + 2) e of itself, a sum of them CHAIN e more;
    # the arguments that matter here are under 120 in size, and smaller exponentials are under e^-100
    eps = (1.5 * 120 + 2 + CHAIN) * E
    loss, eloss = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    ds, eds = torch.zeros_like(s), torch.zeros_like(s)
    counted = torch.zeros(rows, dtype=torch.bool)
    for r in range(rows):
        there = i[r] >= 0
        if (i[r] >= vocab).any():
            counted[r], loss[r], ds[r] = True, math.nan, math.nan
            continue
        if not there.any() or t[r][there].max() == -math.inf:
            continue
        counted[r] = True
        p = torch.softmax(t[r][there], 0)
        at = i[r][there]
        logp, logq = torch.log_softmax(t[r][there], 0), torch.log_softmax(s[r], 0)
        on = p > 0
        loss[r] = temp ** 2 * (p[on] * (logp[on] - logq[at][on])).sum()
        size = p[on] * (2 + logp[on].abs() + logq[at][on].abs() + t[r][there][on].abs().max() + s[r][at][on].abs())
        eloss[r] = temp ** 2 * 2 * eps * size.sum()
        q = logq.exp()
        scattered = torch.zeros(vocab, dtype=torch.float64).index_add_(0, at, p)
        ds[r] = temp * (q - scattered)
        eds[r] = temp * (2 * eps * (q + scattered) + 1e-37)
    count = max(1, int(counted.sum()))
    over = count if reduction == "mean" else 1
    if reduction == "none":
        value, bound = loss, eloss + E * loss.abs()
    else:
        value, bound = loss.sum() / over, eloss.sum() / over + 2 * E * loss.abs().sum() / over
    g = torch.ones(()) if grad is None else grad.detach().cpu()
    g = (g.double().reshape(-1, 1) if reduction == "none" else g.double()) / over
    return {"loss": (value, bound + 1e-37), "ds": _out(ds * g, eds * g.abs() + 4 * E * (ds * g).abs(), dt)}
