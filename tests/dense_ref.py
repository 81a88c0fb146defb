"""Plain 64-bit forms of the dense operators and how far fp32 sums and one rounding to a type may take a result from them.

A sum of k products in fp32, in any order, is off by at most (k + 1) u S, u = 2^-24, S = sum |a b| (first order); an operand held
as three bf16 parts adds at most 4 u S for the parts' products that are left out.  fp32 exp, log1p, expm1, erf and a division are
taken as 8 u relative.  A rounding to T is eps_T / 2 relative, and half the smallest number of T near zero."""
import math

import torch

U = 2.0 ** -24
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def gamma(k):
    return (k + 8) * U


def act(z, name):
    """value, slope, and bounds of the slopes of both."""
    if name == "relu":
        s = (z > 0).double()
        return z * s, s, 1.0, 0.0
    if name == "leaky_relu":
        s = torch.where(z > 0, 1.0, 0.01).double()
        return z * s, s, 1.0, 0.0
    if name == "gelu":
        c = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 1.13, 0.80
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p)), 1.10, 0.50
    return z, torch.ones_like(z), 1.0, 0.0


def rounded(v, tol, dtype):
    """tolerance after v (known to tol) was rounded to dtype"""
    return tol + (v.abs() + tol) * HALF[dtype] + TINY[dtype]


def close(got, want, tol, what=""):
    got = got.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol) & ~(torch.isnan(got) & torch.isnan(want)) & ~((got == want) & torch.isinf(want))
    if bad.any():
        i = torch.nonzero(bad.reshape(-1))[0, 0]
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; first at {int(i)}: got {got.reshape(-1)[i].item()!r}, "
                             f"want {want.reshape(-1)[i].item()!r}, tolerance {tol.expand_as(want).reshape(-1)[i].item()!r}")


def linear(x, w, b, r, name, dy=None):
    """{output: (value, tolerance)} of linear_act and its gradients"""
    dt = x.dtype
    x, w = x.detach().double(), w.detach().double()
    k = x.shape[1]
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, size = z + b.detach().double(), size + b.detach().double().abs()
    ez = gamma(k) * size
    v, slope, s1, s2 = act(z, name)
    ey = s1 * ez + 8 * U * (v.abs() + z.abs())
    if r is not None:
        v = v + r.detach().double()
        ey = ey + U * v.abs()
    out = {"y": (v, rounded(v, ey, dt))}
    if dy is not None:
        dy = dy.double()
        dz = dy * slope
        kept = torch.float32 if dt == torch.float32 else torch.float16  # what the backward pass has of z
        e_slope = s2 * rounded(z, ez, kept) + 16 * U
        edz = rounded(dz, dy.abs() * e_slope, dt)  # the products take dz in dt
        out |= gradients(x, w, dz, edz, dt)
    return out


def gradients(x, w, dz, edz, dt):
    m, n = dz.shape
    big = dz.abs() + edz
    out = {}
    v = dz @ w
    out["dx"] = (v, rounded(v, edz @ w.abs() + gamma(n) * (big @ w.abs()), dt))
    v = dz.t() @ x
    out["dw"] = (v, rounded(v, edz.t() @ x.abs() + gamma(m) * (big.t() @ x.abs()), dt))
    v = dz.sum(0)
    out["db"] = (v, rounded(v, edz.sum(0) + gamma(m) * big.sum(0), dt))
    return out


def logits(x, w, b, keep=None):
    x, w = x.detach().double(), w.detach().double()
    if keep is not None:
        x = torch.where(keep[:, None], x, 0.0)
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        bb = b.detach().double()
        z, size = z + bb, size + torch.where(torch.isinf(bb), 0.0, bb.abs())
    return x, w, z, gamma(x.shape[1]) * size


def cross_entropy(x, w, b, target, ignore, reduction, g=None):
    """{output: (value, tolerance)} of linear_cross_entropy and its gradients; g: dL/dloss"""
    dt = x.dtype
    target = target.long()
    keep = target != ignore
    x, w, z, ez = logits(x, w, b, keep)
    top = torch.where(torch.isinf(z), 0.0, ez).amax(1)
    rows = torch.arange(len(target), device=z.device)
    at = torch.where(keep, target, 0)
    lp = torch.log_softmax(z, 1)
    loss = torch.where(keep, -lp[rows, at], 0.0)
    eloss = torch.where(keep, 2 * top + 8 * U * (1 + loss.abs()) + gamma(z.shape[1]), 0.0)
    many = max(1, int(keep.sum()))
    if reduction == "none":
        out = {"loss": (loss, eloss + U * loss.abs())}
    else:
        div = many if reduction == "mean" else 1
        out = {"loss": (loss.sum() / div, eloss.sum() / div + 4 * U * loss.sum() / div)}
    if g is not None:
        g = g.double()
        row = (g / many if reduction == "mean" else g).expand(len(target)) * keep
        p = lp.exp()
        spread = torch.where(torch.isinf(z), 0.0, (z - z.amax(1, keepdim=True)).abs())
        ep = p * (2 * ez + 2 * top[:, None] + U * spread + 32 * U + gamma(z.shape[1]))
        hot = torch.zeros_like(p)
        hot[rows[keep], at[keep]] = 1.0
        dz = (p - hot) * row[:, None]
        edz = rounded(dz, row.abs()[:, None] * (ep + hot * (eloss[:, None] + 16 * U * (1 - p))) + 4 * U * dz.abs(), dt)
        edz = torch.where(keep[:, None], edz, 0.0)
        out |= gradients(x, w, dz, edz, dt)
    return out
