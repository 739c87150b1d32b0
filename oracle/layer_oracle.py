"""Encoder-layer operators in 64 bits on the CPU (linear, attention, layer norm), each with the bound that a kernel with
32-bit sums and one final rounding has to keep.

Rounding to a type is off by at most u = finfo(type).eps / 2 of the value (plus half the smallest subnormal); an fp32
operation by F = 2^-24 of its result.  A sum of n products in fp32, in any order, is off by at most 2 n F sum |products|
(matrix instructions may truncate where they align: hence the 2)."""
import math

import torch

F = 2.0**-24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _rounded(y, dtype):
    """Most that rounding y to dtype moves it."""
    return half_step(dtype) * y.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


# ---- linear ------------------------------------------------------------------------------------------
def activate(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z**3))
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "tanh":
        return torch.tanh(z)
    return z


# Slope of the activation at most (gelu and its tanh form 1.13, silu 1.10), and how far the fp32 evaluation may be off
# relative to its result: gelu's fit 3.4e-5; the others lose a few fp32 roundings in exp2 and 1 / x (1 ulp each), and
# an argument error of 3 F |a| in e^a with a below 25 where the result is not negligible.  tanh: three terms of its
# series below 0.1 (next term 17/315 x^6 < 5.4e-8), 1 - 2 / (1 + e) above (at 0.1: 4 F / 0.1).
_SLOPE = {"none": 1.0, "relu": 1.0, "gelu": 1.13, "gelu_tanh": 1.13, "silu": 1.1, "tanh": 1.0}
_OWN = {"none": 0.0, "relu": 0.0, "gelu": 3.4e-5 + 100 * F, "gelu_tanh": 100 * F, "silu": 100 * F, "tanh": 60 * F}


def linear(x, w, b=None, act="none", r=None, dtype=torch.bfloat16):
    """-> (y, bound) in float64."""
    x, w = x.double(), w.double()
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    a = activate(z, act)
    err = _SLOPE[act] * 2 * (x.shape[1] + 2) * F * size + _OWN[act] * a.abs() + 1e-30
    y = a
    if r is not None:
        y = a + r.double()
        err = err + F * (a.abs() + r.double().abs())
    return y, _rounded(y, dtype) + (1 + half_step(dtype)) * err


# ---- layer norm --------------------------------------------------------------------------------------
def layer_norm(x, g, b=None, eps=1e-12, r=None, dtype=torch.bfloat16):
    """-> (y, bound).  Sums over lanes and registers: at most n / 64 + 16 additions deep (n / 256 for long rows)."""
    z = x.double() + (r.double() if r is not None else 0)
    n = z.shape[-1]
    depth = n / 64 + 16
    mean = z.mean(-1, keepdim=True)
    d = z - mean
    var = (d * d).mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    y0 = d * rstd * g.double()
    y = y0 + (b.double() if b is not None else 0)
    # deviation: rounding of z, of the mean (a sum), of the difference
    dd = 2 * F * z.abs() + (depth + 2) * F * z.abs().mean(-1, keepdim=True) + F * d.abs()
    # mean square of d + dd, and the sum's roundings, as a relative error of var + eps
    dvar = 2 * (d.abs() * dd).mean(-1, keepdim=True) + (dd * dd).mean(-1, keepdim=True) + (depth + 3) * F * var
    rel = dvar * rstd * rstd
    rel = torch.where(rel < 0.5, rel, torch.full_like(rel, float("inf")))  # (no claim where the variance is all rounding)
    err = dd * rstd * g.double().abs() * (1 + rel) + y0.abs() * (rel + 8 * F) + F * y.abs()
    if n == 1:  # the sum is z and zeros, its mean z / 1 = z: the deviation is exactly 0 and y is beta
        err = F * y.abs()
    return y, _rounded(y, dtype) + (1 + half_step(dtype)) * err + 1e-30


# ---- attention ---------------------------------------------------------------------------------------
def attention(q, k, v, lq, lk, causal=False, prefix=None, scale=None, cap=0.0, slopes=None, table=None, dtype=torch.bfloat16):
    """One document: q [lq.., Hq, D] of which the first lq queries count, k and v [lk.., Hkv, D] likewise.
    -> (o, bound) [len(q), Hq, D]; queries behind lq are zero."""
    n, hq, dim = q.shape
    group = hq // k.shape[1]
    scale = dim**-0.5 if scale is None else scale
    o = torch.zeros(n, hq, dim, dtype=torch.float64)
    bound = torch.zeros_like(o)
    if lq == 0 or lk == 0:
        return o, bound
    u = half_step(dtype)
    dist = torch.arange(lk)[None, :] - (torch.arange(lq)[:, None] + lk - lq)
    seen = torch.ones(lq, lk, dtype=torch.bool)
    if causal:
        seen = dist <= 0
        if prefix:
            seen = seen | (torch.arange(lk) < prefix)[None, :]
    for h in range(hq):
        qh, kh, vh = q[:lq, h].double(), k[:lk, h // group].double(), v[:lk, h // group].double()
        s = scale * (qh @ kh.t())
        ds = 2 * (dim + 4) * F * scale * (qh.abs() @ kh.abs().t())
        if cap:
            s = cap * torch.tanh(s / cap)
            # cap - 2 cap / (1 + e): exp2, 1 / x and two roundings, all of size cap; beyond 64 only where |s| > 0.38 cap, and
            # tanh's series below (a dozen roundings of the result's size): relative to the score
            ds = ds + (8 * F * cap if cap <= 64 else 24 * F * s.abs())
        x = s
        if slopes is not None:
            x = x - slopes[h].double() * dist.abs()
            # a bias linear over a tile of 64 keys may enter the products as their initial value (up to 64 slope), which
            # each of the dim / 16 + 1 accumulations then rounds beside, and leave with the tile's own offset
            ds = ds + 2 * (dim / 16 + 3) * 64 * slopes[h].double().abs() * F
        if table is not None:
            reach = table.shape[1] // 2
            x = x + table[h].double()[dist.clamp(-reach, reach) + reach]
        dx = ds + 6 * F * (s.abs() + (x - s).abs().clamp(max=1e30))
        x = torch.where(seen, x, torch.full_like(x, -math.inf))
        top = x.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        w = torch.exp(x - top)
        # a weight is e^x: off by dx (and that of the row's maximum cancels in the quotient), by the subtraction and by exp2
        rel = torch.where(w > 0, torch.expm1((dx + 3 * F * (x - top).abs()).clamp(max=1.0)) + 4 * F, torch.zeros_like(w))
        total = w.sum(-1, keepdim=True)
        some = total > 0
        p = torch.where(some, w / torch.where(some, total, torch.ones_like(total)), torch.zeros_like(w))
        o[:lq, h] = p @ vh
        # the weight's rounding to the type (u, or half a subnormal of the type where the type has a narrow range), its own
        # error, the same in the sum of weights, and the fp32 sums
        tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
        spread = p @ vh.abs()
        mean_rel = (p * rel).sum(-1, keepdim=True)
        # (weights w (1 + d), |d| <= u, in numerator and denominator alike move o by sum p d (v - o), at most u (spread + |o|))
        err = (p * rel) @ vh.abs() + (u + mean_rel + 4 * (lk + 64) * F) * (spread + o[:lq, h].abs()) + (seen.double() @ vh.abs()) * tiny / torch.where(some, total, torch.ones_like(total))
        bound[:lq, h] = _rounded(o[:lq, h], dtype) + (1 + 4 * u) * err
    return o, bound
