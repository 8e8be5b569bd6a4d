"""The named operators (stablehlo.custom_call @b2x.*) in 64 bits, written from their definitions, with bounds on what rounding may do.

A bound counts roundings: u is half a step of the tensors' type (bf16 2^-8 / 2 per unit of eps/2 = 2^-9 .. 2^-8 of a value), every
rounding of a value x may move it by u |x|; F covers the f32 arithmetic between them (approximate exponentials and tanh, sums in
another order), far below u for the 16-bit types.
"""
from __future__ import annotations

import math

import torch

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def half_step(dtype):
    return torch.finfo(TORCH[dtype]).eps / 2


def heads_first(x, layout):
    return x.transpose(1, 2) if layout == "bshd" else x


# ---- rotary ---------------------------------------------------------------------------------------------------------------

def frequencies(R, base=10000.0, factor=1.0, bands=None):
    f = base ** (-2.0 * torch.arange(R // 2, dtype=torch.float64) / R) if R else torch.zeros(0, dtype=torch.float64)
    if bands is None:
        return f / factor
    low, high, original = bands
    keep = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
    return (1 - keep) * f / factor + keep * f


def _turn(x, positions, layout, R, interleaved, sign, **how):
    a = positions.double()[:, :, None] * frequencies(R, **how)
    a = a[:, :, None] if layout == "bshd" else a[:, None]
    c, s = torch.cos(a), sign * torch.sin(a)
    i = torch.arange(R // 2)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    y, size = x.clone(), x.abs()
    size = size.clone()
    y[..., ia], y[..., ib] = x[..., ia] * c - x[..., ib] * s, x[..., ib] * c + x[..., ia] * s
    size[..., ia] = size[..., ib] = x[..., ia].abs() + x[..., ib].abs()
    return y, size


def rotary(x, positions, weight, dtype, layout, R, interleaved, epsilon, **how):
    """(y, bound) of one tensor.  f32 errors: the angle is good to 2^-24 of a half turn (2e-7 radians), the norm's sum, root and two
    products to 3e-7, the two products and their sum to 2e-7: below 2e-6 of |a| + |b| together."""
    x = x.double()
    n = x if weight is None else x / (x.square().mean(-1, keepdim=True) + epsilon).sqrt() * weight.double()
    y, size = _turn(n, positions, layout, R, interleaved, 1.0, **how)
    return y, half_step(dtype) * y.abs() + 2e-6 * size + 1e-30 + subnormal(dtype)


def subnormal(dtype):
    """Half of the smallest step: what a rounding may do to a value below the normal range."""
    return torch.finfo(TORCH[dtype]).smallest_normal * torch.finfo(TORCH[dtype]).eps / 2


def rotary_gradient(dy, x, positions, weight, dtype, layout, R, interleaved, epsilon, **how):
    """(dx, bound, dw, bound): dw sums tokens and heads in f32, chains of at most a few hundred terms and partial sums: 1e-5 of the
    sum of magnitudes; dx has two more sums over the head than the forward pass: 4e-6 of its terms."""
    dn, size = _turn(dy.double(), positions, layout, R, interleaved, -1.0, **how)
    if weight is None:
        return dn, half_step(dtype) * dn.abs() + 2e-6 * size + 1e-30 + subnormal(dtype), None, None
    x, w = x.double(), weight.double()
    r = 1 / (x.square().mean(-1, keepdim=True) + epsilon).sqrt()
    g = dn * w
    dx = r * (g - x * r * r * (g * x).mean(-1, keepdim=True))
    terms = r * (size * w.abs() + x.abs() * r * r * (size * w.abs() * x.abs()).mean(-1, keepdim=True))
    dw, dw_terms = (dn * x * r).sum((0, 1, 2)), (size * x.abs() * r).sum((0, 1, 2))
    return dx, half_step(dtype) * dx.abs() + 4e-6 * terms + 1e-30 + subnormal(dtype), dw, 1e-5 * dw_terms + 1e-30


# ---- attention --------------------------------------------------------------------------------------------------------------

def seen(B, Sq, Sk, causal=False, query_offset=0, queries_at_end=False, documents=None, prefix=None, lengths=None):
    """([B, Sq, Sk] which keys a query sees, [B, Sq, Sk] how far they are)"""
    key = torch.arange(Sk)[None, None]
    length = lengths.long().clamp(0, Sk)[:, None, None] if lengths is not None else torch.full((B, 1, 1), Sk)
    at = torch.arange(Sq)[None, :, None].expand(B, Sq, 1)
    at = at + (length - Sq if queries_at_end else query_offset)
    see = (key < length).expand(B, Sq, Sk)
    if causal:
        before = key <= at
        if prefix is not None:
            before = before | (key < prefix.long()[:, None, None])
        see = see & before
    if documents is not None:
        inside = (at >= 0) & (at < Sk)
        own = torch.gather(documents.long(), 1, at[:, :, 0].clamp(0, max(Sk - 1, 0))) if Sk else torch.zeros(B, Sq, dtype=torch.long)
        see = see & inside & (own[:, :, None] == documents.long()[:, None, :])
    return see, (at - key).abs()


def attention(q, k, v, dtype, layout, scale, softcap=0.0, slopes=None, do=None, **mask):
    """{name: (value, bound)} of o and lse, and with `do` of dq, dk, dv.

    o: rounded once (u |o|), its weights rounded before the product (u sum w|v|), F sum w|v| for f32.  dv likewise.  dq: dS is rounded
    (u sum |dS||k|), and delta = sum dO O sees the rounding of O and of the weights behind it (2 u sum w|v|)."""
    u, F = half_step(dtype), 2e-4
    q, k, v = (heads_first(x, layout).double() for x in (q, k, v))
    B, Hq, Sq, D = q.shape
    Hk, Sk = k.shape[1], k.shape[2]
    group = Hq // Hk
    see, far = seen(B, Sq, Sk, **mask)
    # what nobody may see is not a number: kept out before it meets one
    hidden = ~see.any(1)                                                             # [B, Sk]
    k, v = (torch.where(hidden[:, None, :, None], 0.0, x) for x in (k, v))
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = q @ kk.transpose(2, 3) * scale
    bend = torch.ones_like(s)
    if softcap:
        t = torch.tanh(s / softcap)
        s, bend = softcap * t, 1 - t * t
    if slopes is not None:
        s = s - slopes.double()[None, :, None, None] * far[:, None]
    s = torch.where(see[:, None], s, -math.inf)
    lse = torch.logsumexp(s, -1) if Sk else torch.full((B, Hq, Sq), -math.inf, dtype=torch.float64)
    w = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None])
    o, ao = w @ vv, w @ vv.abs()
    back = lambda x: heads_first(x, layout)  # noqa: E731
    tiny = subnormal(dtype)
    out = {"o": (back(o), back(u * o.abs() + (u + F) * ao) + tiny), "lse": (lse, 2e-5 + 2e-6 * torch.where(lse.isinf(), 0.0, lse).abs())}
    if do is None:
        return out
    d = heads_first(do, layout).double()
    share = lambda x: x.unflatten(1, (Hk, group)).sum(2)  # noqa: E731
    dv, adv = share(w.transpose(2, 3) @ d), share(w.transpose(2, 3) @ d.abs())
    ds = w * (d @ vv.transpose(2, 3) - (d * o).sum(-1, keepdim=True)) * bend * scale
    # dP and delta are sums of f32 products: F of their terms' magnitudes goes with the weight, too
    off = w * bend * scale * ((d.abs() * (2 * u + F) * ao).sum(-1, keepdim=True) + 1e-5 * (d.abs() @ vv.abs().transpose(2, 3)))
    err = (u + F) * ds.abs() + off
    dq, edq = ds @ kk, err @ kk.abs()
    dk, edk = share(ds.transpose(2, 3) @ q), share(err.transpose(2, 3) @ q.abs())
    # f16 values below its normal range carry an absolute error: one step of 2^-25 per rounded weight or dS
    low = tiny * 2
    out["dq"] = (back(dq), back(u * dq.abs() + edq + low * kk.abs().sum(2, keepdim=True)) + tiny)
    out["dk"] = (back(dk), back(u * dk.abs() + edk + low * share(q.abs().sum(2, keepdim=True))) + tiny)
    out["dv"] = (back(dv), back(u * dv.abs() + (u + F) * adv + low * share(d.abs().sum(2, keepdim=True))) + tiny)
    return out
