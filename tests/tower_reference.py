"""Definitions in 64 bits of the attention-tower operators, with elementwise bounds on what kernels of a given type may be
off.  Every bound follows from the operations alone: e = 2^-24 is half a step of fp32, u half a step of the tensors' type
(one final rounding; for 16-bit types also one of p and one of ds), sums of n fp32 terms are off by at most n e times
the sum of magnitudes."""
import math

import torch

E = 2.0 ** -24
F64 = torch.float64


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the distance of the type's smallest values: what a final rounding is off by below its normal range."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def attention(q, k, v, sl=None, mask=None, scale=None, dout=None):
    """Reference and bounds: dict name -> (value, bound), CPU float64.  q [B,Tq,H,D], k, v [B,Tk,Hkv,D] of the kernel's
    type; keys that are left out are taken out by value, so what they hold plays no part."""
    t = q.dtype
    u, low = half_step(t), 0.0 if t == torch.float32 else half_step(t)
    B, Tq, H, D = q.shape
    Tk, Hkv = k.shape[1], k.shape[2]
    G = H // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    ok = torch.ones(B, Tk, dtype=torch.bool)
    if sl is not None:
        ok &= torch.arange(Tk)[None] < sl.cpu().long()[:, None]
    if mask is not None:
        ok &= mask.cpu() != 0
    keep = ok[:, None, :, None]
    zero = torch.zeros((), dtype=F64)

    def heads(x):
        return x.cpu().to(F64).permute(0, 2, 1, 3)

    Q = heads(q)
    K = torch.where(keep, heads(k), zero).repeat_interleave(G, 1)
    V = torch.where(keep, heads(v), zero).repeat_interleave(G, 1)
    s = scale * (Q @ K.transpose(2, 3))
    s_off = (D + 12) * E * scale * (Q.abs() @ K.abs().transpose(2, 3)) + 4 * E * s.abs()
    s = s.masked_fill(~ok[:, None, None, :], -math.inf)
    top = s.amax(-1, keepdim=True) if Tk else torch.full((B, H, Tq, 1), -math.inf, dtype=F64)
    top = top.masked_fill(top == -math.inf, 0.0)
    w = (s - top).exp()
    total = w.sum(-1, keepdim=True)
    safe = total.masked_fill(total == 0, 1.0)
    p = w / safe
    lse = torch.where(total > 0, top + safe.log(), torch.full_like(top, -math.inf))[..., 0]
    # p's relative error: its own score, the row's sum (a mean of the others') and the exponential's argument and result
    worst = (s_off * (p > 0)).amax(-1, keepdim=True) if Tk else torch.zeros_like(top)
    arg = 4 * E * (s.masked_fill(~ok[:, None, None, :], 0.0).abs().amax(-1, keepdim=True) if Tk else 0.0)
    p_rel = 2 * worst + 2 * arg + (Tk + 16) * E
    # fp16: p times 2^14 and ds times a power of two are held with a last place of 2^-24
    p_abs = 2.0 ** -39 * 2 if t == torch.float16 else 0.0
    out = p @ V
    out_off = (p_rel + low) * (p @ V.abs()) + p_abs * V.abs().sum(2, keepdim=True) + (Tk + 8) * E * (p @ V.abs())
    out_bound = out_off + u * (out.abs() + out_off) + tiny(t)
    back = lambda x: x.permute(0, 2, 1, 3)
    lse_off = (worst + arg)[..., 0] + (Tk + 24) * E * (1 + lse.abs().masked_fill(lse == -math.inf, 0.0))
    res = dict(out=(back(out), back(out_bound)), lse=(lse, lse_off))
    if dout is None:
        return res
    g = heads(dout)
    dp = g @ V.transpose(2, 3)
    dp_off = (D + 12) * E * (g.abs() @ V.abs().transpose(2, 3))
    delta = (g * out).sum(-1, keepdim=True)
    delta_off = (g.abs() * out_bound).sum(-1, keepdim=True) + (D + 4) * E * (g * out).abs().sum(-1, keepdim=True)
    ds = p * (dp - delta)
    pr = p_rel + lse_off[..., None]
    ds_off = (pr + 4 * E + low) * ds.abs() + p * (1 + pr) * (dp_off + delta_off)
    if t == torch.float16:
        ds_off = ds_off + 2.0 ** -37 * (ds.abs().amax() if ds.numel() else 0.0)
    dq = scale * (ds @ K)
    dq_off = scale * (ds_off @ K.abs() + (Tk + 8) * E * (ds.abs() @ K.abs()))
    dk = scale * (ds.transpose(2, 3) @ Q)
    dk_off = scale * (ds_off.transpose(2, 3) @ Q.abs() + (Tq * G + 8) * E * (ds.abs().transpose(2, 3) @ Q.abs()))
    dv = p.transpose(2, 3) @ g
    p_off = (pr + low) * p + p_abs
    dv_off = p_off.transpose(2, 3) @ g.abs() + (Tq * G + 8) * E * (p.transpose(2, 3) @ g.abs())
    share = lambda x: x.reshape(B, Hkv, G, *x.shape[2:]).sum(2)
    dk, dk_off, dv, dv_off = share(dk), share(dk_off), share(dv), share(dv_off)
    for n, x, off in (('dq', dq, dq_off), ('dk', dk, dk_off), ('dv', dv, dv_off)):
        res[n] = (back(x), back(off + u * (x.abs() + off)) + tiny(t))
    return res


def layer_norm(x, gamma=None, beta=None, eps=1e-5, dy=None, into=None):
    """Reference and bounds of layer_norm_fwd / _bwd (into: what an accumulating dx holds).  Sums over a row are 16 terms
    per lane and a tree over at most 1024 lanes (16384 columns; further passes of 1024 packets above), 2 roundings on
    the way: depth.  Sums over rows: a lane's rows, the rows of a block side by side (at most 128) and a tree."""
    t = x.dtype
    u = half_step(t)
    X = x.cpu().to(F64)
    rows, n = X.shape
    w = torch.ones(n, dtype=F64) if gamma is None else gamma.cpu().to(F64)
    b = torch.zeros(n, dtype=F64) if beta is None else beta.cpu().to(F64)
    depth = 30 + n / 1024
    mean = X.mean(1, keepdim=True)
    d = X - mean
    var = (d * d).mean(1, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    xh = d * rstd
    mean_off = depth * E * X.abs().mean(1, keepdim=True) + E * mean.abs()
    d_off = mean_off + E * d.abs()
    r_rel = (depth + 6) * E + 0.5 * (d_off * rstd).square().amax(1, keepdim=True) + 2 * E
    xh_off = rstd * d_off + (r_rel + 2 * E) * xh.abs()
    y = xh * w + b
    y_off = xh_off * w.abs() + 3 * E * ((xh * w).abs() + b.abs())
    res = dict(y=(y, y_off + u * (y.abs() + y_off) + tiny(t)), mean=(mean[:, 0], mean_off[:, 0]),
               rstd=(rstd[:, 0], (r_rel * rstd)[:, 0] + 2 * E * rstd[:, 0]))
    if dy is None:
        return res
    up = dy.cpu().to(F64)
    g = up * w
    s1, s2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    s1_off = depth * E * g.abs().mean(1, keepdim=True)
    s2_off = depth * E * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * xh_off).mean(1, keepdim=True)
    dx = rstd * (g - s1 - xh * s2)
    dx_off = rstd * (6 * E * (g.abs() + s1.abs() + (xh * s2).abs()) + s1_off + xh.abs() * s2_off + xh_off * s2.abs()) \
        + (r_rel + 2 * E) * dx.abs()
    if into is not None:
        dx = dx + into.cpu().to(F64)
        dx_off = dx_off + 2 * E * dx.abs()
    res['dx'] = (dx, dx_off + u * (dx.abs() + dx_off) + tiny(t))
    long = 160 + rows / 64
    res['dgamma'] = ((up * xh).sum(0), (up.abs() * xh_off).sum(0) + long * E * (up * xh).abs().sum(0))
    res['dbeta'] = (up.sum(0), long * E * up.abs().sum(0))
    return res


def within(got, want, what):
    value, bound = want
    got = got.detach().cpu().to(F64)
    assert got.shape == value.shape, (what, got.shape, value.shape)
    same = (got == value) | (got.isnan() & value.isnan())
    off = torch.where(same, torch.zeros_like(value), (got - value).abs())
    bad = ~(off <= bound)
    if bad.any():
        i = int((off / bound.clamp_min(1e-300)).nan_to_num(nan=math.inf).argmax())
        raise AssertionError('%s: %d of %d values off, worst %.9g for %.9g (bound %.3g)'
                             % (what, int(bad.sum()), bad.numel(), got.flatten()[i], value.flatten()[i], bound.flatten()[i]))
