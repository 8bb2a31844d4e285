"""The attention-tower operators as they are used together: candidates and their sample's history through layer norm,
projections, cross attention and a residual, a loss, the whole backward, clipping, an SGD step - against the same tower
in 64 bits with autograd.  fp32 throughout.  Every operator of the chain is held to 1e-5 of its outputs' largest value by
its own tests (the projections) or far below (the rest); two projections follow each other on the way to any gradient:
2e-5."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


class Tower:
    """cand [B,Tq,W], hist [B,Tk,W] -> cand + attention(LN(cand) Wq, LN(hist) Wk, LN(hist) Wv) Wo"""
    NAMES = ('g1', 'b1', 'g2', 'b2', 'Wq', 'Wk', 'Wv', 'Wo')

    def __init__(self, W, H, params):
        from recommendation_amd import ops
        self.ops, self.W, self.H = ops, W, H
        self.p = {n: params[n].to(torch.float32).to(DEV).contiguous() for n in self.NAMES}
        self.g = {n: torch.full_like(t, math.nan) for n, t in self.p.items()}
        self.ws, self.bufs = ops.Workspace(torch.device(DEV)), {}
        self.list, self.norm = ops.GradList(list(self.g.values())), torch.empty(1, device=DEV)

    def buf(self, name, *shape):
        return self.bufs.setdefault(name, torch.full(shape, math.nan, device=DEV))

    def step(self, cand, hist, sl, mask, dy, bound, lr):
        ops, p, g, ws, W, H = self.ops, self.p, self.g, self.ws, self.W, self.H
        B, Tq, Tk, D = cand.shape[0], cand.shape[1], hist.shape[1], W // H
        nq, nk = B * Tq, B * Tk
        c2, h2, dy2 = cand.view(nq, W), hist.view(nk, W), dy.view(nq, W)
        b = self.buf
        stats = {n: b(n, r) for n, r in (('m1', nq), ('r1', nq), ('m2', nk), ('r2', nk))}
        x, m = b('x', nq, W), b('mem', nk, W)
        ops.layer_norm_fwd(c2, x, gamma=p['g1'], beta=p['b1'], mean=stats['m1'], rstd=stats['r1'])
        ops.layer_norm_fwd(h2, m, gamma=p['g2'], beta=p['b2'], mean=stats['m2'], rstd=stats['r2'])
        q, kv, o, y = b('q', nq, W), b('kv', nk, 2 * W), b('o', nq, W), b('y', nq, W)
        ops.gemm(x, p['Wq'], q, ws=ws)
        ops.gemm(m, p['Wk'], kv[:, :W], ws=ws)
        ops.gemm(m, p['Wv'], kv[:, W:], ws=ws)
        heads = lambda t, T: t.view(B, T, -1, D)
        both = kv.view(B, Tk, 2, H, D)
        k4, v4, lse = both[:, :, 0], both[:, :, 1], b('lse', B, H, Tq)
        ops.cross_attn_fwd(heads(q, Tq), k4, v4, heads(o, Tq), lse=lse, sl=sl, mask=mask, ws=ws)
        ops.gemm(o, p['Wo'], y, ws=ws)
        y += c2
        # backward
        do, dq, dkv = b('do', nq, W), b('dq', nq, W), b('dkv', nk, 2 * W)
        ops.dense_wgrad(o, dy2, g['Wo'], ws=ws)
        ops.gemm(dy2, p['Wo'], do, trans_b=True, ws=ws)
        dboth = dkv.view(B, Tk, 2, H, D)
        ops.cross_attn_bwd(heads(do, Tq), heads(q, Tq), k4, v4, heads(o, Tq), lse, heads(dq, Tq), dboth[:, :, 0],
                           dboth[:, :, 1], sl=sl, mask=mask, ws=ws)
        ops.dense_wgrad(x, dq, g['Wq'], ws=ws)
        ops.dense_wgrad(m, dkv[:, :W], g['Wk'], ws=ws)
        ops.dense_wgrad(m, dkv[:, W:], g['Wv'], ws=ws)
        dx, dm = b('dx', nq, W), b('dm', nk, W)
        ops.gemm(dq, p['Wq'], dx, trans_b=True, ws=ws)
        ops.gemm(dkv[:, :W], p['Wk'], dm, trans_b=True, ws=ws)
        ops.gemm(dkv[:, W:], p['Wv'], dm, trans_b=True, accumulate=True, ws=ws)
        dcand = b('dcand', nq, W)
        dcand.copy_(dy2)                                   # the residual branch; the layer norm adds its own
        ops.layer_norm_bwd(dx, c2, stats['m1'], stats['r1'], dcand, gamma=p['g1'], dgamma=g['g1'], dbeta=g['b1'],
                           accumulate=True, ws=ws)
        ops.layer_norm_bwd(dm, h2, stats['m2'], stats['r2'], dm, gamma=p['g2'], dgamma=g['g2'], dbeta=g['b2'], ws=ws)
        ops.clip_grads(self.list, bound, self.norm, ws=ws)
        for n in self.NAMES:
            ops.dense_update(p[n].view(-1), g[n].view(-1), ops.make_opt(_sgd(), lr=lr))
        return dict(y=y, dcand=dcand, dhist=dm)


def _sgd():
    from recommendation_amd import _lib
    return _lib.OPT_SGD


def _reference(P, cand, hist, sl, mask, dy, H, bound, lr):
    P = {n: v.clone().requires_grad_(True) for n, v in P.items()}
    cand, hist = cand.clone().requires_grad_(True), hist.clone().requires_grad_(True)
    B, Tq, W = cand.shape
    Tk, D = hist.shape[1], W // H

    def norm(x, g, b):
        d = x - x.mean(-1, keepdim=True)
        return d / (d.square().mean(-1, keepdim=True) + 1e-5).sqrt() * g + b

    x, m = norm(cand, P['g1'], P['b1']), norm(hist, P['g2'], P['b2'])
    split = lambda t: t.view(B, -1, H, D).transpose(1, 2)
    q, k, v = split(x @ P['Wq']), split(m @ P['Wk']), split(m @ P['Wv'])
    ok = (torch.arange(Tk)[None] < sl[:, None]) & mask
    s = (q @ k.transpose(2, 3) / math.sqrt(D)).masked_fill(~ok[:, None, None], -math.inf)
    w = torch.where(ok.any(1)[:, None, None, None], torch.softmax(s.masked_fill(~ok.any(1)[:, None, None, None], 0.0), -1), 0.0)
    y = cand + (w @ v).transpose(1, 2).reshape(B, Tq, W) @ P['Wo']
    names = list(P)
    grads = torch.autograd.grad(y, [P[n] for n in names] + [cand, hist], dy)
    G = dict(zip(names, grads))
    total = math.sqrt(sum(float(G[n].square().sum()) for n in names))
    by = min(1.0, bound / total)
    new = {n: (P[n] - lr * by * G[n]).detach() for n in names}
    return dict(y=y.detach(), dcand=grads[-2], dhist=grads[-1]), {n: by * G[n] for n in names}, total, new


@pytest.mark.parametrize('B,Tq,Tk,W,H,bound', [(6, 1, 50, 64, 4, 1.0), (5, 20, 37, 128, 2, 0.5), (3, 70, 40, 32, 4, 1e6)])
def test_training_steps_of_a_tower(B, Tq, Tk, W, H, bound):
    r = torch.Generator().manual_seed(B + Tq)
    rand = lambda *s, sc=1.0: (torch.randn(*s, generator=r, dtype=torch.float64) * sc).float().double()
    P = {n: rand(W, W, sc=W ** -0.5) for n in ('Wq', 'Wk', 'Wv', 'Wo')}
    P.update(g1=1 + rand(W, sc=0.1), g2=1 + rand(W, sc=0.1), b1=rand(W, sc=0.1), b2=rand(W, sc=0.1))
    P = {n: v.float().double() for n, v in P.items()}
    tower = Tower(W, H, P)
    for step in range(3):
        cand, hist, dy = rand(B, Tq, W), rand(B, Tk, W), rand(B, Tq, W)
        sl = torch.randint(1, Tk + 1, (B,), generator=r).to(torch.int32)
        sl[0], sl[1] = 0, Tk                               # a user without a history
        mask = torch.rand(B, Tk, generator=r) < 0.8
        want, grads, total, new = _reference(P, cand, hist, sl, mask, dy, H, bound, 0.01)
        dev = lambda t: t.float().to(DEV).contiguous()
        got = tower.step(dev(cand), dev(hist), sl.to(DEV), mask.to(DEV), dev(dy), bound, 0.01)
        close = lambda a, b, n: (a.detach().cpu().double().view(b.shape) - b).abs().max() <= 2e-5 * b.abs().max() or pytest.fail(n)
        for n in want:
            close(got[n], want[n], n)
        for n in grads:
            close(tower.g[n], grads[n], 'd' + n)
            close(tower.p[n], new[n], n)
        assert abs(float(tower.norm) - total) <= 2e-5 * total
        P = {n: t.cpu().double() for n, t in tower.p.items()}
