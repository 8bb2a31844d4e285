"""DIN's masked softmax pooling, backward: dscore = att (datt - sum_j att_j datt_j) / sqrt(H) for the weights it is given,
whatever they add up to (a softmax's weights as if they added up to one exactly), and dK = att dout."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
E = 2.0 ** -24


@pytest.mark.parametrize('total', ['softmax', 'half', 'three', 'signed'])
@pytest.mark.parametrize('B,T,H', [(5, 30, 32), (3, 300, 64), (2, 1, 16), (4, 70, 24), (3, 500, 20)])
def test_scores_of_any_weights(B, T, H, total):
    from recommendation_amd import ops
    g = torch.Generator().manual_seed(T)
    K, dout = torch.randn(B, T, H, generator=g), torch.randn(B, H, generator=g)
    sl = torch.randint(1, T + 1, (B,), generator=g)
    sl[0] = T
    on = torch.arange(T)[None] < sl[:, None]
    att = torch.softmax(torch.randn(B, T, generator=g).masked_fill(~on, -math.inf), 1)
    att = {'softmax': att, 'half': att * 0.5, 'three': att * 3,
           'signed': (torch.randn(B, T, generator=g) * on).float()}[total].contiguous()
    dscore, dK = torch.full((B, T), math.nan, device=DEV), torch.full((B, T, H), math.nan, device=DEV)
    ops.din_attn_pool_bwd(dout.to(DEV), att.to(DEV), sl.to(torch.int32).to(DEV), K.to(DEV), dscore, dK, B=B, T=T, H=H)
    a, d, k = att.double(), dout.double(), K.double()
    datt = (d[:, None] * k).sum(2)
    datt_off = (H + 2) * E * (d.abs()[:, None] * k.abs()).sum(2)
    dot = (a * datt).sum(1, keepdim=True)
    if total == 'softmax':
        assert (a.sum(1) - 1).abs().max() < 2.0 ** -18
        dot = dot / a.sum(1, keepdim=True)
    want = torch.where(on, a * (datt - dot) / math.sqrt(H), 0.0)
    # datt's sum of H products, the sum over positions (fp64, of rounded datt), the subtraction and the two products
    dot_off = (a.abs() * datt_off).sum(1, keepdim=True) + T * 2.0 ** -52 * (a * datt).abs().sum(1, keepdim=True)
    bound = a.abs() / math.sqrt(H) * (datt_off + dot_off) + 6 * E * want.abs()
    off = (dscore.cpu().double() - want).abs()
    assert (off <= torch.where(on, bound, 0.0)).all(), (float(off.max()), float(bound.max()))
    assert ((dK.cpu().double() - a[:, :, None] * d[:, None]).abs() <= E * (a[:, :, None] * d[:, None]).abs()).all()
