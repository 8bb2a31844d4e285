"""Cross attention of few query rows per key head (kernels of their own): what non-finite gradients and queries leave
alone, and three rows, which the kernels for four take."""
import math

import pytest
import torch

from tests.test_gpu_cross_attn import TYPES, _check, _lengths, _make, _run
from tests.tower_reference import attention

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'

# pairs of one wave each, one block to a pair, too long for a block's LDS, split (two, one, four and three rows); tiles,
# tiles with a split row list
FORMS = [(700, 1, 40, 4, 4, 16), (500, 1, 1500, 4, 4, 32), (103, 1, 4200, 10, 10, 8), (3, 1, 600, 4, 2, 64),
         (3, 1, 9000, 2, 2, 64), (3, 4, 700, 2, 2, 128), (3, 3, 120, 4, 4, 40), (3, 40, 130, 2, 2, 64), (3, 300, 70, 4, 1, 32)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('where', ['dout', 'q'])
@pytest.mark.parametrize('B,Tq,Tk,H,Hkv,D', FORMS)
def test_keys_left_out_get_zeros_beside_infinite_gradients_and_queries(B, Tq, Tk, H, Hkv, D, where, dtype):
    """A key that is left out has no part in a row whatever the row holds: infinities and NaN in dout or q of a sample
    leave dk and dv of its keys behind the length and off in the mask at zero, and the other samples as they were."""
    q, k, v, dout = _make(B, Tq, Tk, H, Hkv, D, dtype, seed=41)
    mask = torch.rand(B, Tk, generator=torch.Generator().manual_seed(42)) < 0.7
    mask[:, 3], mask[:, 5] = True, False
    sl = torch.full((B,), Tk - Tk // 4, dtype=torch.int32)
    ok = (mask & (torch.arange(Tk)[None] < sl[:, None])).to(DEV)
    mask, sl = mask.to(DEV), sl.to(DEV)
    clean = _run(q, k, v, dout, sl, mask)
    _check({n: t[:3] for n, t in clean.items()}, attention(q[:3], k[:3], v[:3], sl[:3], mask[:3], dout=dout[:3]))
    bad = dout if where == 'dout' else q
    bad[0, 0, :, 2] = math.inf
    bad[0, Tq - 1, 0, 1] = -math.inf
    bad[1, Tq - 1, :, 4] = math.nan
    got = _run(q, k, v, dout, sl, mask)
    gone = ~ok[:, :, None, None].expand_as(k)
    wrong = {n: int((got[n][gone] != 0).sum()) for n in ('dk', 'dv')}
    assert wrong == dict(dk=0, dv=0)
    for n in got:
        assert torch.equal(got[n][2:], clean[n][2:]), n


# one wave to a pair in one launch, and with keys too many for its share of LDS; one block to a pair, the same two; split
THREE = [(700, 60, 4, 32), (700, 300, 4, 16), (150, 700, 4, 40), (150, 1500, 4, 24), (3, 5000, 2, 64), (2, 2100, 1, 128),
         (2, 1, 3, 8), (5, 37, 2, 96)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('Tq,G', [(3, 1), (1, 3)])
@pytest.mark.parametrize('B,Tk,Hkv,D', THREE)
@pytest.mark.parametrize('masked', [False, True])
def test_three_rows(B, Tk, Hkv, D, Tq, G, masked, dtype):
    q, k, v, dout = _make(B, Tq, Tk, Hkv * G, Hkv, D, dtype, seed=43)
    sl = _lengths(B, Tk)
    mask = (torch.rand(B, Tk, generator=torch.Generator().manual_seed(44)) < 0.8).to(DEV) if masked else None
    _check(_run(q, k, v, dout, sl, mask), attention(q, k, v, sl, mask, dout=dout))
