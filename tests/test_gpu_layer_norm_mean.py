"""Layer norm of rows whose spread is nothing or little beside their mean: the mean's rounding must not be left in the row."""
import math

import pytest
import torch

from tests.test_gpu_layer_norm import TYPES, _make, _run
from tests.tower_reference import E, half_step

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
# every kernel: a part of a wave, a wave, four waves, a block, a walked row; widths that no power of two divides
COLS = [1, 3, 7, 41, 47, 55, 61, 82, 100, 131, 250, 509, 1000, 1531, 2050, 4091, 6001, 9000, 16383, 16385, 20001]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('value', [100.0, 1000.0, -1000.0, 1e-3, 0.0, 60000.0])
@pytest.mark.parametrize('cols', COLS)
def test_constant_rows_give_beta(cols, value, dtype):
    """x - mean is zero.  What is left of it: the mean is off by depth * 2^-24 of its size, the residuals' mean by as much
    of that, so |x - mean| < depth^2 2^-48 |x|, times rstd <= 1 / sqrt(eps) and gamma (below 2) - and the rounding of y."""
    _, _, gamma, beta = _make(1, cols, dtype)
    x = torch.full((5, cols), value).to(dtype).to(DEV)
    got = _run(x, torch.zeros_like(x), gamma, beta)
    depth = 30 + cols / 1024
    left = 2 * (depth * E) ** 2 * x[0, 0].abs().float().item() * 1e-5 ** -0.5
    want = beta.double().expand(5, cols)
    off = (got['y'].double() - want).abs()
    bound = left + half_step(dtype) * (want.abs() + left) + E * want.abs() + torch.finfo(dtype).tiny * half_step(dtype)
    assert (off <= bound).all(), float((off - bound).max())
    assert torch.equal(got['mean'], x[:, 0].float()), (got['mean'][0].item(), x[0, 0].item())
    # var is at most what the squared rounding of the mean leaves beside eps
    assert ((got['rstd'].double() * 1e-5 ** 0.5 - 1).abs() <= (depth * E) ** 2 * float(x[0, 0].float()) ** 2 * 1e5 + 4 * E).all()


@pytest.mark.parametrize('cols', COLS[2:])
def test_one_step_beside_the_mean(cols):
    """Rows of 1000 with one entry a step of fp32 above it: x - mean is known exactly, and |x - mean| rstd too."""
    step = 2.0 ** -14                                     # fp32's at 1000
    x = torch.full((4, cols), 1000.0)
    x[:, cols // 2] += step
    got = _run(x.to(DEV), torch.zeros(4, cols, device=DEV), None, None)
    xd = x.double()
    d = xd - xd.mean(1, keepdim=True)
    rstd = ((d * d).mean(1, keepdim=True) + 1e-5) ** -0.5
    depth = 30 + cols / 1024
    # d: the residual of every entry is exact to 2^-24 of |d| + the mean's offset m (depth 2^-24 * 1000), which is taken
    # out to depth 2^-24 of itself; the variance's two terms are each off by depth 2^-24 of d^2 + m^2
    m = depth * E * 1000
    d_off = 3 * depth * E * (d.abs() + m)
    r_rel = 0.5 * (depth + 4) * E * ((d * d).mean(1, keepdim=True) + 2 * m * m) * rstd ** 2 + 4 * E
    bound = rstd * d_off + d.abs() * rstd * (r_rel + 3 * E)
    off = (got['y'].cpu().double() - d * rstd).abs()
    assert (off <= bound).all(), (float(off.max()), float(bound.max()))


@pytest.mark.parametrize('cols', [41, 1000, 6001, 20001])
def test_backward_of_constant_rows(cols):
    """xh = 0: dgamma is zero, dx is rstd (g - mean g)."""
    x, dy, gamma, beta = _make(9, cols, torch.float32)
    x = torch.full_like(x, 1000.0)
    got = _run(x, dy, gamma, beta)
    assert (got['dgamma'] == 0).all()
    g = dy.double() * gamma.double()
    rstd = got['rstd'].double()[:, None]
    want = rstd * (g - g.mean(1, keepdim=True))
    bound = rstd * ((30 + cols / 1024 + 8) * E * (g.abs() + g.abs().mean(1, keepdim=True)))
    assert ((got['dx'].double() - want).abs() <= bound).all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('cols', COLS)
def test_equal_entries_get_equal_gradients(cols, dtype):
    """Rows of two values, dy following x: dx has two values too, whatever lane or packet an entry lies in."""
    x = torch.where(torch.arange(cols) % 3 == 0, 3.0, -1.5).expand(4, cols).to(dtype).to(DEV).contiguous()
    dy = torch.where(torch.arange(cols) % 3 == 0, 100.3, 99.1).expand(4, cols).to(dtype).to(DEV).contiguous()
    got = _run(x, dy, None, None)
    for n in ('y', 'dx'):
        for first in range(min(cols, 2)):
            same = got[n][:, torch.arange(cols) % 3 == 0] if first == 0 else got[n][:, torch.arange(cols) % 3 != 0]
            assert (same == same[:, :1]).all(), (n, first, same.unique())


@pytest.mark.parametrize('cols', [7, 40, 1000, 6001, 20001])
@pytest.mark.parametrize('value', [math.nan, math.inf, -math.inf])
def test_the_statistics_of_bad_rows(cols, value):
    """A row with a NaN or an infinity keeps no rstd that looks like a number."""
    x, dy, gamma, beta = _make(6, cols, torch.float32)
    x[2, cols - 1] = value
    x[4, 0] = value
    got = _run(x, dy, gamma, beta)
    bad = torch.tensor([False, False, True, False, True, False], device=DEV)
    assert (got['rstd'].isnan() == bad).all() and (got['mean'].isfinite() == ~bad).all()
    assert (got['y'].isnan().all(1) == bad).all() and (got['dx'].isnan().all(1) == bad).all()
