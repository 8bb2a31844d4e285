"""Layer norm (ops.layer_norm_fwd / _bwd) against its definition in 64 bits, within derived bounds."""
import math

import pytest
import torch

from tests.tower_reference import layer_norm, within

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ws():
    from recommendation_amd import ops
    return ops.Workspace(torch.device(DEV))


def _make(rows, cols, dtype, seed=0, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols + pad, generator=g) * 2 + torch.randn(rows, 1, generator=g)).to(dtype).to(DEV)[:, :cols]
    dy = torch.randn(rows, cols + pad, generator=g).to(dtype).to(DEV)[:, :cols]
    return x, dy, (1 + 0.1 * torch.randn(cols, generator=g)).to(DEV), (0.1 * torch.randn(cols, generator=g)).to(DEV)


def _run(x, dy, gamma, beta, eps=1e-5, into=None, ws=None):
    from recommendation_amd import ops
    rows, cols = x.shape
    nan = lambda *s, t=torch.float32: torch.full(s, math.nan, dtype=t, device=DEV)
    r = dict(y=nan(rows, cols, t=x.dtype), mean=nan(rows), rstd=nan(rows), dgamma=nan(cols), dbeta=nan(cols))
    ops.layer_norm_fwd(x, r['y'], gamma=gamma, beta=beta, eps=eps, mean=r['mean'], rstd=r['rstd'])
    r['dx'] = nan(rows, cols, t=x.dtype) if into is None else into.clone()
    ops.layer_norm_bwd(dy, x, r['mean'], r['rstd'], r['dx'], gamma=gamma, dgamma=r['dgamma'], dbeta=r['dbeta'],
                       accumulate=into is not None, ws=ws or _ws())
    return r


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,cols', [(1, 1), (3, 2), (70, 5), (200, 8), (33, 16), (500, 17), (129, 33), (65, 64), (257, 100),
                                       (40, 128), (50, 257), (31, 512), (9, 1001), (21, 1024), (7, 2049), (13, 4096),
                                       (5, 4097), (3, 16384), (2, 16385), (70, 20000), (5000, 24), (1, 1000), (300, 1536), (300000, 20)])
def test_forward_and_gradients(rows, cols, dtype):
    x, dy, gamma, beta = _make(rows, cols, dtype)
    got, want = _run(x, dy, gamma, beta), layer_norm(x, gamma, beta, dy=dy)
    for n in want:
        within(got[n], want[n], n)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,cols', [(600, 2048), (37, 1025), (9, 4104), (530, 8192), (3, 8193), (1, 6001)])
def test_rows_at_the_limits_of_the_kernels(rows, cols, dtype):
    """Rows that just fill half or all of a block's registers, or pass that by an element; more rows than blocks."""
    test_forward_and_gradients(rows, cols, dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,cols,pad', [(40, 24, 3), (33, 128, 1), (17, 999, 25), (6, 5000, 7), (4, 17000, 5)])
def test_rows_of_a_wider_buffer(rows, cols, pad, dtype):
    """Rows that start at any element, results into a wider buffer whose other columns stay."""
    from recommendation_amd import ops
    x, dy, gamma, beta = _make(rows, cols, dtype, seed=1, pad=pad)
    want = layer_norm(x, gamma, beta, dy=dy)
    buf = torch.full((2, rows, cols + pad), 7.0, dtype=dtype, device=DEV)
    y, dx = buf[0, :, 1:cols + 1], buf[1, :, 1:cols + 1]
    mean, rstd = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    dgamma, dbeta = torch.empty(cols, device=DEV), torch.empty(cols, device=DEV)
    ops.layer_norm_fwd(x, y, gamma=gamma, beta=beta, mean=mean, rstd=rstd)
    ops.layer_norm_bwd(dy, x, mean, rstd, dx, gamma=gamma, dgamma=dgamma, dbeta=dbeta, ws=_ws())
    for n, t in (('y', y), ('dx', dx), ('dgamma', dgamma), ('dbeta', dbeta)):
        within(t, want[n], n)
    assert (buf[:, :, 0] == 7).all() and (buf[:, :, cols + 1:] == 7).all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('cols', [30, 2000, 18000])
def test_without_parameters_in_place_and_accumulated(dtype, cols):
    from recommendation_amd import ops
    x, dy, _, _ = _make(25, cols, dtype, seed=2)
    want = layer_norm(x, dy=dy)
    got = _run(x, dy, None, None)
    for n in want:
        within(got[n], want[n], n)
    into = _make(25, cols, dtype, seed=3)[0].contiguous()
    within(_run(x, dy, None, None, into=into)['dx'], layer_norm(x, dy=dy, into=into)['dx'], 'dx added')
    y, g = x.clone(), dy.clone()
    ops.layer_norm_fwd(y, y)
    assert torch.equal(y, got['y'])
    dbeta = torch.empty(cols, device=DEV)
    ops.layer_norm_bwd(g, x, got['mean'], got['rstd'], g, dbeta=dbeta, ws=_ws())
    assert torch.equal(g, got['dx']) and torch.equal(dbeta, got['dbeta'])
    x2 = x.clone()
    ops.layer_norm_bwd(dy, x2, got['mean'], got['rstd'], x2, ws=_ws())
    assert torch.equal(x2, got['dx'])


def test_far_mean_small_spread():
    """The variance is taken around the mean: a spread of 1 at a mean of 4096 keeps its digits."""
    g = torch.Generator().manual_seed(4)
    x = (4096 + torch.randn(20, 700, generator=g)).to(DEV)
    dy = torch.randn(20, 700, generator=g).to(DEV)
    got, want = _run(x, dy, None, None), layer_norm(x, dy=dy)
    for n in want:
        within(got[n], want[n], n)


def test_bad_rows_stay_alone():
    x, dy, gamma, beta = _make(50, 40, torch.float32, seed=5)
    x[7, 3], x[20, 0] = math.nan, math.inf
    got, clean = _run(x, dy, gamma, beta), _run(torch.where(x.isfinite(), x, 0.0), dy, gamma, beta)
    rows = [r for r in range(50) if r not in (7, 20)]
    assert torch.equal(got['y'][rows], clean['y'][rows]) and torch.equal(got['dx'][rows], clean['dx'][rows])
    assert got['y'][7].isnan().all() and got['y'][20].isnan().all()


def test_no_rows():
    x, dy, gamma, beta = _make(0, 12, torch.float32)
    got = _run(x, dy, gamma, beta)
    assert (got['dgamma'] == 0).all() and (got['dbeta'] == 0).all()


@pytest.mark.parametrize('dtype', TYPES)
def test_same_bits_again(dtype):
    for rows, cols in ((5000, 96), (900, 4096)):
        x, dy, gamma, beta = _make(rows, cols, dtype, seed=6)
        a, b = _run(x, dy, gamma, beta), _run(x, dy, gamma, beta)
        for n in a:
            assert torch.equal(a[n], b[n]), n


def test_gradients_against_differences():
    x, dy, gamma, beta = _make(6, 50, torch.float32, seed=7)
    got, want = _run(x, dy, gamma, beta), layer_norm(x, gamma, beta, dy=dy)
    h, g64 = 2.0 ** -7, dy.cpu().double()
    for name, t, grad in (('x', x, 'dx'), ('gamma', gamma, 'dgamma'), ('beta', beta, 'dbeta')):
        u = (torch.randn(t.shape, generator=torch.Generator().manual_seed(8)) * 64).round().div(64).to(DEV)
        ends, exact, noise = [], [], 0.0
        for sign in (1, -1):
            a = dict(x=x, gamma=gamma, beta=beta)
            a[name] = t + sign * h * u
            ends.append(float((_run(dy=dy, **a)['y'].cpu().double() * g64).sum()))
            value, bound = layer_norm(**a)['y']
            exact.append(float((value * g64).sum()))
            noise += float((bound * g64.abs()).sum())
        value, off = want[grad]
        u64 = u.cpu().double()
        allowed = noise / (2 * h) + abs((exact[0] - exact[1]) / (2 * h) - float((value * u64).sum())) \
            + float((off * u64.abs()).sum())
        assert abs((ends[0] - ends[1]) / (2 * h) - float((got[grad].cpu().double() * u64).sum())) <= allowed, name


def test_another_stream_and_replays():
    from recommendation_amd import ops
    x, dy, gamma, beta = _make(700, 96, torch.bfloat16, seed=9)
    ws = _ws()
    want = _run(x, dy, gamma, beta, ws=ws)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _run(x, dy, gamma, beta)
    stream.synchronize()
    for n in want:
        assert torch.equal(got[n], want[n]), n
    r = {n: torch.empty_like(t) for n, t in want.items()}
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.layer_norm_fwd(x, r['y'], gamma=gamma, beta=beta, mean=r['mean'], rstd=r['rstd'])
        ops.layer_norm_bwd(dy, x, r['mean'], r['rstd'], r['dx'], gamma=gamma, dgamma=r['dgamma'], dbeta=r['dbeta'], ws=ws)
    for rep in range(3):
        fresh = _make(700, 96, torch.bfloat16, seed=20 + rep)
        for dst, src in zip((x, dy, gamma, beta), fresh):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        want = _run(x, dy, gamma, beta)
        for n in want:
            assert torch.equal(r[n], want[n]), (rep, n)
