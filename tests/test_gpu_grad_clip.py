"""Global gradient norm and clipping (ops.grad_norm / clip_grads) against 64-bit sums.  The norm is an fp64 sum rounded
once to fp32 (half a step, 2^-24; the sum's own error is below 2^-40); a clipped value is off by the factor's rounding,
the product's and the type's: 2 x 2^-24 plus half a step of the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
TYPES = [torch.float32, torch.bfloat16, torch.float16]
E = 2.0 ** -24


def _ws():
    from recommendation_amd import ops
    return ops.Workspace(torch.device(DEV))


def _make(sizes, types, std=0.1, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * std).to(types[i % len(types)]).to(DEV) for i, n in enumerate(sizes)]


def _norm(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def _check_clipped(outs, grads, bound):
    norm = _norm(grads)
    by = min(1.0, bound / norm) if norm else 1.0
    for o, g in zip(outs, grads):
        want = g.double() * by
        off = (2 * E + torch.finfo(g.dtype).eps / 2 + 2.0 ** -38) * want.abs() + torch.finfo(g.dtype).tiny * torch.finfo(g.dtype).eps / 2
        assert ((o.double() - want).abs() <= (off if by < 1 else 0 * off)).all()


SIZES = [[1], [0], [], [3, 0, 1, 17], [8192, 8193, 16384, 16385, 5], [100000, 7, 4096], [1 + 37 * i for i in range(250)],
         [5] * 96, [5] * 97, [9000000, 3]]


@pytest.mark.parametrize('types', [TYPES[:1], TYPES[1:2], TYPES[2:], TYPES])
@pytest.mark.parametrize('case', range(len(SIZES)))
@pytest.mark.parametrize('bound', [0.25, 1e5])
def test_norm_and_clipping(case, types, bound):
    from recommendation_amd import ops
    grads, ws = _make(SIZES[case], types), _ws()
    norm = torch.full((1,), math.nan, device=DEV)
    ops.grad_norm(grads, norm, ws=ws)
    want = _norm(grads)
    assert abs(float(norm) - want) <= 2 * E * want
    outs = [torch.full_like(g, math.nan) for g in grads]
    kept = [g.clone() for g in grads]
    norm.fill_(math.nan)
    ops.clip_grads(ops.GradList(grads), bound, norm, out=ops.GradList(outs), ws=ws)
    assert abs(float(norm) - want) <= 2 * E * want
    assert all(torch.equal(g, k) for g, k in zip(grads, kept))
    _check_clipped(outs, grads, bound)
    ops.clip_grads(grads, bound, ws=ws)                  # in place, without the norm
    for g, o in zip(grads, outs):
        assert torch.equal(g, o)


@pytest.mark.parametrize('dtype', TYPES)
def test_views_at_any_element(dtype):
    from recommendation_amd import ops
    flat = _make([50000], [dtype], seed=3)[0]
    cuts = [1, 2, 9, 10, 4111, 20000, 45001]
    grads = [flat[a:b - 1] for a, b in zip(cuts, cuts[1:])]           # one element between neighbours stays
    kept, ws, norm = flat.clone(), _ws(), torch.empty(1, device=DEV)
    want = [g.clone() for g in grads]
    ops.clip_grads(grads, 0.5, norm, ws=ws)
    assert abs(float(norm) - _norm(want)) <= 2 * E * _norm(want)
    _check_clipped(grads, want, 0.5)
    for b in cuts:
        assert flat[b - 1] == kept[b - 1]
    assert torch.equal(flat[45001:], kept[45001:])


@pytest.mark.parametrize('value', [1e30, 1e-30, 3e38])
def test_squares_beyond_fp32(value):
    from recommendation_amd import ops
    g = torch.full((1000,), value, device=DEV)
    norm, ws = torch.empty(1, device=DEV), _ws()
    ops.grad_norm([g], norm, ws=ws)
    want = value * math.sqrt(1000)
    assert float(norm) == math.inf if want > 3.5e38 else abs(float(norm) / want - 1) <= 4 * E
    ops.clip_grads([g], 1.0, ws=ws)
    want = min(value, 1 / math.sqrt(1000))
    assert ((g.double() / want - 1).abs() <= 6 * E).all()


@pytest.mark.parametrize('bad', [math.nan, math.inf])
def test_not_finite(bad):
    """As tf.clip_by_global_norm: every result is NaN, so the step shows what happened."""
    from recommendation_amd import ops
    grads, ws, norm = _make([10, 5000], TYPES[:1]), _ws(), torch.empty(1, device=DEV)
    grads[1][77] = bad
    ops.clip_grads(grads, 1.0, norm, ws=ws)
    assert not math.isfinite(float(norm)) and all(g.isnan().all() for g in grads)


def test_zero_gradients():
    from recommendation_amd import ops
    grads, ws, norm = [torch.zeros(100, device=DEV)], _ws(), torch.empty(1, device=DEV)
    ops.clip_grads(grads, 1.0, norm, ws=ws)
    assert float(norm) == 0 and (grads[0] == 0).all()


def test_same_bits_stream_and_replays():
    from recommendation_amd import ops
    grads = _make([70000, 5, 333333, 12], TYPES, seed=5)
    outs, ws, norm = [torch.empty_like(g) for g in grads], _ws(), torch.empty(1, device=DEV)
    gl, ol = ops.GradList(grads), ops.GradList(outs)
    ops.clip_grads(gl, 1.0, norm, out=ol, ws=ws)
    want, n0 = [o.clone() for o in outs], norm.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.clip_grads(gl, 1.0, norm, out=ol, ws=ws)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(norm, n0)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.clip_grads(gl, 1.0, norm, out=ol, ws=ws)
    for rep in range(3):
        for g, f in zip(grads, _make([70000, 5, 333333, 12], TYPES, seed=10 + rep, std=1e-4 if rep == 1 else 0.1)):
            g.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        got, n1 = [o.clone() for o in outs], norm.clone()
        ops.clip_grads(gl, 1.0, norm, out=ol, ws=ws)
        assert all(torch.equal(a, b) for a, b in zip(outs, got)) and torch.equal(norm, n1)


def test_refusals_on_the_device():
    from recommendation_amd import ops
    ws, a = _ws(), torch.ones(100, device=DEV)
    with pytest.raises(ValueError):
        ops.GradList([a, a])
    with pytest.raises(ValueError):
        ops.GradList([a[:60], a[50:]])
    with pytest.raises(ValueError):
        ops.GradList([torch.ones(4, 6, device=DEV).t()])
    with pytest.raises(TypeError):
        ops.GradList([torch.ones(4, dtype=torch.float64, device=DEV)])
    with pytest.raises(ValueError):
        ops.clip_grads([a[:50]], 1.0, out=[a[25:75]], ws=ws)
    with pytest.raises(ValueError):
        ops.clip_grads([a[:50]], 1.0, out=[a[50:90]], ws=ws)
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            ops.clip_grads([a], bad, ws=ws)
    assert (a == 1).all()
