"""Cross attention (ops.cross_attn_fwd / _bwd) against its definition in 64 bits, within bounds that follow from the
operations (tests/tower_reference.py)."""
import math

import pytest
import torch

from tests.tower_reference import attention, within

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ws():
    from recommendation_amd import ops
    return ops.Workspace(torch.device(DEV))


def _make(B, Tq, Tk, H, Hkv, D, dtype, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g) * std).to(dtype).to(DEV)
    return r(B, Tq, H, D), r(B, Tk, Hkv, D), r(B, Tk, Hkv, D), r(B, Tq, H, D)


def _lengths(B, Tk, seed=1):
    g = torch.Generator().manual_seed(seed)
    sl = torch.randint(0, Tk + 1, (B,), generator=g)
    for i, n in enumerate((0, 1, Tk)[:B]):
        sl[i] = n
    return sl.to(torch.int32).to(DEV)


def _run(q, k, v, dout=None, sl=None, mask=None, scale=None, ws=None, outs=None):
    """Everything the operators write, over buffers that hold NaN before."""
    from recommendation_amd import ops
    ws = ws or _ws()
    nan = lambda t: torch.full(t.shape, math.nan, dtype=t.dtype, device=DEV)
    out, lse = nan(q), torch.full((q.shape[0], q.shape[2], q.shape[1]), math.nan, device=DEV)
    ops.cross_attn_fwd(q, k, v, out, lse=lse, sl=sl, mask=mask, scale=scale, ws=ws)
    res = dict(out=out, lse=lse)
    if dout is not None:
        res.update(dq=nan(q), dk=nan(k), dv=nan(v))
        ops.cross_attn_bwd(dout, q, k, v, out, lse, res['dq'], res['dk'], res['dv'], sl=sl, mask=mask, scale=scale, ws=ws)
    return res


def _check(got, want):
    for n in want:
        within(got[n], want[n], n)


SHAPES = [  # B, Tq, Tk, H, Hkv, D
    (1, 1, 1, 1, 1, 8), (2, 1, 50, 4, 4, 32), (3, 1, 200, 4, 2, 16), (4, 1, 77, 8, 1, 64), (2, 1, 700, 8, 2, 128),
    (3, 2, 33, 2, 1, 40), (2, 3, 65, 6, 2, 72), (3, 20, 31, 2, 2, 32), (2, 33, 64, 3, 3, 24), (2, 17, 129, 4, 2, 96),
    (1, 130, 260, 2, 1, 64), (2, 129, 63, 2, 2, 128), (1, 257, 130, 4, 2, 48), (3, 5, 1, 2, 1, 104)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('B,Tq,Tk,H,Hkv,D', SHAPES)
def test_forward_and_gradients(B, Tq, Tk, H, Hkv, D, dtype):
    q, k, v, dout = _make(B, Tq, Tk, H, Hkv, D, dtype)
    _check(_run(q, k, v, dout), attention(q, k, v, dout=dout))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('B,Tq,Tk,H,Hkv,D', [(5, 1, 70, 4, 2, 32), (6, 40, 150, 2, 2, 64), (4, 3, 129, 8, 2, 128),
                                             (7, 1, 33, 2, 2, 16)])
@pytest.mark.parametrize('masked', ['lengths', 'mask', 'both'])
def test_keys_left_out(B, Tq, Tk, H, Hkv, D, dtype, masked):
    """Lengths from zero to all, a mask with a row that leaves nothing; NaN and infinities where no row attends."""
    q, k, v, dout = _make(B, Tq, Tk, H, Hkv, D, dtype, seed=2)
    sl = _lengths(B, Tk) if masked != 'mask' else None
    mask = None
    if masked != 'lengths':
        mask = torch.rand(B, Tk, generator=torch.Generator().manual_seed(3)) < 0.6
        mask[B - 1] = False
        mask = mask.to(DEV)
    want = attention(q, k, v, sl, mask, dout=dout)
    ok = torch.ones(B, Tk, dtype=torch.bool, device=DEV)
    if sl is not None:
        ok &= torch.arange(Tk, device=DEV)[None] < sl[:, None]
    if mask is not None:
        ok &= mask
    fill = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min], device=DEV).to(dtype)
    junk = fill[torch.arange(k.numel(), device=DEV).view(k.shape) % 4]
    k2, v2 = torch.where(ok[:, :, None, None], k, junk), torch.where(ok[:, :, None, None], v, junk)
    got = _run(q, k2, v2, dout, sl, mask)
    _check(got, want)
    gone = ~ok[:, :, None, None].expand_as(k)
    assert (got['dk'][gone] == 0).all() and (got['dv'][gone] == 0).all()
    empty = ~ok.any(1)
    assert empty.any() and (got['out'][empty] == 0).all() and (got['lse'][empty] == -math.inf).all()
    assert (got['dq'][empty] == 0).all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('Tq,G', [(1, 1), (1, 8), (3, 2), (40, 1)])
def test_long_cache_in_splits(Tq, G, dtype):
    q, k, v, dout = _make(2, Tq, 2500, 2 * G, 2, 64, dtype, seed=5)
    sl = torch.tensor([2500, 900], dtype=torch.int32, device=DEV)      # whole splits without a key
    _check(_run(q, k, v, dout, sl), attention(q, k, v, sl, dout=dout))
    _check(_run(q, k, v, dout), attention(q, k, v, dout=dout))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('B,Tq,Tk,H,Hkv,D', [(103, 1, 4200, 10, 10, 8), (300, 1, 33, 4, 4, 16), (40, 4, 260, 3, 3, 128),
                                             (9, 1, 1500, 4, 1, 56)])
def test_few_rows_of_many_pairs(B, Tq, Tk, H, Hkv, D, dtype):
    """One to four rows per key head: whole histories in one block's LDS, too long for it, and split."""
    q, k, v, dout = _make(B, Tq, Tk, H, Hkv, D, dtype, seed=6)
    sl = _lengths(B, Tk)
    _check(_run(q, k, v, dout, sl), attention(q, k, v, sl, dout=dout))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('Tq', [1, 70])
def test_strided_views(dtype, Tq):
    """Keys and values as halves of one projection, heads before time, a query that every sample shares."""
    B, Tk, H, D = 3, 45, 4, 32
    g = torch.Generator().manual_seed(7)
    kv = torch.randn(B, Tk, 2, H, D, generator=g).to(dtype).to(DEV)
    q = torch.randn(1, H, Tq, D, generator=g).to(dtype).to(DEV).transpose(1, 2).expand(B, Tq, H, D)
    dout = torch.randn(B, H, Tq, D, generator=g).to(dtype).to(DEV).transpose(1, 2)
    k, v = kv[:, :, 0], kv[:, :, 1]
    want = attention(q, k, v, dout=dout)
    _check(_run(q, k, v, dout), want)
    from recommendation_amd import ops
    grads = torch.full((B, Tk + 1, 2, H, D), 7.0, dtype=dtype, device=DEV)      # one row more than is written
    wide = torch.full((B, Tq, H, 2 * D), 7.0, dtype=dtype, device=DEV)
    lse, dq, ws = torch.empty(B, H, Tq, device=DEV), torch.empty(B, Tq, H, D, dtype=dtype, device=DEV), _ws()
    out = wide[..., :D]
    ops.cross_attn_fwd(q, k, v, out, lse=lse, ws=ws)
    ops.cross_attn_bwd(dout, q, k, v, out, lse, dq, grads[:, :Tk, 0], grads[:, :Tk, 1], ws=ws)
    _check(dict(out=out, lse=lse, dq=dq, dk=grads[:, :Tk, 0], dv=grads[:, :Tk, 1]), want)
    assert (grads[:, Tk] == 7).all() and (wide[..., D:] == 7).all()


@pytest.mark.parametrize('dtype', TYPES)
def test_large_scores_and_scale(dtype):
    """One key far above the others; a scale of one's own."""
    q, k, v, dout = _make(2, 37, 90, 2, 2, 64, dtype, seed=9, std=2.0)
    k[:, 11] *= 4
    _check(_run(q, k, v, dout, scale=0.7), attention(q, k, v, dout=dout, scale=0.7))


@pytest.mark.parametrize('Tq', [1, 40])
@pytest.mark.parametrize('size', [1e-6, 1e3])
def test_fp16_gradients_keep_their_digits(Tq, size):
    """Gradients far below and above fp16's middle: ds is scaled by a power of two before it is rounded."""
    q, k, v, dout = _make(2, Tq, 300, 2, 1, 64, torch.float16, seed=11)
    dout = (dout.float() * size).half()
    want = attention(q, k, v, dout=dout)
    got = _run(q, k, v, dout)
    _check(got, want)


@pytest.mark.parametrize('dtype', TYPES)
def test_same_bits_again(dtype):
    for B, Tq, Tk, H, Hkv, D in ((2, 1, 3000, 8, 2, 64), (3, 70, 200, 4, 2, 32), (300, 1, 60, 2, 2, 32)):
        q, k, v, dout = _make(B, Tq, Tk, H, Hkv, D, dtype, seed=13)
        a, b = _run(q, k, v, dout), _run(q, k, v, dout)
        for n in a:
            assert torch.equal(a[n], b[n]), n


@pytest.mark.parametrize('Tq', [1, 24])
def test_gradients_against_differences(Tq):
    """(f(x + h u) - f(x - h u)) / 2h for f = <out, dout>, against <gradient, u>.  Off by what the two outputs are off
    by, over 2h, by the quotient's own error (measured on the definition) and by the gradient's bound."""
    q, k, v, dout = _make(2, Tq, 60, 4, 2, 32, torch.float32, seed=17)
    got, want = _run(q, k, v, dout), attention(q, k, v, dout=dout)
    h, g64 = 2.0 ** -7, dout.cpu().double()
    for name, x in (('q', q), ('k', k), ('v', v)):
        u = torch.randn(x.shape, generator=torch.Generator().manual_seed(19)).to(DEV)
        u = (u * 64).round() / 64                       # x +- h u rounds once, by at most 2^-24 of |x|: 4 below
        ends, exact, noise = [], [], 0.0
        for sign in (1, -1):
            args = {'q': q, 'k': k, 'v': v}
            args[name] = x + sign * h * u
            ends.append(float((_run(**args)['out'].cpu().double() * g64).sum()))
            value, bound = attention(**args)['out']
            exact.append(float((value * g64).sum()))
            noise += float((bound * g64.abs()).sum())
        grad, off = want['d' + name]
        u64 = u.cpu().double()
        slope = float((got['d' + name].cpu().double() * u64).sum())
        allowed = noise / (2 * h) + abs((exact[0] - exact[1]) / (2 * h) - float((grad * u64).sum())) \
            + float((off * u64.abs()).sum())
        assert abs((ends[0] - ends[1]) / (2 * h) - slope) <= allowed, name


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('Tq', [1, 40])
@pytest.mark.parametrize('left', ['one key', 'lengths', 'mask'])
def test_a_single_key_has_no_gradient_of_its_score(dtype, Tq, left):
    """softmax over one key is 1 whatever the score: dq and dk are zeros exactly."""
    Tk = 1 if left == 'one key' else 2600
    q, k, v, dout = _make(2, Tq, Tk, 4, 2, 64, dtype, seed=21)
    sl = torch.tensor([1, 1], dtype=torch.int32, device=DEV) if left == 'lengths' else None
    mask = None
    if left == 'mask':
        mask = torch.zeros(2, Tk, dtype=torch.bool, device=DEV)
        mask[0, 2000] = mask[1, 7] = True
    got = _run(q, k, v, dout, sl, mask)
    _check(got, attention(q, k, v, sl, mask, dout=dout))
    assert (got['dq'] == 0).all() and (got['dk'] == 0).all()


def test_no_queries_no_keys_no_samples():
    from recommendation_amd import ops
    for dtype in TYPES:
        q, k, v, dout = _make(2, 3, 0, 2, 2, 32, dtype)
        got = _run(q, k, v, dout)
        assert (got['out'] == 0).all() and (got['lse'] == -math.inf).all() and (got['dq'] == 0).all()
        q, k, v, dout = _make(2, 0, 5, 2, 2, 32, dtype)
        got = _run(q, k, v, dout)
        assert (got['dk'] == 0).all() and (got['dv'] == 0).all()
        q, k, v, dout = _make(0, 3, 5, 2, 2, 32, dtype)
        _run(q, k, v, dout)


def test_infinite_scores():
    """All scores of a row at -infinity: no weight to give, zeros.  NaN in a valid key reaches its own sample only."""
    q, k, v, _ = _make(2, 2, 40, 1, 1, 32, torch.bfloat16)
    k[0], q[0] = -math.inf, 1.0
    k[1, 3, 0, 0] = math.nan
    got = _run(q, k, v)
    assert (got['out'][0] == 0).all() and (got['lse'][0] == -math.inf).all()
    assert got['out'][1].isnan().all()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_another_stream_and_replays(dtype):
    """On a side stream, and captured: every replay over new inputs equals the eager call, with eager work between."""
    from recommendation_amd import ops
    for B, Tq, Tk, H, Hkv, D in ((2, 1, 2100, 4, 2, 64), (2, 40, 90, 2, 2, 32)):
        q, k, v, dout = _make(B, Tq, Tk, H, Hkv, D, dtype, seed=23)
        sl = _lengths(B, Tk, seed=4)
        ws = _ws()
        want = _run(q, k, v, dout, sl)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got = _run(q, k, v, dout, sl, ws=ws)
        stream.synchronize()
        for n in want:
            assert torch.equal(got[n], want[n]), n
        bufs = {n: torch.empty_like(t) for n, t in want.items()}

        def step():
            ops.cross_attn_fwd(q, k, v, bufs['out'], lse=bufs['lse'], sl=sl, ws=ws)
            ops.cross_attn_bwd(dout, q, k, v, bufs['out'], bufs['lse'], bufs['dq'], bufs['dk'], bufs['dv'], sl=sl, ws=ws)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for rep in range(3):
            fresh = _make(B, Tq, Tk, H, Hkv, D, dtype, seed=40 + rep)
            for dst, src in zip((q, k, v, dout), fresh):
                dst.copy_(src)
            sl.copy_(_lengths(B, Tk, seed=60 + rep))
            graph.replay()
            torch.cuda.synchronize()
            want = _run(q, k, v, dout, sl)
            for n in want:
                assert torch.equal(bufs[n], want[n]), (rep, n)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('B,Tq,Tk,H,Hkv,D', [(2, 100, 70, 6, 2, 64), (2, 33, 130, 5, 1, 32), (1, 3, 200, 64, 1, 16),
                                             (2, 70, 90, 14, 2, 96), (1, 1, 300, 40, 1, 128), (2, 9, 40, 33, 1, 24)])
def test_groups_of_any_size(B, Tq, Tk, H, Hkv, D, dtype):
    """3, 5, 7, 33, 40 and 64 query heads to a key head: groups that no tile of rows holds whole."""
    q, k, v, dout = _make(B, Tq, Tk, H, Hkv, D, dtype, seed=25)
    _check(_run(q, k, v, dout), attention(q, k, v, dout=dout))


@pytest.mark.parametrize('Tq', [1, 40])
def test_lengths_out_of_range_and_masks_of_other_forms(Tq):
    """Lengths below zero and beyond Tk are taken as none and all; masks as bytes, one row for all samples, strided rows."""
    q, k, v, dout = _make(3, Tq, 50, 2, 2, 32, torch.bfloat16, seed=27)
    sl = torch.tensor([-3, 70, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    _check(_run(q, k, v, dout, sl), attention(q, k, v, torch.tensor([0, 50, 50]), dout=dout))
    keep = torch.rand(3, 90, generator=torch.Generator().manual_seed(1)) < 0.5
    for mask in ((keep * 255).to(torch.uint8).to(DEV)[:, 7:57], keep.to(DEV)[:1, :50].expand(3, 50), keep.to(DEV)[:, 1:51]):
        _check(_run(q, k, v, dout, None, mask), attention(q, k, v, None, mask, dout=dout))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('Tq,Tk', [(1, 700), (40, 700), (150, 1600), (20, 9000)])
def test_padding_before_the_keys(dtype, Tq, Tk):
    """Whole tiles and whole splits that the mask leaves nothing of, before, between and behind the keys of a sample; one
    sample has its only key at the end."""
    q, k, v, dout = _make(4, Tq, Tk, 2, 1, 64, dtype)
    mask = torch.zeros(4, Tk, dtype=torch.bool)
    mask[0, Tk - 300:] = True
    mask[1, Tk - 1] = True
    mask[2, 5], mask[2, Tk - 2] = True, True
    mask[3, 130:131 + Tk // 3] = True
    mask = mask.to(DEV)
    want = attention(q, k, v, None, mask, dout=dout)
    k2, v2 = k.clone(), v.clone()
    k2[~mask], v2[~mask] = math.nan, math.inf
    _check(_run(q, k2, v2, dout, None, mask), want)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D', [24, 32, 64, 72, 96, 128])
@pytest.mark.parametrize('Tq,Tk', [(20, 70), (50, 30), (33, 64), (5, 33), (130, 20)])
def test_many_pairs_of_few_strips(dtype, D, Tq, Tk):
    """Enough (sample, key head) pairs for blocks of one and two waves, over rows, over keys and over both."""
    B = 260
    q, k, v, dout = _make(B, Tq, Tk, 8, 8, D, dtype)
    sl = _lengths(B, Tk)
    _check(_run(q, k, v, dout, sl), attention(q, k, v, sl, dout=dout))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('Tq', [1, 45])
def test_time_before_batch(dtype, Tq):
    q, k, v, dout = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in _make(3, Tq, 70, 4, 2, 64, dtype, seed=29))
    _check(_run(q, k, v, dout), attention(q, k, v, dout=dout))


@pytest.mark.parametrize('Tq', [1, 40])
def test_offsets_beyond_32_bits(Tq):
    """Rows of a cache 64 MiB apart: the last ones lie beyond 2^31 bytes, a tile's rows beyond 2^31 of its first."""
    Tk, D, far = 40, 32, 1 << 24
    q, k, v, dout = _make(1, Tq, Tk, 1, 1, D, torch.float32, seed=31)
    want = attention(q, k, v, dout=dout)
    cache = torch.empty(Tk * far, device=DEV)
    view = lambda at: cache.as_strided((1, Tk, 1, D), (Tk * far, far, D, 1), at)
    kf, vf = view(0), view(64)
    kf.copy_(k)
    vf.copy_(v)
    got = _run(q, kf, vf)
    _check(got, {n: want[n] for n in ('out', 'lse')})
    from recommendation_amd import ops
    dq, dk, dv = torch.empty_like(q), view(128), view(192)
    ops.cross_attn_bwd(dout, q, kf, vf, got['out'], got['lse'], dq, dk, dv, ws=_ws())
    _check(dict(dq=dq, dk=dk, dv=dv), {n: want[n] for n in ('dq', 'dk', 'dv')})


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('B,Tq,Tk,D', [(70001, 1, 3, 8), (20003, 6, 2, 16)])
def test_very_many_samples(B, Tq, Tk, D, dtype):
    q, k, v, dout = _make(B, Tq, Tk, 1, 1, D, dtype, seed=33)
    sl = (torch.arange(B) % (Tk + 1)).to(torch.int32).to(DEV)
    _check(_run(q, k, v, dout, sl), attention(q, k, v, sl, dout=dout))


def test_two_streams_at_once():
    """Two calls in flight on two streams, each with its own workspace."""
    cases = [_make(2, 1, 3000, 4, 2, 64, torch.bfloat16, seed=35), _make(2, 90, 400, 4, 2, 64, torch.bfloat16, seed=36)]
    want = [_run(*c) for c in cases]
    streams, ws = [torch.cuda.Stream() for _ in cases], [_ws() for _ in cases]
    for rep in range(3):
        got = []
        for s, c, w in zip(streams, cases, ws):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(_run(*c, ws=w))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for n in b:
                assert torch.equal(a[n], b[n]), n
