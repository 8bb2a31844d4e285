"""Outputs of cross attention, layer norm and gradient clipping that share memory with another tensor of the call are
refused, views that only interleave in one buffer are not (CPU tensors: a call that is well formed ends at the check of
the device)."""
import random

import pytest
import torch

from recommendation_amd import ops


class Ws:
    def get(self, n):
        return None, 0


def _elements(t):
    at = torch.tensor([t.storage_offset()])
    for n, stride in zip(t.shape, t.stride()):
        at = (at[:, None] + torch.arange(n)[None] * stride).reshape(-1)
    return set(at.tolist())


@pytest.mark.parametrize('seed', range(8))
def test_share_is_exact(seed):
    """Against the sets of elements, over views of any strides (overlapping and broadcast ones too)."""
    rng = random.Random(seed)
    buf = torch.zeros(4096)

    def view():
        shape = [rng.randint(1, 4) for _ in range(3)] + [rng.choice([1, 2, 4, 8])]
        strides = [rng.choice([0, 4, 8, 12, 16, 24, 32, 48, 64, 96, 128, 200]) for _ in range(3)] + [1]
        return torch.as_strided(buf, shape, strides, rng.choice([0, 4, 8, 16, 32, 64, 100, 300]))

    seen = set()
    for _ in range(400):
        a, b = view(), view()
        want = bool(_elements(a) & _elements(b))
        assert ops._share(a, b) == want, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
        seen.add(want)
    assert seen == {True, False}


def test_share_of_other_types_and_of_no_elements():
    raw = torch.zeros(1024, dtype=torch.uint8)
    a = raw[:64].view(torch.float32)
    assert ops._share(a, raw[63:70]) and not ops._share(a, raw[64:70]) and ops._share(raw[60:62].view(torch.bfloat16), a)


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


B, TQ, TK, H, HKV, D = 3, 6, 5, 4, 2, 16


def _fwd(**kw):
    a = dict(q=_t(B, TQ, H, D), k=_t(B, TK, HKV, D), v=_t(B, TK, HKV, D), out=_t(B, TQ, H, D))
    a.update(kw)
    ops.cross_attn_fwd(**a, ws=Ws())


def _bwd(**kw):
    a = dict(dout=_t(B, TQ, H, D), q=_t(B, TQ, H, D), k=_t(B, TK, HKV, D), v=_t(B, TK, HKV, D), out=_t(B, TQ, H, D),
             lse=_t(B, H, TQ), dq=_t(B, TQ, H, D), dk=_t(B, TK, HKV, D), dv=_t(B, TK, HKV, D))
    a.update(kw)
    ops.cross_attn_bwd(**a, ws=Ws())


def _shifted(shape, by):
    """Two tensors of `shape` in one buffer, the second `by` elements behind the first."""
    n = 1
    for s in shape:
        n *= s
    buf = _t(n + by)
    return buf[:n].view(shape), buf[by:].view(shape)


def test_forward_refuses_shifted_outputs():
    for by in (0, 4, 64, B * TQ * H * D - 4):
        for a, b in (_shifted((B, TQ, H, D), by), _shifted((B, TQ, H, D), by)[::-1]):
            with pytest.raises(ValueError, match='out shares its memory with q'):
                _fwd(q=a, out=b)
    wide = _t(B, TK + 1, HKV, D)
    with pytest.raises(ValueError, match='out shares its memory with v'):
        ops.cross_attn_fwd(_t(B, TK, HKV, D), _t(B, TK, HKV, D), wide[:, :TK], wide[:, 1:], ws=Ws())
    buf = _t(B * H * TQ + B * TQ * H * D)
    lse, out = buf[:B * H * TQ].view(B, H, TQ), buf[B * H * TQ - 4:-4].view(B, TQ, H, D)
    with pytest.raises(ValueError, match='out shares its memory with lse'):
        _fwd(lse=lse, out=out)
    with pytest.raises(ValueError, match='lse shares its memory with q'):
        _fwd(lse=lse, q=out)
    rows = _t(B * TQ * H * D)
    with pytest.raises(ValueError, match='out shares its memory with mask'):
        _fwd(out=rows.view(B, TQ, H, D), mask=rows.view(torch.uint8)[64:64 + B * TK].view(B, TK))
    with pytest.raises(ValueError, match='out shares its memory with sl'):
        _fwd(out=rows.view(B, TQ, H, D), sl=rows.view(torch.int32)[-B:])


def test_backward_refuses_shifted_gradients():
    buf = _t(B, TK + 1, HKV, D)
    with pytest.raises(ValueError, match='dk shares its memory with dv'):
        _bwd(dk=buf[:, :TK], dv=buf[:, 1:])
    for name in ('dout', 'q', 'out'):
        a, b = _shifted((B, TQ, H, D), 64)
        with pytest.raises(ValueError, match='dq shares its memory with ' + name):
            _bwd(**{'dq': b, name: a})
    for name in ('k', 'v'):
        a, b = _shifted((B, TK, HKV, D), 4)
        with pytest.raises(ValueError, match='dk shares its memory with ' + name):
            _bwd(**{'dk': a, name: b})
    rows = _t(B * TQ * H * D)
    with pytest.raises(ValueError, match='dq shares its memory with lse'):
        _bwd(dq=rows.view(B, TQ, H, D), lse=rows[-B * H * TQ:].view(B, H, TQ))


def test_views_that_interleave_are_taken():
    """Parts of a packed projection and of its gradient, columns of a wider buffer, neighbours in one arena."""
    pack = lambda T: _t(B, T, H + 2 * HKV, D).split([H, HKV, HKV], dim=2)
    (q, k, v), (dq, dk, dv) = pack(TK), pack(TK)
    both = _t(B, TK, H, 2 * D)
    out, dout = both[..., :D], both[..., D:]
    lse = _t(B, H, TK)
    with pytest.raises(ValueError, match='must live on the GPU'):
        ops.cross_attn_fwd(q, k, v, out, lse=lse, ws=Ws())
    with pytest.raises(ValueError, match='must live on the GPU'):
        ops.cross_attn_bwd(dout, q, k, v, out, lse, dq, dk, dv, ws=Ws())
    kv = _t(2, B, TK, HKV, D).permute(1, 2, 0, 3, 4)
    with pytest.raises(ValueError, match='must live on the GPU'):
        _bwd(dk=kv[:, :, 0], dv=kv[:, :, 1])
    time_first = _t(TK, B, 2, HKV, D).transpose(0, 1)
    with pytest.raises(ValueError, match='must live on the GPU'):
        _bwd(dk=time_first[:, :, 0], dv=time_first[:, :, 1])
    arena = _t(4 * B * TQ * H * D)
    parts = [arena[i * B * TQ * H * D:(i + 1) * B * TQ * H * D].view(B, TQ, H, D) for i in range(4)]
    with pytest.raises(ValueError, match='must live on the GPU'):
        _bwd(dout=parts[0], q=parts[1], out=parts[2], dq=parts[3])
    shared = _t(1, TQ, H, D).expand(B, TQ, H, D)                       # inputs may be one another
    with pytest.raises(ValueError, match='must live on the GPU'):
        _bwd(dout=shared, q=shared, out=shared)


ROWS, COLS = 4, 6


def _norm_fwd(**kw):
    a = dict(x=_t(ROWS, COLS), y=_t(ROWS, COLS), gamma=_t(COLS), beta=_t(COLS), mean=_t(ROWS), rstd=_t(ROWS))
    a.update(kw)
    ops.layer_norm_fwd(**a)


def _norm_bwd(**kw):
    a = dict(dy=_t(ROWS, COLS), x=_t(ROWS, COLS), mean=_t(ROWS), rstd=_t(ROWS), dx=_t(ROWS, COLS), gamma=_t(COLS),
             dgamma=_t(COLS), dbeta=_t(COLS))
    a.update(kw)
    ops.layer_norm_bwd(**a, ws=Ws())


@pytest.mark.parametrize('by', [1, 3, COLS, 2 * COLS])
def test_layer_norm_refuses_shifted_rows(by):
    a, b = _shifted((ROWS, COLS), by)
    with pytest.raises(ValueError, match='y shares its memory with x'):
        _norm_fwd(x=a, y=b)
    with pytest.raises(ValueError, match='dx shares its memory with x'):
        _norm_bwd(x=b, dx=a)
    with pytest.raises(ValueError, match='dx shares its memory with dy'):
        _norm_bwd(dy=a, dx=b)
    with pytest.raises(ValueError, match='dx shares its memory with x'):
        _norm_bwd(dy=a, dx=a, x=b)


def test_layer_norm_refuses_the_same_start_with_other_rows():
    wide = _t(ROWS * 2 * COLS)
    x, y = wide.view(ROWS, 2 * COLS)[:, :COLS], wide[:ROWS * COLS].view(ROWS, COLS)
    with pytest.raises(ValueError, match='y shares its memory with x'):
        _norm_fwd(x=x, y=y)
    with pytest.raises(ValueError, match='dx shares its memory with dy'):
        _norm_bwd(dy=x, dx=y)


def test_layer_norm_refuses_shared_vectors():
    rows, cols = _t(2 * ROWS), _t(2 * COLS)
    for kw, match in ((dict(mean=rows[:ROWS], rstd=rows[:ROWS]), 'mean shares its memory with rstd'),
                      (dict(mean=rows[:ROWS], rstd=rows[1:ROWS + 1]), 'mean shares its memory with rstd'),
                      (dict(mean=cols[:ROWS], gamma=cols[:COLS]), 'mean shares its memory with gamma'),
                      (dict(rstd=cols[5:5 + ROWS], beta=cols[:COLS]), 'rstd shares its memory with beta')):
        with pytest.raises(ValueError, match=match):
            _norm_fwd(**kw)
    for kw, match in ((dict(dgamma=cols[:COLS], dbeta=cols[:COLS]), 'dgamma shares its memory with dbeta'),
                      (dict(dgamma=cols[:COLS], dbeta=cols[2:COLS + 2]), 'dgamma shares its memory with dbeta'),
                      (dict(dgamma=cols[:COLS], gamma=cols[:COLS]), 'dgamma shares its memory with gamma'),
                      (dict(dbeta=cols[:COLS], mean=cols[:ROWS]), 'dbeta shares its memory with mean')):
        with pytest.raises(ValueError, match=match):
            _norm_bwd(**kw)
    y = _t(ROWS, COLS)
    with pytest.raises(ValueError, match='y shares its memory with mean'):
        _norm_fwd(x=y, y=y, mean=y.view(-1)[:ROWS])


def test_layer_norm_takes_its_rows_in_place_and_columns_side_by_side():
    a = _t(ROWS, COLS)
    both = _t(ROWS, 2 * COLS)
    for call in (lambda: _norm_fwd(x=a, y=a), lambda: _norm_fwd(x=both[:, :COLS], y=both[:, COLS:]),
                 lambda: _norm_fwd(x=both[:, :COLS], y=both[:, :COLS]), lambda: _norm_bwd(dy=a, dx=a),
                 lambda: _norm_bwd(x=a, dx=a), lambda: _norm_bwd(x=a, dy=a, dx=a),
                 lambda: _norm_bwd(dy=both[:, :COLS], dx=both[:, COLS:]),
                 lambda: _norm_fwd(x=_t(1, COLS), y=_t(1, 2 * COLS)[:, :COLS], mean=_t(1), rstd=_t(1))):
        with pytest.raises(ValueError, match='must live on the GPU'):
            call()


def test_a_gradient_list_knows_its_bytes():
    buf = _t(100)
    lst = ops.GradList.__new__(ops.GradList)
    with pytest.raises(ValueError, match='must live on the GPU'):
        lst.__init__([buf[10:20], buf[:0], buf[40:41], buf[30:35]])
    inside = [i for i in range(100) if lst.holds(buf[i:].data_ptr(), 4)]
    assert inside == [*range(10, 20), *range(30, 35), 40]
    assert lst.holds(buf[20:].data_ptr() - 1, 4) and not lst.holds(buf[20:].data_ptr(), 4)
    none = ops.GradList([])
    assert not none.holds(buf.data_ptr(), 4)


@pytest.mark.gpu
def test_the_norm_may_not_be_a_gradient():
    dev = 'cuda:0'
    ws = ops.Workspace(torch.device(dev))
    buf, out = torch.ones(50, device=dev), torch.ones(52, device=dev)
    grads, outs = ops.GradList([buf[:20], buf[30:]]), ops.GradList([out[:20], out[32:]])
    for norm in (buf[19:20], buf[30:31], buf[49:]):
        with pytest.raises(ValueError, match='norm shares its memory'):
            ops.grad_norm(grads, norm, ws=ws)
        with pytest.raises(ValueError, match='norm shares its memory'):
            ops.clip_grads(grads, 1.0, norm, ws=ws)
    with pytest.raises(ValueError, match='norm shares its memory'):
        ops.clip_grads(grads, 1.0, out[5:6], out=outs, ws=ws)
    ops.grad_norm(grads, buf[20:21], ws=ws)
    ops.clip_grads(grads, 1.0, out[20:21], out=outs, ws=ws)
    assert abs(buf[20].item() - 40 ** 0.5) < 1e-6 and out[20] == buf[20] and (buf[:20] == 1).all() and out[21] == 1
