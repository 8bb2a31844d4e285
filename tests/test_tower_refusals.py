"""What cross attention, layer norm and gradient clipping refuse, before anything is launched: through the operators (CPU
tensors: every check of shapes, dtypes and strides comes before the device's) and through the C ABI (addresses that are
never followed)."""
import ctypes as C
import math

import pytest
import torch

from recommendation_amd import _lib, ops

F = torch.float32
P = 1 << 20                      # an address on a 16-byte boundary


class Ws:
    def get(self, n):
        return None, 0


def _attn(B=2, Tq=3, Tk=5, H=4, Hkv=2, D=16, dtype=F):
    z = lambda *s: torch.zeros(*s, dtype=dtype)
    return dict(q=z(B, Tq, H, D), k=z(B, Tk, Hkv, D), v=z(B, Tk, Hkv, D), out=z(B, Tq, H, D)), z


def _fwd(**kw):
    a, _ = _attn()
    a.update(kw)
    ops.cross_attn_fwd(a.pop('q'), a.pop('k'), a.pop('v'), a.pop('out'), ws=Ws(), **a)


@pytest.mark.parametrize('kw,error', [
    (dict(q=torch.zeros(2, 3, 16)), ValueError),
    (dict(q=torch.zeros(3, 3, 4, 16)), ValueError),                      # another batch
    (dict(q=torch.zeros(2, 3, 5, 16)), ValueError),                      # 5 heads over 2
    (dict(k=torch.zeros(2, 5, 2, 24)), ValueError),                      # another head size
    (dict(v=torch.zeros(2, 6, 2, 16)), ValueError),
    (dict(v=torch.zeros(2, 5, 2, 16, dtype=torch.bfloat16)), TypeError),
    (dict(out=torch.zeros(2, 3, 4, 16, dtype=torch.float16)), TypeError),
    (dict(out=torch.zeros(2, 4, 4, 16)), ValueError),
    (dict(q=torch.zeros(2, 3, 16, 4).transpose(2, 3)), ValueError),      # strided last dimension
    (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError), (dict(scale=math.nan), ValueError),
    (dict(scale=math.inf), ValueError),
    (dict(sl=torch.zeros(2, dtype=torch.int64)), ValueError), (dict(sl=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(mask=torch.zeros(2, 5)), TypeError), (dict(mask=torch.zeros(2, 4, dtype=torch.bool)), ValueError),
    (dict(mask=torch.zeros(5, 2, dtype=torch.bool).t()), ValueError),
    (dict(lse=torch.zeros(2, 3, 4)), ValueError), (dict(lse=torch.zeros(2, 4, 3, dtype=torch.float64)), ValueError),
    (dict(), ValueError),                                                # well formed, but not on the GPU
])
def test_cross_attention_refuses(kw, error):
    with pytest.raises(error):
        _fwd(**kw)


@pytest.mark.parametrize('scale', [1e-40, 2.4e38])
def test_cross_attention_refuses_scales_that_leave_fp32(scale):
    """scale / ln 2 has to be an ordinary fp32 number."""
    with pytest.raises(ValueError, match='1e-30'):
        _fwd(scale=scale)
    assert _abi_fwd(shape=_shape(scale=scale)) == -1 and b'1e-30' in _lib.load().ctr_last_error()


@pytest.mark.parametrize('D', [4, 12, 20, 136, 256])
def test_cross_attention_refuses_head_sizes(D):
    a, z = _attn(D=D)
    with pytest.raises(ValueError, match='head size'):
        _fwd(**a)


def test_cross_attention_refuses_other_types_and_shared_outputs():
    a, z = _attn(dtype=torch.float64)
    with pytest.raises(TypeError):
        _fwd(**a)
    a, z = _attn(H=2)
    with pytest.raises(ValueError, match='shares'):
        _fwd(q=a['q'], k=a['k'], v=a['v'], out=a['q'])
    g = [torch.zeros_like(a['q']), torch.zeros_like(a['k']), torch.zeros_like(a['v'])]
    lse = torch.zeros(2, 2, 3)
    call = lambda dq, dk, dv: ops.cross_attn_bwd(torch.zeros_like(a['q']), a['q'], a['k'], a['v'], a['out'], lse, dq, dk, dv, ws=Ws())
    for grads in ((a['q'], g[1], g[2]), (g[0], a['k'], g[2]), (g[0], g[1], g[1]), (a['out'], g[1], g[2])):
        with pytest.raises(ValueError, match='shares'):
            call(*grads)
    with pytest.raises(ValueError, match='GPU'):
        call(*g)


def _shape(**kw):
    d = dict(B=2, Tq=3, Tk=5, H=4, Hkv=2, D=16, dtype=0, scale=0.25, sl=0, mask=0, mask_ld=0)
    d.update(kw)
    return _lib.ATTN.pack(*d.values())


def _view(p=P, b=4096, t=256, h=16):
    return _lib.HEADS.pack(p, b, t, h)


def _abi_fwd(shape=None, q=None, k=None, v=None, out=None, ws=None, n=0):
    ok = _view()
    return _lib.load().ctr_cross_attn_fwd(shape or _shape(), q or ok, k or ok, v or ok, out or ok, None, ws, n, None)


@pytest.mark.parametrize('kw', [
    dict(shape=_shape(dtype=3)), dict(shape=_shape(dtype=-1)), dict(shape=_shape(B=-1)), dict(shape=_shape(Tk=-1)),
    dict(shape=_shape(Hkv=3)), dict(shape=_shape(Hkv=0)), dict(shape=_shape(H=0)), dict(shape=_shape(D=0)),
    dict(shape=_shape(D=12)), dict(shape=_shape(D=136)), dict(shape=_shape(scale=0.0)), dict(shape=_shape(scale=math.nan)),
    dict(shape=_shape(scale=math.inf)), dict(shape=_shape(mask=P, mask_ld=-1)), dict(shape=_shape(Tq=1 << 30, H=4)),
    dict(shape=_shape(Tk=1 << 30)), dict(shape=_shape(B=1 << 29)),
    dict(q=_view(p=0)), dict(k=_view(p=P + 8)), dict(v=_view(t=18)), dict(q=_view(b=-4096)), dict(out=_view(h=2)),
    dict(out=_view(t=0)), dict(out=_view(h=0)), dict(out=_view(h=8)), dict(out=_view(b=256)), dict(out=_view(t=32)),
])
def test_abi_refuses_attention(kw):
    assert _abi_fwd(**kw) == -1
    assert _lib.load().ctr_last_error()


def test_abi_attention_workspace():
    lib = _lib.load()
    long = _shape(Tq=9, Tk=100000)
    need = lib.ctr_cross_attn_fwd_workspace_bytes(long)
    assert need > 0 and _abi_fwd(shape=long) == -2
    assert _abi_fwd(shape=long, ws=P, n=need - 1) == -2
    assert lib.ctr_cross_attn_fwd_workspace_bytes(_shape(D=12)) == 0
    v = _view(b=1 << 30)
    bwd = lambda ws, n, lse=P: lib.ctr_cross_attn_bwd(long, v, v, v, v, v, lse, v, v, v, ws, n, None)
    need = lib.ctr_cross_attn_bwd_workspace_bytes(long)
    assert bwd(None, 0) == -2 and bwd(P, need - 1) == -2 and bwd(P, need, None) == -1
    assert _abi_fwd(shape=_shape(B=0), q=_view(p=0)) == 0 and _abi_fwd(shape=_shape(Tq=0), q=_view(p=0), out=_view(p=0)) == 0


@pytest.mark.parametrize('call', [
    lambda x, y: ops.layer_norm_fwd(x[0], y[0]),
    lambda x, y: ops.layer_norm_fwd(x, y[:3]),
    lambda x, y: ops.layer_norm_fwd(x, y.half()),
    lambda x, y: ops.layer_norm_fwd(x.double(), y.double()),
    lambda x, y: ops.layer_norm_fwd(x.t(), y.t()),
    lambda x, y: ops.layer_norm_fwd(x[:, :0], y[:, :0]),
    lambda x, y: ops.layer_norm_fwd(x, torch.zeros(1, 6).expand(4, 6)),
    lambda x, y: ops.layer_norm_fwd(x, y, gamma=torch.zeros(5)),
    lambda x, y: ops.layer_norm_fwd(x, y, gamma=torch.zeros(6).half()),
    lambda x, y: ops.layer_norm_fwd(x, y, beta=torch.zeros(12)[::2]),
    lambda x, y: ops.layer_norm_fwd(x, y, mean=torch.zeros(5)),
    lambda x, y: ops.layer_norm_fwd(x, y, eps=-1e-5),
    lambda x, y: ops.layer_norm_fwd(x, y, eps=math.nan),
    lambda x, y: ops.layer_norm_fwd(x, y),
    lambda x, y: ops.layer_norm_bwd(x, x, None, None, y, ws=Ws()),
    lambda x, y: ops.layer_norm_bwd(x, x, torch.zeros(4), torch.zeros(4), y[:3], ws=Ws()),
    lambda x, y: ops.layer_norm_bwd(x, x, torch.zeros(4), torch.zeros(4), y, dgamma=torch.zeros(5), ws=Ws()),
    lambda x, y: ops.layer_norm_bwd(x, x, torch.zeros(4), torch.zeros(4), y, ws=Ws()),
])
def test_layer_norm_refuses(call):
    with pytest.raises((ValueError, TypeError)):
        call(torch.zeros(4, 6), torch.zeros(4, 6))


def test_abi_refuses_layer_norm():
    lib = _lib.load()
    f = lambda x=P, xl=8, rows=4, cols=8, t=0, eps=1e-5, y=P, yl=8: lib.ctr_layer_norm_fwd(x, xl, rows, cols, t, None, None, eps, y, yl, None, None, None)
    for kw in (dict(rows=-1), dict(cols=0), dict(t=7), dict(eps=-1.0), dict(x=None), dict(y=None), dict(xl=7), dict(yl=7)):
        assert f(**kw) == -1, kw
    assert f(rows=0, x=None, y=None) == 0
    b = lambda dy=P, x=P, m=P, r=P, rows=4, cols=8, dx=P, ld=8, dg=P, ws=P, n=1 << 20: lib.ctr_layer_norm_bwd(dy, ld, x, 8, m, r, rows, cols, 0, None, dx, 8, 0, dg, None, ws, n, None)
    for kw in (dict(dy=None), dict(x=None), dict(m=None), dict(r=None), dict(dx=None), dict(ld=7), dict(cols=0)):
        assert b(**kw) == -1, kw
    need = lib.ctr_layer_norm_bwd_workspace_bytes(4, 8)
    assert need > 0 and b(n=need - 1) == -2 and b(ws=None) == -2
    assert b(rows=0, dg=None) == 0


def test_gradient_lists_refuse():
    a = torch.zeros(10)
    for bad in ([a.double()], [torch.zeros(4, 4).t()], [a[:6], a[5:]], [a, a], [a]):
        with pytest.raises((ValueError, TypeError)):
            ops.GradList(bad)
    for bound in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            ops.clip_grads([], bound, ws=Ws())


def test_abi_refuses_gradient_lists():
    lib = _lib.load()
    ptr, cnt, typ = (C.c_void_p * 2)(P, P), (C.c_int64 * 2)(5, 6), (C.c_int * 2)(0, 1)
    need = lib.ctr_grad_norm_workspace_bytes(2)
    norm = lambda p=ptr, c=cnt, t=typ, n=2, out=P, ws=P, b=need: lib.ctr_grad_norm(p, c, t, n, out, ws, b, None)
    neg, huge, kind, null = (C.c_int64 * 2)(5, -1), (C.c_int64 * 2)(5, 1 << 43), (C.c_int * 2)(0, 9), (C.c_void_p * 2)(P, None)
    for kw in (dict(p=None), dict(c=None), dict(t=None), dict(n=-1), dict(c=neg), dict(c=huge), dict(t=kind), dict(p=null), dict(out=None)):
        assert norm(**kw) == -1, kw
    assert norm(b=need - 1) == -2 and norm(ws=None) == -2
    clip = lambda o=ptr, m=1.0, c=cnt, b=need: lib.ctr_clip_grads(ptr, o, c, typ, 2, m, None, P, b, None)
    for kw in (dict(m=0.0), dict(m=-1.0), dict(m=math.nan), dict(m=math.inf), dict(o=None), dict(o=null), dict(c=neg)):
        assert clip(**kw) == -1, kw
    assert clip(b=need - 1) == -2
