"""Every refusal of cross attention, layer norm and gradient clipping by its own words and its own exception: a call that
slipped past a check would end at another one (CPU tensors: at the device's at the latest) and must not count as refused
here.  The checks of the device itself see CPU tensors that say they live on a GPU."""
import ctypes as C
import math
import re

import pytest
import torch

from recommendation_amd import _lib, ops

P = 1 << 20                      # an address on a 16-byte boundary
BF, HF, F64 = torch.bfloat16, torch.float16, torch.float64


class Ws:
    def get(self, n):
        return None, 0


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def _refuses(call, error, message, kw):
    with pytest.raises(error, match=re.escape(message)) as info:
        call(**kw)
    assert info.type is error and 'must live on the GPU' not in str(info.value)


# ---------------------------------------------------------------------------------------- cross attention: 2 x 3 x 4 x 16
def _fwd(**kw):
    a = dict(q=_t(2, 3, 4, 16), k=_t(2, 5, 2, 16), v=_t(2, 5, 2, 16), out=_t(2, 3, 4, 16))
    a.update(kw)
    ops.cross_attn_fwd(**a, ws=Ws())


def _bwd(**kw):
    a = dict(dout=_t(2, 3, 4, 16), q=_t(2, 3, 4, 16), k=_t(2, 5, 2, 16), v=_t(2, 5, 2, 16), out=_t(2, 3, 4, 16),
             lse=_t(2, 4, 3), dq=_t(2, 3, 4, 16), dk=_t(2, 5, 2, 16), dv=_t(2, 5, 2, 16))
    a.update(kw)
    ops.cross_attn_bwd(**a, ws=Ws())


TOGETHER = 'do not belong together'
QK = [  # what both directions check of q, k, sl, mask and scale
    (dict(q=_t(2, 3, 16)), ValueError, 'q must be [B, Tq, H, D] and k [B, Tk, Hkv, D]'),
    (dict(k=_t(2, 5, 32)), ValueError, 'q must be [B, Tq, H, D] and k [B, Tk, Hkv, D]'),
    (dict(q=_t(3, 3, 4, 16)), ValueError, TOGETHER), (dict(q=_t(2, 3, 5, 16)), ValueError, TOGETHER),
    (dict(k=_t(2, 5, 2, 24)), ValueError, TOGETHER), (dict(k=_t(2, 5, 0, 16)), ValueError, TOGETHER),
    (dict(q=_t(2, 3, 4, 20), k=_t(2, 5, 2, 20)), ValueError, 'head size 20 is not a multiple of 8 up to 128'),
    (dict(q=_t(2, 3, 4, 136), k=_t(2, 5, 2, 136)), ValueError, 'head size 136 is not a multiple of 8 up to 128'),
    (dict(q=_t(2, 3, 4, 16, dtype=F64)), TypeError, 'q: expected float32, bfloat16 or float16, got torch.float64'),
    (dict(q=_t(1, 1, 1, 8).expand(1, 1 << 30, 1, 8), k=_t(1, 1, 1, 8)), ValueError, 'more than 2^30'),
    (dict(q=_t(1, 1, 1, 8), k=_t(1, 1, 1, 8).expand(1, 1 << 30, 1, 8)), ValueError, 'more than 2^30'),
    (dict(q=_t(1, 1, 1, 8).expand(1 << 30, 1, 1, 8), k=_t(1, 1, 1, 8).expand(1 << 30, 1, 1, 8)), ValueError, 'more than 2^30'),
] + [(dict(scale=s), ValueError, 'scale must lie between 1e-30 and 1e30') for s in (0.0, -1.0, math.nan, math.inf, 1e-31, 1e31)] + [
    (dict(sl=_t(2, dtype=torch.int64)), ValueError, 'sl must be a contiguous int32 [B] tensor'),
    (dict(sl=_t(3, dtype=torch.int32)), ValueError, 'sl must be a contiguous int32 [B] tensor'),
    (dict(sl=_t(4, dtype=torch.int32)[::2]), ValueError, 'sl must be a contiguous int32 [B] tensor'),
    (dict(mask=_t(2, 5)), TypeError, 'mask: expected bool or uint8, got torch.float32'),
    (dict(mask=_t(2, 4, dtype=torch.bool)), ValueError, 'mask must be [B, Tk] with a contiguous last dimension'),
    (dict(mask=_t(5, 2, dtype=torch.bool).t()), ValueError, 'mask must be [B, Tk] with a contiguous last dimension'),
]


@pytest.mark.parametrize('call', [_fwd, _bwd])
@pytest.mark.parametrize('kw,error,message', QK)
def test_what_q_and_k_decide(call, kw, error, message):
    _refuses(call, error, message, kw)


ROWS, KEYS = '[2, 3, 4, 16]', '[2, 5, 2, 16]'


@pytest.mark.parametrize('call,name,shape', [
    (_fwd, 'v', KEYS), (_fwd, 'out', ROWS), (_bwd, 'dout', ROWS), (_bwd, 'v', KEYS), (_bwd, 'out', ROWS), (_bwd, 'dq', ROWS),
    (_bwd, 'dk', KEYS), (_bwd, 'dv', KEYS)])
def test_every_tensor_has_the_shape_type_and_layout(call, name, shape):
    dims = [int(n) for n in shape[1:-1].split(', ')]
    for axis in range(4):
        other = list(dims)
        other[axis] += 8
        _refuses(call, ValueError, '%s must be %s, got %s' % (name, shape, other), {name: _t(*other)})
    _refuses(call, ValueError, '%s must be %s' % (name, shape), {name: _t(*dims[:3])})
    _refuses(call, TypeError, '%s: expected torch.float32, got torch.bfloat16' % name, {name: _t(*dims, dtype=BF)})
    apart = _t(*dims[:2], dims[3], dims[2]).transpose(2, 3)
    _refuses(call, ValueError, '%s must have a contiguous last dimension' % name, {name: apart})


@pytest.mark.parametrize('call', [_fwd, _bwd])
def test_q_and_k_have_the_layout_and_one_type(call):
    for name, dims in (('q', (2, 3, 4, 16)), ('k', (2, 5, 2, 16))):
        apart = _t(*dims[:2], dims[3], dims[2]).transpose(2, 3)
        _refuses(call, ValueError, '%s must have a contiguous last dimension' % name, {name: apart})
    _refuses(call, TypeError, 'k: expected torch.float32, got torch.float16', dict(k=_t(2, 5, 2, 16, dtype=HF)))


@pytest.mark.parametrize('call', [_fwd, _bwd])
@pytest.mark.parametrize('lse', [_t(2, 3, 4), _t(2, 4, 3, dtype=F64), _t(2, 4, 2), _t(2, 3, 4).transpose(1, 2), _t(24)])
def test_lse(call, lse):
    _refuses(call, ValueError, 'lse must be contiguous float32 [B, H, Tq]', dict(lse=lse))


@pytest.mark.parametrize('call', [_fwd, _bwd])
def test_a_well_formed_call_ends_at_the_device(call):
    with pytest.raises(ValueError, match='must live on the GPU'):
        call()


# ---------------------------------------------------------------------------------------- layer norm: 4 x 6
def _norm_fwd(**kw):
    a = dict(x=_t(4, 6), y=_t(4, 6), gamma=_t(6), beta=_t(6), mean=_t(4), rstd=_t(4))
    a.update(kw)
    ops.layer_norm_fwd(**a)


def _norm_bwd(**kw):
    a = dict(dy=_t(4, 6), x=_t(4, 6), mean=_t(4), rstd=_t(4), dx=_t(4, 6), gamma=_t(6), dgamma=_t(6), dbeta=_t(6))
    a.update(kw)
    ops.layer_norm_bwd(**a, ws=Ws())


VIEW = 'layer norm wants a [rows, cols] view with at least one column'


@pytest.mark.parametrize('call', [_norm_fwd, _norm_bwd])
@pytest.mark.parametrize('kw,error,message', [
    (dict(x=_t(6)), ValueError, VIEW), (dict(x=_t(4, 0)), ValueError, VIEW), (dict(x=_t(2, 2, 6)), ValueError, VIEW),
    (dict(x=_t(1, 1).expand(1, 1 << 30)), ValueError, VIEW),
    (dict(x=_t(4, 6, dtype=F64)), TypeError, 'x: expected float32, bfloat16 or float16, got torch.float64'),
    (dict(x=_t(6, 4).t()), ValueError, 'x must have a contiguous last dimension and rows that do not overlap'),
    (dict(x=_t(1, 6).expand(4, 6)), ValueError, 'x must have a contiguous last dimension and rows that do not overlap')])
def test_layer_norm_rows(call, kw, error, message):
    _refuses(call, error, message, kw)


@pytest.mark.parametrize('call,name', [(_norm_fwd, 'y'), (_norm_bwd, 'dy'), (_norm_bwd, 'dx')])
def test_layer_norm_tensors(call, name):
    for other in ((3, 6), (4, 7), (4, 6, 1), (24,)):
        _refuses(call, ValueError, '%s must be [4, 6], got %s' % (name, list(other)), {name: _t(*other)})
    _refuses(call, TypeError, '%s: expected torch.float32, got torch.float16' % name, {name: _t(4, 6, dtype=HF)})
    layout = '%s must have a contiguous last dimension and rows that do not overlap' % name
    _refuses(call, ValueError, layout, {name: _t(6, 4).t()})
    _refuses(call, ValueError, layout, {name: _t(1, 6).expand(4, 6)})
    _refuses(call, ValueError, layout, {name: _t(30).as_strided((4, 6), (5, 1))})


@pytest.mark.parametrize('call,name,n', [(_norm_fwd, 'gamma', 6), (_norm_fwd, 'beta', 6), (_norm_fwd, 'mean', 4),
                                         (_norm_fwd, 'rstd', 4), (_norm_bwd, 'mean', 4), (_norm_bwd, 'rstd', 4),
                                         (_norm_bwd, 'gamma', 6), (_norm_bwd, 'dgamma', 6), (_norm_bwd, 'dbeta', 6)])
def test_layer_norm_vectors(call, name, n):
    for bad in (_t(n - 1), _t(n + 1), _t(0), _t(2 * n)[::2]):
        _refuses(call, ValueError, '%s must be contiguous with %d entries' % (name, n), {name: bad})
    _refuses(call, TypeError, '%s: expected torch.float32, got torch.float16' % name, {name: _t(n, dtype=HF)})


def test_layer_norm_eps_and_statistics():
    for eps in (-1e-5, math.nan, math.inf):
        _refuses(_norm_fwd, ValueError, 'eps must be finite and not negative', dict(eps=eps))
    for kw in (dict(mean=None), dict(rstd=None)):
        _refuses(_norm_bwd, ValueError, 'layer_norm_bwd needs the mean and rstd that layer_norm_fwd kept', kw)


@pytest.mark.parametrize('call', [_norm_fwd, _norm_bwd])
def test_a_well_formed_norm_ends_at_the_device(call):
    with pytest.raises(ValueError, match='must live on the GPU'):
        call()


# ---------------------------------------------------------------------------------------- gradient lists
def test_gradient_lists():
    a = _t(10)
    for bad, error, message in (
            ([a, a.double()], TypeError, 'tensor 1: expected float32, bfloat16 or float16, got torch.float64'),
            ([_t(4, 4).t()], ValueError, 'tensor 0 must be contiguous'),
            ([a[:6], a[5:]], ValueError, 'tensors 0 and 1 share memory'),
            ([a[5:], a[:6]], ValueError, 'tensors 1 and 0 share memory'),
            ([a, _t(3), a], ValueError, 'share memory')):
        _refuses(lambda tensors: ops.GradList(tensors), error, message, dict(tensors=bad))
    for bound in (0.0, -1.0, math.inf, math.nan, 3.1e38):
        _refuses(lambda b: ops.clip_grads([], b, ws=Ws()), ValueError, 'max_norm must be positive and finite', dict(b=bound))
    _refuses(lambda: ops.grad_norm([], None, ws=Ws()), ValueError, 'grad_norm needs a norm tensor', {})
    for norm in (_t(2), _t(1, dtype=F64)):
        _refuses(lambda n: ops.grad_norm([], n, ws=Ws()), ValueError, 'norm must be a float32 tensor of one element', dict(n=norm))


# ---------------------------------------------------------------------------------------- devices
class On(torch.Tensor):
    """A CPU tensor that says that it lives on a GPU: enough for checks that come before any launch."""
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device('cuda', self.at))

    def get_device(self):
        return self.at


def _on(t, at=0):
    t = t.as_subclass(On)
    t.at = at
    return t


@pytest.fixture
def first_gpu(monkeypatch):
    monkeypatch.setattr(torch._C, '_cuda_getDevice', lambda: 0, raising=False)
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 0)


def test_tensors_of_a_call_live_on_the_current_device(first_gpu):
    a = dict(q=_t(2, 3, 4, 16), k=_t(2, 5, 2, 16), v=_t(2, 5, 2, 16), out=_t(2, 3, 4, 16), lse=_t(2, 4, 3),
             sl=_t(2, dtype=torch.int32), mask=_t(2, 5, dtype=torch.bool))
    for name in list(a)[1:]:
        kw = {n: _on(t, 1 if n == name else 0) for n, t in a.items()}
        _refuses(_fwd, ValueError, '%s lives on cuda:1, q on cuda:0' % name, kw)
        kw[name] = a[name]
        with pytest.raises(ValueError, match='%s must live on the GPU' % name):
            _fwd(**kw)
    _refuses(_fwd, ValueError, 'q lives on cuda:1, the current device is cuda:0', {n: _on(t, 1) for n, t in a.items()})
    rows = dict(x=_t(4, 6), y=_t(4, 6), gamma=_t(6), beta=_t(6), mean=_t(4), rstd=_t(4))
    for name in list(rows)[1:]:
        _refuses(_norm_fwd, ValueError, '%s lives on cuda:1, x on cuda:0' % name,
                 {n: _on(t, 1 if n == name else 0) for n, t in rows.items()})


def test_gradient_lists_live_on_one_device(first_gpu):
    a, b, out = _t(10), _t(7), _t(17)
    _refuses(lambda tensors: ops.GradList(tensors), ValueError, 'tensor 1 lives on cuda:1, the others on cuda:0',
             dict(tensors=[_on(a), _on(b, 1)]))
    lst = lambda at=0: ops.GradList([_on(a, at), _on(b, at)])
    clip = lambda **kw: ops.clip_grads(kw.pop('g', None) or lst(), 1.0, ws=Ws(), **kw)
    away = 'the gradients or norm live on cuda:1, the current device is cuda:0'
    _refuses(clip, ValueError, away, dict(g=lst(1)))
    _refuses(clip, ValueError, away, dict(norm=_on(_t(1), 1)))
    with pytest.raises(ValueError, match='norm must live on the GPU'):
        clip(norm=_t(1))
    for norm in (a[3:4], b[6:]):
        _refuses(clip, ValueError, 'norm shares its memory with a tensor of the list', dict(norm=_on(norm)))
        _refuses(lambda n: ops.grad_norm(lst(), n, ws=Ws()), ValueError, 'norm shares its memory with a tensor of the list',
                 dict(n=_on(norm)))
    results = ops.GradList([_on(out[:10]), _on(out[10:])])
    _refuses(clip, ValueError, 'norm shares its memory with a tensor of the list', dict(out=results, norm=_on(out[16:])))
    for other in ([a], [_t(10), _t(8)], [_t(10), _t(7, dtype=BF)], [_t(7), _t(10)]):
        _refuses(clip, ValueError, 'out must hold tensors of the same sizes and dtypes', dict(out=[_on(t) for t in other]))
    _refuses(clip, ValueError, 'out shares memory with the gradients without being them', dict(out=[_on(_t(10)), _on(b)]))
    both = _t(30)
    grads, shifted = ops.GradList([_on(both[:10]), _on(both[20:27])]), [_on(both[12:22]), _on(both[1:8])]
    _refuses(clip, ValueError, 'out shares memory with the gradients without being them', dict(g=grads, out=shifted))


# ---------------------------------------------------------------------------------------- the C ABI
def _shape(**kw):
    d = dict(B=2, Tq=3, Tk=5, H=4, Hkv=2, D=16, dtype=0, scale=0.25, sl=0, mask=0, mask_ld=0)
    d.update(kw)
    return _lib.ATTN.pack(*d.values())


def _view(p=P, b=4096, t=256, h=16):
    return _lib.HEADS.pack(p, b, t, h)


def _says(rc, text, code=-1):
    said = _lib.load().ctr_last_error().decode()
    assert rc == code and text in said, (rc, said)


SIZES = 'Hkv must divide H'


@pytest.mark.parametrize('kw,text', [
    (dict(dtype=3), 'unknown dtype 3'), (dict(dtype=-1), 'unknown dtype -1'), (dict(B=-1), SIZES), (dict(Tq=-1), SIZES),
    (dict(Tk=-1), SIZES), (dict(Hkv=3), SIZES), (dict(Hkv=0), SIZES), (dict(H=0), SIZES),
    (dict(D=0), 'head size 0'), (dict(D=12), 'head size 12'), (dict(D=136), 'head size 136'),
    (dict(scale=0.0), '1e-30'), (dict(scale=math.nan), '1e-30'), (dict(scale=math.inf), '1e-30'),
    (dict(mask=P, mask_ld=-1), 'the mask has a negative stride'), (dict(Tq=1 << 30, H=4), 'more than 2^30'),
    (dict(Tk=1 << 30), 'more than 2^30'), (dict(B=1 << 29), 'more than 2^30')])
def test_abi_attention_shapes(kw, text):
    ok = _view()
    lib, shape = _lib.load(), _shape(**kw)
    _says(lib.ctr_cross_attn_fwd(shape, ok, ok, ok, ok, None, None, 0, None), text)
    _says(lib.ctr_cross_attn_bwd(shape, ok, ok, ok, ok, ok, P, ok, ok, ok, None, 0, None), text)


def _abi_fwd(**kw):
    v = [kw.get(n, _view()) for n in ('q', 'k', 'v', 'out')]
    return _lib.load().ctr_cross_attn_fwd(_shape(), *v, None, None, 0, None)


def _abi_bwd(**kw):
    v = [kw.get(n, _view()) for n in ('dout', 'q', 'k', 'v', 'out', 'dq', 'dk', 'dv')]
    return _lib.load().ctr_cross_attn_bwd(_shape(), *v[:5], P, *v[5:], None, 0, None)


@pytest.mark.parametrize('call,name,output', [
    (_abi_fwd, 'q', False), (_abi_fwd, 'k', False), (_abi_fwd, 'v', False), (_abi_fwd, 'out', True), (_abi_bwd, 'dout', False),
    (_abi_bwd, 'q', False), (_abi_bwd, 'k', False), (_abi_bwd, 'v', False), (_abi_bwd, 'out', False), (_abi_bwd, 'dq', True),
    (_abi_bwd, 'dk', True), (_abi_bwd, 'dv', True)])
def test_abi_attention_views(call, name, output):
    _says(call(**{name: None}), '%s is missing' % name)
    _says(call(**{name: _view(p=0)}), '%s is NULL' % name)
    for bad in (_view(p=P + 8), _view(b=4098), _view(t=18), _view(h=17)):
        _says(call(**{name: bad}), '%s and its rows must lie on 16-byte boundaries' % name)
    for bad in (_view(b=-4096), _view(t=-256), _view(h=-16)):
        _says(call(**{name: bad}), '%s has a negative stride' % name)
    if output:
        for bad in (_view(b=0), _view(t=0), _view(h=0), _view(h=8), _view(b=256), _view(t=16)):
            _says(call(**{name: bad}), '%s holds an element twice' % name)


def test_abi_layer_norm_and_lists():
    lib = _lib.load()
    f = lambda x=P, xl=8, rows=4, cols=8, t=0, eps=1e-5, y=P, yl=8: lib.ctr_layer_norm_fwd(x, xl, rows, cols, t, None, None, eps, y, yl, None, None, None)
    missing = 'layer_norm_fwd: missing x / y or a leading dimension below cols'
    for kw, text in ((dict(rows=-1), 'rows -1'), (dict(cols=0), 'cols 0'), (dict(t=7), 'unknown dtype 7'), (dict(eps=-1.0), 'eps'),
                     (dict(eps=math.nan), 'eps'), (dict(x=None), missing), (dict(y=None), missing), (dict(xl=7), missing),
                     (dict(yl=7), missing)):
        _says(f(**kw), text)
    b = lambda dy=P, gl=8, x=P, xl=8, m=P, r=P, rows=4, cols=8, t=0, dx=P, dl=8: lib.ctr_layer_norm_bwd(dy, gl, x, xl, m, r, rows, cols, t, None, dx, dl, 0, None, None, None, 0, None)
    missing = 'layer_norm_bwd: missing tensor or a leading dimension below cols'
    for kw, text in ((dict(rows=-1), 'rows -1'), (dict(cols=0), 'cols 0'), (dict(t=7), 'unknown dtype 7')) + tuple(
            (kw, missing) for kw in (dict(dy=None), dict(x=None), dict(m=None), dict(r=None), dict(dx=None), dict(gl=7), dict(xl=7), dict(dl=7))):
        _says(b(**kw), text)
    ptr, cnt, typ = (C.c_void_p * 2)(P, P), (C.c_int64 * 2)(5, 6), (C.c_int * 2)(0, 1)
    need = lib.ctr_grad_norm_workspace_bytes(2)
    norm = lambda p=ptr, c=cnt, t=typ, n=2, out=P: lib.ctr_grad_norm(p, c, t, n, out, P, need, None)
    for kw, text in ((dict(p=None), '2 tensors without their lists'), (dict(c=None), '2 tensors without their lists'),
                     (dict(t=None), '2 tensors without their lists'), (dict(n=-1), '-1 tensors'),
                     (dict(c=(C.c_int64 * 2)(5, -1)), 'tensor 1 has -1 elements'),
                     (dict(c=(C.c_int64 * 2)(1 << 43, 5)), 'tensor 0 has 8796093022208 elements'),
                     (dict(t=(C.c_int * 2)(0, 9)), 'tensor 1 has unknown dtype 9'),
                     (dict(p=(C.c_void_p * 2)(P, None)), 'tensor 1 is NULL'), (dict(out=None), 'norm_out is NULL')):
        _says(norm(**kw), text)
    clip = lambda o=ptr, m=1.0: lib.ctr_clip_grads(ptr, o, cnt, typ, 2, m, None, P, need, None)
    for m in (0.0, -1.0, math.nan, math.inf):
        _says(clip(m=m), 'max_norm must be positive and finite')
    _says(clip(o=None), 'out_host is NULL')
    _says(clip(o=(C.c_void_p * 2)(P, None)), 'output 1 is NULL')
