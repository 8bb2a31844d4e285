"""DIN with args.clip_norm: a step's gradients scaled as tf.clip_by_global_norm scales them (dense variables, and the
slices of the item, category and bias lookups), eager and replayed."""
import math

import numpy as np
import pytest
import torch

from oracle import ctr_oracle as O

pytestmark = pytest.mark.gpu
B, T, H, ITEMS, CATES = 24, 13, 32, 50, 7


def _model(sess, clip_norm, P, cate_list):
    import recommendation_amd as ra
    ra.enable_zoo_imports()
    from DIN import DIN
    cfg = O.default_cfg('DIN')
    cfg.hidden_units, cfg.clip_norm = H, clip_norm
    m = DIN.DIN(cfg, 5, ITEMS, CATES, cate_list)
    m.initialize(sess, params=P)
    return m


def _case(seed=0):
    rng = np.random.default_rng(seed)
    cate_list = rng.integers(0, CATES, ITEMS)
    cfg = O.default_cfg('DIN')
    cfg.hidden_units = H
    P = O.din_init_params(cfg, 5, ITEMS, CATES, seed=seed + 1)
    for k in P:
        if k.endswith('bias') or k.endswith('beta') or 'alphadice' in k or k.endswith('item_b'):
            P[k] = rng.standard_normal(P[k].shape) * 0.2
    sl = rng.integers(1, T + 1, B)
    hist = rng.integers(0, ITEMS, (B, T)) * (np.arange(T) < sl[:, None])
    uij = (np.zeros(B, dtype=np.int64), rng.integers(0, ITEMS, B), rng.integers(0, 2, B), hist, sl)
    return P, cate_list, uij


@pytest.mark.parametrize('share', [0.1, 0.9, 10.0])
def test_a_clipped_step_is_a_shorter_step(sess, share):
    """SGD is linear in the gradient: every variable moves by bound / norm of the unclipped step's way, or all of it."""
    P, cate_list, uij = _case()
    free = _model(sess, None, P, cate_list)
    before = free.get_params()
    free.train(sess, uij, 0.5)
    b = free._bufs[(B, T)]
    norm = math.sqrt(sum(float(t.double().square().sum()) for t in (free.dense.grad, b['demb'], b['dlogit'])))
    orc = O.OracleDIN(_cfg(), cate_list, P, dtype=torch.float64)
    _, g, _ = orc.loss_and_grads(uij)
    dense = math.sqrt(sum(float(v.square().sum()) for k, v in g.items() if k in free.dense_shapes))
    got = math.sqrt(float(free.dense.grad.double().square().sum()))
    assert abs(got - dense) <= 1e-5 * dense
    m = _model(sess, share * norm, P, cate_list)
    m.train(sess, uij, 0.5)
    assert abs(float(m.grad_norm) - norm) <= 1e-5 * norm
    by = min(1.0, share)
    moved, want = m.get_params(), free.get_params()
    for k in want:
        way = want[k].astype(np.float64) - before[k]
        # each of the two updates rounds the parameter once, the factor and the product twice
        off = 2.0 ** -23 * np.abs(before[k]) + 2.0 ** -22 * np.abs(way) + 2.0 ** -22 * by * 1e-5
        assert (np.abs(moved[k] - before[k] - by * way) <= 2 * off + 1e-5 * np.abs(way)).all(), k


def _cfg():
    cfg = O.default_cfg('DIN')
    cfg.hidden_units = H
    return cfg


def test_replayed_equals_eager(sess):
    P, cate_list, uij = _case(3)
    models = [_model(sess, 0.05, P, cate_list) for _ in range(2)]
    for rep in range(4):
        _, _, other = _case(10 + rep)
        args = [m._dev_i32(other[1]) for m in models[:1]] + [torch.as_tensor(other[2].astype(np.float32)).to(sess.device),
                                                            models[0]._dev_i32(other[3]), models[0]._dev_i32(other[4])]
        models[0].train_step(*args, 0.3)
        models[1].train_step_graphed(*args, 0.3)
        torch.cuda.synchronize()
        assert float(models[0].grad_norm) == float(models[1].grad_norm) > 0.05
        a, b = (m.get_params() for m in models)
        for k in a:
            assert np.array_equal(a[k], b[k]), (rep, k)
    for m in models:
        m.close()


@pytest.mark.parametrize('bad', [0.0, -1.0, math.inf, math.nan])
def test_bad_bounds(sess, bad):
    P, cate_list, _ = _case()
    with pytest.raises(ValueError, match='clip_norm'):
        _model(sess, bad, P, cate_list)
