"""Refusals of the policy entry points, which come before any GPU call."""
import ctypes as C

import pytest

import graphzero_b200 as gz

L = gz._lib
X = 0x1000  # an address that nothing follows


def rows(**kw):
    return gz.PolicyRows(**(dict(logits=X, mask=None, logits_stride=7, mask_stride=0, rows=2, actions=7, dtype=gz.F32) | kw))


BAD_ROWS = [dict(rows=-1), dict(rows=2**31), dict(actions=0), dict(actions=gz.POLICY_MAX_ACTIONS + 1), dict(dtype=3),
            dict(dtype=-1), dict(logits_stride=-7), dict(mask_stride=-1), dict(logits=None)]


@pytest.mark.parametrize("kw", BAD_ROWS, ids=str)
def test_rows(kw):
    cfg, r = gz.SampleConfig(1.0, 1.0, 0.0, 0), rows(**kw)
    assert L.gz_policy_sample(C.byref(r), C.byref(cfg), None, 0, X, X, None) == gz.ERR_INVALID_ARG
    assert L.gz_policy_loss(C.byref(r), X, 7, None, None, 1.0, X, X, 7, None) == gz.ERR_INVALID_ARG
    assert L.gz_last_error()


@pytest.mark.parametrize("cfg", [(-1.0, 1.0, 0.0, 0), (float("nan"), 1.0, 0.0, 0), (1.0, 1.1, 0.0, 0), (1.0, -0.1, 0.0, 0),
                                 (1.0, float("nan"), 0.0, 0), (1.0, 1.0, -0.5, 0), (1.0, 1.0, 1.5, 0), (1.0, 1.0, 0.0, -1)])
def test_sample_settings(cfg):
    r, c = rows(), gz.SampleConfig(*cfg)
    assert L.gz_policy_sample(C.byref(r), C.byref(c), None, 0, X, X, None) == gz.ERR_INVALID_ARG


def test_other_arguments():
    r, c = rows(), gz.SampleConfig(1.0, 1.0, 0.0, 0)
    assert L.gz_policy_sample(None, C.byref(c), None, 0, X, X, None) == gz.ERR_INVALID_ARG
    assert L.gz_policy_sample(C.byref(r), None, None, 0, X, X, None) == gz.ERR_INVALID_ARG
    assert L.gz_policy_sample(C.byref(r), C.byref(c), X, -7, X, X, None) == gz.ERR_INVALID_ARG
    assert L.gz_policy_sample(C.byref(r), C.byref(c), None, 0, None, X, None) == gz.ERR_INVALID_ARG
    for target, label, loss, gstride in ((None, None, X, 7), (X, X, X, 7), (X, None, None, 7), (X, None, X, 6), (X, None, X, -7)):
        assert L.gz_policy_loss(C.byref(r), target, 7, label, None, 1.0, loss, X, gstride, None) == gz.ERR_INVALID_ARG
    # no rows: nothing to do, on a machine without a GPU too
    r = rows(rows=0, logits=None)
    assert L.gz_policy_sample(C.byref(r), C.byref(c), None, 0, None, None, None) == gz.OK
    assert L.gz_policy_loss(C.byref(r), None, 0, None, None, 1.0, None, None, 0, None) == gz.OK


def tensor(**kw):
    return gz.AdamWTensor(**(dict(param=X, copy=None, m=X, v=X, m_scale=X, v_scale=X, n=8, weight_decay=0.0, lr_scale=1.0,
                                  copy_dtype=0) | kw))


@pytest.mark.parametrize("kw,bits", [(dict(n=-1), 32), (dict(n=2**62), 32), (dict(param=None), 32), (dict(m=None), 32),
                                     (dict(v=None), 32), (dict(weight_decay=-1.0), 32), (dict(lr_scale=float("nan")), 32),
                                     (dict(copy=X, copy_dtype=gz.F32), 32), (dict(m_scale=None), 8), (dict(m=X + 8), 8),
                                     (dict(), 16)], ids=str)
def test_adamw_tensors(kw, bits):
    t, h = (gz.AdamWTensor * 1)(tensor(**kw)), C.c_void_p()
    assert L.gz_adamw_create(t, 1, bits, 0, C.byref(h)) == gz.ERR_INVALID_ARG
    assert not h


def test_adamw_other_arguments():
    h = C.c_void_p()
    assert L.gz_adamw_create(None, 1, 32, 0, C.byref(h)) == gz.ERR_INVALID_ARG
    assert L.gz_adamw_create((gz.AdamWTensor * 1)(tensor()), -1, 32, 0, C.byref(h)) == gz.ERR_INVALID_ARG
    assert L.gz_adamw_create((gz.AdamWTensor * 1)(tensor()), 1, 32, 0, None) == gz.ERR_INVALID_ARG
    cfg = gz.AdamWConfig(1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, 1, 0)
    assert L.gz_adamw_step(None, None, None, C.byref(cfg), None, None) == gz.ERR_INVALID_ARG
    assert L.gz_adamw_destroy(None) == gz.OK
