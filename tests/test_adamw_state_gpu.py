"""AdamW: its states' types, gradients and norms that are not finite, captures
replayed, and tensors that have moved."""
import gc

import numpy as np
import pytest
import torch

import graphzero_b200 as gz
from test_adamw_gpu import U, gradients, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("default", [torch.bfloat16, torch.float16, torch.float64])
def test_states_do_not_follow_the_default_type(cuda, bits, default):
    """States, scales and norm are 32-bit floats (or the 8-bit ones) whatever type torch gives new tensors."""
    shapes = [(300, 3), (17,)]
    a, b, gs = make(shapes), make(shapes), gradients(shapes, 1)
    want = gz.AdamW(a, state_bits=bits, max_norm=0.01)
    torch.set_default_dtype(default)
    try:
        got = gz.AdamW(b, state_bits=bits, max_norm=0.01)
        for k in ("m", "v", "m_scale", "v_scale"):
            t, u = getattr(got, k), getattr(want, k)
            assert (t is None and u is None) or (t.dtype == u.dtype and t.shape == u.shape)
        norm = got.step(gs)
    finally:
        torch.set_default_dtype(torch.float32)
    assert norm.dtype == torch.float32 and torch.equal(norm, want.step(gs))
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(want.m.float(), got.m.float())


@pytest.mark.parametrize("bits", [8, 32])
def test_tensors_that_have_moved_are_refused(cuda, bits):
    """A plan holds its tensors' addresses: a step after one got other memory
    raises and changes nothing (the old memory is kept here throughout)."""
    shapes = [(300, 3), (17,)]
    gs = gradients(shapes, 1)

    def moved(take, put):
        params = make(shapes)
        copies = [p.to(torch.bfloat16) for p in params]
        opt = gz.AdamW(params, state_bits=bits, copies=copies)
        opt.step(gs)
        t = take(opt, params, copies)
        old = t.data
        kept = old.float().clone()
        put(t)
        with pytest.raises(ValueError, match="moved"):
            opt.step(gs)
        assert opt.steps == 1 and torch.equal(old.float(), kept)
        t.data = old  # back again
        opt.step(gs)
        assert opt.steps == 2

    other = lambda t: setattr(t, "data", t.data.clone())  # noqa: E731
    moved(lambda o, p, c: p[1], other)
    moved(lambda o, p, c: p[0], other)
    moved(lambda o, p, c: c[1], other)
    moved(lambda o, p, c: o.m, other)
    moved(lambda o, p, c: o.v, other)
    moved(lambda o, p, c: p[1], lambda t: t.set_(t.clone()))
    if bits == 8:
        moved(lambda o, p, c: o.m_scale, other)
        moved(lambda o, p, c: o.v_scale, other)


@pytest.mark.parametrize("bits", [8, 32])
def test_states_are_restored_in_place(cuda, bits):
    shapes = [(300, 3), (17,)]
    a, gs = make(shapes), gradients(shapes, 1)
    opt = gz.AdamW(a, state_bits=bits)
    opt.step(gs)
    saved = {k: getattr(opt, k).clone() for k in ("m", "v", "m_scale", "v_scale") if getattr(opt, k) is not None}
    weights = [p.clone() for p in a]
    opt.step(gs)
    for k, t in saved.items():
        with pytest.raises(AttributeError):
            setattr(opt, k, t)
    again = gz.AdamW(weights, state_bits=bits)
    for k, t in saved.items():
        getattr(again, k).copy_(t)
    again.steps = 1
    again.step(gs)
    assert all(torch.equal(p, q) for p, q in zip(a, weights)) and torch.equal(opt.m.float(), again.m.float())
    with pytest.raises(AttributeError):
        opt.params = weights
    with pytest.raises(TypeError):
        opt.params[0] = weights[0]


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("many", [False, True])
def test_clipping_by_a_norm_that_is_not_finite(cuda, bits, many):
    """A NaN among the gradients makes every clipped gradient, and so every
    weight that has one, NaN; an infinity alone scales the finite ones to 0
    (and itself to NaN)."""
    shapes = [(300, 3), (17,), (256,)] + [(5,)] * (900 if many else 0)
    gs = gradients(shapes, 1)
    gs[2] = None
    gs[1][4] = float("nan")
    params = make(shapes)
    before = params[2].clone()
    norm = gz.AdamW(params, state_bits=bits, max_norm=1.0).step(gs)
    assert norm.isnan()
    assert all(p.isnan().all() for k, p in enumerate(params) if k != 2) and torch.equal(params[2], before)

    gs[1][4] = float("inf")
    params, still = make(shapes), make(shapes)
    norm = gz.AdamW(params, state_bits=bits, max_norm=1.0).step(gs)
    assert float(norm) == float("inf")
    gz.AdamW(still, state_bits=bits).step([None if g is None else torch.zeros_like(g) for g in gs])
    assert params[1][4].isnan()
    params[1][4] = still[1][4]
    assert all(torch.equal(p, q) for p, q in zip(params, still))


@pytest.mark.parametrize("bits", [8, 32])
def test_an_infinite_limit_only_measures_the_norm(cuda, bits):
    shapes = [(300, 3), (17,)]
    gs = gradients(shapes, 1)
    for bad in (None, float("inf")):
        if bad:
            gs[1][4] = bad
        a, b = make(shapes), make(shapes)
        norm = gz.AdamW(a, state_bits=bits, max_norm=float("inf")).step(gs)
        gz.AdamW(b, state_bits=bits).step(gs)
        want = float(torch.sqrt(sum((g.double() ** 2).sum() for g in gs)))
        assert float(norm) == want if bad else abs(float(norm) - want) <= 2 * U * want
        for p, q in zip(a, b):
            np.testing.assert_array_equal(p.cpu().numpy(), q.cpu().numpy())


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("max_norm", [0.0, 0.01])
def test_replays_of_a_capture_are_steps(cuda, bits, max_norm):
    """Calls, replays and calls again are the same steps as as many calls: bias
    corrections, rounding numbers and the count go on from wherever they are."""
    shapes = [(500, 20), (33,)]
    a, b = make(shapes), make(shapes)
    kw = dict(state_bits=bits, max_norm=max_norm, lr=1e-2, betas=(0.8, 0.95), seed=3)
    x, y = gz.AdamW(a, **kw), gz.AdamW(b, **kw)
    gs = gradients(shapes, 0)

    def new_gradients(t):
        for g, h in zip(gs, gradients(shapes, 10 + t)):
            g.copy_(h)

    t = 0
    for _ in range(2):
        new_gradients(t)
        x.step(gs), y.step(gs)
        t += 1
    assert x.steps == y.steps == 2
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = y.step(gs)
    assert y.steps == 2  # a capture is not a step
    for _ in range(4):
        new_gradients(t)
        n = x.step(gs)
        graph.replay()
        t += 1
        assert norm is None or torch.equal(n, norm)
    assert x.steps == y.steps == t == 6
    for _ in range(2):
        new_gradients(t)
        x.step(gs), y.step(gs)
        t += 1
    new_gradients(t)
    x.step(gs)
    graph.replay()
    assert x.steps == y.steps == 9
    # restored to another place
    x.steps = y.steps = 100
    new_gradients(t)
    x.step(gs)
    graph.replay()
    assert x.steps == y.steps == 101
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert torch.equal(x.m.float(), y.m.float()) and torch.equal(x.v.float(), y.v.float())


def test_a_restored_count_is_where_a_capture_starts(cuda):
    a, b = make([(700,)]), make([(700,)])
    x, y = gz.AdamW(a, state_bits=8), gz.AdamW(b, state_bits=8)
    gs = gradients([(700,)], 2)
    x.steps = y.steps = 40
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y.step(gs)
    for _ in range(3):
        x.step(gs)
        graph.replay()
    assert x.steps == y.steps == 43
    assert torch.equal(a[0], b[0]) and torch.equal(x.v.float(), y.v.float())


def test_capture_of_a_plan_in_several_launches(cuda):
    shapes = [(k % 37 + 1, 11) for k in range(1000)] + [(0,)]
    a, b, gs = make(shapes), make(shapes), gradients(shapes, 7)
    gs[999] = gs[0] = None
    x, y = gz.AdamW(a, state_bits=8, max_norm=0.3), gz.AdamW(b, state_bits=8, max_norm=0.3)
    x.step(gs), y.step(gs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y.step(gs)
    for _ in range(3):
        x.step(gs)
        graph.replay()
    assert x.steps == y.steps == 4
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_steps_of_a_plan_without_gradients_count(cuda):
    p = make([(9,)])
    opt = gz.AdamW(p)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step([None])
    graph.replay()
    graph.replay()
    assert opt.steps == 2
    opt.step([None])
    assert opt.steps == 3
    for bad in (-1, 2**63):
        with pytest.raises((ValueError, gz.GZError)):
            opt.steps = bad
    assert opt.steps == 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-38, 1e-30, 1e-22, 1e-15, 1e15, 1e19, 1e22, 1e30, 1e34])
def test_norm_over_the_range_of_the_gradients(cuda, size, dtype):
    """Squares that 32 bits do not hold count too, in whole blocks and ragged ends.
    The sum is taken in 64 bits and rounded once; a norm below 2^-126 to a
    multiple of 2^-149."""
    shapes = [(4, 256), (301,)]
    gs = [(g / 1e-3 * size).to(dtype) for g in gradients(shapes, 3)]
    params = make(shapes)
    norm = gz.AdamW(params, max_norm=1.0).step(gs)
    want = float(torch.sqrt(sum((g.double() ** 2).sum() for g in gs)))
    assert abs(float(norm) - want) <= 2 * U * want + 2.0**-149
    assert all(p.isfinite().all() for p in params)


def test_a_captured_plan_outlives_its_object(cuda, monkeypatch):
    """A graph's replays read the plan: collecting the AdamW must not free it (close() does)."""
    freed = []
    destroy = gz._lib.gz_adamw_destroy
    monkeypatch.setattr(gz._lib, "gz_adamw_destroy", lambda plan: freed.append(plan.value) or destroy(plan))
    for capture in (False, True):
        params, gs = make([(300,)]), gradients([(300,)], 1)
        opt = gz.AdamW(params)
        if capture:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step(gs)
            del graph
        else:
            opt.step(gs)
        plan = opt._plan.value
        del opt
        gc.collect()
        assert (plan in freed) == (not capture)
    destroy(plan)  # (nothing uses it any more here)
    opt = gz.AdamW(params)
    plan = opt._plan.value
    opt.close()
    assert freed[-1] == plan


def test_steps_take_any_whole_number(cuda):
    opt = gz.AdamW(make([(9,)]))
    for n in (3, np.int64(4), torch.tensor(5)):
        opt.steps = n
        assert opt.steps == int(n) and type(opt.steps) is int
    with pytest.raises(TypeError):
        opt.steps = 2.5
    assert opt.steps == 5
