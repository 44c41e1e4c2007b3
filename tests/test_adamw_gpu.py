"""AdamW over many tensors on the GPU: bit for bit against the same 32-bit
operations in numpy (tests/policy_ref.py; every operation of both is correctly
rounded, so equality is the tolerance), against the formulas in 64 bits, and
the properties of the 8-bit states.

Against 64 bits: a step makes about ten roundings of relative 2^-24 in the
update and two in the weight, so after s steps the weights are within
s (16 lr + 2 |p|) 2^-24 of it.  With clipping, the norm may round to a
neighbour of the 64-bit one: 2^-23 relative on every gradient, the same bound
with a few more roundings."""
import numpy as np
import pytest
import torch

import graphzero_b200 as gz
import policy_ref as ref

pytestmark = pytest.mark.gpu
U = 2.0**-24
SHAPES = [(4, 256), (256,), (2, 256), (1,), (255,), (257,), (33, 67), (4096,), (1000, 3), (0,), (7,)]


def make(shapes, seed=1, offset=0):
    """Weights as slices of one buffer, `offset` elements off its start."""
    g = torch.Generator().manual_seed(seed)
    flat = torch.randn(sum(int(np.prod(s)) for s in shapes) + offset, generator=g).cuda() * 0.05
    out, at = [], offset
    for s in shapes:
        n = int(np.prod(s))
        out.append(flat[at:at + n].view(s))
        at += n
    return out


def gradients(shapes, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * torch.exp(torch.randn(s, generator=g))).mul(1e-3).to(dtype).cuda() for s in shapes]


def same_state(opt, r, bits):
    for k, (p, at) in enumerate(zip(opt.params, opt.offsets)):
        n = p.numel()
        np.testing.assert_array_equal(p.cpu().numpy().reshape(-1), r.p[k], err_msg=str(k))
        pad = r.m[k].size
        np.testing.assert_array_equal(opt.m[at:at + pad].float().cpu().numpy()[:n], r.m[k][:n], err_msg=str(k))
        np.testing.assert_array_equal(opt.v[at:at + pad].float().cpu().numpy()[:n], r.v[k][:n], err_msg=str(k))
        if bits == 8:
            np.testing.assert_array_equal(opt.m_scale[at // 256:(at + pad) // 256].cpu().numpy(), r.ms[k])
            np.testing.assert_array_equal(opt.v_scale[at // 256:(at + pad) // 256].cpu().numpy(), r.vs[k])


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 2])
def test_steps_bit_for_bit(cuda, bits, dtype, offset):
    params = make(SHAPES, offset=offset)
    copies = [torch.zeros(p.shape, dtype=torch.bfloat16 if k % 2 else torch.float16, device="cuda") for k, p in enumerate(params)]
    decays, scales = [0.01 * (k % 3) for k in range(len(SHAPES))], [1.0 + 0.5 * (k % 2) for k in range(len(SHAPES))]
    opt = gz.AdamW(params, lr=3e-3, betas=(0.8, 0.99), eps=1e-7, weight_decay=decays, lr_scale=scales, state_bits=bits,
                   copies=copies, seed=5)
    r = ref.AdamW([p.cpu().numpy() for p in params], bits, 3e-3, (0.8, 0.99), 1e-7, decays, scales, 0.0, 5)
    for t in range(4):
        gs = gradients(SHAPES, 100 + t, dtype)
        opt.step(gs, grad_scale=0.75)
        r.step([g.float().cpu().numpy() for g in gs], grad_scale=0.75)
    same_state(opt, r, bits)
    for p, c in zip(params, copies):
        assert torch.equal(c, p.to(c.dtype))


@pytest.mark.parametrize("bits", [8, 32])
def test_gradients_at_any_alignment(cuda, bits):
    for dtype in (torch.float32, torch.bfloat16):
        got = []
        for off in (0, 1, 3):
            params, flat = make([(3000,)]), torch.zeros(3010, dtype=dtype, device="cuda")
            g = flat[off:off + 3000]
            g.copy_(gradients([(3000,)], 9, dtype)[0])
            opt = gz.AdamW(params, state_bits=bits)
            opt.step([g])
            got.append((params[0].clone(), opt.m.float()))
        assert all(torch.equal(a, b) for x in got[1:] for a, b in zip(x, got[0]))


def test_against_64_bits(cuda):
    params = make(SHAPES)
    p = [x.double().cpu() for x in params]
    m, v = [torch.zeros_like(x) for x in p], [torch.zeros_like(x) for x in p]
    opt = gz.AdamW(params, lr=1e-3, weight_decay=0.1, max_norm=0.05)
    for t in range(1, 6):
        gs = gradients(SHAPES, 200 + t)
        norm = opt.step(gs)
        g64 = [g.double().cpu() for g in gs]
        want = float(torch.sqrt(sum((g * g).sum() for g in g64)))
        assert abs(float(norm) - want) <= 2 * U * want
        coef = min(1.0, 0.05 / (want + 1e-6))
        for k, g in enumerate(g64):
            g = g * coef
            m[k], v[k] = 0.9 * m[k] + 0.1 * g, 0.999 * v[k] + 0.001 * g * g
            p[k] = p[k] * (1 - 1e-3 * 0.1) - 1e-3 * (m[k] / (1 - 0.9**t)) / ((v[k] / (1 - 0.999**t)).sqrt() + 1e-8)
    for a, b in zip(params, p):
        assert ((a.double().cpu() - b).abs() <= 5 * (40 * 1e-3 + 2 * b.abs()) * U).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_clipping_and_norm(cuda, bits):
    shapes = [(300, 300), (777,), (5,)]
    params = make(shapes)
    opt = gz.AdamW(params, state_bits=bits, max_norm=1.0, seed=3)
    r = ref.AdamW([p.cpu().numpy() for p in params], bits, 1e-3, (0.9, 0.999), 1e-8, [0.01] * 3, [1.0] * 3, 1.0, 3)
    for t, size in enumerate((1.0, 1e4)):  # the first below the limit: not scaled up
        gs = [g * size for g in gradients(shapes, 300 + t)]
        norm = opt.step(gs)
        want = np.sqrt(sum(float((g.double() ** 2).sum()) for g in gs))
        assert abs(float(norm) - want) <= 2 * U * want
        f = np.float32
        r.step([g.cpu().numpy() for g in gs], coef=min(f(1.0) / (f(norm.item()) + f(1e-6)), f(1)))
    same_state(opt, r, bits)


def test_norm_is_reproducible(cuda):
    got = set()
    for _ in range(5):
        opt = gz.AdamW(make([(1000, 1000), (3,)]), max_norm=1.0)
        got.add(float(opt.step(gradients([(1000, 1000), (3,)], 4))))
    assert len(got) == 1


@pytest.mark.parametrize("bits", [8, 32])
def test_more_tensors_than_one_launch_takes(cuda, bits):
    shapes = [(k % 37 + 1, 11) for k in range(1000)]
    params = make(shapes)
    opt = gz.AdamW(params, state_bits=bits, max_norm=0.3, seed=1)
    r = ref.AdamW([p.cpu().numpy() for p in params], bits, 1e-3, (0.9, 0.999), 1e-8, [0.01] * 1000, [1.0] * 1000, 0.3, 1)
    gs = gradients(shapes, 7)
    gs[3] = gs[500] = gs[999] = None
    norm = opt.step(gs)
    want = np.sqrt(sum(float((g.double() ** 2).sum()) for g in gs if g is not None))
    assert abs(float(norm) - want) <= 2 * U * want
    f = np.float32
    r.step([None if g is None else g.cpu().numpy() for g in gs], coef=min(f(0.3) / (f(norm.item()) + f(1e-6)), f(1)))
    same_state(opt, r, bits)


def test_missing_gradients_leave_everything(cuda):
    params = make([(100,), (50,)])
    opt = gz.AdamW(params)
    before = [p.clone() for p in params]
    opt.step([None, gradients([(50,)], 1)[0]])
    assert torch.equal(params[0], before[0]) and not torch.equal(params[1], before[1])
    assert (opt.m[:256] == 0).all()
    params[0].grad, params[1].grad = torch.ones(100, device="cuda"), None
    opt.step()
    assert not torch.equal(params[0], before[0])
    opt.max_norm = 1.0
    assert float(opt.step([None, None])) == 0


@pytest.mark.parametrize("bits", [8, 32])
def test_bad_gradients_stay_where_they_are(cuda, bits):
    """A NaN or infinity spoils its own weight, not its block."""
    params = make([(512,)])
    clean = make([(512,)])
    opt, other = gz.AdamW(params, state_bits=bits), gz.AdamW(clean, state_bits=bits)
    g = gradients([(512,)], 1)
    h = g[0].clone()
    h[3], h[200] = float("nan"), float("inf")
    opt.step([h])
    other.step(g)
    spoilt = torch.zeros(512, dtype=torch.bool, device="cuda")
    spoilt[[3, 200]] = True
    assert params[0][spoilt].isnan().all() and params[0][~spoilt].isfinite().all()
    assert torch.equal(params[0][~spoilt], clean[0][~spoilt])
    assert opt.m[:512].float()[~spoilt].isfinite().all() and opt.v[:512].float()[~spoilt].isfinite().all()
    if bits == 8:
        assert opt.m_scale.isfinite().all() and opt.v_scale.isfinite().all()


def test_8bit_blocks_of_every_magnitude(cuda):
    """Blocks from 1e-30 to 1e18 and of zeros: the largest of a block lies in
    (224, 448] of its scale, a root never becomes zero, zeros stay zero."""
    n = 256 * 40
    params = make([(n,)])
    opt = gz.AdamW(params, state_bits=8)
    r = ref.AdamW([params[0].cpu().numpy()], 8, 1e-3, (0.9, 0.999), 1e-8, [0.01], [1.0], 0.0, 0)
    g = gradients([(n,)], 3)[0] * torch.logspace(-27, 20, 40, device="cuda").repeat_interleave(256)
    g[256:512] = 0
    g[512:768] = 0
    g[600] = 1e-12
    opt.step([g])
    with np.errstate(under="ignore"):
        r.step([g.cpu().numpy()])
    same_state(opt, r, 8)
    m, v = opt.m.float().view(-1, 256), opt.v.float().view(-1, 256)
    big = torch.ones(40, dtype=torch.bool)
    big[1] = False
    assert (m[1] == 0).all() and (v[1] == 0).all()
    assert (m.abs().amax(1)[big] <= 448).all() and (m.abs().amax(1)[big] >= 208).all()
    roots = g.view(-1, 256)
    assert ((v > 0) | ((0.001 * roots.double() ** 2).sqrt() < 1e-22)).all()


def test_8bit_rounding_is_unbiased(cuda):
    """The mean over 2^18 weights of the rounded first moment is the exact
    one's within 5 standard deviations (a grain is at most 1/8 of the value)."""
    n = 1 << 18
    params = make([(n,)])
    opt = gz.AdamW(params, state_bits=8, seed=11)
    g = torch.full((n,), 0.0123, device="cuda")
    g[::256] = 0.05  # sets the scale
    opt.step([g])
    m = (opt.m.float().view(-1, 256) * opt.m_scale[:, None])[:, 1:].double()
    assert m.unique().numel() == 2
    exact = float(np.float32(0.0123) * np.float32(0.1))
    assert abs(float(m.mean()) - exact) <= 5 * float(m.std()) / np.sqrt(m.numel())


def test_8bit_states_follow_small_changes(cuda):
    """Without gradients the root of v falls by sqrt(beta2) a step, far below
    a grain: the mean over the weights follows within 3 %, and m vanishes."""
    n = 256 * 64
    params = make([(n,)])
    opt = gz.AdamW(params, state_bits=8, lr=0.0)
    opt.step([torch.ones(n, device="cuda")])
    first = (opt.v.float().view(-1, 256) * opt.v_scale[:, None]).double().mean()
    zero = torch.zeros(n, device="cuda")
    for _ in range(400):
        opt.step([zero])
    now = (opt.v.float().view(-1, 256) * opt.v_scale[:, None]).double().mean()
    assert abs(float(now / first) / 0.999**200 - 1) < 0.03
    assert float((opt.m.float().view(-1, 256) * opt.m_scale[:, None]).abs().max()) < 1e-6


def test_8bit_states_train_like_32bit_ones(cuda):
    """A regression's loss with 8-bit states stays within a factor of 2 of that
    with 32-bit states while both fall (the update's noise, one grain of m and
    of the root, is at most 1/8 of a step and unbiased)."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = torch.randn(4096, 64, device="cuda", generator=g), torch.randn(64, 8, device="cuda", generator=g)
    losses = {}
    for bits in (8, 32):
        p = torch.zeros(64, 8, device="cuda")
        opt = gz.AdamW([p], lr=0.005, weight_decay=0.0, state_bits=bits)
        losses[bits] = []
        for _ in range(100):
            r = x @ (p - w)
            losses[bits].append(float((r * r).mean()))
            opt.step([x.t() @ r / 4096])
    for a, b in zip(losses[8], losses[32]):
        assert b / 2 <= a <= b * 2
    assert losses[8][-1] < losses[8][0] and losses[32][-1] < losses[32][0]


def test_streams_and_graphs(cuda):
    shapes = [(500, 20), (33,)]
    a, b, gs = make(shapes), make(shapes), gradients(shapes, 5)
    x, y = gz.AdamW(a, state_bits=8, max_norm=0.01), gz.AdamW(b, state_bits=8, max_norm=0.01)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x.step(gs)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y.step(gs)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(x.m.float(), y.m.float())


def test_refusals(cuda):
    p = torch.zeros(4, 4, device="cuda")
    for call in (lambda: gz.AdamW([]), lambda: gz.AdamW([p.cpu()]), lambda: gz.AdamW([p.half()]), lambda: gz.AdamW([p.t()[:2].t()]),
                 lambda: gz.AdamW([p], state_bits=16), lambda: gz.AdamW([p], copies=[p]),
                 lambda: gz.AdamW([p], copies=[torch.zeros(4, device="cuda").half()]), lambda: gz.AdamW([p], weight_decay=[0.1, 0.2]),
                 lambda: gz.AdamW([p]).step([p.double()]), lambda: gz.AdamW([p]).step([p[0]]), lambda: gz.AdamW([p]).step([p, p]),
                 lambda: gz.AdamW([p]).step([p.cpu()])):
        with pytest.raises(ValueError):
            call()
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(max_norm=-1.0), dict(lr=float("nan"))):
        opt = gz.AdamW([p], **kw)
        with pytest.raises(gz.GZError) as e:
            opt.step([p])
        assert e.value.status == gz.ERR_INVALID_ARG and opt.steps == 0
    for kw in (dict(weight_decay=-0.1), dict(lr_scale=float("inf"))):
        with pytest.raises(gz.GZError):
            gz.AdamW([p], **kw)
