"""Drawing actions from policy rows and the policy loss on the GPU, against
plain restatements in 64 bits (tests/policy_ref.py).

Actions are compared exactly.  The scores that decide are 32-bit sums of two
rounded terms of a magnitude below 32, so a draw could differ from the 64-bit
one only where two scores lie within 4e-6 of each other: about one row in 1e5
of random input, and the inputs here are fixed.

Tolerances, with u = 2^-24: logp is d - log z, d a rounded difference and
quotient (2 u |d|), z an integer sum of exponentials of 2 ulp each, floored to
2^-44 (a relative 6 u + actions 2^-44), the logarithm within 2 ulp: 16 u (1 +
|logp| + |d|) covers them, with |d| <= |logp| + log(actions).  The loss sums
actions / 32 terms or fewer in a row and a tree over them: a relative (actions
/ 32 + 64) u of the terms' sizes.  The gradient's p carries z's and the
exponential's error: (actions / 32 + 64) u (1 + max |d|) of p's share, plus the
output type's rounding (half an ulp, or half its smallest number)."""
import numpy as np
import pytest
import torch

import graphzero_b200 as gz
import policy_ref as ref

pytestmark = pytest.mark.gpu
U = 2.0**-24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def rows_of(n, a, seed, dtype=torch.float32, pad=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, a + pad, generator=g) * spread).to(dtype)


def legal(n, a, share, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(n, a, generator=g) < share).to(torch.uint8)


def check_sample(x, noise, mask=None, **kw):
    """Runs policy_sample on CPU tensors' copies and compares."""
    dev = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    action, logp = gz.policy_sample(x.cuda(), None if noise is None else noise.cuda(),
                                    mask=None if mask is None else mask.cuda(), **dev)
    kw = {k: v.numpy() if isinstance(v, torch.Tensor) else np.float32(v) if isinstance(v, float) else v
          for k, v in kw.items()}
    a, lp = ref.sample(x.float().numpy(), None if mask is None else mask.numpy(),
                       None if noise is None else noise.numpy(), **kw)
    got = logp.cpu().numpy()
    np.testing.assert_array_equal(action.cpu().numpy(), a)
    fine = np.isfinite(lp)
    np.testing.assert_array_equal(np.isfinite(got), fine)
    bound = 16 * U * (1 + 2 * np.abs(lp[fine]) + np.log(x.shape[1]))
    assert (np.abs(got[fine] - lp[fine]) <= bound).all(), np.abs(got[fine] - lp[fine]).max()
    return action, logp


SIZES = [1, 2, 7, 9, 31, 32, 33, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 1000, 1024, 1025, 2047, 2049, 4672,
         8191, 8192, 8193, 12289, 16385, 20000, 32768, 32769, 50001, 65537, 100003, 131072, 262144]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("a", SIZES)
def test_sample_sizes(cuda, a, dtype):
    n = 5 if a <= 8192 else 2
    check_sample(rows_of(n, a, a, dtype), ref.gumbel((n, a), a + 1))
    check_sample(rows_of(n, a, a, dtype), ref.gumbel((n, a), a + 1), top_k=min(a, 5), top_p=0.8)


FILTERS = [dict(temperature=0.0), dict(temperature=0.3), dict(temperature=4.0), dict(top_k=1), dict(top_k=3),
           dict(top_k=100), dict(top_k=100000), dict(top_p=0.0), dict(top_p=1e-6), dict(top_p=0.5), dict(top_p=0.999),
           dict(min_p=0.3), dict(min_p=1.0), dict(temperature=1.7, top_k=40, top_p=0.7, min_p=0.01),
           dict(temperature=0.5, top_p=0.95, min_p=0.05), dict(temperature=1e-6), dict(temperature=1e30)]


@pytest.mark.parametrize("kw", FILTERS, ids=str)
@pytest.mark.parametrize("a,share", [(7, 0.7), (300, None), (4672, 0.01), (4672, None), (9001, None), (9001, 0.5),
                                     (70001, None)])
def test_sample_filters(cuda, a, share, kw):
    n = 6 if a < 70000 else 2
    x, noise = rows_of(n, a, 11 + a, torch.bfloat16 if a == 300 else torch.float32), ref.gumbel((n, a), 12 + a)
    check_sample(x, noise, None if share is None else legal(n, a, share, 13), **kw)


@pytest.mark.parametrize("spread", [0.05, 0.5, 1.5])
@pytest.mark.parametrize("a", [65, 100, 256, 500, 1100, 2048, 2049, 5000, 9001, 40000])
def test_sample_flat_rows(cuda, a, spread):
    """Kept shares from a few actions to nearly all, in lists of every length and beyond them."""
    n = 4 if a <= 9001 else 2
    for dtype in (torch.float32, torch.bfloat16):
        x, noise = rows_of(n, a, a, dtype, spread=spread), ref.gumbel((n, a), a + 2)
        for kw in (dict(top_p=0.02), dict(top_p=0.3), dict(top_p=0.9), dict(top_p=0.9, temperature=0.7), dict(top_k=a // 3),
                   dict(top_k=a - 1, top_p=0.95), dict(top_k=40, top_p=0.5), dict(top_p=0.8, min_p=0.2)):
            check_sample(x, noise, **kw)


@pytest.mark.parametrize("a", [400, 4672, 5121, 40000])
def test_sample_masks_of_every_density(cuda, a):
    """From none to all of a block's rows with more visible actions than a list holds."""
    n = 9
    x, noise = rows_of(n, a, 3, torch.float16), ref.gumbel((n, a), 4)
    share = torch.tensor([0.0, 0.001, 0.02, 0.05, 0.2, 0.5, 0.9, 1.0, 0.01])
    g = torch.Generator().manual_seed(5)
    mask = (torch.rand(n, a, generator=g) < share[:, None]).to(torch.uint8) * 255
    for kw in (dict(), dict(top_p=0.9), dict(top_k=70), dict(top_k=300, top_p=0.7, min_p=0.01), dict(temperature=0.0)):
        check_sample(x, noise, mask, **kw)


def test_sample_many_rows_per_row_settings(cuda):
    n, a = 700, 129
    g = torch.Generator().manual_seed(5)
    x, noise, mask = rows_of(n, a, 1), ref.gumbel((n, a), 2), legal(n, a, 0.4, 3)
    mask[::50] = 0
    kw = dict(temperature=torch.rand(n, generator=g) * 2, top_k=torch.randint(0, 30, (n,), generator=g, dtype=torch.int32),
              top_p=torch.rand(n, generator=g) * 1.2, min_p=torch.rand(n, generator=g) * 0.2)
    kw["temperature"][::7] = 0
    check_sample(x, noise, mask, **kw)


def test_sample_settings_out_of_range_take_the_nearest_end(cuda):
    n, a = 8, 50
    x, noise = rows_of(n, a, 1), ref.gumbel((n, a), 2)
    minus, two = torch.full((n,), -1.0), torch.full((n,), 2.0)
    none = gz.policy_sample(x.cuda(), noise.cuda())
    best = gz.policy_sample(x.cuda(), noise.cuda(), temperature=0.0)
    for kw, want in ((dict(temperature=minus), best), (dict(top_p=two), none), (dict(top_p=minus), best),
                     (dict(min_p=minus), none), (dict(min_p=two), best),
                     (dict(top_k=torch.full((n,), -3, dtype=torch.int32)), none)):
        got = gz.policy_sample(x.cuda(), noise.cuda(), **{k: v.cuda() for k, v in kw.items()})
        assert torch.equal(got[0], want[0]), kw


@pytest.mark.parametrize("a", [7, 500, 4672, 40000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_hidden_and_extreme_scores(cuda, a, dtype):
    """Whatever lies under the mask has no influence; NaN is -inf, +inf the
    largest float, the type's lowest value an ordinary score."""
    lowest = torch.finfo(dtype).min
    x = rows_of(12, a, 21, dtype)
    mask = legal(12, a, 0.5, 22)
    mask[:, 0], mask[:, 1], mask[:, 2] = 1, 0, 1
    bad = torch.tensor([float("nan"), float("inf"), float("-inf"), lowest, -lowest])
    g = torch.Generator().manual_seed(3)
    x = torch.where(mask == 0, bad[torch.randint(0, 5, x.shape, generator=g)], x.float()).to(dtype)
    x[1] = float("-inf")  # nothing visible
    x[2] = float("nan")
    x[3] = lowest  # all alike: uniform
    x[4, 2] = lowest
    x[5] = lowest
    x[5, 2] = 0
    x[6, 0] = float("nan")
    x[7, 2] = float("inf")
    x[8, 0], x[8, 2] = float("inf"), float("inf")
    x[9, 0], x[9, 2] = -lowest, lowest
    mask[10] = 0
    mask[11] = 0
    mask[11, a - 1] = 255
    noise = ref.gumbel((12, a), 23)
    noise[0, 0] = float("nan")
    for kw in (dict(), dict(temperature=0.4), dict(top_k=3), dict(top_p=0.6), dict(temperature=0.0),
               dict(top_k=a // 2 + 1, top_p=0.9, min_p=0.001)):
        check_sample(x, noise, mask, **kw)


@pytest.mark.parametrize("a", [50, 1000, 4672, 30000, 131072])
def test_sample_ties_go_to_the_lowest_index(cuda, a):
    x, noise = torch.zeros(3, a), ref.gumbel((3, a), 31)
    x[1, ::2] = -1.0
    x[2] = torch.randint(0, 3, (a,), generator=torch.Generator().manual_seed(1)).float() / 4
    for kw in (dict(top_k=10), dict(top_k=a // 2 + 3), dict(top_p=0.25), dict(top_k=a // 2, top_p=0.5), dict()):
        check_sample(x, noise, **kw)
    check_sample(x, None)
    check_sample(x, torch.zeros(3, a), top_k=7)


@pytest.mark.parametrize("a", [33, 4672, 20000])
def test_sample_strides_and_alignment(cuda, a):
    for dtype in DTYPES:
        wide = rows_of(4, a, 41, dtype, pad=3).cuda()
        noise = ref.gumbel((4, a + 5), 42).cuda()
        mask = legal(4, a + 1, 0.3, 43).cuda()
        for off in (0, 1, 2, 3):
            x, m = wide[:, off:off + a], mask[:, off % 2:off % 2 + a]
            nz = noise[:, off:off + a]
            want = gz.policy_sample(x.contiguous(), nz.contiguous(), mask=m.contiguous(), top_p=0.9)
            got = gz.policy_sample(x, nz, mask=m, top_p=0.9)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            got = gz.policy_sample(x, nz, mask=m.bool(), top_p=0.9)
            assert torch.equal(got[0], want[0])
        t = wide[:, :a].t().contiguous().t()  # rows that are not contiguous
        assert torch.equal(gz.policy_sample(t)[0], gz.policy_sample(wide[:, :a])[0])
        one = wide[:1, :a].expand(4, a)  # one row for all
        got = gz.policy_sample(one, noise[:, :a], mask=mask[:1, :a].expand(4, a))
        want = gz.policy_sample(one.contiguous(), noise[:, :a].contiguous(), mask=mask[:1, :a].repeat(4, 1))
        assert torch.equal(got[0], want[0])


@pytest.mark.parametrize("a,n", [(7, 40), (130, 300), (4672, 50), (30000, 9)])
def test_sample_row_does_not_depend_on_its_batch(cuda, a, n):
    x, noise = rows_of(n, a, 51).cuda(), ref.gumbel((n, a), 52).cuda()
    whole = gz.policy_sample(x, noise, top_p=0.9)
    for i in (0, n // 2, n - 1):
        one = gz.policy_sample(x[i:i + 1], noise[i:i + 1], top_p=0.9)
        assert torch.equal(one[0], whole[0][i:i + 1]) and torch.equal(one[1], whole[1][i:i + 1])


def test_sample_frequencies(cuda):
    """Draws follow the kept distribution: 5 standard deviations per action."""
    n = 40000
    x = torch.tensor([[0.0, 1.0, -1.0, 0.5, 2.0, -3.0, 0.1]]).cuda()
    noise = -torch.empty(n, 7, device="cuda").exponential_(generator=torch.Generator("cuda").manual_seed(6)).log()
    for kw, keep in ((dict(), 7), (dict(top_k=3), 3)):
        action, logp = gz.policy_sample(x.expand(n, 7), noise, **kw)
        p = torch.softmax(x[0].double(), 0).cpu()
        p[torch.argsort(p, descending=True)[keep:]] = 0
        p /= p.sum()
        got = torch.bincount(action.long().cpu(), minlength=7).double() / n
        assert ((got - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()
        assert (logp.double().cpu() - p.log()[action.long().cpu()]).abs().max() < 1e-5


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_step_of_shared_memory(cuda, dtype):
    """Rows whose shared memory lies on either side of what a launch gets without asking."""
    per = 4 // dtype.itemsize * 4  # actions of a 16-byte vector
    for vecs in (2500, 2900, 3000, 3072, 3500, 5900, 5980, 6050, 6144, 6300, 12200, 24576, 24577):
        a = vecs * per
        if a > gz.POLICY_MAX_ACTIONS:
            continue
        x = rows_of(2, a, vecs, dtype)
        check_sample(x, ref.gumbel((2, a), 1), top_k=3)
        n = 150  # as many rows as multiprocessors: none is split for want of rows
        y = x[:1].cuda().expand(n, a)
        loss, grad = gz.policy_loss(y, label=torch.zeros(n, dtype=torch.int32, device="cuda"))
        want, wgrad, terms = ref.loss(x[:1].float().numpy(), None, label=np.zeros(1, np.int64))
        assert (np.abs(loss.cpu().numpy() - want[0]) <= (a / 32 + 64) * U * terms[0]).all()
        assert torch.equal(grad[0], grad[-1])


def test_keywords_and_streams_by_number(cuda):
    x, noise = rows_of(3, 300, 1).cuda(), ref.gumbel((3, 300), 2).cuda()
    want = gz.policy_sample(x, noise, top_p=0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (side, side.cuda_stream):
        got = gz.policy_sample(logits=x, noise=noise, top_p=0.5, stream=stream)
        side.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        loss, _ = gz.policy_loss(logits=x.t().contiguous().t(), label=want[0], stream=stream)
        side.synchronize()
        assert torch.equal(loss, gz.policy_loss(x, label=want[0])[0])


def test_offsets_beyond_32_bits(cuda):
    """Rows further apart than 2^31 elements."""
    a, stride = 1000, 2**31 + 24
    buf = torch.empty(2 * stride + a, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(buf, (3, a), (stride, 1))
    x.copy_(rows_of(3, a, 61, torch.bfloat16))
    noise = ref.gumbel((3, a), 62).cuda()
    got, want = gz.policy_sample(x, noise, top_k=20), gz.policy_sample(x.contiguous(), noise, top_k=20)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    label = torch.arange(3, dtype=torch.int32, device="cuda")
    got, want = gz.policy_loss(x, label=label), gz.policy_loss(x.contiguous(), label=label)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_no_rows(cuda):
    action, logp = gz.policy_sample(torch.empty(0, 7, device="cuda"))
    assert action.shape == logp.shape == (0,)
    loss, grad = gz.policy_loss(torch.empty(0, 7, device="cuda"), label=torch.empty(0, dtype=torch.int32, device="cuda"))
    assert loss.shape == (0,) and grad.shape == (0, 7)


def check_loss(x, mask=None, target=None, label=None, weight=None, grad_scale=1.0):
    up = lambda t: None if t is None else t.cuda()  # noqa: E731
    loss, grad = gz.policy_loss(x.cuda(), target=up(target), label=up(label), mask=up(mask), weight=up(weight),
                                grad_scale=grad_scale)
    arr = lambda t: None if t is None else t.numpy()  # noqa: E731
    xs = x.float().numpy()
    want, wgrad, terms = ref.loss(xs, arr(mask), arr(target), arr(label), arr(weight), grad_scale)
    a = x.shape[1]
    few = (a / 32 + 64) * U
    assert (np.abs(loss.cpu().numpy() - want) <= few * terms + 1e-38).all(), np.abs(loss.cpu().numpy() - want).max()
    got = grad.float().cpu().numpy()
    half, least = {torch.float32: (U, 2.0**-149), torch.float16: (2.0**-11, 2.0**-25),
                   torch.bfloat16: (2.0**-8, 2.0**-134)}[x.dtype]
    seen = np.ones_like(xs, bool) if mask is None else mask.numpy() != 0
    finite = xs[seen & np.isfinite(xs)]
    depth = float(finite.max() - finite.min()) if finite.size else 0.0
    t = np.zeros_like(want)
    w = np.ones(len(xs)) if weight is None else np.abs(weight.numpy().astype(np.float64))
    if target is not None:
        t = np.abs(np.where(seen, target.numpy().astype(np.float64), 0))
    else:
        t = np.zeros_like(wgrad)
        ok = (label.numpy() >= 0) & (label.numpy() < a)
        t[np.nonzero(ok)[0], label.numpy()[ok]] = 1
        t = np.where(seen, t, 0)
    p = np.abs(wgrad + grad_scale * w[:, None] * t) + grad_scale * w[:, None] * t
    bound = few * (1 + depth) * p + half * np.abs(wgrad) + least
    assert (np.abs(got - wgrad) <= bound).all(), np.max(np.abs(got - wgrad) / np.maximum(bound, 1e-300))
    assert (got[~seen] == 0).all()
    # the loss alone is the same
    alone, none = gz.policy_loss(x.cuda(), target=up(target), label=up(label), mask=up(mask), weight=up(weight),
                                 need_grad=False)
    assert none is None and torch.equal(alone, loss)
    return loss, grad


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("a", SIZES)
def test_loss_sizes(cuda, a, dtype):
    n = 4 if a <= 8192 else 2
    g = torch.Generator().manual_seed(a)
    x = rows_of(n, a, a, dtype)
    target = torch.rand(n, a, generator=g) ** 4
    check_loss(x, target=target / target.sum(1, keepdim=True), grad_scale=1 / n)
    check_loss(x, label=torch.randint(0, a, (n,), generator=g, dtype=torch.int32), weight=torch.randn(n, generator=g))


@pytest.mark.parametrize("a,n,share", [(7, 64, 0.7), (130, 37, 0.1), (4672, 20, 0.008), (20000, 5, 0.5), (131072, 3, 0.9)])
def test_loss_masks(cuda, a, n, share):
    g = torch.Generator().manual_seed(a)
    mask = legal(n, a, share, 71)
    mask[1] = 0  # nothing legal
    mask[2] = 0
    mask[2, a - 1] = 7  # one legal action: loss 0, gradient 0
    x = rows_of(n, a, 72)
    x[mask == 0] = float("nan")
    x[0, mask[0] == 0] = float("inf")
    target = torch.rand(n, a, generator=g)
    target[mask == 0] = float("nan")
    loss, grad = check_loss(x, mask, target=target)
    assert loss[1] == 0 and (grad[1] == 0).all()
    label = torch.randint(0, a, (n,), generator=g, dtype=torch.int32)
    label[0], label[n - 1] = -1, a  # outside the row
    loss, grad = check_loss(x, mask, label=label, weight=torch.randn(n, generator=g), grad_scale=0.25)
    assert loss[0] == 0 and (grad[0] == 0).all() and loss[n - 1] == 0 and (grad[n - 1] == 0).all()


@pytest.mark.parametrize("a", [5, 300, 9000, 60000])
def test_loss_extreme_scores(cuda, a):
    x = rows_of(8, a, 81)
    x[0] += 5000  # large scores, ordinary differences
    x[1, :] = torch.finfo(torch.float32).min
    x[2, 1:] = float("-inf")
    x[3, 0] = float("-inf")
    x[4] = float("-inf")
    target = torch.zeros(8, a)
    target[:, 1] = 1.0
    target[2, :2] = torch.tensor([1.0, 0.0])
    target[6] = 0
    target[7] = -0.5
    check_loss(x, target=target)
    y = rows_of(3, a, 82)
    y[0, 2], y[1, 2] = float("nan"), float("inf")
    loss, grad = gz.policy_loss(y.cuda(), label=torch.zeros(3, dtype=torch.int32).cuda())
    assert loss[:2].isnan().all() and grad[:2].isnan().all() and grad[2].isfinite().all()
    z = torch.zeros(1, a)
    z[0, 0] = float("-inf")
    loss, grad = gz.policy_loss(z.cuda(), label=torch.zeros(1, dtype=torch.int32).cuda())
    assert loss[0] == float("inf") and grad[0, 0] == -1 and abs(float(grad[0, 1:].sum()) - 1) < 1e-4


@pytest.mark.parametrize("a", [9, 5000])
def test_loss_gradient_matches_differences(cuda, a):
    """Central differences of the loss at step h: the third derivative of a
    cross-entropy is at most 1 (h^2 / 6), and two losses of about 10 carry
    (a / 32 + 64) u each."""
    h, x = 0.125, rows_of(1, a, 91)
    at = torch.randperm(a, generator=torch.Generator().manual_seed(1))[:9]
    target = torch.rand(1, a) / a
    rows = x.repeat(18, 1)
    rows[torch.arange(9), at] += h
    rows[torch.arange(9, 18), at] -= h
    both = gz.policy_loss(rows.cuda(), target=target.cuda().expand(18, a))[0].double().cpu()
    grad = gz.policy_loss(x.cuda(), target=target.cuda())[1][0].double().cpu()[at]
    diff = (both[:9] - both[9:]) / (2 * h)
    assert (diff - grad).abs().max() <= h * h / 6 + 40 * (a / 32 + 64) * U / (2 * h)
    # a smaller step on a steeper direction, relative
    big = (diff - grad).abs() <= 0.02 * grad.abs() + 40 * (a / 32 + 64) * U / (2 * h)
    assert big.all()


@pytest.mark.parametrize("a", [33, 4672, 20001])
def test_loss_strides_and_alignment(cuda, a):
    for dtype in DTYPES:
        wide, mask = rows_of(4, a, 95, dtype, pad=3).cuda(), legal(4, a + 3, 0.5, 96).cuda()
        target = torch.rand(4, a + 3, generator=torch.Generator().manual_seed(2)).cuda()
        want = gz.policy_loss(wide[:, :a].contiguous(), target=target[:, :a].contiguous(), mask=mask[:, :a].contiguous())
        for off in (1, 2, 3):
            x, m, t = (torch.roll(v, off, 1)[:, off:off + a] for v in (wide, mask, target))
            got = gz.policy_loss(x, target=t, mask=m)
            assert (got[0] - want[0]).abs().max() <= 4 * (a / 32 + 64) * U * want[0].abs().max()
            assert (got[1].float() - want[1].float()).abs().max() <= 2.0**-7 * want[1].float().abs().max()


def test_loss_gradient_into_wider_rows(cuda):
    """The C entry writes gradients with a stride of their own, nothing beside them."""
    import ctypes as C
    n, a = 5, 77
    x, label = rows_of(n, a, 5).cuda(), torch.arange(n, dtype=torch.int32).cuda()
    out = torch.full((n, a + 6), 3.0, device="cuda")
    loss = torch.empty(n, device="cuda")
    rows = gz.PolicyRows(x.data_ptr(), None, a, 0, n, a, gz.F32)
    s = torch.cuda.current_stream().cuda_stream
    assert gz._lib.gz_policy_loss(C.byref(rows), None, 0, label.data_ptr(), None, 1.0, loss.data_ptr(), out.data_ptr() + 12,
                                  a + 6, s) == gz.OK
    want = gz.policy_loss(x, label=label)[1]
    assert (out[:, 3:3 + a] - want).abs().max() <= 1e-6
    assert (out[:, :3] == 3).all() and (out[:, 3 + a:] == 3).all()


def test_streams_and_graphs(cuda):
    x, noise = rows_of(64, 4672, 1).cuda(), ref.gumbel((64, 4672), 2).cuda()
    label = torch.arange(64, dtype=torch.int32).cuda()
    want, wl = gz.policy_sample(x, noise, top_p=0.9), gz.policy_loss(x, label=label)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, gl = gz.policy_sample(x, noise, top_p=0.9), gz.policy_loss(x, label=label)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(gl[1], wl[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, gl = gz.policy_sample(x, noise, top_p=0.9), gz.policy_loss(x, label=label)
    x.copy_(x.flip(0).clone())
    want, wl = gz.policy_sample(x, noise, top_p=0.9), gz.policy_loss(x, label=label)
    graph.replay()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(gl[0], wl[0]) and torch.equal(gl[1], wl[1])


def test_wrapper_refusals(cuda):
    x, cpu = torch.zeros(2, 7, device="cuda"), torch.zeros(2, 7)
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    for call in (lambda: gz.policy_sample(cpu), lambda: gz.policy_sample(x.double()), lambda: gz.policy_sample(x[0]),
                 lambda: gz.policy_sample(x, cpu), lambda: gz.policy_sample(x, x.half()), lambda: gz.policy_sample(x, x[:, :5]),
                 lambda: gz.policy_sample(x, mask=x), lambda: gz.policy_sample(x, mask=cpu.bool()),
                 lambda: gz.policy_sample(x, temperature=torch.ones(3, device="cuda")),
                 lambda: gz.policy_sample(x, top_k=torch.ones(2, device="cuda")), lambda: gz.policy_loss(x),
                 lambda: gz.policy_loss(x, target=x, label=i), lambda: gz.policy_loss(x, label=i.long()),
                 lambda: gz.policy_loss(x, target=x[:1]), lambda: gz.policy_loss(x, label=i, weight=i)):
        with pytest.raises(ValueError):
            call()
    for kw in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=1.5), dict(top_p=-0.1),
               dict(min_p=2.0), dict(min_p=float("nan"))):
        with pytest.raises(gz.GZError) as e:
            gz.policy_sample(x, **kw)
        assert e.value.status == gz.ERR_INVALID_ARG
    with pytest.raises(gz.GZError):
        gz.policy_sample(torch.zeros(1, gz.POLICY_MAX_ACTIONS + 1, device="cuda"))
