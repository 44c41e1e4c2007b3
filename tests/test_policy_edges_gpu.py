"""The policy loss and sampling at the edges of their inputs, against the plain
restatements in 64 bits (tests/policy_ref.py)."""
import ctypes as C
import threading

import numpy as np
import pytest
import torch

import graphzero_b200 as gz
import policy_ref as ref
from test_policy_gpu import DTYPES, U, check_loss, check_sample, legal, rows_of

pytestmark = pytest.mark.gpu


def hidden_prefixes(n, a, slice_size, prefix):
    """[n][a]: each slice's first `prefix` actions hidden; in odd rows those of every second slice."""
    j = torch.arange(a)
    hide = (j % slice_size < prefix).repeat(n, 1)
    hide[1::2] &= j // slice_size % 2 == 0
    return hide


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,a,slice_size,prefix", [
    (150, 4672, 4672, 1500),     # a block a row, which looks at 512 actions first
    (151, 20001, 20001, 7000),
    (40, 131072, 131072, 20000),  # four or eight slices a row
    (2, 262144, 16384, 9000),    # sixteen
])
def test_loss_rows_that_begin_with_hidden_actions(cuda, n, a, slice_size, prefix, dtype):
    """More visible actions than are listed one by one, all behind those that
    the first look at a row sees: masked ones, and visible ones at -inf."""
    g = torch.Generator().manual_seed(a)
    hide = hidden_prefixes(n, a, slice_size, prefix)
    some = torch.rand(n, a, generator=g) < 0.7
    target = torch.rand(n, a, generator=g)
    label = torch.full((n,), a - 1, dtype=torch.int32)
    x = rows_of(n, a, a + 1, dtype)
    mask = (some & ~hide).to(torch.uint8)
    mask[:, a - 1] = 1
    x[mask == 0] = float("nan")
    loss, grad = check_loss(x, mask, target=target)
    assert (loss > 0).all() and (grad != 0).any(1).all()
    loss, grad = check_loss(x, mask, label=label, grad_scale=1 / n)
    assert (loss > 0).all() and (grad[:, a - 1] < 0).all()
    x = rows_of(n, a, a + 2, dtype)
    x[hide] = float("-inf")
    mask = some.to(torch.uint8)
    mask[:, a - 1] = 1
    loss, grad = check_loss(x, mask, target=torch.where(hide, torch.zeros(()), target))
    assert (loss > 0).all() and (grad != 0).any(1).all()
    loss, grad = check_loss(x, mask, label=label)
    assert (loss > 0).all() and (grad[:, a - 1] < 0).all()


LARGE = [2.0**29, 1e9, 2.0**30, 2.0**31 - 128, 2.0**31, 5e9, 1e10, 1e11, 1e15, 1e20, 1e29, 1e30, 3e38]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,a,share", [
    (3 * 2 * len(LARGE), 300, None), (3 * 2 * len(LARGE), 300, 0.5),  # a warp a row
    (3 * 2 * len(LARGE), 4672, 0.02),                                 # listed
    (6 * 2 * len(LARGE), 9000, 0.5), (3 * 2 * len(LARGE), 60000, 0.5),   # through a mask: a block a row, slices
    (6 * 2 * len(LARGE), 9000, None), (3 * 2 * len(LARGE), 60000, None),  # without
])
def test_loss_of_scores_of_any_magnitude(cuda, n, a, share, dtype):
    """Rows around +-2^29 to +-3e38: all alike (a finished game in a batch that
    hides moves by a large negative score), with a third of the scores lower
    still, and ordinary scores beside a third at the large negative value.

    Tolerance: that of check_loss with the depth of scores that count (24; e^-24
    of the sum is below u).  From 2^30 on neighbouring floats lie 64 or more
    apart, so all but the best have shares below e^-64 and may come out as
    anything up to 2^-64."""
    base = torch.tensor([s * v for v in LARGE for s in (1, -1)])
    kind = torch.arange(n) // len(base) % 3
    base = base.repeat(-(-n // len(base)))[:n, None].to(dtype).float()
    low = torch.arange(a)[None, :] % 3 == 1
    x = base.repeat(1, a)
    x = torch.where((kind == 1)[:, None] & low, (base - 0.1 * base.abs()).to(dtype).float(), x)
    ordinary = rows_of(n, a, a).clamp(-6, 6)
    x = torch.where((kind == 2)[:, None], torch.where(low, -base.abs(), ordinary), x).to(dtype)
    g = torch.Generator().manual_seed(1)
    mask = None
    if share is not None:
        mask = (torch.rand(n, a, generator=g) < share).to(torch.uint8)
        mask[:, 0] = mask[:, 1] = 1
    target = torch.where(low, torch.zeros(()), torch.rand(n, a, generator=g)) / a
    label = torch.zeros(n, dtype=torch.int32)
    xs = x.float().numpy()
    few = (a / 32 + 64) * U
    half, least = {torch.float32: (U, 2.0**-149), torch.bfloat16: (2.0**-8, 2.0**-134)}[dtype]
    for t, l in ((target, None), (None, label)):
        up = lambda v: None if v is None else v.cuda()  # noqa: E731
        arr = lambda v: None if v is None else v.numpy()  # noqa: E731
        loss, grad = gz.policy_loss(x.cuda(), target=up(t), label=up(l), mask=up(mask))
        want, wgrad, terms = ref.loss(xs, arr(mask), arr(t), arr(l))
        assert (np.abs(loss.cpu().numpy() - want) <= few * terms + 1e-38).all()
        amount = np.zeros_like(wgrad)
        if t is None:
            amount[:, 0] = 1.0
        else:
            amount = np.where(np.ones_like(xs, bool) if mask is None else mask.numpy() != 0, t.numpy(), 0.0)
        p = np.abs(wgrad + amount) + amount
        bound = 25 * few * p + half * np.abs(wgrad) + least + 2.0**-64
        assert (np.abs(grad.float().cpu().numpy() - wgrad) <= bound).all()


@pytest.mark.parametrize("n,a,share", [(40, 300, None), (40, 4672, 0.01), (40, 9000, 0.5), (200, 9000, None), (5, 131072, None),
                                       (5, 131072, 0.5)])
def test_loss_of_a_row_does_not_depend_on_other_rows(cuda, n, a, share):
    """In calls of as many rows: the same bits whatever the others hold, and again for the same call."""
    mask = None if share is None else legal(n, a, share, 1).cuda()
    x, label = rows_of(n, a, 2, torch.bfloat16).cuda(), torch.arange(n, dtype=torch.int32, device="cuda")
    loss, grad = gz.policy_loss(x, label=label, mask=mask)
    again = gz.policy_loss(x, label=label, mask=mask)
    assert torch.equal(loss, again[0]) and torch.equal(grad, again[1])
    for i in (0, n // 2, n - 1):
        y = rows_of(n, a, 3 + i, torch.bfloat16, spread=9.0).cuda()
        y[i] = x[i]
        got = gz.policy_loss(y, label=label, mask=mask)
        assert torch.equal(got[0][i], loss[i]) and torch.equal(got[1][i], grad[i])


def test_a_wait_that_runs_out_leaves_nan(cuda):
    """Blocks that share a row wait for sums that nothing sends: the waits give
    up after their limit, the results are NaN, and the next call is right."""
    assert gz.selftest_cluster_wait_timeout(0, 20000) == gz.ERR_TIMEOUT
    assert gz.selftest_cluster_wait_timeout(0, 0) == gz.ERR_INVALID_ARG
    check_loss(rows_of(3, 60000, 1), label=torch.arange(3, dtype=torch.int32))


def test_loss_from_several_threads(cuda):
    """Calls at once, whose rows want different amounts of shared memory, do not refuse each other."""
    calls, refused = [], []
    for a in (24000, 50000, 30000, 44000):
        x = torch.zeros(1, a, dtype=torch.bfloat16, device="cuda").expand(200, a)
        label, loss = torch.zeros(200, dtype=torch.int32, device="cuda"), torch.empty(200, device="cuda")
        rows = gz.PolicyRows(x.data_ptr(), None, 0, 0, 200, a, gz.BF16)
        calls.append((x, label, loss, rows, torch.cuda.Stream()))
    torch.cuda.synchronize()

    def work(x, label, loss, rows, stream):
        for _ in range(4000):
            status = gz._lib.gz_policy_loss(C.byref(rows), None, 0, label.data_ptr(), None, 1.0, loss.data_ptr(), None, 0,
                                            stream.cuda_stream)
            if status != gz.OK:
                refused.append(status)

    threads = [threading.Thread(target=work, args=c) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not refused
    for x, _, loss, _, _ in calls:
        assert (loss - np.log(x.shape[1])).abs().max() <= 1e-4


@pytest.mark.parametrize("a,share", [(7, None), (500, None), (4672, 0.01), (20000, None), (20000, 0.5)])
def test_sample_settings_of_nan_keep_the_best(cuda, a, share):
    """A NaN in a row's setting is taken as the value that keeps the fewest actions."""
    n = 6
    x, noise = rows_of(n, a, 1).cuda(), ref.gumbel((n, a), 2).cuda()
    mask = None if share is None else (torch.rand(n, a, device="cuda") < share).to(torch.uint8)
    best = gz.policy_sample(x, noise, mask=mask, temperature=0.0)
    plain = gz.policy_sample(x, noise, mask=mask)
    for kw, rest in (("temperature", 1.0), ("top_p", 1.0), ("min_p", 0.0)):
        v = torch.full((n,), float("nan"), device="cuda")
        v[::2] = rest
        got = gz.policy_sample(x, noise, mask=mask, **{kw: v})
        for k in (0, 1):
            assert torch.equal(got[k][1::2], best[k][1::2]), kw
            assert torch.equal(got[k][::2], plain[k][::2]), kw


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("a,share", [(300, None), (2000, None), (4672, 0.9), (9001, None), (40000, None), (40000, 0.9)])
def test_sample_scores_of_infinity_tie(cuda, a, share, dtype):
    """Scores of +inf are the largest float: of many such, and of the largest
    finite score beside them, the filters keep the lowest indices."""
    n = 6
    g = torch.Generator().manual_seed(a)
    x, noise = rows_of(n, a, a, dtype), ref.gumbel((n, a), a + 3)
    for i, many in enumerate((2, 9, 44, 44, a // 2, a)):
        x[i, torch.randperm(a, generator=g)[:many]] = float("inf")
    x[3, torch.randperm(a, generator=g)[:20]] = torch.finfo(dtype).max
    x[3, :a // 8] = float("nan")
    mask = None if share is None else legal(n, a, share, 5)
    for kw in (dict(top_p=0.5), dict(top_k=a - 1, top_p=0.95, temperature=0.001), dict(top_k=a - 1, top_p=0.9, temperature=0.3),
               dict(top_k=30), dict(top_k=a // 3), dict(top_p=0.95, min_p=0.5), dict()):
        check_sample(x, noise, mask, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("a,share", [(7, None), (60, 0.9), (300, None), (2000, None), (4672, 0.9), (9001, None), (40001, None),
                                     (40001, 0.9)])
def test_sample_nan_beside_infinity_is_never_picked(cuda, a, share, dtype):
    """Rows of NaN but for a few scores of +inf, of the largest float, or ordinary ones."""
    n = 12
    g = torch.Generator().manual_seed(a)
    x, noise = torch.full((n, a), float("nan"), dtype=dtype), ref.gumbel((n, a), a + 4)
    for i in range(n):
        at = torch.randperm(a, generator=g)[:1 + i // 3]
        x[i, at] = (float("inf"), torch.finfo(dtype).max, 1.5)[i % 3]
    mask = None if share is None else legal(n, a, share, 6)
    for kw in (dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0), dict(top_k=2), dict(top_p=0.4), dict(min_p=1.0), dict()):
        check_sample(x, noise, mask, **kw)
    check_sample(x, None, mask)
