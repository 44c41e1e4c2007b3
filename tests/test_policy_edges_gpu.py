"""The policy loss and sampling at the edges of their inputs, against the plain
restatements in 64 bits (tests/policy_ref.py)."""
import pytest
import torch

from test_policy_gpu import DTYPES, check_loss, rows_of

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
