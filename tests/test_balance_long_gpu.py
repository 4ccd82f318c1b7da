"""balance_loss over many long groups."""
import pytest
import torch

from test_hip_parity import DEV, _ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('experts, rows', [(512, 1 << 18), (5, 1 << 24)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_mean_probabilities_of_long_groups(experts, rows, dtype):
    """257 groups, whose rows are all alike (an expanded tensor, so that they take no memory): the mean probabilities are the
    row's.  Equal addends round the same way again and again, the worst that a running float32 sum can meet: n of them are off by up
    to (n / 2) 2^-24 of the sum, and a lane adds no more than 1024."""
    ops = _ops()
    gen = torch.Generator().manual_seed(5)
    row = torch.randn(experts, generator=gen).to(dtype)
    x = row.to(DEV).expand(257, rows, experts)
    loss, counts, prob = ops.balance_loss(x, 1)
    p = torch.softmax(row.double(), 0)
    far = float(row.double().max() - row.double().min())
    most = 512 * 2.0 ** -24 + (far + 68) * 2.0 ** -24            # + a probability's own roundings and the joins'
    want = torch.zeros(experts, dtype=torch.int64)
    want[int(p.argmax())] = rows
    assert torch.equal(counts.cpu(), want.expand(257, experts))
    assert float(((prob.double().cpu() - p) / p).abs().max()) <= most
    assert abs(float(loss) - experts * float(p.max())) <= most * experts * float(p.max())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('experts', [5, 24, 200, 600])
def test_a_row_does_not_go_by_the_rows_beside_it(experts, dtype):
    """The gradient of ordinary rows is the same, bit by bit, whether other rows lie near zero or far from it (where the softmax takes
    its difference to the maximum in two steps), as long as those choose alike."""
    ops = _ops()
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(64, experts, generator=gen).to(dtype)
    moved = x.clone()
    moved[::3] = torch.where(torch.arange(experts) == x[::3].float().argmax(1, keepdim=True), 1e9, -1e9).to(dtype)
    keep = torch.ones(64, dtype=torch.bool)
    keep[::3] = False
    out = []
    for z in (x, moved):
        z = z.to(DEV).requires_grad_(True)
        loss, counts, _ = ops.balance_loss(z, 1)
        grad, = torch.autograd.grad(loss, z)
        out.append((counts, grad.cpu()[keep]))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1]) and bool(torch.isfinite(out[0][1]).all())
