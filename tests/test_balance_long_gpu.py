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
