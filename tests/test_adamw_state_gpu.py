"""optim.AdamW and the update's operators on the GPU: steps that are left out, states loaded under a captured step, memory that is shared."""
import copy
import math

import pytest
import torch

from test_hip_parity import DEV, _ops
from test_train_ops_gpu import _bytes

pytestmark = pytest.mark.gpu


def _fresh(bits, sizes=(5000, 300), dtypes=(torch.float32, torch.bfloat16)):
    """p, g and adamw8_step's four lists of zero moments."""
    ops = _ops()
    ps = [torch.randn(n, generator=torch.Generator().manual_seed(n)).to(DEV, d) for n, d in zip(sizes, dtypes)]
    gs = [torch.randn(n, generator=torch.Generator().manual_seed(n + 1)).to(DEV, d) for n, d in zip(sizes, dtypes)]
    none = torch.empty(0, device=DEV)
    st = [ops.adamw8_state(p) if bits == 8 else (torch.zeros_like(p, dtype=torch.float32), none, torch.zeros_like(p, dtype=torch.float32), none)
          for p in ps]
    return ps, gs, [list(x) for x in zip(*st)]


@pytest.mark.parametrize('bits', [32, 8])
def test_a_step_that_is_left_out_keeps_the_count_on_the_device(bits):
    """NaN for a clip factor: the next update is the one that a first update would have been, bit by bit."""
    ops = _ops()
    (p, g, s), (q, _, r) = _fresh(bits), _fresh(bits)
    count = torch.zeros(1, dtype=torch.int64, device=DEV)
    bad, good = torch.tensor(math.nan, device=DEV), torch.tensor(0.5, device=DEV)
    for clip, want in ((bad, 0), (good, 1), (bad, 1), (bad, 1), (good, 2), (None, 3)):
        ops.adamw8_step(p, g, *s, count, clip=clip, seed=3)
        assert int(count) == want
        if clip is not bad:
            ops.adamw8_step(q, g, *r, want, clip=clip, seed=3)
        for a, b in zip(p + sum(s, []), q + sum(r, [])):
            assert torch.equal(_bytes(a), _bytes(b)), want
