"""A train step replayed as a HIP graph against the step launch by launch, gradient by gradient: in deterministic mode bit by bit, with
float atomics within what their order alone does.  Freed memory is filled with NaN between the replays."""
import pytest
import torch

from conftest import Opts

KINDS = [{}, dict(optimizer='adamw', optimizer_args=dict(max_norm=0.1, state_bits=8), balance_coef=0.25)]


def _exact(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


def _close(got, want):
    """The whole gradient within 0.6 of its norm.  Two bfloat16 steps launch by launch, at the size below, differ by up to 0.24 (the
    first from new weights; 0.06 and less afterwards); a gradient that is missing or doubled is off by 1, another step's by more."""
    a, b = (torch.cat([g.double().reshape(-1) for g in gs]) for gs in (got, want))
    return bool(torch.isfinite(a).all()) and float((a - b).norm()) < 0.6 * float(b.norm())


@pytest.mark.parametrize('check', [_exact, _close])
def test_the_checks_find_what_they_are_for(check):
    gen = torch.Generator().manual_seed(0)
    want, before = ([torch.randn(n, generator=gen) for n in (300, 5, 4000)] for _ in range(2))
    assert check([g.clone() for g in want], want)
    for wrong in ([torch.zeros_like(g) for g in want], [2 * g for g in want], before, [g + 1e30 for g in want], [g * float('nan') for g in want]):
        assert not check(wrong, want)
    for i in range(3):
        assert not _exact(want[:i] + [before[i]] + want[i + 1:], want)


def _replays(dtype, kw, shape, tasks, check, steps=6):
    from repmode_amd.model import Model
    make = lambda graph: Model(Opts(), lr=1e-3, gpu_ids=0, mult_chan=4, dtype=dtype, hip_graph=graph, **kw)
    torch.manual_seed(0)
    m, e = make(True), make(False)
    gen = torch.Generator().manual_seed(1)
    for t in range(steps):
        hold = [torch.full((n,), float('nan'), device='cuda') for n in (200, 5000, 100000, 2000000) for _ in range(20)]
        torch.cuda.synchronize()
        del hold
        x, y = (torch.randn(len(tasks), 1, *shape, generator=gen) for _ in range(2))
        e.net.load_state_dict(m.net.state_dict())
        m.do_train_iter(x, y, torch.tensor(tasks))
        e.do_train_iter(x, y, torch.tensor(tasks))
        assert check([p.grad for p in m.net.parameters()], [p.grad for p in e.net.parameters()]), t
    assert next(iter(m._graphs.values()))['graph'] is not None
    return m, e


@pytest.mark.gpu
@pytest.mark.parametrize('kw', KINDS)
@pytest.mark.parametrize('shape', [(16, 16, 32), (32, 64, 64)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_replays_are_the_eager_step_bit_by_bit(dtype, shape, kw):
    from test_hip_parity import _ops
    ops = _ops()
    ops.set_deterministic(True)
    try:
        m, e = _replays(dtype, kw, shape, [1, 5, 1], _exact)
        assert torch.equal(m.last_loss, e.last_loss)
    finally:
        ops.set_deterministic(False)


@pytest.mark.gpu
@pytest.mark.parametrize('kw', KINDS)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_replays_with_float_atomics(dtype, kw):
    from test_hip_parity import _ops
    _ops()
    _replays(dtype, kw, (32, 64, 64), [1, 5, 1, 0, 7, 2, 3, 9], _close)


@pytest.mark.gpu
@pytest.mark.parametrize('graph', [False, True])
def test_model_adds_the_gates_balance_term(graph):
    """The gates' gradients with balance_coef are those without plus gate_balance's own, and nothing else moves; last_balance has its
    value and counts."""
    from repmode_amd.model import Model
    from repmode_amd.nn_modules.RepMode import MoDEConv
    from test_hip_parity import _ops
    ops = _ops()
    coef, tasks = 0.25, [1, 5, 1]
    ops.set_deterministic(True)
    try:
        make = lambda c: Model(Opts(), lr=1e-3, gpu_ids=0, mult_chan=2, dtype=torch.float32, hip_graph=graph and c > 0, balance_coef=c)
        torch.manual_seed(0)
        m, e = make(coef), make(0.0)
        gen = torch.Generator().manual_seed(1)
        for t in range(4):
            x, y = (torch.randn(3, 1, 16, 16, 16, generator=gen) for _ in range(2))
            e.net.load_state_dict(m.net.state_dict())
            term, counts, _ = e.net.gate_balance(tasks, coef)
            gates = [q for b in e.net.modules() if isinstance(b, MoDEConv) for q in (b.gate.weight, b.gate.bias)]
            own = dict(zip(map(id, gates), torch.autograd.grad(term, gates)))
            value = term.detach()
            del term
            m.do_train_iter(x, y, torch.tensor(tasks))
            e.do_train_iter(x, y, torch.tensor(tasks))
            assert torch.equal(m.last_loss, e.last_loss) and torch.equal(m.last_balance[0], value) and torch.equal(m.last_balance[1], counts)
            # experts that are used alike give coef; a term lies between 0 and 5 coef
            assert 0 < float(value) <= 5 * coef and e.last_balance is None
            for p, q in zip(m.net.parameters(), e.net.parameters()):
                if id(q) in own:
                    want = q.grad.double() + own[id(q)].double()
                    assert bool(own[id(q)].any()) and float((p.grad - want).abs().max()) <= 2.0 ** -24 * float(want.abs().max()) * 2
                else:
                    assert torch.equal(p.grad, q.grad)
    finally:
        ops.set_deterministic(False)
