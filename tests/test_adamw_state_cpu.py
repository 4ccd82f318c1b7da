"""optim.AdamW's state where a captured step holds it by address, without a GPU: the kernels are replaced, a capture is pretended."""
import copy

import pytest
import torch

from test_train_ops_cpu import _FakeOps


def _captured(monkeypatch, sizes=(5000, 7), groups=None, **kw):
    """An optimizer after one step launch by launch and one that was captured, and its parameters."""
    from repmode_amd import ops, optim
    monkeypatch.setattr(ops, 'list_ops', lambda: _FakeOps())
    ps = [torch.nn.Parameter(torch.zeros(n)) for n in sizes]
    opt = optim.AdamW(groups(ps) if groups else ps, capturable=True, **kw)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    with monkeypatch.context() as m:
        m.setattr(optim, '_capturing', lambda: True)
        opt.step()
    return opt, ps


def _tensors(opt, ps):
    return {(i, k): t for i, p in enumerate(ps) for k, t in opt.state[p].items() if k != 'step'}


def _loaded(bits, sizes=(5000, 7), steps=(3, 3)):
    """A state dict of an optimizer of that many bits whose moments are not zero."""
    from repmode_amd import ops, optim
    ps = [torch.nn.Parameter(torch.zeros(n)) for n in sizes]
    opt = optim.AdamW(ps, state_bits=bits)
    for p, n in zip(ps, steps):
        opt._state(p, opt.param_groups[0])['step'] = torch.tensor(float(n))
        for k, t in opt.state[p].items():
            if k != 'step':
                t.view(torch.uint8).fill_(60)
    return opt.state_dict()


def _bytes(t):
    return t.reshape(-1).view(torch.uint8)


@pytest.mark.parametrize('bits', [32, 8])
def test_a_state_goes_into_what_a_captured_step_holds(monkeypatch, bits):
    opt, ps = _captured(monkeypatch, state_bits=bits)
    held, count = _tensors(opt, ps), opt._step_dev[0]
    saved = _loaded(bits)
    opt.load_state_dict(copy.deepcopy(saved))
    now = _tensors(opt, ps)
    assert sorted(now) == sorted(held) and all(now[k] is held[k] for k in held) and opt._step_dev[0] is count and int(count) == 3
    for i, p in enumerate(ps):
        for k, t in saved['state'][i].items():
            if k != 'step':
                assert torch.equal(_bytes(opt.state[p][k]), _bytes(t))


@pytest.mark.parametrize('bits', [32, 8])
def test_a_dict_without_state_rewinds_what_a_captured_step_holds(monkeypatch, bits):
    """What a new optimizer's state dict has: no moments, no counts.  Zero moments, zero codes with the scale 1."""
    from repmode_amd import ops, optim
    opt, ps = _captured(monkeypatch, state_bits=bits)
    opt.load_state_dict(copy.deepcopy(_loaded(bits)))
    held, count = _tensors(opt, ps), opt._step_dev[0]
    opt.load_state_dict(optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], state_bits=bits).state_dict())
    now = _tensors(opt, ps)
    assert sorted(now) == sorted(held) and all(now[k] is held[k] for k in held) and opt._step_dev[0] is count and int(count) == 0
    for p in ps:
        fresh = dict(zip(('exp_avg', 'exp_avg_scale', 'exp_avg_sq', 'exp_avg_sq_scale'), ops.adamw8_state(p)))
        for k, t in opt.state[p].items():
            if k == 'step':
                assert int(t) == 0
            else:
                assert torch.equal(_bytes(t), _bytes(fresh[k]) if t.dtype != torch.float32 else torch.zeros(4 * p.numel(), dtype=torch.uint8)), k


@pytest.mark.parametrize('have, loads', [(8, 32), (32, 8)])
def test_moments_of_other_bits_are_refused_under_a_captured_step(monkeypatch, have, loads):
    opt, ps = _captured(monkeypatch, state_bits=have)
    held, before = _tensors(opt, ps), copy.deepcopy(opt.state_dict())
    with pytest.raises(ValueError, match='captured'):
        opt.load_state_dict(_loaded(loads))
    now, after = _tensors(opt, ps), opt.state_dict()
    assert all(now[k] is held[k] for k in held) and after['param_groups'] == before['param_groups']
    for i, st in before['state'].items():
        assert all(torch.equal(_bytes(t), _bytes(after['state'][i][k])) for k, t in st.items())


def test_other_shapes_and_counts_that_differ_are_refused_under_a_captured_step(monkeypatch):
    opt, ps = _captured(monkeypatch)
    held, count = _tensors(opt, ps), opt._step_dev[0]
    for saved in (_loaded(32, sizes=(5001, 7)), _loaded(32, steps=(3, 4))):
        with pytest.raises(ValueError, match='captured'):
            opt.load_state_dict(saved)
    half = _loaded(32)
    del half['state'][1]                                 # (one parameter at step 3, the other at none)
    with pytest.raises(ValueError, match='captured'):
        opt.load_state_dict(half)
    assert all(t is held[k] for k, t in _tensors(opt, ps).items()) and opt._step_dev[0] is count and int(count) == 0


@pytest.mark.parametrize('have, loads', [(8, 32), (32, 8)])
def test_before_a_capture_moments_keep_the_bits_they_were_saved_with(monkeypatch, have, loads):
    """Nothing holds them yet: as without ``capturable``."""
    from repmode_amd import ops, optim
    monkeypatch.setattr(ops, 'list_ops', lambda: _FakeOps())
    ps = [torch.nn.Parameter(torch.zeros(n)) for n in (5000, 7)]
    opt = optim.AdamW(ps, capturable=True, state_bits=have)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    opt.load_state_dict(_loaded(loads))
    assert ('exp_avg_scale' in opt.state[ps[0]]) == (loads == 8) and int(opt._step_dev[0]) == 3


@pytest.mark.parametrize('saved_lr', [0.25, torch.tensor(0.25), torch.tensor(0.25, dtype=torch.float64)])
def test_a_learning_rate_on_the_device_stays_where_it_is(monkeypatch, saved_lr):
    """The tensor that replays read takes the loaded value, whatever the state has it as; also before a capture."""
    lr = torch.tensor(0.5)
    opt, ps = _captured(monkeypatch, groups=lambda p: [dict(params=p[:1], lr=lr), dict(params=p[1:], lr=0.125)])
    saved = opt.state_dict()
    saved = dict(saved, param_groups=[dict(g, lr=saved_lr) for g in saved['param_groups']])
    opt.load_state_dict(saved)
    assert opt.param_groups[0]['lr'] is lr and float(lr) == 0.25 and lr.dtype == torch.float32
    assert float(opt.param_groups[1]['lr']) == 0.25
    if torch.is_tensor(saved_lr):                        # (neither the dict's own tensor nor its type)
        assert opt.param_groups[1]['lr'] is not saved_lr and opt.param_groups[1]['lr'].dtype == torch.float32
        assert opt.param_groups[1]['lr'].device == ps[0].device


def test_a_saved_learning_rate_on_the_device_becomes_a_number_without_capturable(monkeypatch):
    from repmode_amd import ops, optim
    monkeypatch.setattr(ops, 'list_ops', lambda: _FakeOps())
    p = torch.nn.Parameter(torch.zeros(3))
    opt = optim.AdamW([p])
    saved = opt.state_dict()
    saved['param_groups'][0]['lr'] = torch.tensor(0.25)
    opt.load_state_dict(saved)
    p.grad = torch.ones(3)
    opt.step()
    assert opt.param_groups[0]['lr'] == 0.25 and not torch.is_tensor(opt.param_groups[0]['lr'])


def test_a_scheduler_fills_the_captured_learning_rate_after_a_load(monkeypatch):
    lr = torch.tensor(0.5)
    opt, ps = _captured(monkeypatch, lr=lr)
    opt.load_state_dict(copy.deepcopy(opt.state_dict()))
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda t: 0.5 ** t)
    sched.step()
    assert opt.param_groups[0]['lr'] is lr and float(lr) == 0.25


class _Skips(_FakeOps):
    """Gradient norms that are not finite in the steps that are named."""

    def __init__(self, bad):
        super().__init__()
        self.bad = bad

    def grad_norm(self, tensors, max_norm):
        super().grad_norm(tensors, max_norm)
        return torch.tensor(2.0), torch.tensor(float('nan') if len(self.norms) in self.bad else 0.5)


def test_steps_that_are_left_out_are_not_counted(monkeypatch):
    """Counts on the host: taken back before they are next used, of the parameters that had a gradient in that step."""
    from repmode_amd import ops, optim
    fake = _Skips({1, 3, 4, 6})
    monkeypatch.setattr(ops, 'list_ops', lambda: fake)
    a, b = (torch.nn.Parameter(torch.zeros(n)) for n in (5, 6))
    opt = optim.AdamW([a, b], max_norm=1.0)
    counts = []
    for t in range(1, 7):
        a.grad, b.grad = torch.ones(5), None if t == 3 else torch.ones(6)
        opt.step()
        counts.append([(c['n'], c['step']) for c in fake.steps])
        fake.steps.clear()
    assert counts == [[(2, 1)], [(2, 1)], [(1, 2)], [(2, 2)], [(2, 2)], [(2, 3)]]
    assert [int(s['step']) for s in opt.state_dict()['state'].values()] == [2, 2]
    assert [int(s['step']) for s in copy.deepcopy(opt).state.values()] == [2, 2]


def test_a_load_forgets_the_step_before_it(monkeypatch):
    from repmode_amd import ops, optim
    fake = _Skips({1})
    monkeypatch.setattr(ops, 'list_ops', lambda: fake)
    p = torch.nn.Parameter(torch.zeros(5))
    opt = optim.AdamW([p], max_norm=1.0)
    p.grad = torch.ones(5)
    opt.step()
    opt.load_state_dict(_loaded(32, sizes=(5,), steps=(3,)))
    opt.step()
    assert fake.steps[-1]['step'] == 4 and int(opt.state[p]['step']) == 4


@pytest.mark.parametrize('capturable', [False, True])
def test_moments_saved_in_another_order(monkeypatch, capturable):
    """float32 moments take their parameter's strides, as torch.optim.AdamW's would; 8-bit ones, whose scales go by the order in memory,
    are refused where it is another."""
    from repmode_amd import ops, optim
    monkeypatch.setattr(ops, 'list_ops', lambda: _FakeOps())
    shape = (3, 8, 5, 5)
    def one(fmt, bits, **kw):
        p = torch.nn.Parameter(torch.zeros(shape).to(memory_format=fmt))
        p.grad = torch.ones_like(p)
        opt = optim.AdamW([p], state_bits=bits, min_8bit_numel=1, **kw)
        opt.step()
        return opt, p
    plain, last = torch.contiguous_format, torch.channels_last
    opt, p = one(plain, 32)
    opt.state[p]['exp_avg'].copy_(torch.arange(600.).view(shape))
    into, q = one(last, 32, capturable=capturable)
    into.load_state_dict(opt.state_dict())
    for k in ('exp_avg', 'exp_avg_sq'):
        assert torch.equal(into.state[q][k], opt.state[p][k]) and into.state[q][k].stride() == q.stride()
    opt, p = one(plain, 8)
    into, q = one(last, 8, capturable=capturable)
    was = dict(into.state[q])
    with pytest.raises(ValueError, match='order'):
        into.load_state_dict(opt.state_dict())
    assert all(into.state[q][k] is t for k, t in was.items())
    other, r = one(last, 8)
    other.state[r]['exp_avg'].view(torch.uint8).copy_((torch.arange(600) % 120).view(shape))
    into.load_state_dict(other.state_dict())
    assert torch.equal(into.state[q]['exp_avg'].view(torch.uint8), other.state[r]['exp_avg'].view(torch.uint8))
    assert into.state[q]['exp_avg'].stride() == q.stride()


# ---------------------------------------------------------------------------------------------- the plain Adam

class _FakeAdam:
    """Stands for the operator library's Adam: the update is left out, but for the moments."""

    def adam_step_dev(self, params, grads, exp_avgs, exp_avg_sqs, *rest):
        for t in (*exp_avgs, *exp_avg_sqs):
            t.add_(1)


def _captured_adam(monkeypatch):
    from repmode_amd import ops, optim
    monkeypatch.setattr(ops, 'torch_ops', lambda: _FakeAdam())
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    ps = [torch.nn.Parameter(torch.zeros(n)) for n in (50, 7)]
    opt = optim.Adam(ps, capturable=True)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    monkeypatch.setattr(torch.cuda, 'is_initialized', lambda: True)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    opt.step()
    monkeypatch.undo()
    return opt, ps


def _stock_adam(steps=3, sizes=(50, 7)):
    ps = [torch.nn.Parameter(torch.zeros(n)) for n in sizes]
    opt = torch.optim.Adam(ps)
    for t in range(steps):
        for p in ps:
            p.grad = torch.full_like(p, t + 1.0)
        opt.step()
    return opt, ps


def test_a_state_goes_into_what_a_captured_adam_step_holds(monkeypatch):
    opt, ps = _captured_adam(monkeypatch)
    held, count, hyper = _tensors(opt, ps), opt._step_dev, opt._hyper_dev
    stock, qs = _stock_adam()
    saved = stock.state_dict()
    opt.load_state_dict(saved)
    assert all(t is held[k] for k, t in _tensors(opt, ps).items()) and opt._step_dev is count and opt._hyper_dev is hyper and int(count) == 3
    for p, q in zip(ps, qs):
        assert all(torch.equal(opt.state[p][k], stock.state[q][k]) for k in ('step', 'exp_avg', 'exp_avg_sq'))
        assert opt.state[p]['exp_avg'].data_ptr() != stock.state[q]['exp_avg'].data_ptr()
    opt.load_state_dict(torch.optim.Adam(ps).state_dict())       # (no moments at all: rewound)
    assert all(t is held[k] and not bool(t.any()) for k, t in _tensors(opt, ps).items()) and int(count) == 0
    assert opt._step_dev is count and [int(opt.state[p]['step']) for p in ps] == [0, 0]


def test_a_state_that_does_not_fit_a_captured_adam_step_is_refused(monkeypatch):
    opt, ps = _captured_adam(monkeypatch)
    held, count = _tensors(opt, ps), opt._step_dev
    opt.load_state_dict(_stock_adam()[0].state_dict())
    half = _stock_adam(2)[0].state_dict()
    half['state'][1]['step'] += 1
    for saved in (half, _stock_adam(sizes=(51, 7))[0].state_dict()):
        with pytest.raises(ValueError, match='captured'):
            opt.load_state_dict(saved)
    assert all(t is held[k] for k, t in _tensors(opt, ps).items()) and opt._step_dev is count and int(count) == 3
