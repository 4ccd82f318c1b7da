"""The train step's operators without a GPU: what they refuse (balance_loss, grad_norm, adamw_step, adamw8_step -- the operator
library's checks and the C ABI's), and optim.AdamW's bookkeeping, with the kernels replaced."""
import ctypes
import math

import pytest
import torch

from conftest import Opts


def _ops():
    from repmode_amd import ops
    return ops


def test_cpu_tensors_are_refused():
    ops = _ops()
    x = torch.randn(4, 8)
    for call in (lambda: ops.balance_loss(x, 2), lambda: ops.grad_norm([x]),
                 lambda: ops.adamw_step([x], [x.clone()], [x.clone()], [x.clone()], 1),
                 lambda: ops.adamw8_step([x], [x.clone()], *[[t] for t in ops.adamw8_state(x)], 1)):
        with pytest.raises(RuntimeError, match='no CPU fallback'):
            call()
    with pytest.raises(RuntimeError, match='no tensors'):
        ops.grad_norm([])
    with pytest.raises(RuntimeError, match='max_norm'):
        ops.grad_norm([x], max_norm=float('nan'))
    with pytest.raises(RuntimeError, match='list lengths'):
        ops.adamw_step([x], [], [x], [x], 1)
    ops.adamw_step([], [], [], [], 1)                    # (nothing to do)
    for bad in ([1], [None], x, 'x', None):
        with pytest.raises(TypeError):
            ops.adamw_step([x], bad, [x], [x], 1)
    with pytest.raises(TypeError, match='no tensor'):
        ops.grad_norm([x, 3])
    with pytest.raises(TypeError, match='clip'):
        ops.adamw_step([x], [x], [x], [x], 1, clip=0.5)


def test_adamw8_state_layout():
    ops = _ops()
    for n in (1, 255, 256, 257, 5000):
        m, ms, v, vs = ops.adamw8_state(torch.zeros(n, dtype=torch.bfloat16))
        assert m.dtype == torch.float8_e4m3fn and v.dtype == torch.float8_e5m2 and m.shape == v.shape == (n,)
        assert ms.dtype == vs.dtype == torch.float8_e8m0fnu and ms.shape == vs.shape == (-(-n // ops.ADAMW_BLOCK),)
        assert float(m.float().abs().sum()) == 0 and float(v.float().abs().sum()) == 0 and bool((ms.float() == 1).all())


def _call(name, *args):
    from repmode_amd import _lib
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.repmode_last_error().decode()


FAKE = 0x10000          # an address that is only looked at: every call below is refused before a launch


def _arrays(n, value=FAKE):
    return (ctypes.c_void_p * n)(*[value] * n)


def _adamw_multi(n=1, dtype=0, bits=32, p=FAKE, m=FAKE, numel=5, scales=True, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, decay=0.0, step=1):
    k = max(1, min(n, 100))
    numels = (ctypes.c_long * k)(*[numel] * k)
    pos = (ctypes.c_int * k)(*range(k))
    s = _arrays(k) if scales else None
    return _call('repmode_adamw_multi', n, dtype, bits, _arrays(k, p), _arrays(k), _arrays(k, m), s, _arrays(k), s, numels, pos, lr, beta1, beta2,
                 eps, decay, step, 0, None, None, None)


@pytest.mark.parametrize('bad, says', [
    (dict(n=0), 'tensors per call'), (dict(n=61), 'tensors per call'), (dict(dtype=2), 'bad dtype'), (dict(bits=16), '32 or 8 bits'),
    (dict(bits=8, scales=False), 'null pointer'), (dict(p=FAKE + 2), 'aligned'), (dict(dtype=1, p=FAKE + 1), 'aligned'), (dict(m=FAKE + 1), 'aligned'),
    (dict(p=None), 'bad tensor'), (dict(numel=0), 'bad tensor'), (dict(numel=-3), 'bad tensor'), (dict(numel=1 << 44), 'grid too large'),
    (dict(step=0), 'starts at 1'), (dict(lr=-1.0), 'hyper-parameters'), (dict(lr=math.inf), 'hyper-parameters'), (dict(beta1=1.0), 'hyper-parameters'),
    (dict(beta2=-0.1), 'hyper-parameters'), (dict(eps=-1e-8), 'hyper-parameters'), (dict(eps=math.nan), 'hyper-parameters'),
    (dict(decay=-0.1), 'hyper-parameters')])
def test_adamw_abi_refuses(bad, says):
    rc, why = _adamw_multi(**bad)
    assert rc == 1 and says in why, why


@pytest.mark.parametrize('n, dtype, numel, capacity, says', [
    (0, 0, 5, 9, 'tensors per call'), (201, 0, 5, 999, 'tensors per call'), (1, 3, 5, 9, 'bad dtype'), (1, 0, 0, 9, 'bad tensor'),
    (2, 0, 8193, 3, '4 partial sums needed'), (1, 1, 1 << 46, 9, 'grid too large')])
def test_grad_norm_abi_refuses(n, dtype, numel, capacity, says):
    k = max(1, n)
    used = ctypes.c_long(0)
    rc, why = _call('repmode_grad_norm_partial', n, dtype, _arrays(k), (ctypes.c_long * k)(*[numel] * k), FAKE, capacity, ctypes.byref(used), None)
    assert rc == 1 and says in why, why
    for args in ((FAKE, 1, -1.0, FAKE, FAKE), (FAKE, 1, math.nan, FAKE, FAKE), (None, 1, 1.0, FAKE, FAKE), (FAKE, 1, 1.0, None, FAKE)):
        assert _call('repmode_grad_norm_finish', *args, None)[0] == 1


@pytest.mark.parametrize('bad, says', [
    (dict(dtype=2), 'bad dtype'), (dict(groups=0), 'groups'), (dict(groups=65536), 'groups'), (dict(rows=-1), 'rows'), (dict(experts=0), 'experts'),
    (dict(experts=1025), 'experts'), (dict(top_k=0), 'top_k'), (dict(top_k=9), 'top_k'), (dict(rows=1 << 31), 'too many rows'),
    (dict(ws_bytes=8), 'workspace'), (dict(ws=FAKE + 4), 'workspace'), (dict(x=None), 'null pointer'), (dict(loss=None), 'null pointer')])
def test_balance_abi_refuses(bad, says):
    a = dict(x=FAKE, dtype=0, groups=1, rows=4, experts=8, top_k=2, ws=FAKE, ws_bytes=1 << 40, loss=FAKE)
    a.update(bad)
    rc, why = _call('repmode_balance_fwd', a['x'], a['dtype'], a['groups'], a['rows'], a['experts'], 32, 8, 1, None, 0, 0, a['top_k'], 1.0, a['ws'],
                    a['ws_bytes'], a['loss'], FAKE, FAKE, FAKE, None)
    assert rc == 1 and says in why, why


def test_adamw_refuses_bad_settings():
    from repmode_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(3))
    for kw in (dict(lr=-1), dict(eps=-1), dict(betas=(1.0, 0.9)), dict(weight_decay=-1), dict(max_norm=0), dict(max_norm=-1), dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    opt = AdamW([p])
    opt.param_groups[0]['amsgrad'] = True
    p.grad = torch.zeros(3)
    with pytest.raises(RuntimeError, match='amsgrad'):
        opt.step()
    opt = AdamW([p], lr=torch.tensor(1e-3))
    with pytest.raises(RuntimeError, match='capturable'):
        opt.step()


def test_model_refuses_bad_settings():
    from repmode_amd.model import Model
    for kw in (dict(optimizer='sgd'), dict(optimizer_args=dict(max_norm=1.0)), dict(balance_coef=-1.0), dict(balance_coef=float('nan'))):
        with pytest.raises(ValueError):
            Model(Opts(), gpu_ids=-1, **kw)


class _FakeOps:
    """Stands for the operator library: records the calls; the update is left out."""

    def __init__(self):
        self.steps, self.norms = [], []

    def grad_norm(self, tensors, max_norm):
        self.norms.append((len(tensors), max_norm))
        return torch.tensor(2.0), torch.tensor(0.5)

    def adamw_step(self, p, g, m, ms, v, vs, lr, b1, b2, eps, wd, step, step_dev, lr_dev, clip, seed):
        self.steps.append(dict(n=len(p), m=[t.dtype for t in m], scales=len(ms), lr=lr, wd=wd, step=step, clip=clip, seed=seed))
        for t in m:
            if t.dtype == torch.float32:
                t.add_(1)


def test_adamw_bookkeeping(monkeypatch):
    """Groups with their own settings, clipping over all of them, small tensors with float32 moments, parameters grouped by the
    number of updates they have seen."""
    from repmode_amd import ops, optim
    fake = _FakeOps()
    monkeypatch.setattr(ops, 'list_ops', lambda: fake)
    big, small, other = (torch.nn.Parameter(torch.randn(n)) for n in (5000, 7, 9000))
    opt = optim.AdamW([dict(params=[big, small]), dict(params=[other], weight_decay=0.0, state_bits=32)], lr=2e-3, max_norm=1.5, state_bits=8, seed=9)
    for p in (big, small, other):
        p.grad = torch.randn_like(p)
    opt.step()
    assert fake.norms == [(3, 1.5)] and float(opt.last_norm) == 2.0
    a, b = fake.steps
    assert a['n'] == 2 and a['m'] == [torch.float8_e4m3fn, torch.float32] and a['scales'] == 2 and a['wd'] == 1e-2 and a['step'] == 1
    assert b['n'] == 1 and b['m'] == [torch.float32] and b['scales'] == 0 and b['wd'] == 0.0
    assert float(a['clip']) == 0.5 and a['seed'] != b['seed'] and a['lr'] == 2e-3
    small.grad = None
    opt.step()
    small.grad = torch.randn(7)
    opt.step()
    assert [(c['n'], c['step']) for c in fake.steps[2:]] == [(1, 2), (1, 2), (1, 3), (1, 2), (1, 3)]
    assert fake.norms[1:] == [(2, 1.5), (3, 1.5)]
    opt.zero_grad()
    opt.step()                                           # no gradients at all: nothing happens
    assert len(fake.steps) == 7


def test_adamw_state_dicts(monkeypatch, tmp_path):
    """8-bit moments and the float32 moments of bfloat16 parameters survive save / load as they are; float32 states
    interchange with torch.optim.AdamW's."""
    from repmode_amd import ops, optim
    monkeypatch.setattr(ops, 'list_ops', lambda: _FakeOps())
    make = lambda: [torch.nn.Parameter(torch.zeros(n, dtype=d)) for n, d in ((5000, torch.bfloat16), (300, torch.bfloat16), (20, torch.float32))]
    ps, qs = make(), make()
    opt, back = optim.AdamW(ps, state_bits=8), optim.AdamW(qs)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    st = opt.state[ps[0]]
    st['exp_avg'].view(torch.uint8).copy_(torch.arange(5000) % 120)
    st['exp_avg_sq'].view(torch.uint8).copy_(torch.arange(5000) % 100)
    st['exp_avg_scale'].view(torch.uint8).copy_(torch.arange(20) + 100)
    opt.state[ps[1]]['exp_avg'].fill_(1 + 2.0 ** -20)
    torch.save(opt.state_dict(), tmp_path / 'opt.pt')
    back.load_state_dict(torch.load(tmp_path / 'opt.pt', weights_only=True))
    assert back.param_groups[0]['state_bits'] == 8
    for p, q in zip(ps, qs):
        assert sorted(opt.state[p]) == sorted(back.state[q])
        for k, t in opt.state[p].items():
            u = back.state[q][k]
            assert t.dtype == u.dtype and t.shape == u.shape and torch.equal(t.reshape(-1).view(torch.uint8), u.reshape(-1).view(torch.uint8)), k
            assert t.data_ptr() != u.data_ptr()
    # a stock optimizer's dict and back
    r = [torch.nn.Parameter(torch.randn(6)) for _ in range(2)]
    stock = torch.optim.AdamW(r, lr=3e-3, weight_decay=0.2)
    for p in r:
        p.grad = torch.randn(6)
    stock.step()
    mine = optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in r])
    mine.load_state_dict(stock.state_dict())
    g = mine.param_groups[0]
    assert g['lr'] == 3e-3 and g['weight_decay'] == 0.2 and g['state_bits'] == 32 and g['min_8bit_numel'] == 4096
    for p, q in zip(r, g['params']):
        assert torch.equal(stock.state[p]['exp_avg_sq'], mine.state[q]['exp_avg_sq']) and int(mine.state[q]['step']) == 1
        q.grad = torch.zeros(6)
    mine.step()
    again = torch.optim.AdamW(r)
    again.load_state_dict(mine.state_dict())
    again.step()
    assert float(again.state[r[0]]['step']) == 3.0


def test_adamw_copies(monkeypatch):
    """copy.deepcopy (pickle's way) keeps the settings; 8-bit moments are refused by the plain Adam."""
    import copy
    from repmode_amd import ops, optim
    monkeypatch.setattr(ops, 'list_ops', lambda: _FakeOps())
    p = torch.nn.Parameter(torch.zeros(5000))
    opt = optim.AdamW([p], max_norm=2.0, state_bits=8, seed=7)
    p.grad = torch.ones(5000)
    opt.step()
    other = copy.deepcopy(opt)
    q = other.param_groups[0]['params'][0]
    assert other.max_norm == 2.0 and other.seed == 7 and other.device_step is False and other.state[q]['exp_avg'].dtype == torch.float8_e4m3fn
    q.grad = torch.ones(5000)
    other.step()
    assert int(other.state[q]['step']) == 2 and int(opt.state[p]['step']) == 1
    with pytest.raises(ValueError, match='8 bits'):
        optim.Adam([p]).load_state_dict(opt.state_dict())


def test_list_ops_arguments():
    ops = _ops()
    with pytest.raises(TypeError, match='16 arguments'):
        ops.list_ops().adamw_step([])
    with pytest.raises(TypeError):
        ops.list_ops().grad_norm([torch.zeros(1)], 'x')
    with pytest.raises(TypeError):
        ops.list_ops().adamw_step([], [], [], [], [], [], 1e-3, 0.9, 0.99, 1e-8, 0.0, 'x', None, None, None, 0)


def test_graph_alive_sees_a_held_graph():
    ops = _ops()
    p = torch.nn.Parameter(torch.ones(3))
    assert not ops.torch_ops().graph_alive([p])
    held = (p * 2).sum()
    assert ops.torch_ops().graph_alive([p])
    del held
    assert not ops.torch_ops().graph_alive([p, torch.zeros(2)])
