"""optim.AdamW and the update's operators on the GPU: steps that are left out, states loaded under a captured step, memory that is shared."""
import copy
import math

import pytest
import torch

from test_hip_parity import DEV, _ops
from test_train_ops_gpu import HYPER, _bytes, _check_guards, _grid, _noise, _tensors, _update64

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


def _with_grads(ps, gs, at=None):
    for p, g in zip(ps, gs):
        p.grad = g.clone()
    if at is not None:
        ps[0].grad[at] = math.inf


@pytest.mark.parametrize('capturable', [False, True])
@pytest.mark.parametrize('bits', [32, 8])
def test_the_optimizer_does_not_count_steps_that_are_left_out(bits, capturable):
    """Gradients that are not finite before, between and after ordinary steps: parameters, moments and counts of a twin that never had
    those steps."""
    from repmode_amd.optim import AdamW
    ps, gs, _ = _fresh(bits)
    make = lambda: [torch.nn.Parameter(p.clone()) for p in ps]
    a, b = make(), make()
    opt, twin = (AdamW(q, lr=1e-2, max_norm=1.0, state_bits=bits, seed=5, capturable=capturable) for q in (a, b))
    for t, bad in enumerate((True, False, True, True, False, False, True)):
        g = [x * (t + 1) for x in gs]
        _with_grads(a, g, 7 if bad else None)
        opt.step()
        assert math.isfinite(float(opt.last_norm)) != bad
        if not bad:
            _with_grads(b, g)
            twin.step()
        for p, q in zip(a, b):
            assert torch.equal(_bytes(p.detach()), _bytes(q.detach())), t
    for st, want in zip(opt.state_dict()['state'].values(), twin.state_dict()['state'].values()):
        assert int(st['step']) == 3
        assert sorted(st) == sorted(want) and all(torch.equal(_bytes(st[k]), _bytes(want[k])) for k in st if k != 'step')


def test_a_captured_step_is_left_out_of_its_count():
    from repmode_amd.optim import AdamW
    ps, gs, _ = _fresh(32)
    a, b = ([torch.nn.Parameter(p.clone()) for p in ps] for _ in range(2))
    opt, twin = AdamW(a, lr=1e-2, max_norm=1.0, capturable=True), AdamW(b, lr=1e-2, max_norm=1.0)
    _with_grads(a, gs)
    _with_grads(b, gs)
    opt.step()
    twin.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    for t, bad in enumerate((False, True, False, True, False)):
        for p, g in zip(a, gs):
            p.grad.copy_(g * (t + 2))
        if bad:
            a[1].grad[11] = math.nan
        graph.replay()
        if not bad:
            _with_grads(b, [g * (t + 2) for g in gs])
            twin.step()
        torch.cuda.synchronize()
        for p, q in zip(a, b):
            assert torch.equal(_bytes(p.detach()), _bytes(q.detach())), t
    assert all(int(s['step']) == 4 for s in opt.state_dict()['state'].values())


def test_gradients_that_share_memory_with_what_is_written():
    """Refused where threads would race; neighbours, gradients that two parameters share and gradients that are copied first are not."""
    ops = _ops()
    z = lambda n=64, d=torch.float32: torch.zeros(n, device=DEV, dtype=d)
    p, g, m, v = z(), z(), z(), z()
    m8, e8, v8, f8 = ops.adamw8_state(p)
    wide = z(200)
    bad = [
        lambda: ops.adamw_step([p], [p], [m], [v], 1), lambda: ops.adamw_step([p], [m], [m], [v], 1), lambda: ops.adamw_step([p], [v], [m], [v], 1),
        lambda: ops.adamw_step([wide[:64]], [wide[63:127]], [m], [v], 1), lambda: ops.adamw_step([wide[63:127]], [wide[:64]], [m], [v], 1),
        lambda: ops.adamw_step([z(), p], [p, z()], [z(), m], [z(), v], 1), lambda: ops.adamw_step([p], [g], [m], [v], 1, clip=p[:1]),
        lambda: ops.adamw_step([p], [g], [m], [v], 1, clip=v[63]),
        lambda: ops.adamw8_step([p[:16]], [m8.view(torch.float32)], [m8[:16]], [e8], [v8[:16]], [f8], 1)]
    for call in bad:
        with pytest.raises(RuntimeError, match='shares memory'):
            call()
    assert float(p.abs().sum() + m.abs().sum() + v.abs().sum() + wide.abs().sum()) == 0
    q, w = (torch.randn(k, generator=torch.Generator().manual_seed(k)).to(DEV) for k in (64, 200))
    def step(ps, gs):
        ms, vs = ([torch.zeros_like(x, dtype=torch.float32) for x in ps] for _ in range(2))
        ops.adamw_step(ps, gs, ms, vs, 1)
        return [_bytes(x.clone()) for x in ps + ms + vs]
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))
    part = lambda x: (x[:64], x[64:128])
    apart = step([part(w.clone())[0].clone()], [w[64:128].clone()])
    assert same(step(*[[x] for x in part(w.clone())]), apart)                                    # neighbours
    assert same(step([q.clone(), w[:64].clone()], [w[64:128]] * 2)[1::2], step([w[:64].clone()], [w[64:128]]))
    # of another order: as they were at the call, also where parameters of another type are updated first
    def mixed():
        a, b = q.clone().view(8, 8), q[:16].bfloat16()
        return [a, b], [a.t(), a.view(-1).view(torch.bfloat16)[1::2][:16]]
    ps, gs = mixed()
    gs = [g.clone(memory_format=torch.contiguous_format) for g in gs]
    assert same(step(*mixed()), step(ps, gs))


def test_what_is_written_moves_its_version():
    """Parameters, moments and scales; autograd then refuses a graph that has saved one of them.  Gradients are only read."""
    ops = _ops()
    for bits in (32, 8):
        p, g, s = _fresh(bits)
        w = torch.ones(5000, device=DEV, requires_grad=True)
        graph = (w * s[0][0].float()).sum() if bits == 8 else (w * s[0][0]).sum()
        written = [t for t in p + sum(s, []) if t.numel()]
        was, read = [t._version for t in written], [t._version for t in g]
        count = torch.zeros(1, dtype=torch.int64, device=DEV)
        written, was = written + [count], was + [count._version]
        ops.adamw8_step(p, g, *s, count)
        assert all(t._version > v for t, v in zip(written, was)) and [t._version for t in g] == read
        if bits == 32:
            with pytest.raises(RuntimeError, match='modified by an inplace operation'):
                graph.backward()


def test_views_that_are_negated_when_read():
    """Views whose memory holds the negated values (what .imag of a conjugate is): read as what they stand for, not written."""
    ops = _ops()
    p, g, s = _fresh(32, (300,), (torch.float32,))
    neg = torch._neg_view(g[0])
    assert neg.is_neg() and torch.equal(neg, -g[0])
    other = [x.clone() for x in (p[0], s[0][0], s[2][0])]
    ops.adamw_step(p, [neg], s[0], s[2], 1)
    ops.adamw_step([other[0]], [-g[0]], [other[1]], [other[2]], 1)
    for a, b in zip((p[0], s[0][0], s[2][0]), other):
        assert torch.equal(a, b)
    assert torch.equal(ops.grad_norm([neg])[0], ops.grad_norm(g)[0])
    x = torch.randn(40, 12, generator=torch.Generator().manual_seed(1)).to(DEV)
    for a, b in zip(ops.balance_loss(torch._neg_view(x), 3), ops.balance_loss(-x, 3)):
        assert torch.equal(a, b)
    up, y = torch.tensor(-2.0, device=DEV), -x
    grads = [torch.autograd.grad(ops.balance_loss(z, 3)[0], z, grad_outputs=u) for z, u in
             ((y.requires_grad_(True), -up), (torch._neg_view(x).requires_grad_(True), -up), (y, torch._neg_view(up)))]
    assert all(torch.equal(a[0], grads[0][0]) for a in grads)
    for bad in (lambda: ops.adamw_step([torch._neg_view(p[0])], g, s[0], s[2], 1), lambda: ops.adamw_step(p, g, [torch._neg_view(s[0][0])], s[2], 1),
                lambda: ops.adamw_step(p, g, s[0], [torch._neg_view(s[2][0])], 1),
                lambda: ops.adamw_step(p, g, s[0], s[2], 1, clip=torch._neg_view(torch.ones((), device=DEV)))):
        with pytest.raises(RuntimeError, match='negated'):
            bad()


def _captured(bits, **kw):
    """An optimizer over two parameters whose step is in a graph, after one step launch by launch, and a twin without one."""
    from repmode_amd.optim import AdamW
    ps, gs, _ = _fresh(bits, dtypes=(torch.float32, torch.float32))
    a, b = ([torch.nn.Parameter(p.clone()) for p in ps] for _ in range(2))
    opt = AdamW(a, max_norm=1.0, state_bits=bits, seed=5, capturable=True, **kw)
    _with_grads(a, gs)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    for p, q in zip(a, b):
        q.data.copy_(p.detach())
    return graph, opt, a, b, gs


@pytest.mark.parametrize('through', ['device', 'host'])
@pytest.mark.parametrize('bits', [32, 8])
def test_replays_go_on_from_a_loaded_state(bits, through):
    """Rewound to a new optimizer's state, then loaded with a twin's, with memory that was freed taken and filled in between: each replay
    is the twin's step, and a learning rate on the device is the one that a scheduler fills."""
    from repmode_amd.optim import AdamW
    graph, opt, a, b, gs = _captured(bits, lr=torch.tensor(1e-2, device=DEV))
    twin = AdamW(b, lr=float(torch.tensor(1e-2, dtype=torch.float32)), max_norm=1.0, state_bits=bits, seed=5)
    lr = opt.param_groups[0]['lr']
    def load(state):
        opt.load_state_dict({k: v for k, v in state.items()} if through == 'device' else torch.utils._pytree.tree_map(
            lambda t: t.cpu() if torch.is_tensor(t) else t, state))
        hold = [torch.full((n,), math.nan, device=DEV) for n in (1, 64, 300, 1280, 5000) for _ in range(20)]
        torch.cuda.synchronize()
        del hold
    def both(n):
        for t in range(n):
            for p, g in zip(a, gs):
                p.grad.copy_(g * (t + 2))
            _with_grads(b, [g * (t + 2) for g in gs])
            graph.replay()
            twin.step()
            torch.cuda.synchronize()
            for p, q in zip(a, b):
                assert torch.equal(p.detach(), q.detach()), t
                assert all(torch.equal(_bytes(opt.state[p][k]), _bytes(v)) for k, v in twin.state[q].items() if k != 'step')
    load(twin.state_dict())                              # (no step yet: no moments)
    both(3)
    for q, g in zip(b, gs):                              # the twin goes on alone, and then its state is loaded
        q.grad = g.clone()
    twin.step()
    for p, q in zip(a, b):
        p.data.copy_(q.detach())
    load(copy.deepcopy(twin.state_dict()))
    assert opt.param_groups[0]['lr'] is lr
    both(2)
    lr.fill_(3e-3)
    twin.param_groups[0]['lr'] = float(lr)
    both(2)
    assert all(int(s['step']) == 8 for s in opt.state_dict()['state'].values())


def test_replays_of_the_plain_adam_go_on_from_a_loaded_state():
    from repmode_amd.optim import Adam
    ps, gs, _ = _fresh(32, dtypes=(torch.float32, torch.float32))
    a, b = ([torch.nn.Parameter(p.clone()) for p in ps] for _ in range(2))
    opt, twin = Adam(a, lr=1e-2, capturable=True), torch.optim.Adam(b, lr=1e-2)
    _with_grads(a, gs)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    for n in (2, 3):                                     # rewound first, then loaded with the twin's state
        for p, q in zip(a, b):
            p.data.copy_(q.detach())
        opt.load_state_dict(copy.deepcopy(twin.state_dict()))
        hold = [torch.full((k,), math.nan, device=DEV) for k in (1, 300, 5000) for _ in range(20)]
        torch.cuda.synchronize()
        del hold
        for t in range(n):
            for p, g in zip(a, gs):
                p.grad.copy_(g * (t + 2))
            _with_grads(b, [g * (t + 2) for g in gs])
            graph.replay()
            twin.step()
            torch.cuda.synchronize()
            for p, q in zip(a, b):
                # a step moves by lr m / sqrt(v), at most about 1e-2: both sides' roundings of it, and the parameter's
                assert float((p.detach() - q.detach()).abs().max()) < 5 * (2.0 ** -24 * float(q.detach().abs().max()) + 64 * 2.0 ** -24 * 1e-2)
    assert int(opt._step_dev) == 5


@pytest.mark.parametrize('offset', [0, 1])
@pytest.mark.parametrize('sizes', [(1, 3, 4), (1, 1, 1, 1, 2, 2, 2, 2), (9, 8, 7, 6, 5)])
def test_bfloat16_parameters_of_a_few_elements(sizes, offset):
    """Every element of the smallest tensors is the neighbour that its random bits choose (float64 definition), but where those lie
    within the arithmetic's own error of the border; over all steps nearly none does."""
    ops = _ops()
    gen = torch.Generator().manual_seed(21)
    (p, g, m, v), guards = _tensors(sizes, torch.bfloat16, gen, offset)
    sure_of, total = 0, 0
    for t in range(1, 30):
        was = [[x.clone() for x in lst] for lst in (p, g, m, v)]
        ops.adamw_step(p, g, m, v, t, seed=11, **HYPER)
        for i, n in enumerate(sizes):
            p1, _, _, dp, _, _ = _update64(*(lst[i] for lst in was), t, **HYPER)
            low, step = _grid(p1.abs(), 7, -126)
            bits = _noise(11, t, i, torch.arange(n))[1].double() / 65536
            frac = (p1.abs() - low) / step
            sure = (frac + bits - 1).abs() > dp / step + 2.0 ** -20
            want = torch.copysign(low + step * (frac + bits >= 1), p1)
            assert bool((p[i].cpu().double() == want)[sure].all()), (t, i)
            sure_of, total = sure_of + int(sure.sum()), total + n
    assert sure_of > 0.9 * total
    _check_guards([x for x in guards if x[0].dtype == torch.bfloat16])


def test_the_look_at_the_last_step_under_another_default_device():
    """What is copied to the host lies there whatever device new tensors go to by default."""
    from repmode_amd.optim import AdamW
    _ops()
    p = torch.nn.Parameter(torch.ones(8, device=DEV))
    opt = AdamW([p], max_norm=1.0)
    with torch.device(DEV):
        for g, want in ((math.inf, 0), (1.0, 1), (math.nan, 1), (1.0, 2)):
            p.grad = torch.full((8,), g)
            opt.step()
            assert int(opt.state_dict()['state'][0]['step']) == want
