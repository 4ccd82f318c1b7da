"""The train step's operators on the GPU -- balance_loss (csrc/balance.hip), grad_norm (csrc/grad_norm.hip), adamw_step and
adamw8_step (csrc/adamw.hip) -- against their definitions in float64, and together: optim.AdamW and Model.

Tolerances count roundings: U = 2^-24 is half a float32 step relative to the value, half a bfloat16 step is 2^-8."""
import math

import pytest
import torch

from conftest import Opts
from test_hip_parity import DEV, _ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


# ---------------------------------------------------------------------------------------------- balance_loss

def _balance_ref(x, top_k, mask, coef, up=1.0):
    """float64 on the CPU, [groups, rows, experts]: loss, counts, prob, gradient, and the bounds of prob's and the gradient's error."""
    x = x.detach().double().cpu()
    g, n, e = x.shape
    on = torch.ones(g, n, dtype=torch.bool) if mask is None else mask.cpu().clone()
    on &= ~(x == -math.inf).all(2)
    x = torch.where(on[..., None], x, 0.0)
    p = torch.softmax(x, 2) * on[..., None]
    # the top_k of a row: value descending, index ascending, never a -inf
    order = torch.sort(x, dim=2, descending=True, stable=True).indices[..., :top_k]
    chosen = torch.zeros(x.shape, dtype=torch.bool).scatter_(2, order, True) & on[..., None] & (x > -math.inf)
    rows = on.sum(1)
    some = rows.clamp(min=1).double()[:, None]
    counts, prob = chosen.sum(1), p.sum(1) / some
    f = counts / (some * top_k)
    scale = coef * e / max(1, int((rows > 0).sum()))
    loss = scale * (f * prob).sum()
    w = up * scale * f / some
    dot = (p * w[:, None]).sum(2, keepdim=True)
    grad = p * (w[:, None] - dot)
    # a probability: the rounding of its distance D to the maximum (times log2(e), in one step with it: D U and, of log2(e) itself,
    # 0.23 D U, taken from the 28 U for D < 20; above, the probability is below 2e-9), exp within 4 U, at most 20 sums, reciprocal, product
    far = torch.where(p > 0, x.amax(2, keepdim=True) - x, torch.zeros(())).clamp(max=110)
    rel = (far + 28) * U
    off = (p * rel).sum(2, keepdim=True) + rel                       # (the sum's own error, weighted by what it sums)
    dprob = (p * off).sum(1) / some + 40 * U * prob                  # + the column sums
    dgrad = p * (w[:, None] + dot) * (2 * off + 30 * U) + p * (p * w[:, None] * off).sum(2, keepdim=True)
    return dict(loss=loss, counts=counts, prob=prob, grad=grad, dprob=dprob, dgrad=dgrad, dloss=scale * (f * dprob).sum() + 4 * U * abs(loss))


def _check_balance(x, top_k, mask=None, coef=0.5):
    ops = _ops()
    x = x.detach().requires_grad_(True)
    up = torch.tensor(1.75, device=DEV)
    loss, counts, prob = ops.balance_loss(x, top_k, mask=mask, coef=coef)
    grad, = torch.autograd.grad(loss, x, grad_outputs=up)
    x3 = x if x.dim() == 3 else x[None]
    r = _balance_ref(x3, top_k, mask if mask is None or x.dim() == 3 else mask[None], coef, 1.75)
    shape = x.shape[:-2] + x.shape[-1:]
    assert counts.dtype == torch.int64 and counts.shape == prob.shape == shape and grad.dtype == x.dtype and grad.shape == x.shape
    assert torch.equal(counts.cpu().view(r['counts'].shape), r['counts'])
    assert abs(float(loss.detach()) - float(r['loss'])) <= float(r['dloss']) + 1e-30
    assert bool(((prob.cpu().double().view(r['prob'].shape) - r['prob']).abs() <= r['dprob'] + 1e-37).all())
    got = grad.cpu().double().view(r['grad'].shape)
    half = 2.0 ** -8 if x.dtype == torch.bfloat16 else U
    bound = r['dgrad'] + half * r['grad'].abs() * 1.01 + 1e-37
    assert bool(((got - r['grad']).abs() <= bound).all()), float(((got - r['grad']).abs() / bound).max())
    return r


BALANCE_SHAPES = [
    # (groups or None, rows, experts, top_k)
    (None, 1, 1, 1), (None, 1, 8, 2), (None, 3, 5, 1), (None, 257, 5, 5), (None, 64, 8, 3), (None, 1000, 7, 2), (None, 130, 16, 4),
    (None, 33, 17, 17), (None, 500, 64, 6), (None, 77, 96, 8), (None, 40, 100, 3), (None, 65, 128, 1), (None, 129, 256, 8), (None, 19, 300, 12),
    (None, 9, 512, 33), (None, 5, 513, 2), (None, 7, 1000, 16), (None, 6, 1024, 5),
    (1, 70, 32, 2), (3, 41, 8, 2), (5, 1, 24, 4), (70, 3, 12, 1), (2, 2500, 40, 5),
]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('groups, rows, experts, top_k', BALANCE_SHAPES)
def test_balance_loss(groups, rows, experts, top_k, dtype):
    gen = torch.Generator().manual_seed(rows * 1000 + experts)
    shape = (rows, experts) if groups is None else (groups, rows, experts)
    x = (torch.randn(shape, generator=gen) * 2 + torch.randn(experts, generator=gen)).to(DEV, dtype)
    _check_balance(x, top_k)
    mask = (torch.rand(shape[:-1], generator=gen) < 0.6).to(DEV)
    _check_balance(torch.where(mask[..., None], x, math.nan), top_k, mask)               # masked rows hold NaN: not read, gradient 0


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_balance_loss_strides(dtype):
    """Experts the slowest axis, every second row, rows of a wider tensor (at an address off 16 bytes), an expanded group axis of the
    mask; the gradient comes back for each."""
    gen = torch.Generator().manual_seed(5)
    base = torch.randn(6, 48, 90, generator=gen).to(DEV, dtype)
    for x in (base.transpose(1, 2), base[:, ::2, :64], base[:, :, 1:41], base[::2, 3:, :], base[1].t(), base[2][:, 8:72], base.permute(2, 0, 1),
              base[0][:0], base[:, :1, :16]):
        _check_balance(x, 3)
    mask = (torch.rand(90, generator=gen) < 0.5).to(DEV)
    _check_balance(base.transpose(1, 2), 3, mask.expand(6, 90))
    _check_balance(base[:, ::2, :64], 3, (torch.rand(6, 48, generator=gen) < 0.5).to(DEV)[:, ::2])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('groups, rows, experts, top_k', [
    (None, 1, 9, 2), (None, 513, 16, 2), (None, 1100, 17, 3), (2, 300, 33, 4), (None, 257, 64, 6), (3, 129, 100, 2), (None, 130, 256, 8),
    (None, 33, 300, 1), (2, 70, 512, 9), (None, 17, 513, 2), (None, 40, 1024, 16), (None, 20000, 24, 2)])
def test_balance_loss_rows_adjacent(groups, rows, experts, top_k, dtype):
    """Logits whose rows are neighbours in memory, experts the slow axis; with a mask, and rows that a tile's end cuts."""
    gen = torch.Generator().manual_seed(rows + experts)
    shape = (experts, rows) if groups is None else (groups, experts, rows)
    x = (torch.randn(shape, generator=gen) * 2).to(DEV, dtype).transpose(-2, -1)
    _check_balance(x, top_k)
    mask = (torch.rand(x.shape[:-1], generator=gen) < 0.6).to(DEV)
    _check_balance(torch.where(mask[..., None], x, math.nan).transpose(-2, -1).contiguous().transpose(-2, -1), top_k, mask)


@pytest.mark.parametrize('experts', [4, 8, 40, 256, 640])
def test_balance_loss_ties_and_infinities(experts):
    """Equal logits go to the lowest index; -inf is never chosen, even where fewer than top_k experts are left; a row of -inf alone
    does not count; the type's lowest value is a value."""
    x = torch.zeros(12, experts)
    x[1] = torch.arange(experts) % 3
    x[2, 1:] = -math.inf                                  # one expert left for top_k = 3
    x[3] = -math.inf                                      # none: the row does not count
    x[4, ::2] = -math.inf
    x[5] = torch.finfo(torch.float32).min
    x[6] = torch.finfo(torch.float32).min
    x[6, experts - 1] = 0.0
    x[7] = 3e38
    x[8, experts // 2] = 80.0
    x[9] = -0.0
    x[9, experts - 2] = 0.0                               # (equal to -0)
    for dtype in (torch.float32, torch.bfloat16):
        y = x.clamp(min=torch.finfo(dtype).min).masked_fill(x == -math.inf, -math.inf).to(DEV, dtype)
        r = _check_balance(y, 3)
        assert int(r['counts'].sum()) < 12 * 3


@pytest.mark.parametrize('experts', [5, 24, 200, 600])
def test_balance_loss_far_from_zero(experts):
    """Logits of any common offset, up to the types' ends: only their differences count."""
    gen = torch.Generator().manual_seed(experts)
    tops = [2.0 ** e for e in (10, 18, 19.999, 20, 21, 24, 31, 40, 80, 126)] + [1e10, 1.9e38, 3.3e38]
    x = torch.tensor([s * t for t in tops for s in (1, -1)])[:, None].expand(-1, experts).clone()
    step = x.abs() * torch.finfo(torch.float32).eps
    x = x - (torch.randint(0, 6, x.shape, generator=gen) * torch.maximum(step, torch.tensor(0.25))) * (torch.rand(x.shape, generator=gen) < 0.7)
    x = x.clamp(-3.3e38, 3.3e38)
    _check_balance(x.to(DEV), 3)
    _check_balance(x.to(DEV).bfloat16(), 3)
    _check_balance(x.t().contiguous().t().to(DEV), 2)


def test_balance_loss_empty_groups():
    """Groups without a row that counts add nothing and do not count in the mean; with none at all loss and gradient are zero."""
    ops = _ops()
    x = torch.randn(4, 6, 8, device=DEV)
    mask = torch.ones(4, 6, dtype=torch.bool, device=DEV)
    mask[1] = False
    mask[3, 1:] = False
    _check_balance(x, 2, mask)
    alone = ops.balance_loss(x[:1], 2)[0] + ops.balance_loss(x[2:3], 2)[0] + ops.balance_loss(x[3:, :1], 2)[0]
    assert abs(float(ops.balance_loss(x, 2, mask=mask)[0]) - float(alone) / 3) < 8 * U * float(alone)
    for y, m in ((x, torch.zeros_like(mask)), (x[:, :0], None), (x[:, :0], mask[:, :0])):
        y = y.detach().requires_grad_(True)
        loss, counts, prob = ops.balance_loss(y, 2, mask=m)
        grad, = torch.autograd.grad(loss, y)
        assert float(loss.detach()) == 0 and int(counts.sum()) == 0 and float(prob.sum()) == 0 and float(grad.abs().sum()) == 0


def test_balance_loss_not_finite():
    """A NaN or +inf in a row that counts makes the loss NaN; the counts stay within the rows."""
    ops = _ops()
    for bad in (math.nan, math.inf):
        x = torch.randn(50, 24, device=DEV)
        x[17, 5] = bad
        loss, counts, _ = ops.balance_loss(x, 2)
        assert math.isnan(float(loss)) and 0 <= int(counts.min()) and int(counts.sum()) <= 100


def test_balance_loss_gradient_against_differences():
    """Directional differences in float64 of the definition with the counts held (they are constants of the gradient)."""
    ops = _ops()
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, 37, 11, generator=gen)
    y = x.to(DEV).requires_grad_(True)
    loss, counts, _ = ops.balance_loss(y, 2, coef=3.0)
    grad, = torch.autograd.grad(loss, y)
    f = counts.cpu().double() / (37 * 2)
    value = lambda z: 3.0 * 11 * (f * torch.softmax(z, 2).mean(1)).sum() / 2
    for _ in range(4):
        d = torch.randn(x.shape, generator=gen).double()
        want = (value(x.double() + 1e-5 * d) - value(x.double() - 1e-5 * d)) / 2e-5
        got = (grad.cpu().double() * d).sum()
        # (each element within about 150 U of p (w + dot), some five times the gradient p (w - dot))
        assert abs(float(got - want)) < 5e-5 * float(grad.cpu().double().norm() * d.norm())


def test_balance_loss_checks():
    ops = _ops()
    x = torch.randn(3, 4, 8, device=DEV)
    for call, says in ((lambda: ops.balance_loss(x, 0), 'top_k'), (lambda: ops.balance_loss(x, 9), 'top_k'),
                       (lambda: ops.balance_loss(x[0, 0], 1), 'logits are'), (lambda: ops.balance_loss(x.half(), 1), 'float32 or bfloat16'),
                       (lambda: ops.balance_loss(x, 1, mask=torch.ones(4, 3, dtype=torch.bool, device=DEV)), 'mask'),
                       (lambda: ops.balance_loss(x, 1, mask=torch.ones(3, 4, device=DEV)), 'mask'),
                       (lambda: ops.balance_loss(x, 1, mask=torch.ones(3, 4, dtype=torch.bool)), 'mask'),
                       (lambda: ops.balance_loss(x, 1, coef=math.nan), 'coef'), (lambda: ops.balance_loss(x[..., :0], 1), 'experts'),
                       (lambda: ops.balance_loss(torch.zeros(1, 1025, device=DEV), 1), 'experts'), (lambda: ops.balance_loss(x[:0], 1), 'groups')):
        with pytest.raises(RuntimeError, match=says):
            call()


def test_balance_loss_autograd_limits():
    """Logits or mask changed in place after the forward pass, and a second derivative, are errors; two backward passes are not."""
    ops = _ops()
    x = torch.randn(40, 12, device=DEV, requires_grad=True)
    mask = torch.ones(40, dtype=torch.bool, device=DEV)
    loss = ops.balance_loss(x, 2, mask=mask)[0]
    a, = torch.autograd.grad(loss, x, retain_graph=True)
    b, = torch.autograd.grad(loss, x, retain_graph=True)
    assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match='second derivative'):
        torch.autograd.grad(loss, x, create_graph=True)
    mask[3] = False
    with pytest.raises(RuntimeError, match='modified by an inplace'):
        torch.autograd.grad(loss, x)
    loss = ops.balance_loss(x, 2)[0]
    with torch.no_grad():
        x += 1
    with pytest.raises(RuntimeError, match='modified by an inplace'):
        torch.autograd.grad(loss, x)
    counts, prob = ops.balance_loss(x, 2)[1:]
    assert not counts.requires_grad and not prob.requires_grad
    y = x.detach().expand(3, 40, 12)
    _check_balance(y, 2)


def test_balance_loss_repeats_itself_on_any_stream():
    ops = _ops()
    x = torch.randn(3, 5000, 72, device=DEV, dtype=torch.bfloat16).requires_grad_(True)
    def once():
        loss, counts, prob = ops.balance_loss(x, 4)
        return (loss.detach(), counts, prob) + torch.autograd.grad(loss, x)
    first = once()
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in side:
        with torch.cuda.stream(s):
            got.append(once())
    torch.cuda.synchronize()
    for other in got + [once()]:
        assert all(torch.equal(a, b) for a, b in zip(first, other))


def test_balance_loss_in_a_graph():
    """Captured forward and backward, replayed with other logits and eager calls in between."""
    ops = _ops()
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(2, 300, 48, generator=gen).to(DEV).requires_grad_(True)
    up = torch.tensor(0.5, device=DEV)
    def once():
        loss, counts, prob = ops.balance_loss(x, 3)
        return (loss.detach(), counts, prob) + torch.autograd.grad(loss, x, grad_outputs=up)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, once()))
    for _ in range(3):
        for graph, out in graphs:
            with torch.no_grad():
                x.copy_(torch.randn(2, 300, 48, generator=gen))
            graph.replay()
            want = once()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_balance_loss_offsets_past_32_bits():
    """2^32 logits and some: the last rows and the counts."""
    ops = _ops()
    rows, experts = (1 << 24) + 3, 256
    x = torch.zeros(rows, experts, dtype=torch.bfloat16, device=DEV)
    x[:, 7] = 4.0
    x[-2:, 7], x[-2:, 200] = 0.0, 4.0
    x.requires_grad_(True)
    loss, counts, prob = ops.balance_loss(x, 1)
    grad, = torch.autograd.grad(loss, x, grad_outputs=torch.tensor(float(rows), device=DEV))
    want = torch.zeros(experts, dtype=torch.int64)
    want[7], want[200] = rows - 2, 2
    assert torch.equal(counts.cpu(), want)
    e4 = math.exp(4.0)
    assert abs(float(prob[7]) - e4 / (e4 + 255)) < 1e-5
    p = torch.softmax(torch.cat([x[:1], x[-2:]]).detach().double().cpu(), 1)
    w = experts * want.double() / rows
    g = p * (w - (p * w).sum(1, keepdim=True))
    got = torch.cat([grad[:1], grad[-2:]]).double().cpu()
    assert float((got - g).abs().max()) < 2.0 ** -8 * float(g.abs().max()) * 1.1
    del x, grad


# ---------------------------------------------------------------------------------------------- grad_norm

def _norm_ref(ts):
    return math.sqrt(sum(float(t.detach().double().cpu().square().sum()) for t in ts))


@pytest.mark.parametrize('sizes', [(1,), (3, 5, 0, 8192, 8193), (16384, 16385, 70001, 2), tuple(range(1, 420)), (1 << 22,), (0,)])
@pytest.mark.parametrize('dtypes', [(torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16)])
def test_grad_norm(sizes, dtypes):
    ops = _ops()
    gen = torch.Generator().manual_seed(len(sizes))
    ts = [(torch.randn(n, generator=gen) * 10.0 ** float(torch.randn((), generator=gen))).to(DEV, dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]
    want = _norm_ref(ts)
    norm, clip = ops.grad_norm(ts, max_norm=0.75)
    assert norm.dtype == clip.dtype == torch.float32 and norm.shape == clip.shape == ()
    # (float64 sums: what is left is the rounding of the result)
    assert abs(float(norm) - want) <= 1.001 * U * want
    assert abs(float(clip) - min(1.0, 0.75 / (want + 1e-6))) <= 1.001 * U
    again = ops.grad_norm(ts, max_norm=0.75)
    assert torch.equal(norm, again[0]) and torch.equal(clip, again[1])
    assert float(ops.grad_norm(ts)[1]) == 1.0


def test_grad_norm_views_and_range():
    """Addresses off 16 bytes, strides, values whose squares leave float32's range, and what is not finite."""
    ops = _ops()
    base = torch.randn(40000, device=DEV)
    b16 = torch.randn(300, 200, device=DEV).bfloat16()
    ts = [base[1:30001], base[::3], b16[:, 3:150], b16.t(), b16.reshape(-1)[1:], base[:35000].view(7, 5000).t()]
    assert abs(float(ops.grad_norm(ts)[0]) - _norm_ref(ts)) <= 1.001 * U * _norm_ref(ts)
    for scale in (1e-30, 1e30):
        t = torch.full((1000,), scale, device=DEV)
        assert abs(float(ops.grad_norm([t])[0]) / (scale * math.sqrt(1000)) - 1) < 4 * U
    huge = torch.full((1 << 20,), 3e38, device=DEV)                      # the norm leaves float32, the clip factor does not
    norm, clip = ops.grad_norm([huge], max_norm=1.0)
    # (3.3e-42 is below float32's smallest normal value: its step there is 2^-149, 4e-4 of it; or it is flushed to zero)
    assert math.isinf(float(norm)) and (abs(float(clip) * 3e38 * 1024 - 1) < 1e-3 or float(clip) == 0.0)
    for bad in (math.nan, math.inf, -math.inf):
        t = torch.ones(9000, device=DEV)
        t[8999] = bad
        norm, clip = ops.grad_norm([base, t], max_norm=1.0)
        assert not math.isfinite(float(norm)) and math.isnan(float(clip))
    with pytest.raises(RuntimeError, match='float32 or bfloat16'):
        ops.grad_norm([base.double()])
    with pytest.raises(RuntimeError, match='max_norm'):
        ops.grad_norm([base], max_norm=-1.0)


# ---------------------------------------------------------------------------------------------- AdamW

HYPER = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)
M32 = 0xFFFFFFFF


def _mix(x):
    x = ((x ^ (x >> 16)) * 0x455c2ed3) & M32
    x = ((x ^ (x >> 15)) * 0x55a35cd1) & M32
    return x ^ (x >> 16)


def _noise(seed, step, position, index):
    """(32 bits for the 8-bit moments, 16 for a bfloat16 parameter) of the elements ``index`` (int64)."""
    base = _mix((step & M32) ^ _mix((step >> 32) ^ _mix((seed & M32) ^ _mix(((seed >> 32) + 1) & M32))))
    key = _mix((base + position) & M32)
    hi = index >> 32
    keys = torch.where(hi > 0, _mix((key + hi) & M32), key)
    return _mix((index & M32) ^ keys), _mix((index & M32) ^ _mix(keys ^ 0x6f002d25)) & 0xFFFF


def _update64(p, g, m, v, step, clip=1.0, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0):
    """float64: p, m, v after the step and the bounds of their float32 errors."""
    p, g, m, v = (t.detach().double().cpu() for t in (p, g, m, v))
    b1, b2 = betas
    g = g * clip
    m1, v1 = m + (1 - b1) * (g - m), b2 * v + (1 - b2) * g * g
    root = (v1 / (1 - b2 ** step)).sqrt() + eps
    s = lr / (1 - b1 ** step)
    p1 = p * (1 - lr * weight_decay) - s * m1 / root
    # roundings: g clip, g - m, times w1 (itself rounded), the sum; beta2 v, w2 g g (three products), the sum; sqrt and two
    # quotients, the step's product and constants, p's product and difference
    dm, dv = 6 * U * (m.abs() + g.abs()), 7 * U * v1
    dp = 4 * U * (p.abs() + p1.abs()) + s * (dm + 12 * U * m1.abs()) / root
    return p1, m1, v1, dp + 1e-40, dm + 1e-40, dv + 1e-40


def _grid(x, man, low):
    """(largest grid value <= |x|, the step there) of a float with ``man`` mantissa bits and smallest exponent ``low``; x float64 >= 0."""
    e = (torch.frexp(x)[1] - 1).clamp(min=low).double()
    step = torch.exp2(e - man)
    return torch.floor(x / step) * step, step


def _tensors(sizes, dtype, gen, offset=0):
    """p, g, m, v lists at addresses ``offset`` elements off an aligned one, and the guarded buffers they lie in."""
    out, guards = [[], [], [], []], []
    for n in sizes:
        for k, (t, lst) in enumerate(zip((dtype, dtype, torch.float32, torch.float32), out)):
            buf = torch.randn(n + offset + 300, generator=gen)
            if k == 3:
                buf = buf.square() * 0.1
            buf = (buf * 0.3).to(DEV, t)
            lst.append(buf[offset:offset + n])
            if k != 1:
                guards.append((buf, offset, n, buf.clone()))
    return out, guards


def _check_guards(guards):
    for buf, o, n, was in guards:
        assert torch.equal(buf[:o].view(torch.uint8), was[:o].view(torch.uint8)) and torch.equal(buf[o + n:].view(torch.uint8), was[o + n:].view(torch.uint8))


SIZES = (1, 3, 4, 255, 256, 257, 4095, 4096, 4097, 12289, 70001)


@pytest.mark.parametrize('clip', [None, 0.3])
@pytest.mark.parametrize('offset', [0, 1])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_adamw_step(dtype, offset, clip):
    ops = _ops()
    gen = torch.Generator().manual_seed(3)
    (p, g, m, v), guards = _tensors(SIZES, dtype, gen, offset)
    was = [[t.clone() for t in lst] for lst in (p, g, m, v)]
    factor = None if clip is None else torch.tensor(clip, device=DEV)
    c = 1.0 if clip is None else float(factor)
    ops.adamw_step(p, g, m, v, 4, clip=factor, seed=11, **HYPER)
    _check_guards(guards)
    drift, count = 0.0, 0
    for i in range(len(SIZES)):
        p1, m1, v1, dp, dm, dv = _update64(*(lst[i] for lst in was), 4, c, **HYPER)
        assert bool(((m[i].cpu().double() - m1).abs() <= dm).all()) and bool(((v[i].cpu().double() - v1).abs() <= dv).all())
        got = p[i].cpu().double()
        if dtype == torch.float32:
            assert bool(((got - p1).abs() <= dp).all())
        else:
            # one of the two neighbours, and which of them is the random bits' choice: up with the cut-off part's probability
            low, step = _grid(p1.abs(), 7, -126)
            assert bool(((got - p1).abs() <= step + dp).all())
            bits = _noise(11, 4, i, torch.arange(SIZES[i]))[1].double() / 65536
            frac = (p1.abs() - low) / step
            sure = (frac + bits - 1).abs() > dp / step + 2.0 ** -20
            want = torch.copysign(low + step * (frac + bits >= 1), p1)
            assert bool((got == want)[sure].all()) and float(sure.double().mean()) > 0.9 or SIZES[i] < 10
            drift, count = drift + float(((got.abs() - p1.abs()) / step).sum()), count + SIZES[i]
    if count:
        assert abs(drift / count) < 5 * 0.5 / math.sqrt(count)               # (a step's rounding has at most half a step of deviation)


def _random_states8(sizes, gen, offset=0):
    """Codes over the whole range (no NaN, no infinity), scales 2^-20 .. 2^-4."""
    ms, es, vs, fs = [], [], [], []
    for n in sizes:
        blocks = -(-n // 256)
        code = lambda top, sign: torch.randint(0, top, (n + offset,), generator=gen) + (torch.randint(0, 2, (n + offset,), generator=gen) * 128 if sign else 0)
        ms.append(code(0x79, True).to(torch.uint8).to(DEV)[offset:].view(torch.float8_e4m3fn))
        vs.append(code(0x79, False).to(torch.uint8).to(DEV)[offset:].view(torch.float8_e5m2))
        es.append(torch.randint(107, 124, (blocks,), generator=gen).to(torch.uint8).to(DEV).view(torch.float8_e8m0fnu))
        fs.append(torch.randint(87, 104, (blocks,), generator=gen).to(torch.uint8).to(DEV).view(torch.float8_e8m0fnu))
    return ms, es, vs, fs


def _bytes(t):
    return t.detach().reshape(-1).view(torch.uint8).cpu()


def _decode(x8, e8):
    n = x8.numel()
    return x8.reshape(-1).cpu().float().double() * torch.repeat_interleave(torch.exp2(_bytes(e8).double() - 127), 256)[:n]


def _encode(x, noise, man, low, room, least):
    """float32 magnitudes as (grid value, sure?) and the blocks' exponents; ``noise`` in [0, 1): up where the cut-off part and it reach 1."""
    n = x.numel()
    pad = torch.zeros(-(-n // 256) * 256, dtype=torch.float64)
    pad[:n] = torch.where(torch.isfinite(x), x, 0.0)
    most = pad.view(-1, 256).amax(1)
    e = torch.where(most > 0, (torch.frexp(most)[1] - 1).double() - room, -math.inf).clamp(min=-126)
    scale = torch.repeat_interleave(torch.exp2(e), 256)[:n]
    lowv, step = _grid(x / scale, man, low)
    frac = (x / scale - lowv) / step
    y = lowv + step * (frac + noise >= 1)
    return torch.where(x > 0, y.clamp(min=least), y) * scale, e, frac


@pytest.mark.parametrize('clip', [None, 0.3])
@pytest.mark.parametrize('offset', [0, 1])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_adamw8_step(dtype, offset, clip):
    """Against the definition: float32 arithmetic on the decoded moments (each operation rounded once, so the CPU's float32 agrees to
    the bit), the blocks' powers of two and every code."""
    ops = _ops()
    gen = torch.Generator().manual_seed(4)
    (p, g, _, _), guards = _tensors(SIZES, dtype, gen, offset)
    ms, es, vs, fs = _random_states8(SIZES, gen, offset)
    for t in g:
        t.mul_(0.01)
    was = [[t.clone() for t in lst] for lst in (p, g)]
    dec = [(_decode(a, b), _decode(c, d)) for a, b, c, d in zip(ms, es, vs, fs)]
    factor = None if clip is None else torch.tensor(clip, device=DEV)
    ops.adamw8_step(p, g, ms, es, vs, fs, 4, clip=factor, seed=(5 << 32) + 11, **HYPER)
    _check_guards([x for k, x in enumerate(guards) if k % 3 == 0])
    up, count = 0.0, 0
    f32 = lambda x: torch.tensor(x, dtype=torch.float32)
    b1, b2 = HYPER['betas']
    for i, n in enumerate(SIZES):
        m0, v0 = (t.float() for t in dec[i])
        gi = was[1][i].cpu().float()
        if clip is not None:
            gi = gi * f32(clip)
        m1 = m0 + f32(1 - b1) * (gi - m0)
        v1 = v0 * f32(b2) + f32(1 - b2) * gi * gi
        p1, _, _, dp, _, _ = _update64(was[0][i], was[1][i], *dec[i], 4, 1.0 if clip is None else float(f32(clip)), **HYPER)
        h, hp = _noise((5 << 32) + 11, 4, i, torch.arange(n))
        got = p[i].cpu().double()
        assert bool(((got - p1).abs() <= dp + (_grid(p1.abs(), 7, -126)[1] if dtype == torch.bfloat16 else 0)).all())
        wm, em, fm = _encode(m1.abs().double(), ((h & 0xFFFF).double() + 0.5) / 65536, 3, -6, 7, 0.0)
        wv, ev, _ = _encode(v1.double(), ((h >> 16).double() + 0.5) / 65536, 2, -14, 14, 2.0 ** -16)
        assert torch.equal(_bytes(es[i]).double() - 127, em) and torch.equal(_bytes(fs[i]).double() - 127, ev)
        assert torch.equal(_decode(ms[i], es[i]), torch.copysign(wm, m1.double())) and torch.equal(_decode(vs[i], fs[i]), wv)
        up, count = up + float(((_decode(ms[i], es[i]).abs() > m1.abs().double()).double() - fm).sum()), count + n
    assert abs(up / count) < 5 * 0.5 / math.sqrt(count)              # rounded up as often as the cut-off parts say


def test_adamw8_zero_state_and_zero_gradients():
    """From zero moments; blocks that never saw a gradient stay zero (and their parameters only decay); a second moment above zero
    is never rounded to zero, however far below the block's largest."""
    ops = _ops()
    p = torch.ones(1024, device=DEV)
    g = torch.zeros(1024, device=DEV)
    g[256:512] = 1e-9
    g[256] = 1e3
    m, e, v, f = ops.adamw8_state(p)
    for t in range(1, 40):
        ops.adamw8_step([p], [g], [m], [e], [v], [f], t, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
        assert bool((v.view(torch.uint8)[256:512] > 0).all())
        g[257:300] = 0.0                                     # (the first step only: m / sqrt(v) must not blow up afterwards)
    assert bool((_bytes(m)[:256] == 0).all()) and bool((_bytes(v)[512:] == 0).all()) and bool((p[:256] == 1).all()) and bool((p[512:] == 1).all())
    assert bool((p > 0.9).all()) and bool((p <= 1.0).all())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_adamw8_second_moments_near_zero(dtype):
    """Blocks whose second moments span what e5m2 does not, that underflow as a whole, or that are alike: every code by the definition, and
    none above zero becomes zero."""
    ops = _ops()
    gen = torch.Generator().manual_seed(8)
    g = torch.randn(7, 256, generator=gen)
    g[0] *= torch.logspace(-12, 0, 256)                  # beside ordinary ones
    g[1, 1:] = 0.0                                       # one value and zeros
    g[2, :200] *= 1e-7
    g[3] *= 1e-19                                        # squares below the normal range
    g[4] *= 1e-25                                        # squares that are zero
    g[5, 100] = 1e15
    g = g.reshape(-1)[:7 * 256 - 31].to(dtype)
    p = torch.zeros(g.numel(), device=DEV, dtype=dtype)
    m, e, v, f = ops.adamw8_state(p)
    ops.adamw8_step([p], [g.to(DEV)], [m], [e], [v], [f], 1, seed=21, **HYPER)
    f32 = lambda x: torch.tensor(x, dtype=torch.float32)
    gi = g.float()
    v1 = torch.zeros(()) * f32(HYPER['betas'][1]) + f32(1 - HYPER['betas'][1]) * gi * gi
    h, _ = _noise(21, 1, 0, torch.arange(g.numel()))
    wv, ev, _ = _encode(v1.double(), ((h >> 16).double() + 0.5) / 65536, 2, -14, 14, 2.0 ** -16)
    assert torch.equal(_bytes(f).double() - 127, ev) and torch.equal(_decode(v, f), wv)
    assert bool(((wv > 0) == (v1 > 0)).all()) and int((v1 == 0).sum()) > 400


def test_adamw8_follows_the_gradients():
    """What rounding to the nearest would lose: with beta2 = 0.999 every step moves v by far less than half of a code's step, and
    the mean of v still follows 1 - 0.999^t (its deviation over 65536 elements is below 1 %)."""
    ops = _ops()
    p = torch.zeros(65536, device=DEV)
    g = torch.ones(65536, device=DEV)
    st = ops.adamw8_state(p)
    for t in range(1, 3001):
        ops.adamw8_step([p], [g], *[[s] for s in st], t, lr=0.0)
    want = 1 - 0.999 ** 3000
    got = float(_decode(st[2], st[3]).mean())
    assert abs(got / want - 1) < 0.03, got
    m = _decode(st[0], st[1])
    assert abs(float(m.mean()) - 1) < 0.01


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_adamw_not_finite(bits, dtype):
    """A NaN clip factor leaves everything as it is; without one an element that is not finite spoils itself alone."""
    ops = _ops()
    def fresh():
        gen = torch.Generator().manual_seed(6)
        p, g = (torch.randn(1000, generator=gen).to(DEV, dtype) for _ in range(2))
        if bits == 8:
            return p, g, list(ops.adamw8_state(p)), lambda s, t, **k: ops.adamw8_step([p], [g], *[[x] for x in s], t, **k)
        return p, g, [torch.zeros(1000, device=DEV) for _ in range(2)], lambda s, t, **k: ops.adamw_step([p], [g], *[[x] for x in s], t, **k)
    p, g, s, call = fresh()
    was = [x.clone() for x in (p, *s)]
    call(s, 1, clip=torch.tensor(math.nan, device=DEV))
    assert all(torch.equal(_bytes(a), _bytes(b)) for a, b in zip((p, *s), was))
    call(s, 1)
    good = [_bytes(x) for x in (p, *s)]
    p, g, s, call = fresh()
    g[100], g[700], g[701] = math.nan, math.inf, -math.inf
    call(s, 1)
    for a, b, x in zip((_bytes(y) for y in (p, *s)), good, (p, *s)):
        per = a.numel() // x.numel()
        if x.numel() == 1000:
            keep = torch.ones(1000, dtype=torch.bool)
            keep[[100, 700, 701]] = False
            if bits == 32 or x is p:
                assert torch.equal(a.view(1000, per)[keep], b.view(1000, per)[keep])
            assert not bool(torch.isfinite(x.float())[~keep].any()) if x is not p else bool(torch.isfinite(p.float())[keep].all())


def test_adamw_lists_layouts_and_types():
    """More tensors than a launch takes, empty ones among them, float32 and bfloat16, 8- and 32-bit moments in one list, channels-last
    parameters, gradients of other strides: the same values as tensor by tensor (position 0 .. n - 1 kept by empty tensors)."""
    ops = _ops()
    gen = torch.Generator().manual_seed(8)
    ps, gs, ms, es, vs, fs, kinds = [], [], [], [], [], [], []
    for i in range(150):
        shape = [(0,), (33, 7), (4, 3, 2, 5, 6), (513,), (2, 8, 5, 5)][i % 5]
        dtype = torch.bfloat16 if i % 3 == 1 else torch.float32
        p = torch.randn(shape, generator=gen).to(DEV, dtype)
        g = torch.randn(shape, generator=gen).to(DEV, dtype)
        if len(shape) == 5:
            p = p.contiguous(memory_format=torch.channels_last_3d)
        if len(shape) == 4:
            p, g = p.contiguous(memory_format=torch.channels_last), g.transpose(2, 3)
        if len(shape) == 2:
            p = p.t()
            g = torch.randn(tuple(p.shape), generator=gen).to(DEV, dtype)
        if i % 2:
            m, e, v, f = ops.adamw8_state(p)
            assert m.stride() == p.stride()
        else:
            m, v = (torch.zeros_like(p, dtype=torch.float32) for _ in range(2))
            e = f = torch.empty(0, device=DEV)
        for lst, x in zip((ps, gs, ms, es, vs, fs), (p, g, m, e, v, f)):
            lst.append(x)
    single = [[x.clone() for x in lst] for lst in (ps, gs, ms, es, vs, fs)]
    before = [p._version for p in ps]
    ops.adamw8_step(ps, gs, ms, es, vs, fs, 1, seed=3, **HYPER)
    assert all(p._version > b for p, b in zip(ps, before))
    empty = [torch.zeros(0, device=DEV) for _ in range(2)]
    for i in range(150):
        one = [lst[i] for lst in single]
        assert one[0].stride() == ps[i].stride()
        z = [empty[0]] * i
        none = [torch.empty(0, device=DEV, dtype=torch.float32)] * i
        ops.adamw8_step(z + [one[0]], z + [one[1]], none + [one[2]], none + [one[3]], none + [one[4]], none + [one[5]], 1, seed=3, **HYPER)
        for a, b in zip((ps, ms, es, vs, fs), (one[0], one[2], one[3], one[4], one[5])):
            assert torch.equal(a[i].contiguous().reshape(-1).view(torch.uint8), b.contiguous().reshape(-1).view(torch.uint8)), i


def test_adamw_refusals():
    ops = _ops()
    z = lambda n=8, d=torch.float32: torch.zeros(n, device=DEV, dtype=d)
    p, g, m, v = z(), z(), z(), z()
    m8, e8, v8, f8 = ops.adamw8_state(p)
    bad = [
        (lambda: ops.adamw_step([p, p], [g, g], [m, z()], [v, z()], 1), 'share memory'),
        (lambda: ops.adamw_step([p], [g], [m], [m], 1), 'share memory'),
        (lambda: ops.adamw_step([p[:5], p[4:]], [g[:5], g[4:]], [m[:5], m[4:]], [v[:5], v[4:]], 1), 'share memory'),
        (lambda: ops.adamw_step([p[::2]], [g[::2]], [m[::2]], [v[::2]], 1), 'dense'),
        (lambda: ops.adamw_step([z(1).expand(8)], [g], [m], [v], 1), 'dense'),
        (lambda: ops.adamw_step([p.half()], [g.half()], [m], [v], 1), 'float32 or bfloat16'),
        (lambda: ops.adamw_step([p], [g.bfloat16()], [m], [v], 1), 'gradient 0'), (lambda: ops.adamw_step([p], [g[:4]], [m], [v], 1), 'gradient 0'),
        (lambda: ops.adamw_step([p], [g.cpu()], [m], [v], 1), 'gradient 0'), (lambda: ops.adamw_step([p], [g], [m.bfloat16()], [v], 1), 'moments'),
        (lambda: ops.adamw_step([p], [g], [m8], [v], 1), 'moments'), (lambda: ops.adamw_step([p], [g], [m[:4]], [v], 1), 'moments'),
        (lambda: ops.adamw_step([p], [g], [m8], [v8], 1), 'need their scales'),
        (lambda: ops.adamw8_step([p], [g], [m8], [e8.view(torch.uint8)], [v8], [f8], 1), 'scales'),
        (lambda: ops.adamw8_step([p], [g], [m8], [z(2).to(torch.float8_e8m0fnu)], [v8], [f8], 1), 'scales'),
        (lambda: ops.adamw8_step([p], [g], [m8], [e8], [v8], [e8], 1), 'share memory'),
        (lambda: ops.adamw_step([p], [g], [m], [v], 0), 'starts at 1'), (lambda: ops.adamw_step([p], [g], [m], [v], 1, lr=-1.0), 'hyper-parameters'),
        (lambda: ops.adamw_step([p], [g], [m], [v], 1, clip=torch.ones(1)), 'clip'), (lambda: ops.adamw_step([p], [g], [m], [v], 1, clip=z(2)), 'clip'),
        (lambda: ops.adamw_step([p], [g], [m], [v], torch.zeros(1, device=DEV)), 'step count'),
        (lambda: ops.adamw_step([p], [g], [m], [v], 1, lr=torch.tensor(1e-3, device=DEV)), 'learning rate')]
    for call, says in bad:
        with pytest.raises(RuntimeError, match=says):
            call()
    assert float(p.abs().sum() + m.abs().sum() + v.abs().sum()) == 0


def test_adamw8_offsets_past_32_bits():
    """A tensor of more than 2^32 elements: the elements around that border and the last ones."""
    ops = _ops()
    n = (1 << 32) + 4096 + 77
    p = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    g = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    at = torch.tensor([0, 5, (1 << 31) + 9, (1 << 32) - 1, 1 << 32, (1 << 32) + 4000, n - 2, n - 1])
    g[at.to(DEV)] = torch.arange(1, 9, device=DEV).bfloat16()
    assert abs(float(ops.grad_norm([g])[0]) - math.sqrt(204)) < 1e-5
    m, e, v, f = ops.adamw8_state(p)
    ops.adamw8_step([p], [g], [m], [e], [v], [f], 1, lr=0.5, weight_decay=0.0, seed=3)
    assert int((m.view(torch.uint8) != 0).sum()) == 8 and int((v.view(torch.uint8) != 0).sum()) == 8
    for j, i in enumerate(at.tolist()):
        h, hp = _noise(3, 1, 0, torch.tensor([i]))
        # m = 0.1 g, v = 0.001 g^2, p = -lr (sign of g)
        assert abs(float(p[i]) + 0.5) <= 2.0 ** -8, i
        for x8, e8, want, man in ((m, e, 0.1 * (j + 1), 3), (v, f, 0.001 * (j + 1) ** 2, 2)):
            got = float(x8[i].float()) * float(e8[i // 256].float())
            assert abs(got - want) <= want * 2.0 ** -man, (i, got, want)
        bits = float(h & 0xFFFF)
        scale = 2.0 ** (math.floor(math.log2(0.1 * max(k + 1 for k, o in enumerate(at.tolist()) if o // 256 == i // 256))) - 7)
        low, step = _grid(torch.tensor([float(torch.tensor(0.1) * (j + 1)) / scale], dtype=torch.float64), 3, -6)
        frac = float((torch.tensor(0.1) * (j + 1)).double() / scale - low) / float(step)
        if abs(frac + (bits + 0.5) / 65536 - 1) > 1e-4:
            assert float(m[i].float()) == float(low + step * (frac + (bits + 0.5) / 65536 >= 1)), i
    assert int((p != 0).sum()) == 8


@pytest.mark.parametrize('bits', [32, 8])
def test_adamw_in_a_graph(bits):
    """norm + step captured once, with the count and the learning rate on the device, replayed between eager steps of a second copy:
    bit for bit the same."""
    ops = _ops()
    gen = torch.Generator().manual_seed(9)
    sizes, dtypes = (5000, 300, 70001, 64), (torch.float32, torch.bfloat16, torch.float32, torch.bfloat16)
    def make():
        ps = [torch.randn(n, generator=torch.Generator().manual_seed(n)).to(DEV, d) for n, d in zip(sizes, dtypes)]
        gs = [torch.zeros_like(p) for p in ps]
        st = [ops.adamw8_state(p) if bits == 8 else (torch.zeros_like(p, dtype=torch.float32), torch.zeros(0, device=DEV),
                                                    torch.zeros_like(p, dtype=torch.float32), torch.zeros(0, device=DEV)) for p in ps]
        return ps, gs, [list(x) for x in zip(*st)]
    a, b = make(), make()
    count, lr = torch.zeros(1, dtype=torch.int64, device=DEV), torch.tensor(1e-2, device=DEV)
    def step(s, t, rate):
        norm, clip = ops.grad_norm(s[1], max_norm=5.0)
        ops.adamw8_step(s[0], s[1], *s[2], t, lr=rate, clip=clip, seed=77)
        return norm
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        norm = step(a, count, lr)
    for t in range(1, 6):
        for x, y in zip(a[1], b[1]):
            x.copy_(torch.randn(x.numel(), generator=gen))
            y.copy_(x)
        rate = 1e-2 / t
        lr.fill_(rate)
        graph.replay()
        want = step(b, t, float(torch.tensor(rate, dtype=torch.float32)))
        torch.cuda.synchronize()
        assert int(count) == t and torch.equal(norm, want)
        for x, y in zip(a[0] + sum(a[2], []), b[0] + sum(b[2], [])):
            assert torch.equal(_bytes(x), _bytes(y)), t


def test_adamw_optimizer_in_a_graph():
    """optim.AdamW(capturable=True): two groups (8- and 32-bit moments, one learning rate on the device) captured and replayed against a
    twin that steps launch by launch; a state loaded in between goes into the tensors that the graph holds; what a capture must not
    hold is refused."""
    import copy
    from repmode_amd.optim import AdamW
    _ops()
    def make(capturable):
        ps = [torch.nn.Parameter(torch.randn(n, generator=torch.Generator().manual_seed(n)).to(DEV)) for n in (5000, 300, 9000)]
        lr = torch.tensor(1e-2, device=DEV) if capturable else 1e-2
        return ps, AdamW([dict(params=ps[:2], state_bits=8), dict(params=ps[2:], lr=lr)], lr=2e-3, max_norm=1.0, capturable=capturable, seed=4)
    (ps, opt), (qs, twin) = make(True), make(False)
    gen = torch.Generator().manual_seed(1)
    def grads():
        for p, q in zip(ps, qs):
            g = torch.randn(p.shape, generator=gen).to(DEV)
            q.grad = g.clone()
            if p.grad is None:
                p.grad = g
            else:
                p.grad.copy_(g)
    def same():
        for p, q in zip(ps, qs):
            assert torch.equal(p, q)
            for k, v in twin.state[q].items():
                if k != 'step':
                    assert torch.equal(_bytes(opt.state[p][k]), _bytes(v)), k
    twin.param_groups[1]['lr'] = float(torch.tensor(1e-2, dtype=torch.float32))
    grads()
    opt.step()
    twin.step()
    same()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    saved = None
    for t in range(4):
        if t == 2:
            saved = copy.deepcopy(twin.state_dict()), [q.detach().clone() for q in qs]
        grads()
        opt.param_groups[1]['lr'].fill_(1e-2 / (t + 1))
        twin.param_groups[1]['lr'] = float(torch.tensor(1e-2 / (t + 1), dtype=torch.float32))
        graph.replay()
        twin.step()
        same()
    sd = opt.state_dict()
    assert all(int(s['step']) == 5 for s in sd['state'].values())
    held = opt.param_groups[1]['lr']
    opt.load_state_dict(saved[0])
    twin.load_state_dict(copy.deepcopy(saved[0]))
    opt.param_groups[1]['lr'] = held
    with torch.no_grad():
        for p, q, v in zip(ps, qs, saved[1]):
            p.copy_(v)
            q.copy_(v)
    twin.param_groups[1]['lr'] = float(held)
    grads()
    graph.replay()
    twin.step()
    same()
    late = torch.nn.Parameter(torch.zeros(8, device=DEV))
    late.grad = torch.zeros(8, device=DEV)
    for bad, says in ((AdamW([late]), 'needs capturable'), (AdamW([late], capturable=True), 'must not be a captured one')):
        with pytest.raises(RuntimeError, match=says):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                bad.step()
    torch.cuda.synchronize()


def test_adamw_on_device_counts_are_a_groups():
    """capturable: a parameter whose first gradient comes after the others' would be corrected by their step count: refused."""
    from repmode_amd.optim import AdamW
    _ops()
    ps = [torch.nn.Parameter(torch.ones(8, device=DEV)) for _ in range(2)]
    opt = AdamW(ps, capturable=True)
    ps[0].grad = torch.ones(8, device=DEV)
    opt.step()
    ps[1].grad = torch.ones(8, device=DEV)
    with pytest.raises(RuntimeError, match='same number of steps'):
        opt.step()
    assert torch.equal(ps[1].detach(), torch.ones(8, device=DEV))


def test_operators_take_strided_tensors():
    ops = _ops()
    t = torch.zeros(4, 4, device=DEV)
    s = torch.sparse_coo_tensor(torch.zeros(2, 1, dtype=torch.long, device=DEV), torch.ones(1, device=DEV), (4, 4))
    for call in (lambda: ops.grad_norm([t, s]), lambda: ops.balance_loss(s, 1), lambda: ops.adamw_step([s], [t], [t.clone()], [t.clone()], 1),
                 lambda: ops.adamw_step([t], [s], [t.clone()], [t.clone()], 1)):
        with pytest.raises(RuntimeError, match='strided|dense|gradient 0'):
            call()


# ---------------------------------------------------------------------------------------------- together

def _stock_twin(params, **kw):
    twins = [torch.nn.Parameter(p.detach().float().cpu().clone()) for p in params]
    return twins, torch.optim.AdamW(twins, **kw)


def test_optimizer_against_torch_adamw():
    """optim.AdamW with two groups and clipping against torch.optim.AdamW + clip_grad_norm_ on the CPU."""
    from repmode_amd.optim import AdamW
    _ops()
    gen = torch.Generator().manual_seed(12)
    shapes = [(64, 33), (7,), (3, 5, 5, 5, 5), (10000,)]
    ps = [torch.nn.Parameter(torch.randn(s, generator=gen).to(DEV)) for s in shapes]
    twins = [torch.nn.Parameter(p.detach().cpu().clone()) for p in ps]
    split = lambda q: [dict(params=q[:2]), dict(params=q[2:], weight_decay=0.0, lr=5e-3)]
    ours, stock = AdamW(split(ps), lr=1e-2, max_norm=1.0), torch.optim.AdamW(split(twins), lr=1e-2)
    for t in range(4):
        for p, q in zip(ps, twins):
            q.grad = torch.randn(q.shape, generator=gen)
            p.grad = q.grad.to(DEV)
        if t == 2:
            ps[1].grad = twins[1].grad = None
        want = torch.nn.utils.clip_grad_norm_([q for q in twins if q.grad is not None], 1.0)
        ours.step()
        stock.step()
        assert abs(float(ours.last_norm) - float(want)) < 1e-5 * float(want)
        for p, q in zip(ps, twins):
            # a step moves by lr m / sqrt(v): both sides' roundings of it, and p's
            assert float((p.detach().cpu() - q.detach()).abs().max()) < (t + 1) * (8 * U * float(q.detach().abs().max()) + 64 * U * 1e-2 * 4)
    assert [int(ours.state[p]['step']) for p in ps] == [4, 3, 4, 4]


@pytest.mark.parametrize('graph', [False, True])
@pytest.mark.parametrize('bits', [32, 8])
def test_model_trains_with_the_operators(bits, graph):
    """Model with AdamW, clipping and the gates' balance term, launch by launch and as a replayed graph: each step's update is
    the definition's, from the step's own gradients."""
    from repmode_amd.model import Model
    _ops()
    torch.manual_seed(0)
    m = Model(Opts(), lr=1e-3, gpu_ids=0, mult_chan=2, dtype=torch.float32, hip_graph=graph, optimizer='adamw', balance_coef=0.25,
              optimizer_args=dict(max_norm=0.01, weight_decay=0.05, state_bits=bits, min_8bit_numel=512, seed=5))
    gen = torch.Generator().manual_seed(1)
    tasks = torch.tensor([1, 5, 1])
    params = list(m.net.parameters())
    for t in range(1, 6):
        x, y = (torch.randn(3, 1, 16, 16, 32, generator=gen) for _ in range(2))
        before = [p.detach().clone() for p in params]
        state = [{k: v.clone() for k, v in m.optimizer.state[p].items()} if p in m.optimizer.state else None for p in params]
        m.do_train_iter(x, y, tasks)
        grads = [p.grad for p in params]
        norm = _norm_ref(grads)
        assert abs(float(m.optimizer.last_norm) - norm) < 4 * U * norm
        clip = min(1.0, 0.01 / (norm + 1e-6))
        assert clip < 1
        for p, b, s, g in zip(params, before, state, grads):
            eight = bits == 8 and p.numel() >= 512
            st = m.optimizer.state[p]
            assert (st['exp_avg'].dtype == torch.float8_e4m3fn) == eight
            if s is None:
                m0 = v0 = torch.zeros(p.shape)
            elif eight:
                m0, v0 = _decode(s['exp_avg'], s['exp_avg_scale']).view(p.shape), _decode(s['exp_avg_sq'], s['exp_avg_sq_scale']).view(p.shape)
            else:
                m0, v0 = s['exp_avg'], s['exp_avg_sq']
            p1, _, _, dp, _, _ = _update64(b, g, m0, v0, t, clip, lr=1e-3, weight_decay=0.05)
            assert bool(((p.detach().cpu().double() - p1).abs() <= 2 * dp).all())
        assert m.last_balance[1].shape == (19, 5) and int(m.last_balance[1].sum()) == 3 * sum(q.out_chan for q in m.net.modules() if hasattr(q, 'gate'))
        assert float(m.last_balance[0]) >= 0.25 * (1 - 1e-5) * 0.2
    if graph:
        assert int(m.optimizer._step_dev[0]) == 5
    sd = m.get_state()['optimizer_state']
    assert all(int(s['step']) == 5 for s in sd['state'].values())


def test_model_graph_refuses_a_held_graph():
    """An autograd graph of the network that is alive when the step is to be captured would end the process: refused instead."""
    from repmode_amd.model import Model
    _ops()
    torch.manual_seed(0)
    m = Model(Opts(), lr=1e-3, gpu_ids=0, mult_chan=2, dtype=torch.float32, hip_graph=True, optimizer='adamw', balance_coef=0.1)
    x, y, tasks = torch.randn(2, 1, 16, 16, 16), torch.randn(2, 1, 16, 16, 16), torch.tensor([0, 3])
    for _ in range(Model.GRAPH_WARMUP):
        m.do_train_iter(x, y, tasks)
    held = m.net.gate_balance([0, 3])[0]
    with pytest.raises(RuntimeError, match='release it'):
        m.do_train_iter(x, y, tasks)
    del held
    for _ in range(3):
        m.do_train_iter(x, y, tasks)
    assert math.isfinite(float(m.last_loss))


def test_gate_balance_against_the_definition():
    """Net.gate_balance: value, counts and the gates' gradients against float64 autograd of the definition."""
    from repmode_amd.nn_modules.RepMode import MoDEConv, Net
    _ops()
    torch.manual_seed(3)
    net = Net(Opts(), mult_chan=3).to(DEV)
    tasks = [4, 0, 4, 11]
    loss, counts, prob = net.gate_balance(tasks, coef=0.5, top_k=2)
    loss.backward()
    blocks = [m for m in net.modules() if isinstance(m, MoDEConv)]
    total = 0.0
    leaves = []
    for b, (m, c) in enumerate(zip(blocks, counts)):
        w, bias = (t.detach().double().cpu().requires_grad_(True) for t in (m.gate.weight, m.gate.bias))
        leaves.append((m, w, bias, 2 * 4 * 0.5 * 5 / len(blocks) / (m.out_chan * 4)))
        x = (w[:, tasks] + bias[:, None]).view(5, -1).t()
        p = torch.softmax(x, 1)
        f = c.cpu().double() / (x.shape[0] * 2)
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :2]
        assert torch.equal(torch.bincount(order.reshape(-1), minlength=5), c.cpu())
        total = total + 0.5 * 5 * (f * p.mean(0)).sum() / len(blocks)
    total.backward()
    assert abs(float(loss) - float(total)) < 40 * U * float(total)
    for m, w, bias, most in leaves:
        for got, want in ((m.gate.weight.grad, w.grad), (m.gate.bias.grad, bias.grad)):
            # up to 4 samples' terms p (w + dot) <= 2 coef E / (blocks rows), each within about 150 U of it
            assert float((got.cpu().double() - want).abs().max()) < 150 * U * most + 8 * U * float(want.abs().max())
