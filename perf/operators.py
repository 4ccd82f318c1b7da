"""The operators of a train step around the network -- the mixture's balance loss with its per-expert counts and gradient, the
norm of the gradients, and AdamW over many tensors with states in 32 or in 8 bits -- as cases, in plain torch operations and as
calls of this package.

``own`` False: ``run`` computes an operator from elementary torch operations in 32 bits; True: it calls ``repmode_amd.ops``.
"""
import math
import random

import torch

own = False

DEV = 'cuda'
BLOCK = 256                      # elements of one block of the 8-bit states
DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16}
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
M32 = 0xFFFFFFFF


# ---------------------------------------------------------------------------------------------- parameter lists

def _net(mult_chan, tasks=12):
    """numel of every parameter of this repository's U-Net: 19 blocks of five experts and a gate, 8 stride-2 stages, 26 norms."""
    m = mult_chan
    sub = [(1, m), (m, 2 * m), (2 * m, 4 * m), (4 * m, 8 * m), (8 * m, 16 * m), (16 * m, 8 * m), (8 * m, 4 * m), (4 * m, 2 * m), (2 * m, m)]
    out = []
    for i, (ci, co) in enumerate(sub):
        for a in (ci, co):
            out += [co * a * 125, co * a * 27, co * a, co * a, co * a, co, co, 5 * co * tasks, 5 * co]
        if i < 4:
            out += [co * co * 8, co, co]
        elif i < 8:
            out += [co * (co // 2) * 8, co // 2, co // 2]
    return out + [m * 125, m * 27, m, m, m, 5 * tasks, 5]


def _stack(width, layers):
    """numel of a generic stack: four square projections, two of the feed-forward, two norms and their biases a layer."""
    return [w * width for _ in range(layers) for w in (width, width, width, width, 4 * width, 4 * width, 1, 1, 1, 4)]


def _ragged(total, tensors, seed):
    """``tensors`` odd sizes, spread over their logarithm, that add up to about ``total``."""
    r = random.Random(seed)
    w = [math.exp(r.uniform(0, 6)) for _ in range(tensors)]
    return [max(1, int(total * x / sum(w))) for x in w]


def _numels(c):
    if c['list'] == 'net':
        return _net(c['width'])
    if c['list'] == 'stack':
        return _stack(c['width'], c['layers'])
    return _ragged(c['total'], c['tensors'], c['list_seed'])


# ---------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # the gate of one block of the smallest network: what a user with a single small tensor pays per step
        dict(name='adamw f32 one bias', op='adamw', bits=32, dtype='f32', list='ragged', total=161, tensors=1, list_seed=1, clip=False),
        # a train step's update of this repository's network at its own width, clipped by the norm
        dict(name='adamw f32 net', op='adamw', bits=32, dtype='f32', list='net', width=32, clip=True),
        # bfloat16 parameters with 32-bit states
        dict(name='adamw bf16 stack', op='adamw', bits=32, dtype='bf16', list='stack', width=2048, layers=4, clip=False),
        # the smallest call on 8-bit states: one odd tensor, its last block ragged
        dict(name='adamw8 f32 one tensor', op='adamw', bits=8, dtype='f32', list='ragged', total=5003, tensors=1, list_seed=1, clip=False),
        # the same network as above with states in 8 bits
        dict(name='adamw8 f32 net', op='adamw', bits=8, dtype='f32', list='net', width=32, clip=True),
        # the largest: a bfloat16 model whose states have to be small
        dict(name='adamw8 bf16 stack', op='adamw', bits=8, dtype='bf16', list='stack', width=2048, layers=8, clip=False),
        # the norm of a small network's gradients (the width that the tests train): latency
        dict(name='norm f32 small net', op='norm', dtype='f32', list='net', width=2),
        # the norm of many odd bfloat16 gradients
        dict(name='norm bf16 ragged', op='norm', dtype='bf16', list='ragged', total=300_000_001, tensors=199, list_seed=5),
        # one token through a small router
        dict(name='balance one row', op='balance', dtype='f32', groups=1, rows=1, experts=8, top_k=2, order='row', masked=False),
        # the gates of this network's widest block for a batch of 8 tasks: 5 experts, the expert the slow axis
        dict(name='balance gates', op='balance', dtype='f32', groups=1, rows=4096, experts=5, top_k=1, order='expert', masked=False),
        # a padded batch of sequences, balanced sequence by sequence
        dict(name='balance sequences', op='balance', dtype='bf16', groups=8, rows=4099, experts=64, top_k=6, order='row', masked=True),
        # a large batch through a wide router
        dict(name='balance wide', op='balance', dtype='f32', groups=1, rows=262144, experts=256, top_k=8, order='row', masked=False),
    ]


def draw(rng):
    while True:
        c = _drawn(rng)
        if work(c)['bytes'] <= 4e9:                  # no more than the largest listed ones
            return c


def _drawn(rng):
    log = lambda a, b: int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))  # noqa: E731
    op = rng.choice(['adamw', 'adamw', 'norm', 'balance', 'balance'])
    dtype = rng.choice(['f32', 'bf16'])
    if op == 'balance':
        experts = log(5, 512)
        groups = rng.choice([1, 1, log(2, 64)])
        rows = max(1, log(1, 60_000_000) // (groups * experts))
        return dict(op=op, dtype=dtype, groups=groups, rows=rows, experts=experts, top_k=min(experts // 2, rng.choice([1, 2, log(1, 16)])),
                    order=rng.choice(['row', 'row', 'expert']), masked=rng.random() < 0.5)
    c = dict(op=op, dtype=dtype)
    kind = rng.choice(['ragged', 'ragged', 'stack', 'net'])
    if kind == 'net':
        c.update(list='net', width=rng.randint(1, 31))
    elif kind == 'stack':
        c.update(list='stack', width=log(33, 2047), layers=log(1, 8))
    else:
        c.update(list='ragged', total=log(7, 300_000_000), tensors=log(1, 250), list_seed=rng.randrange(1 << 20))
    if op == 'adamw':
        c.update(bits=rng.choice([8, 32]), clip=rng.random() < 0.5)
    return c


# ---------------------------------------------------------------------------------------------- rounding with given bits
# What is rounded to fewer bits is rounded up with the probability of what is cut off.  The bits are a function of (seed, step,
# position of the tensor, element): two multiply-xorshift rounds over counters.

def _mix_int(x):
    x = (x ^ (x >> 16)) * 0x455c2ed3 & M32
    x = (x ^ (x >> 15)) * 0x55a35cd1 & M32
    return x ^ (x >> 16)


def _mix(x):
    x = ((x ^ (x >> 16)) * 0x455c2ed3) & M32
    x = ((x ^ (x >> 15)) * 0x55a35cd1) & M32
    return x ^ (x >> 16)


def _base(seed, step):
    return _mix_int((step & M32) ^ _mix_int((step >> 32) ^ _mix_int((seed & M32) ^ _mix_int((seed >> 32) + 1 & M32))))


def _bits(s):
    """The random numbers of this step, int64 [blocks, BLOCK]: 32 bits an element for the 8-bit states, 16 for a bfloat16 parameter."""
    key = _mix((s['tensor_of'] + _base(s['seed'], s['t'])) & M32)
    return _mix(s['index'] ^ key), _mix(s['index'] ^ _mix(key ^ 0x6f002d25)) & 0xFFFF


def _to_float8(x, up, man, bias, top, inverse, nan):
    """Magnitudes ``x`` [blocks, BLOCK] as 8-bit codes: x times the block's power of two, its low bits cut off after ``up`` is added."""
    cut = 23 - man
    x = x * inverse
    least = 2.0 ** (1 - bias)                       # the smallest normal value; below it the steps stay as they are there
    low = x < least
    bits = (x + torch.where(low, least, 0.0)).view(torch.int32)
    code = ((bits + up) >> cut) - torch.where(low, (128 - bias) << man, (127 - bias) << man)
    return torch.where(torch.isfinite(x), code.clamp(max=top), torch.where(torch.isnan(x), nan[0], nan[1]))


def _scale(x, room):
    """Biased exponent [blocks, 1] of the power of two that brings each block's largest magnitude to [2^room, 2^(room + 1))."""
    most = torch.where(torch.isfinite(x), x, 0.0).amax(1, keepdim=True)
    return ((most.view(torch.int32) >> 23) - room).clamp(min=1)


def _power(e):
    return (e << 23).view(torch.float32)            # 2^(e - 127) from its biased exponent, 1 <= e <= 254


def _encode(m, v, h):
    """The 8-bit states of m and v (float32 [blocks, BLOCK]) with 32 bits h an element: e4m3 and e5m2 values, and their blocks' powers of two."""
    em, ev = _scale(m.abs(), 7), _scale(v, 14)
    m8 = _to_float8(m.abs(), ((h & 0xFFFF) << 4) + 8, 3, 7, 0x7E, _power(254 - em), (0x7F, 0x7F))
    m8 = torch.where(torch.signbit(m), m8 | 0x80, m8).to(torch.uint8).view(torch.float8_e4m3fn)
    v8 = _to_float8(v, ((h >> 16) << 5) + 16, 2, 15, 0x7B, _power(254 - ev), (0x7E, 0x7C))
    v8 = torch.where(v > 0, v8.clamp(min=1), v8).to(torch.uint8).view(torch.float8_e5m2)   # a second moment that is not zero stays so
    e8 = lambda e: e.reshape(-1).to(torch.uint8).view(torch.float8_e8m0fnu)  # noqa: E731
    return m8, e8(em), v8, e8(ev)


def _decode(x8, e8):
    return x8.view(-1, BLOCK).float() * _power(e8.view(torch.uint8).to(torch.int32)).view(-1, 1)


# ---------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    c = case
    g = torch.Generator(DEV).manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device=DEV)  # noqa: E731
    rand = lambda *shape: torch.rand(shape, generator=g, device=DEV)  # noqa: E731
    dtype = DTYPES[c['dtype']]
    if c['op'] == 'balance':
        n, e, k = c['rows'], c['experts'], c['groups']
        x = randn(k, n, e) * 1.5 + randn(k, 1, e)                       # some experts are liked more than others
        mask = None
        if c['masked']:
            if e > c['top_k']:
                x[:, :, 0] = -math.inf                                   # an expert that is switched off
            length = (rand(k, 1) * (n + 1)).long()
            mask = torch.arange(n, device=DEV)[None] < length
            x = torch.where(mask[:, :, None], x, math.nan)               # what stands in padded rows is not to be read
        x = x.to(dtype)
        if c['order'] == 'expert':
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        return dict(case=c, x=x.detach().requires_grad_(True), mask=mask, up=1 + rand(1)[0])

    numels = _numels(c)
    blocks = [-(-n // BLOCK) for n in numels]
    first = [0]
    for b in blocks:
        first.append(first[-1] + b)
    nb = first[-1]
    count = torch.tensor(blocks, device=DEV)
    tensor_of = torch.repeat_interleave(torch.arange(len(numels), device=DEV), count)
    block_in = torch.arange(nb, device=DEV) - torch.tensor(first[:-1], device=DEV)[tensor_of]
    index = block_in[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)
    here = index < torch.tensor(numels, device=DEV)[tensor_of][:, None]     # False: the space behind a tensor's end
    sigma = torch.exp(-5 + 1.5 * randn(len(numels)))[tensor_of][:, None] * here
    grad = randn(nb, BLOCK) * sigma * (rand(nb, 1) > 0.05)                    # some blocks saw nothing in this step
    views = lambda flat: [flat.view(-1)[f * BLOCK:f * BLOCK + n] for f, n in zip(first, numels)]  # noqa: E731
    s = dict(case=c, here=here, grad=grad.to(dtype), n=sum(numels))
    s['grads'] = views(s['grad'])
    if c['op'] == 'norm':
        return s
    s.update(tensor_of=tensor_of[:, None], index=index, seed=seed * 7919 + 3, t=100, p=(randn(nb, BLOCK) * 0.02 * here).to(dtype))
    m, v = 0.3 * sigma * randn(nb, BLOCK), sigma.square() * torch.exp(randn(nb, BLOCK))
    s['ps'] = views(s['p'])
    if c['bits'] == 32:
        s.update(m=m, v=v, ms=views(m), vs=views(v))
    else:
        half = torch.full((1, 1), 0x80008000, dtype=torch.int64, device=DEV)
        m8, em, v8, ev = _encode(m, v, half)
        part = lambda e: [e[f:f + b] for f, b in zip(first, blocks)]  # noqa: E731
        s.update(m8=m8, em=em, v8=v8, ev=ev, ms=views(m8), vs=views(v8), ems=part(em), evs=part(ev))
    return s


# ---------------------------------------------------------------------------------------------- one pass

def run(s):
    return {'balance': _balance, 'norm': _norm, 'adamw': _adamw}[s['case']['op']](s)


def _norm(s):
    """The norm of all gradients together and the factor that brings it to at most 1."""
    if own:
        from repmode_amd import ops
        norm, clip = ops.grad_norm(s['grads'], max_norm=1.0)
        return dict(norm=norm, clip=clip)
    norm = s['grad'].float().square().sum(1).double().sum().sqrt()
    return dict(norm=norm.float(), clip=torch.clamp(1.0 / (norm + 1e-6), max=1.0).float())


def _adamw(s):
    c = s['case']
    s['t'] += 1
    if own:
        from repmode_amd import ops
        clip = ops.grad_norm(s['grads'], max_norm=1.0)[1] if c['clip'] else None
        how = dict(lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, clip=clip, seed=s['seed'])
        if c['bits'] == 32:
            ops.adamw_step(s['ps'], s['grads'], s['ms'], s['vs'], s['t'], **how)
        else:
            ops.adamw8_step(s['ps'], s['grads'], s['ms'], s['ems'], s['vs'], s['evs'], s['t'], **how)
        return {k: s[k] for k in ('p', 'm', 'v', 'm8', 'em', 'v8', 'ev') if k in s}
    g = s['grad'].float()
    if c['clip']:
        g = g * _norm(s)['clip']
    if c['bits'] == 32:
        m, v = s['m'], s['v']
    else:
        m, v = _decode(s['m8'], s['em']), _decode(s['v8'], s['ev'])
    m = m + (1 - BETA1) * (g - m)
    v = v * BETA2 + (1 - BETA2) * g * g
    root = v.sqrt() / math.sqrt(1 - BETA2 ** s['t']) + EPS
    p = s['p'].float() * (1 - LR * DECAY) - (LR / (1 - BETA1 ** s['t'])) * (m / root)
    if c['dtype'] == 'bf16':
        bits = p.view(torch.int32)
        bits = torch.where(torch.isfinite(p), bits + _bits(s)[1].to(torch.int32), bits)
        p = (bits & -65536).view(torch.float32)
    s['p'].copy_(p)
    if c['bits'] == 32:
        s['m'].copy_(m)
        s['v'].copy_(v)
        return dict(p=s['p'], m=s['m'], v=s['v'])
    for name, x in zip(('m8', 'em', 'v8', 'ev'), _encode(m, v, _bits(s)[0])):
        s[name].view(torch.uint8).copy_(x.view(torch.uint8).view_as(s[name]))
    return {k: s[k] for k in ('p', 'm8', 'em', 'v8', 'ev')}


COEF = 0.01


def _balance(s):
    """loss = COEF * E * mean over the groups with rows of sum_e f_e P_e: f the share of choices that went to expert e, P its mean probability."""
    c = s['case']
    if own:
        from repmode_amd import ops
        loss, counts, prob = ops.balance_loss(s['x'], c['top_k'], mask=s['mask'], coef=COEF)
        grad, = torch.autograd.grad(loss, s['x'], grad_outputs=s['up'])
        return dict(loss=loss.detach(), counts=counts, prob=prob, grad=grad)
    x = s['x'].detach().float()
    k, n, e = x.shape
    if s['mask'] is None:
        rows = torch.full((k, 1), float(n), device=DEV)
    else:
        x = torch.where(s['mask'][:, :, None], x, 0.0)
        rows = s['mask'].sum(1, keepdim=True).float()
    y = torch.exp(x - x.amax(2, keepdim=True))
    p = y / y.sum(2, keepdim=True)
    if s['mask'] is not None:
        p = p * s['mask'][:, :, None]
    order = torch.sort(x, dim=2, descending=True, stable=True).indices[:, :, :c['top_k']]      # ties: the lowest index first
    chosen = torch.zeros_like(x).scatter_(2, order, 1.0) * (p > 0)
    counts = chosen.sum(1, dtype=torch.float64)
    some = rows.clamp(min=1)
    prob = p.sum(1) / some
    share = (counts / (some * c['top_k'])).float()
    groups = (rows > 0).sum().clamp(min=1)
    loss = COEF * e * (share * prob).sum() / groups
    dp = share[:, None] * (COEF * e / groups / some)[:, None] * s['up']
    grad = p * (dp - (p * dp).sum(2, keepdim=True))
    return dict(loss=loss, counts=counts.long(), prob=prob, grad=grad.to(s['x'].dtype))


# ---------------------------------------------------------------------------------------------- in 64 bits

def _grid(x, u, man, low, e):
    """x >= 0 in units of 2^e to a float of ``man`` bits whose smallest exponent is ``low``, up where the cut-off part and u in [0, 1) reach 1."""
    x = x * torch.exp2(-e)
    step = torch.exp2(torch.frexp(x)[1].double().sub_(1).clamp_(min=low) - man)
    return torch.floor(x / step + u) * step


def _exponent(x):
    """Of each block's largest value, as whole numbers; a block of zeros has none (the smallest there is)."""
    most = x.amax(1, keepdim=True)
    return torch.where(most > 0, torch.frexp(most)[1].double() - 1, -math.inf)


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c['op'] == 'norm':
        norm = s['grad'].double().pow(2).sum().sqrt()
        return dict(norm=norm, clip=(1 / (norm + 1e-6)).clamp(max=1))
    if c['op'] == 'balance':
        x = s['x'].detach().double()
        valid = torch.ones(x.shape[:2], dtype=torch.bool, device=DEV) if s['mask'] is None else s['mask']
        n = valid.sum(1).double()
        lse = torch.logsumexp(x, 2, keepdim=True)
        p = torch.where(valid[..., None], torch.exp(x - lse), 0.0)
        rank = torch.argsort(torch.argsort(torch.nan_to_num(x, nan=0.0, neginf=-1e300), dim=2, descending=True, stable=True), dim=2)
        f = ((rank < c['top_k']) & (p > 0)).sum(1) / (n * c['top_k']).clamp(min=1)[:, None]
        prob = p.sum(1) / n.clamp(min=1)[:, None]
        a = COEF * c['experts'] / max(1, int((n > 0).sum()))
        q = p * s['up'].double() * a / n.clamp(min=1)[:, None, None]
        return dict(loss=a * (f * prob).sum(), counts=None, prob=prob, grad=q * (f[:, None] - (p * f[:, None]).sum(2, keepdim=True)))
    s['t'] += 1
    t, (h, low) = s['t'], _bits(s)
    g = s['grad'].double()
    if c['clip']:
        g = g * (1 / (g.pow(2).sum().sqrt() + 1e-6)).clamp(max=1)
    if c['bits'] == 32:
        m, v = s['m'].double(), s['v'].double()
    else:
        at = lambda e8: torch.exp2(e8.view(torch.uint8).double() - 127)[:, None]  # noqa: E731
        m, v = s['m8'].double() * at(s['em']), s['v8'].double() * at(s['ev'])
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    p = s['p'].double()
    p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    if c['dtype'] == 'bf16':
        p = torch.copysign(_grid(p.abs(), low.double() / 65536, 7, -126, torch.zeros_like(p[:, :1])), p)
    if c['bits'] == 32:
        return dict(p=p, m=m, v=v)
    em, ev = (_exponent(m.abs()) - 7).clamp(min=-126), (_exponent(v) - 14).clamp(min=-126)
    m8 = torch.copysign(_grid(m.abs(), ((h % 65536).double() + 0.5) / 65536, 3, -6, em), m)
    v8 = _grid(v, ((h // 65536).double() + 0.5) / 65536, 2, -14, ev)
    v8 = torch.where(v > 0, v8.clamp(min=2.0 ** -16), v8)
    return dict(p=p, m8=m8.view(-1), em=torch.exp2(em.view(-1)), v8=v8.view(-1), ev=torch.exp2(ev.view(-1)))


# ---------------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    size = 4 if c['dtype'] == 'f32' else 2
    if c['op'] == 'balance':
        rows = c['groups'] * c['rows']
        values = rows * c['experts']
        return dict(bytes=2 * size * values + (rows if c['masked'] else 0) + 12 * c['groups'] * c['experts'] + 8, flops=12 * values)
    n = sum(_numels(c))
    if c['op'] == 'norm':
        return dict(bytes=size * n + 8, flops=2 * n)
    state = 16 if c['bits'] == 32 else 4 + 4 / BLOCK
    return dict(bytes=int((3 * size + state) * n), flops=(17 if c['clip'] else 15) * n)
