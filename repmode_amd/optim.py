"""The optimizer of the train step -- ``torch.optim.Adam(net.parameters(), lr)`` of the reference harness
(fnet/fnet_model.py:55, stepped at :112) -- running through this build's own kernels (csrc/adam.hip).

``Adam`` IS a ``torch.optim.Adam`` (same constructor defaults, same ``state`` layout: ``step`` / ``exp_avg`` / ``exp_avg_sq``
per parameter, so ``state_dict()`` / ``load_state_dict()`` interchange with the stock optimizer and with the reference's
checkpoints, fnet_model.py:57-65); only ``step()`` differs: one call into the operator library, which updates every
parameter with two kernel families and -- for the 5x5x5 / 3x3x3 experts of the blocks that run the per-expert formulation --
emits the updated experts as the convolution kernels' bf16 operands in the same pass (``repmode_adam_expert_frags``), so the
next forward pass has no layout launch.  No CPU path: parameters must live on the HIP device.

``AdamW`` is for what the reference does not train with: decoupled weight decay, clipping by the gradients' common norm, bfloat16
parameters and moments in 8 bits.
"""
import math

import torch


def _foreign_step_hook(optimizer, args, kwargs):
    """Any OTHER optimizer stepping (the reference harness's own ``torch.optim.Adam``, a stock fused one): its foreach / fused
    kernels write the parameters without moving autograd's version counters (measured: torch's fused Adam left the expert
    operands kept across steps looking current -- stale filters, a 4 % worse loss after 55 steps), so the operator library's
    store of expert operands is emptied and the next forward pass lays them out again."""
    if not isinstance(optimizer, Adam):
        from . import _lib
        if _lib.torch_ops_loaded():
            torch.ops.repmode.clear_frag_store()


_hook_handle = None


def install_foreign_step_hook():
    """Registered once, when the operator library is loaded (``_lib.load_torch_ops``)."""
    global _hook_handle
    if _hook_handle is None:
        from torch.optim.optimizer import register_optimizer_step_post_hook
        _hook_handle = register_optimizer_step_post_hook(_foreign_step_hook)


def _capturing():
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


def _kept_as(v):
    """The type a saved moment is kept in: float32 for anything of 16 bits (a stock optimizer's of bfloat16 parameters)."""
    return torch.float32 if v.dtype in (torch.bfloat16, torch.float16) else v.dtype


def _check_captured(who, opt, state_dict):
    """Raises, before anything has changed, where a state does not fit the tensors that a captured step holds."""
    for saved, group in zip(state_dict['param_groups'], opt.param_groups):
        counts = set()
        for key, p in zip(saved['params'], group['params']):
            st, there = state_dict['state'].get(key, {}), opt.state.get(p, {})
            if st or there:
                counts.add(int(st.get('step', 0)))
            if not st or not there:                      # (no moments yet; or none saved: those that are there become zero)
                continue
            new = {k: (_kept_as(v), v.shape) for k, v in st.items() if k != 'step' and torch.is_tensor(v)}
            if new != {k: (t.dtype, t.shape) for k, t in there.items() if k != 'step'}:
                raise ValueError('repmode_amd.optim.%s: a captured step holds this optimizer\'s moments, and the state has others (another '
                                 'number of bits, other shapes): load it into a new optimizer and capture again' % who)
        if len(counts) > 1:
            raise ValueError('repmode_amd.optim.%s: a captured step holds one step count for a group, and the state\'s counts differ: load it '
                             'into a new optimizer and capture again' % who)


class Adam(torch.optim.Adam):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, capturable=False):
        """``capturable``: the step count ALSO lives on the device (one int64 for the whole parameter list) and the kernels take
        the step's constants from device memory (``repmode_adam_hyper_dev``), so that ``step()`` can be part of a captured HIP
        graph: a replay advances the count itself.  The host counters of ``state`` are brought up to date by ``sync_steps()``
        (``state_dict()`` calls it).  The learning rate is a launch argument: changing it needs a new capture."""
        # (the stock single-tensor bookkeeping: `step` counters are host scalars -- no device read to learn the step count)
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=0, amsgrad=False, foreach=False, fused=False,
                         capturable=False)
        self.device_step = bool(capturable)
        self._step_dev = self._hyper_dev = None
        self._captured = False       # a step was captured: some graph may hold moments, count and constants by address

    def sync_steps(self):
        """Device step count -> the host counters of ``state`` (after graph replays, which run no host code).  One device read."""
        if self._step_dev is not None:
            t = int(self._step_dev.item())
            for st in self.state.values():
                if 'step' in st:
                    st['step'] = torch.tensor(float(t))

    def state_dict(self):
        self.sync_steps()
        return super().state_dict()

    def load_state_dict(self, state_dict):
        """As torch.optim.Adam; `step` counters that a fused / capturable optimizer kept on the device come to the host (one
        copy at load time, so that ``step()`` never reads the device to learn the step count)."""
        if any('exp_avg_scale' in st for st in state_dict['state'].values()):
            raise ValueError('repmode_amd.optim.Adam: these moments are in 8 bits (optim.AdamW)')
        if self._captured:
            _check_captured('Adam', self, state_dict)
        held = {p: dict(st) for p, st in self.state.items()} if self._captured else {}
        super().load_state_dict(state_dict)
        for p, st in held.items():                 # (what a captured step holds by address takes the loaded values; none: zeros)
            new = self.state[p]
            for k in ('exp_avg', 'exp_avg_sq'):
                st[k].copy_(new[k]) if k in new else st[k].zero_()
                new[k] = st[k]
            new.setdefault('step', torch.tensor(0.0))
        for group in self.param_groups:            # (a stock optimizer's groups say fused / capturable; this one's bookkeeping is neither)
            group['fused'], group['capturable'], group['foreach'] = False, False, False
        for st in self.state.values():
            if torch.is_tensor(st.get('step')) and st['step'].is_cuda:
                st['step'] = st['step'].detach().cpu()
        if self._step_dev is not None:
            # A captured step holds the device count and the constants' buffer BY ADDRESS: they stay where they are and take the
            # loaded count in place.  Counters that disagree cannot be one device count: where nothing was captured the buffers go,
            # and the next step says so (as a first step would).
            loaded = {int(st['step']) for st in self.state.values() if 'step' in st}
            if len(loaded) <= 1:
                self._step_dev.fill_(loaded.pop() if loaded else 0)
            else:
                self._step_dev = self._hyper_dev = None

    @torch.no_grad()
    def step(self, closure=None):
        from . import ops as ops_
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            if group['weight_decay'] != 0 or group['amsgrad'] or group.get('maximize', False):
                raise RuntimeError('repmode_amd.optim.Adam: the reference trains with plain Adam (no weight decay / amsgrad / maximize)')
            params, grads, exp_avgs, exp_avg_sqs, max_sqs, steps = [], [], [], [], [], []
            self._init_group(group, params, grads, exp_avgs, exp_avg_sqs, max_sqs, steps)
            if not params:
                continue
            beta1, beta2 = group['betas']
            lr = float(group['lr'])
            if self.device_step:
                if len(self.param_groups) != 1:
                    raise RuntimeError('repmode_amd.optim.Adam(capturable=True): one parameter group (one device step count)')
                if self._step_dev is None:
                    # first step (launch by launch, never under capture): the device count starts where the host counters are
                    t0 = {int(s) for s in steps}
                    if len(t0) != 1:
                        raise RuntimeError('repmode_amd.optim.Adam(capturable=True): every parameter must have seen the same '
                                           'number of steps')
                    if _capturing():
                        raise RuntimeError('repmode_amd.optim.Adam(capturable=True): run one step launch by launch before capturing')
                    self._step_dev = torch.full((1,), t0.pop(), dtype=torch.int64, device=params[0].device)
                    self._hyper_dev = torch.zeros(8, dtype=torch.float32, device=params[0].device)
                self._captured |= _capturing()
                for s in steps:
                    s += 1              # (host mirror: exact while steps run launch by launch; sync_steps() after replays)
                ops_.torch_ops().adam_step_dev(params, grads, exp_avgs, exp_avg_sqs, lr, float(beta1), float(beta2), float(group['eps']),
                                               self._step_dev, self._hyper_dev)
                continue
            # parameters that have seen the same number of updates go together (normally: all of them)
            by_step = {}
            for i, s in enumerate(steps):
                if s.is_cuda:                                       # (a counter created under another optimizer's policy)
                    s = self.state[params[i]]['step'] = s.detach().cpu()
                s += 1                                              # (host scalar tensor, in place: the state's counter)
                by_step.setdefault(int(s), []).append(i)
            for t, idx in by_step.items():
                sel = (lambda xs: xs) if len(idx) == len(params) else (lambda xs: [xs[i] for i in idx])
                ops_.torch_ops().adam_step(sel(params), sel(grads), sel(exp_avgs), sel(exp_avg_sqs), lr, float(beta1), float(beta2),
                                           float(group['eps']), t)
        return loss


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over all tensors at once, with the gradients clipped by their common norm in the same step
    and the moments in float32 or in 8 bits (csrc/adamw.hip, csrc/grad_norm.hip).  float32 and bfloat16 parameters.

    ``max_norm``: the gradients of all groups together are scaled by ``min(1, max_norm / (norm + 1e-6))`` on their way into the
    update (``.grad`` itself stays as it is; ``last_norm`` is the norm, a device scalar).  Where a gradient is not finite the step
    is left out: it changes no parameter, no moment and no step count.  (A count on the host learns of it afterwards: the next ``step()``
    waits until the GPU is past this one's norm and takes it back, as ``sync_steps()`` and ``state_dict()`` do.)
    ``state_bits``: 32, or 8 -- e4m3 / e5m2 values with a power of two for each 256 elements, rounded stochastically: 2 bytes a
    parameter instead of 8.  Tensors of fewer than ``min_8bit_numel`` elements (biases, norms) keep float32 moments.  Both may be
    set per group.
    ``seed``: of the stochastic roundings (8-bit moments, bfloat16 parameters); a run with the same seed repeats itself.
    ``capturable``: the step count of each group lives on the device, so that ``step()`` can be part of a captured HIP graph (after
    one step launch by launch); a group's ``lr`` may then be a float32 tensor of one value on the device, which replays read (every other
    setting, and an ``lr`` that is a number, stays what it was at the capture).

    The state of a float32 parameter with 32-bit moments is ``torch.optim.AdamW``'s (``step``, ``exp_avg``, ``exp_avg_sq``): their state
    dicts interchange.  Loaded moments keep the bits they were saved with.  No CPU path."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_norm=None, state_bits=32, min_8bit_numel=4096,
                 capturable=False, seed=0):
        if not (torch.is_tensor(lr) or lr >= 0) or not eps >= 0 or not weight_decay >= 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError('repmode_amd.optim.AdamW: bad hyper-parameters')
        if max_norm is not None and not max_norm > 0:
            raise ValueError('repmode_amd.optim.AdamW: max_norm must be positive, got %r' % (max_norm,))
        self.max_norm, self.seed, self.device_step, self.last_norm = max_norm, int(seed), bool(capturable), None
        self._step_dev = {}          # group index -> int64[1] on the device (capturable)
        self._captured = False       # a step was captured: some graph may hold moments and counts by address
        self._last = self._flag = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      min_8bit_numel=min_8bit_numel))

    def add_param_group(self, group):
        super().add_param_group(group)
        if self.param_groups[-1]['state_bits'] not in (8, 32):
            bits = self.param_groups.pop()['state_bits']
            raise ValueError('repmode_amd.optim.AdamW: moments in 8 or 32 bits, got %r' % (bits,))

    def __getstate__(self):
        self.sync_steps()
        return {**super().__getstate__(), 'max_norm': self.max_norm, 'seed': self.seed, 'device_step': self.device_step, 'last_norm': None,
                '_step_dev': {}, '_captured': False, '_last': None, '_flag': None}

    def _state(self, p, group):
        st = self.state[p]
        if not st:
            from . import ops as ops_
            if self.device_step and _capturing():
                # (the zeros would be part of the graph, and every replay begin with them)
                raise RuntimeError('repmode_amd.optim.AdamW(capturable=True): a parameter\'s first step must not be a captured one')
            st['step'] = torch.tensor(0.0)
            if group['state_bits'] == 8 and p.numel() >= group['min_8bit_numel']:
                st['exp_avg'], st['exp_avg_scale'], st['exp_avg_sq'], st['exp_avg_sq_scale'] = ops_.adamw8_state(p)
            else:
                st['exp_avg'] = torch.zeros_like(p, dtype=torch.float32)
                st['exp_avg_sq'] = torch.zeros_like(p, dtype=torch.float32)
        return st

    def _watch(self, clip):
        """Keeps a step's clip factor -- of one on the GPU: what will be on the host behind an event -- and the list of the counters
        that it moves, for ``_settle``.  Called between norm and update, so that the event does not wait for the update."""
        event = None
        if clip.is_cuda:
            if self._flag is None:
                self._flag = torch.empty((), dtype=torch.float32, device='cpu', pin_memory=True), torch.cuda.Event()
            (flag, event), stream = self._flag, torch.cuda.current_stream(clip.device)
            clip = flag.copy_(clip, non_blocking=True)
            event.record(stream)
        self._last = clip, event, []
        return self._last[2]

    def _settle(self):
        """Takes the last step back from the host counters of its parameters if it was left out."""
        if self._last is not None:
            clip, event, steps = self._last
            self._last = None
            if event is not None:
                event.synchronize()
            if math.isnan(clip):
                for s in steps:
                    s -= 1

    def sync_steps(self):
        """What the GPU knows of the step counts -> the host counters of ``state``: device counts (after graph replays, which run no host
        code; one read a group), and whether the last step was left out."""
        self._settle()
        for gi, dev in self._step_dev.items():
            t = float(dev.item())
            for p in self.param_groups[gi]['params']:
                if 'step' in self.state.get(p, {}):
                    self.state[p]['step'] = torch.tensor(t)

    def state_dict(self):
        self.sync_steps()
        return super().state_dict()

    def _check_loaded(self, state_dict):
        """Raises, before anything has changed, where 8-bit moments lie in another order than their parameter (their scales are those of
        neighbours in memory), or where a state does not fit the tensors that a captured step holds."""
        for saved, group in zip(state_dict['param_groups'], self.param_groups):
            for key, p in zip(saved['params'], group['params']):
                st = state_dict['state'].get(key, {})
                for v in (st.get('exp_avg'), st.get('exp_avg_sq')):
                    if (torch.is_tensor(v) and v.dtype.itemsize == 1 and v.shape == p.shape and v.stride() != p.stride() and
                            not (v.is_contiguous() and p.is_contiguous())):
                        raise ValueError('repmode_amd.optim.AdamW: 8-bit moments whose order in memory is not their parameter\'s')
        if self._captured:
            _check_captured('AdamW', self, state_dict)

    def load_state_dict(self, state_dict):
        """As torch.optim.AdamW's, with the moments as they were saved.  After a captured step the state goes into the tensors that the
        graph holds -- a parameter without state gets zero moments -- and one that does not fit them is refused.  A group's learning rate
        on the device stays the tensor that it is and takes the loaded value."""
        self._check_loaded(state_dict)
        self._settle()
        own = [{k: g[k] for k in ('state_bits', 'min_8bit_numel', 'lr')} for g in self.param_groups]
        # (captured steps hold the moments by address, as they do the step counts: what fits goes into the tensors that are there)
        held = {p: dict(st) for p, st in self.state.items()} if self.device_step else {}
        super().load_state_dict(state_dict)
        for group, mine in zip(self.param_groups, own):          # (a stock optimizer's groups have neither)
            lr = mine.pop('lr')
            for k, v in mine.items():
                group.setdefault(k, v)
            if torch.is_tensor(lr):
                group['lr'] = lr.fill_(float(group['lr']))
            elif torch.is_tensor(group['lr']):
                group['lr'] = (group['lr'].to(next(iter(group['params']), group['lr']).device, torch.float32) if self.device_step
                               else float(group['lr']))
        # (the base class casts floating moments to the parameter's type: 8-bit codes and the float32 moments of bfloat16
        # parameters are taken from the dict as they are)
        for saved, group in zip(state_dict['param_groups'], self.param_groups):
            for key, p in zip(saved['params'], group['params']):
                for k, v in state_dict['state'].get(key, {}).items():
                    if k == 'step':
                        self.state[p][k] = torch.tensor(float(v))
                    elif torch.is_tensor(v):
                        # (a moment of its parameter's shape takes its strides too)
                        v = torch.empty_like(p if v.shape == p.shape else v, dtype=_kept_as(v), device=p.device,
                                             requires_grad=False).copy_(v.detach())
                        there = held.get(p, {}).get(k)
                        if torch.is_tensor(there) and there.dtype == v.dtype and there.shape == v.shape:
                            v = there.copy_(v)
                        self.state[p][k] = v
                if self._captured and held.get(p) and not self.state.get(p):
                    self.state[p] = held[p]
                    self._rewind(held[p])
        for gi, dev in list(self._step_dev.items()):
            counts = {int(self.state[p]['step']) for p in self.param_groups[gi]['params'] if 'step' in self.state.get(p, {})}
            if len(counts) <= 1:
                dev.fill_(counts.pop() if counts else 0)
            else:                        # (no step was captured: the next one says that they differ)
                del self._step_dev[gi]

    @staticmethod
    def _rewind(st):
        """A parameter's state as before its first step, in place."""
        for k, t in st.items():
            if k == 'step':
                st[k] = torch.tensor(0.0)
            elif t.dtype == torch.float32:
                t.zero_()
            else:
                t.view(torch.uint8).fill_(127 if t.dtype == torch.float8_e8m0fnu else 0)

    def _count_on_device(self, gi, steps, device):
        """The group's step count on the device; ``steps``: its parameters' host counters, which go on as well."""
        t0 = {int(s) for s in steps}
        if len(t0) != 1:                       # (also where a parameter has its first gradient after the others)
            raise RuntimeError('repmode_amd.optim.AdamW(capturable=True): the parameters of a group must have seen the same number of steps')
        if gi not in self._step_dev:
            if _capturing():
                raise RuntimeError('repmode_amd.optim.AdamW(capturable=True): run one step launch by launch before capturing')
            self._step_dev[gi] = torch.full((1,), t0.pop(), dtype=torch.int64, device=device)
        for s in steps:
            s += 1
        return self._step_dev[gi]

    @torch.no_grad()
    def step(self, closure=None):
        from . import ops as ops_
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work, grads = [], []
        for gi, group in enumerate(self.param_groups):
            if group.get('amsgrad', False) or group.get('maximize', False):
                raise RuntimeError('repmode_amd.optim.AdamW: no amsgrad, no maximize')
            ps = [p for p in group['params'] if p.grad is not None]
            if any(p.grad.is_sparse for p in ps):
                raise RuntimeError('repmode_amd.optim.AdamW: dense gradients only')
            if ps:
                work.append((gi, group, ps))
                grads += [p.grad for p in ps]
        if not work:
            return loss
        if not self.device_step and _capturing():
            raise RuntimeError('repmode_amd.optim.AdamW: a captured step needs capturable=True')
        clip = None
        if self.max_norm is not None:
            self._settle()
            self.last_norm, clip = ops_.grad_norm(grads, self.max_norm)
        counted = [] if clip is None or self.device_step else self._watch(clip)
        none = torch.empty(0)
        for gi, group, ps in work:
            states = [self._state(p, group) for p in ps]
            if self.device_step:
                calls = [(self._count_on_device(gi, [st['step'] for st in states], ps[0].device), range(len(ps)))]
                self._captured |= _capturing()
            else:
                # parameters that have seen the same number of updates go together (normally: all of them)
                if torch.is_tensor(group['lr']):
                    raise RuntimeError('repmode_amd.optim.AdamW: a learning rate on the device needs capturable=True')
                by_step = {}
                for i, st in enumerate(states):
                    st['step'] += 1
                    counted.append(st['step'])
                    by_step.setdefault(int(st['step']), []).append(i)
                calls = by_step.items()
            for count, idx in calls:
                eight = any('exp_avg_scale' in states[i] for i in idx)
                scales = (lambda k: [states[i].get(k, none) for i in idx]) if eight else (lambda k: [])
                ops_.adamw8_step([ps[i] for i in idx], [ps[i].grad for i in idx], [states[i]['exp_avg'] for i in idx], scales('exp_avg_scale'),
                                 [states[i]['exp_avg_sq'] for i in idx], scales('exp_avg_sq_scale'), count, lr=group['lr'],
                                 betas=group['betas'], eps=group['eps'], weight_decay=group['weight_decay'], clip=clip,
                                 seed=(gi << 32) + (self.seed & 0xffffffff))
        return loss
