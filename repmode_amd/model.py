"""Training / inference harness around the MI355X MoDE network -- counterpart of the reference's
``fnet/fnet_model.py`` ``Model`` for the rows of SURVEY.md section 8 that call the hot path:

  * ``do_train_iter(signal, target, task)``  -- fnet_model.py:96-132 (zero_grad, autocast forward,
    MSELoss('none') -> mean, backward, Adam step, per-sample loss);
  * ``predict(signal, task, patch_size)``    -- fnet_model.py:149-223 (50 %-overlap tiling, LIFO
    batches of ``opts.batch_size_eval``, Gaussian-weighted blend);
  * ``get_state/save_state/load_state``      -- fnet_model.py:57-94 (same dict keys, so checkpoints
    are interchangeable through ``nn_state``).

Differences that are the point of the build: bfloat16 instead of fp16 autocast (no GradScaler), the
task ids stay on the host until the slot plan is built (no device->host sync per sample), the loss
stays on the device (no ``.item()`` per iteration unless asked), the Gaussian blend accumulates on
the GPU, and data-parallel training is one process per GPU with RCCL all-reduce (DistributedData
Parallel) instead of single-process ``nn.DataParallel`` (fnet_model.py:40-44).
"""
import math
import os

import numpy as np
import torch

from .nn_modules import RepMode as _repmode


def get_gaussian(patch_size, sigma_scale=1.0 / 8):
    """Importance map of fnet_model.py:242-252.

    A centred delta filtered by scipy's separable ``gaussian_filter(mode='constant')`` equals the
    outer product of three 1-D Gaussians truncated at 4 sigma (scipy's default); it is
    max-normalised and zeros are replaced by the smallest non-zero value.
    """
    from scipy.ndimage import gaussian_filter
    tmp = np.zeros(patch_size)
    tmp[tuple(i // 2 for i in patch_size)] = 1
    gm = gaussian_filter(tmp, [i * sigma_scale for i in patch_size], 0, mode='constant', cval=0)
    gm = (gm / np.max(gm)).astype(np.float32)
    gm[gm == 0] = np.min(gm[gm != 0])
    return gm


def patch_grid(img_size, patch_size, overlap=0.5):
    """(starts, ends) of every patch in enumeration order -- fnet_model.py:156-193."""
    strides = [int(math.ceil(p * (1 - overlap))) for p in patch_size]
    steps = [int(math.ceil((i - p) / s + 1)) for i, p, s in zip(img_size, patch_size, strides)]
    grid = []
    for a in range(steps[0]):
        for b in range(steps[1]):
            for c in range(steps[2]):
                starts = [i * s for i, s in zip((a, b, c), strides)]
                ends = [min(s + p, im) for s, p, im in zip(starts, patch_size, img_size)]
                starts = [max(e - p, 0) for e, p in zip(ends, patch_size)]
                grid.append((starts, ends))
    return grid


class Model(object):
    def __init__(self, opts, nn_module='RepMode', init_weights=True, lr=0.001, criterion_fn=torch.nn.MSELoss,
                 gpu_ids=0, mult_chan=32, dtype=torch.bfloat16, distributed=False, hip_graph=False, grad_compress=None,
                 optimizer='adam', optimizer_args=None, balance_coef=0.0):
        # optimizer: 'adam' (the reference's) or 'adamw' (optim.AdamW: weight decay, clipping by the gradients' norm, moments in 8
        # bits; optimizer_args goes to its constructor).  balance_coef > 0 adds Net.gate_balance's term to the loss.
        if optimizer not in ('adam', 'adamw'):
            raise ValueError("optimizer must be 'adam' or 'adamw', got %r" % (optimizer,))
        if optimizer == 'adam' and optimizer_args:
            raise ValueError('optimizer_args go with optimizer=\'adamw\': the reference trains with plain Adam')
        if not balance_coef >= 0:
            raise ValueError('balance_coef must not be negative, got %r' % (balance_coef,))
        self.optimizer_name, self.optimizer_args, self.balance_coef = optimizer, dict(optimizer_args or {}), float(balance_coef)
        self.last_balance = None
        self.opts = opts
        self.nn_module = nn_module
        self.lr = lr
        self.count_iter = 0
        self.count_epoch = 0
        self.gpu_ids = [gpu_ids] if isinstance(gpu_ids, int) else gpu_ids
        if self.gpu_ids[0] < 0:
            raise RuntimeError('repmode_amd.Model needs a HIP device; there is no CPU path')
        self.device = torch.device('cuda', self.gpu_ids[0])
        self.patch_size = (32, 128, 128)                       # fnet_model.py:34
        self.mult_chan = mult_chan
        self.dtype = dtype
        self.distributed = distributed
        # The gradient buckets are float32 by default -- what the reference averages in (DataParallel + Adam, fnet_model.py:40-44,
        # 112) -- and stay float32 unless the caller opts in: grad_compress='bf16' (or REPMODE_GRAD_COMPRESS=bf16) sends them as
        # bfloat16; 'auto' lets the RULE decide (distributed.pick_grad_dtype): float32 until two measured
        # backward passes say that the per-link ring estimate of the float32 all-reduce exceeds 0.6 of the backward it has to
        # hide under, then bfloat16 (the decision is printed; the measured backward includes the wait for the collectives it
        # overlaps, which only makes the rule keep float32 longer).
        gc = grad_compress or os.environ.get('REPMODE_GRAD_COMPRESS') or 'fp32'
        if gc in (torch.bfloat16, 'bf16', 'bfloat16'):     # one spelling for both data-parallel paths (a typo must not run silently)
            gc = 'bf16'
        elif gc in ('none', 'fp32', 'f32', torch.float32):
            gc = None
        elif gc != 'auto':
            raise ValueError("grad_compress / REPMODE_GRAD_COMPRESS must be 'bf16', 'fp32' or 'auto', got %r" % (gc,))
        self.grad_compress_rule = 'auto' if gc == 'auto' else 'pinned'
        self.grad_compress = None if gc == 'auto' else gc
        self._bwd_events = []                                  # (start, end) of the first distributed backward passes
        # hip_graph: replay the whole train step (forward, backward, Adam: ~415 launches, 13 ms of host time) as ONE
        # HIP graph per (input shape, number of distinct tasks) -- see _graph_train_iter.  Single-GPU training only.
        self.hip_graph = bool(hip_graph)
        if self.hip_graph and distributed:
            raise ValueError('hip_graph covers single-GPU training (the collectives are not captured)')
        self._graphs = {}
        self._graph_pool = None
        self._capture_stream = None
        self.count_dist_steps = 0
        self.criterion = criterion_fn(reduction='none')        # fnet_model.py:36
        self._fused_mse = criterion_fn is torch.nn.MSELoss     # the reference's criterion: fused HIP pass (csrc/pipeline.hip)
        self._last_log = None
        self._init_model()

    def _init_model(self):
        if self.nn_module != 'RepMode':
            raise ValueError('only the RepMode network is provided (got %r)' % self.nn_module)
        from . import distributed as dist_
        from . import ops as ops_
        # a rebuild (load_state): the previous network's reducer hooks / communication buckets and DDP wrapper go first
        if getattr(self, 'reducer', None) is not None:
            self.reducer.remove()
            ops_.set_grad_sink(None)
        self.ddp = self.reducer = None
        self.net = _repmode.Net(self.opts, mult_chan=self.mult_chan, dtype=self.dtype).to(self.device)
        if self.distributed in ('reducer', 'reducer-always'):
            # gradients are produced inside the communication buckets and averaged under backward (distributed.py);
            # measured equal to the stock wrapper on one rank, not yet run on eight -> opt-in
            self.reducer = dist_.GradReducer(self.net, always_reduce=self.distributed == 'reducer-always',
                                             comm_dtype=torch.bfloat16 if self.grad_compress == 'bf16' else None)
        elif self.distributed:
            self.ddp = dist_.wrap_ddp(self.net, self.device,
                                      grad_compress='auto' if self.grad_compress_rule.startswith('auto') else self.grad_compress)
        # process-wide (one training process per GPU): where the MoDE gradient kernels put the parameter gradients
        ops_.set_grad_sink(self.reducer)
        ops_.torch_ops().clear_frag_store()          # (expert operands kept across steps belong to the previous network)
        # process-wide, like the gradient sink (one training process per GPU).  A graph replay updates the parameters with no
        # version counter and no optimizer hook to say so: with the STOCK optimizer a model that replays its step lays the
        # per-expert blocks' operands out at every forward pass (store off); with the build's own optimizer the captured pass
        # writes the stored operands itself, replay after replay (repmode_ops.cpp op_prepare_filters)
        own_adam = self.optimizer_name == 'adam' and os.environ.get('REPMODE_ADAM', '1') != '0'
        ops_.torch_ops().set_frag_store((own_adam or not self.hip_graph) and os.environ.get('REPMODE_FRAG_STORE', '1') != '0')
        if self.optimizer_name == 'adamw':
            # (writes no expert operands: as with a stock optimizer, the next forward pass lays them out)
            from .optim import AdamW
            self.optimizer = AdamW(self.net.parameters(), lr=self.lr, capturable=self.hip_graph, **self.optimizer_args)
        elif not own_adam:
            # (REPMODE_ADAM=0: the stock fused optimizer, for A/B; capturable: its step counters live on the device)
            self.optimizer = torch.optim.Adam(self.net.parameters(), lr=self.lr, fused=True, capturable=self.hip_graph)
        else:
            # fnet_model.py:55 through the build's own kernels (csrc/adam.hip): same state layout as torch.optim.Adam.  Under
            # hip_graph the step count also lives on the device (capturable) and the captured pass keeps the per-expert blocks'
            # operands current in every replay: the graph IS the eager step, operand store included.
            from .optim import Adam
            self.optimizer = Adam(self.net.parameters(), lr=self.lr, capturable=self.hip_graph)

    # ---- checkpoint: fnet_model.py:57-94 (same keys)
    def get_state(self):
        return dict(nn_module=self.nn_module, opts=self.opts, nn_state=self.net.state_dict(),
                    optimizer_state=self.optimizer.state_dict(), count_iter=self.count_iter,
                    count_epoch=self.count_epoch)

    def save_state(self, path_save):
        dirname = os.path.dirname(path_save)
        if dirname and not os.path.exists(dirname):
            os.makedirs(dirname)
        state = self.get_state()
        state['nn_state'] = {k: v.cpu() for k, v in state['nn_state'].items()}
        torch.save(state, path_save)

    def load_state(self, path_load, gpu_ids=None):
        """fnet_model.py:82-94: the checkpoint decides the network (``nn_module``, ``opts``), the model is rebuilt from it
        and moved to ``gpu_ids``.  The reference's default ``gpu_ids=-1`` means the CPU, which this build does not have:
        ``None`` (default) keeps the model's current device; a negative id raises like the constructor does."""
        state = torch.load(path_load, map_location='cpu', weights_only=False)
        if gpu_ids is not None:
            ids = [gpu_ids] if isinstance(gpu_ids, int) else list(gpu_ids)
            if ids[0] < 0:
                raise RuntimeError('repmode_amd.Model needs a HIP device; there is no CPU path')
            self.gpu_ids = ids
            self.device = torch.device('cuda', ids[0])
        if state.get('nn_module') is not None:
            self.nn_module = state['nn_module']
        if state.get('opts') is not None:
            self.opts = state['opts']
        self.opts.gpu_ids = self.gpu_ids[0]                  # (also when the checkpoint carries no opts)
        self._init_model()
        self.net.load_state_dict(state['nn_state'])
        if 'optimizer_state' in state:
            self.optimizer.load_state_dict(state['optimizer_state'])
        self.count_iter = state.get('count_iter', 0)
        self.count_epoch = state.get('count_epoch', 0)
        self._graphs, self._graph_pool = {}, None           # (captured steps hold the previous network's tensors)

    # ---- training step: fnet_model.py:96-132
    def _train_step(self, signal, target, task):
        """zero_grad, forward, MSELoss('none') -> mean, backward, (all-reduce), Adam.  ``task``: ints or a TaskPlan."""
        from . import ops as ops_
        module = self.ddp if self.ddp is not None else self.net
        # fnet_model.py:102 calls net.train() every iteration; the guard is on the INNER network, the module whose mode
        # predict() changes (a DistributedDataParallel wrapper keeps its own flag and would hide an eval-mode net)
        if not self.net.training or not module.training:
            module.train()               # (walks the whole module tree: ~0.6 ms, not needed every step)
        plan = task if isinstance(task, ops_.TaskPlan) else ops_.TaskPlan(task, self.net.num_tasks, self.device, True)
        self.optimizer.zero_grad(set_to_none=True)
        output = module(signal, plan)
        if self._fused_mse:
            # one pass: loss, d loss / d output, per-sample and per-task means (fnet_model.py:108-109, 115-122), all on the device
            loss, loss_sample, task_mean, task_count = ops_.torch_ops().mse_loss(output, target, plan.sample_task, self.net.num_tasks)
        else:
            loss_nomean = self.criterion(output, target)
            loss = torch.mean(loss_nomean)
            loss_sample = torch.mean(loss_nomean.detach(), dim=(1, 2, 3, 4))
            task_mean = task_count = None
        measure = self.grad_compress_rule == 'auto' and self.distributed and self.count_dist_steps < self.RULE_STEPS
        if measure:
            ev = (torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True))
            ev[0].record()
        if self.balance_coef:
            # (the logged loss stays the criterion's; the term and the counts are in last_balance)
            balance, counts, _ = self.net.gate_balance(plan, self.balance_coef)
            self.last_balance = (balance.detach(), counts)
            (loss + balance).backward()
        else:
            loss.backward()
        if measure:
            ev[1].record()
            self._bwd_events.append(ev)
        if self.reducer is not None:
            self.reducer.finish()
        self.optimizer.step()
        if self.distributed:
            self.count_dist_steps += 1
            if self.grad_compress_rule == 'auto' and self.count_dist_steps == self.RULE_STEPS:
                self._apply_grad_dtype_rule()
        self.last_loss = loss.detach()
        self._last_log = (self.last_loss, loss_sample, task_mean, task_count, plan.tasks_host)
        return output.detach(), loss_sample

    RULE_STEPS = 4      # distributed steps before the buckets' dtype is chosen (the first two warm the allocator and are skipped)

    def _apply_grad_dtype_rule(self):
        """Choose the gradient buckets' dtype from what was measured (distributed.pick_grad_dtype); every rank takes the MAX of
        the backward times, so all ranks decide alike.  One synchronisation, once."""
        import torch.distributed as tdist
        from . import distributed as dist_
        self.grad_compress_rule = 'auto: float32 kept'
        if not (tdist.is_available() and tdist.is_initialized()) or not self._bwd_events:
            return
        torch.cuda.synchronize(self.device)
        ms = [a.elapsed_time(b) for a, b in self._bwd_events[2:]] or [a.elapsed_time(b) for a, b in self._bwd_events]
        self._bwd_events = []
        bwd = dist_.max_over_ranks(float(np.median(ms)), self.device)
        nbytes = 4 * sum(p.numel() for p in self.net.parameters() if p.requires_grad)
        world = tdist.get_world_size()
        pick = dist_.pick_grad_dtype(nbytes, world, bwd, tdist.get_backend())
        self.grad_compress_rule = 'auto: ring estimate %.2f ms vs backward %.2f ms -> %s' % (
            dist_.ring_allreduce_ms(nbytes, world), bwd, pick or 'float32')
        if tdist.get_rank() == 0:
            import sys
            print('repmode_amd: gradient buckets -- %s' % self.grad_compress_rule, file=sys.stderr, flush=True)
        if pick == 'bf16' and self.grad_compress != 'bf16':
            self.grad_compress = 'bf16'
            if self.reducer is not None:
                self.reducer.comm_dtype = torch.bfloat16
            elif self.ddp is not None:
                self.ddp.grad_dtype_switch.dtype = 'bf16'      # (one wrapper for the whole run: the hook reads this flag)

    def loss_log(self):
        """The dict the reference hands to ``wandb.log`` and its per-sample DataFrame (fnet_model.py:115-130) for the last
        ``do_train_iter``.  The values were computed on the device during the step; THIS call copies them to the host
        (one synchronisation, when and if the caller wants the numbers -- the reference pays ~4 per iteration)."""
        import pandas as pd
        if self._last_log is None:
            raise RuntimeError('loss_log(): no train iteration has run yet')
        loss, loss_sample, task_mean, task_count, tasks = self._last_log
        names = self.opts.adopted_datasets
        per = loss_sample.float().cpu().numpy()
        # (count_iter is the caller's: main.py:250 sets it before the call)
        log = {'X-axis/iter': self.count_iter, 'loss/iter': float(loss)}
        if task_mean is not None:
            tm = task_mean.cpu().numpy()
            for i in sorted(set(tasks)):
                log['loss_iter/%s' % names[i]] = float(tm[i])
        else:
            for i in sorted(set(tasks)):
                log['loss_iter/%s' % names[i]] = float(per[[j for j, t in enumerate(tasks) if t == i]].mean())
        frame = pd.DataFrame({'dataset': [names[i] for i in tasks], 'loss': list(per)})
        return log, frame

    def do_train_iter(self, signal, target, task, sync=False, eager=False):
        """One optimisation step.  ``task`` should be a CPU int tensor (as the DataLoader yields it):
        the slot plan is then built without touching the device.  Returns (output, per-sample loss);
        both stay on the device unless ``sync`` (then they are copied to the host like the reference
        does).  With ``hip_graph`` the step is a graph replay (``eager=True``: this step launch by launch) and the
        returned tensors are overwritten by the next replay of the same shape."""
        signal = signal.to(self.device, non_blocking=True)
        target = target.to(self.device, non_blocking=True)
        if torch.is_tensor(task) and not task.is_cuda:
            task = [int(t) for t in task.tolist()]   # plain ints: DDP's input scatter would move a tensor to the GPU
        if self.hip_graph and not eager:
            output, loss_sample = self._graph_train_iter(signal, target, task)
        else:
            output, loss_sample = self._train_step(signal, target, task)
        if sync:
            return output.cpu(), loss_sample.cpu()
        return output, loss_sample

    GRAPH_WARMUP = 2     # launch-by-launch steps on the capture stream before a shape is captured

    def _graph_train_iter(self, signal, target, task):
        """The train step as a HIP graph.  One graph per (input shape, number of distinct tasks): that pair fixes every
        launch's grid, every buffer size and which levels take the per-expert formulation; WHICH tasks they are is
        data (three small index vectors, updated in place before the replay).  The first GRAPH_WARMUP steps of a
        signature run launch by launch on the capture stream (they create the optimizer state, the library's
        per-stream scratch and the zero pool's plan), the next one is captured -- into a private memory pool, so the
        step's activations keep their addresses -- and replayed; from then on a step costs the host three small
        copies and one graph launch."""
        from . import ops as ops_
        plan = task if isinstance(task, ops_.TaskPlan) else None
        host = list(plan.tasks_host) if plan is not None else [int(t) for t in (task.tolist() if torch.is_tensor(task) else task)]
        key = (tuple(signal.shape), signal.dtype, len(set(host)))
        st = self._graphs.get(key)
        if st is None:
            st = self._graphs[key] = {'calls': 0, 'graph': None}
        cur = torch.cuda.current_stream(self.device)
        if self._capture_stream is None:
            self._capture_stream = torch.cuda.Stream(self.device)
        cs = self._capture_stream
        if st['graph'] is None:
            st['calls'] += 1
            if st['calls'] <= self.GRAPH_WARMUP:
                cs.wait_stream(cur)
                with torch.cuda.stream(cs):
                    out = self._train_step(signal, target, ops_.TaskPlan(host, self.net.num_tasks, self.device, True))
                cur.wait_stream(cs)
                return out
            if ops_.torch_ops().graph_alive(list(self.net.parameters())):
                raise RuntimeError('Model(hip_graph=True): an autograd graph of the network is alive (an output or a gate_balance loss '
                                   'that was computed with gradients and is still held): release it before a step is captured')
            st['signal'], st['target'] = signal.clone(), target.clone()
            st['plan'] = ops_.TaskPlan(host, self.net.num_tasks, self.device, True)
            graph = torch.cuda.CUDAGraph()
            cs.wait_stream(cur)
            # every captured signature shares ONE private memory pool (replays never overlap: they run in stream
            # order), so a new number of distinct tasks costs its peak once, not a whole extra step of activations
            if self._graph_pool is None:
                self._graph_pool = torch.cuda.graph_pool_handle()
            with torch.cuda.graph(graph, stream=cs, pool=self._graph_pool):
                st['out'] = self._train_step(st['signal'], st['target'], st['plan'])
            st['graph'], st['last_loss'] = graph, self.last_loss
            # the per-expert blocks' operands kept across steps were captured BY ADDRESS: whoever holds the graph holds them
            # (the store may drop its entries -- another optimizer steps, another Model is built -- while replays go on)
            st['operands'] = ops_.torch_ops().pinned_operands()
            st['log'] = self._last_log[:4]
            st['balance'], st['norm'] = self.last_balance, getattr(self.optimizer, 'last_norm', None)
            st['plan'].bn_counted = False
        else:
            st['signal'].copy_(signal, non_blocking=True)
            st['target'].copy_(target, non_blocking=True)
        sp = st['plan']
        if host != sp.tasks_host:
            new = ops_.TaskPlan(host, self.net.num_tasks, self.device, True)
            sp.slot_task.copy_(new.slot_task, non_blocking=True)
            sp.sample_slot.copy_(new.sample_slot, non_blocking=True)
            sp.sample_task.copy_(new.sample_task, non_blocking=True)
            sp.tasks_host, sp.slot_task_host = new.tasks_host, new.slot_task_host
        st['graph'].replay()
        self.last_loss, self.last_balance = st['last_loss'], st['balance']
        if st['norm'] is not None:
            self.optimizer.last_norm = st['norm']
        self._last_log = st['log'] + (host,)
        return st['out']

    # ---- sliding-window inference: fnet_model.py:149-223
    def predict(self, signal, task, patch_size=None):
        patch_size = tuple(patch_size or self.patch_size)
        signal = signal.to(self.device)
        self.net.eval()
        img_size = signal.shape[-3:]
        gauss = torch.from_numpy(get_gaussian(patch_size)).to(self.device)
        pred_sum = torch.zeros(signal.shape, device=self.device)
        weight_sum = torch.zeros(signal.shape, device=self.device)
        patches = patch_grid(img_size, patch_size)
        task_id = int(task.reshape(-1)[0]) if torch.is_tensor(task) else int(task)
        bs = int(self.opts.batch_size_eval)
        from . import ops as ops_
        # eval mode: one task, one merged filter per block -- computed for the first batch of patches, re-used for the rest
        with torch.no_grad(), ops_.eval_filter_cache():
            # one volume of one channel (what the reference's test set holds): the batch's crops and its Gaussian blend are
            # one kernel launch each (csrc/pipeline.hip); any other shape takes the reference's indexing expressions
            single = (signal.is_cuda and signal.shape[0] == 1 and signal.shape[1] == 1 and signal.dtype == torch.float32 and
                      all(i >= p for i, p in zip(img_size, patch_size)))
            while patches:                                      # LIFO batches, fnet_model.py:196-200
                batch = [patches.pop() for _ in range(min(bs, len(patches)))]
                if single:
                    starts = [s for s, _ in batch]
                    out = self.net(ops_.patch_gather(signal, starts, patch_size), [task_id] * len(batch))
                    if out.dtype not in (torch.float32, torch.bfloat16):
                        out = out.float()
                    ops_.patch_blend(out, gauss, starts, pred_sum, weight_sum)
                    continue
                crops = torch.cat([signal[:, :, s[0]:e[0], s[1]:e[1], s[2]:e[2]] for s, e in batch], dim=0)
                out = self.net(crops, [task_id] * len(batch))
                for i, (s, e) in enumerate(batch):
                    pred_sum[:, :, s[0]:e[0], s[1]:e[1], s[2]:e[2]] += out[i:i + 1] * gauss
                    weight_sum[:, :, s[0]:e[0], s[1]:e[1], s[2]:e[2]] += gauss
        return (pred_sum / weight_sum).cpu()
