"""AdamW over all tensors of a network in one launch, with moments in 32 or in 8 bits."""
import struct
from collections import defaultdict

import numpy as np
import torch as ch

from . import _native as N

_BLOCK = N.ADAMW_BLOCK
_address = ch.Tensor.data_ptr


class AdamW(ch.optim.Optimizer):
    """Adam with decoupled weight decay.

    Parameters
    ----------
    params : iterable
        Parameters or groups of them, all of one floating type and on one GPU.
    lr, betas, eps, weight_decay
        As in ``torch.optim.AdamW``; each may differ from group to group and change from step to step.
    state_bits : 32 or 8
        8 keeps the first moment as an e4m3 and the second as an e5m2 number, with one power of two as scale per 256
        values, rounded stochastically.
    max_grad_norm : float
        Gradients are scaled down together so that their norm is at most this.  Where the norm is not finite, the step
        changes nothing (but counts).  ``grad_norm`` holds the last step's norm, on the GPU.
        A value that is not finite, without such a bound, makes its block of 256 values none with 8-bit moments, and itself with 32.
    seed : int
        Of the stochastic rounding: the same seed, steps and gradients give the same weights.

    16-bit parameters have 32-bit masters, which the steps are made on.  Values that were written to a parameter since (by
    ``load_state_dict`` of a network, by a swap for its average, by clamping) take their masters' place at the next step; what is written
    through ``p.data`` autograd does not know of, and ``masters_from_parameters`` has to be called behind it.  The state lies in flat tensors, ``exp_avg``,
    ``exp_avg_sq``, ``scales`` (8 bits) and ``master`` (16-bit parameters), of which ``state[p]`` has views; every
    parameter begins a block of 256 values, the rest of its last block is zero.  A parameter without a gradient is left alone,
    and its step is not counted.  The kernels read the current learning rates from the groups and take gradients and
    parameters wherever they lie at the time of the step.  Where the order of a parameter's values in memory has changed
    (``model.to(memory_format=...)``) its state is brought into that order, moments in 8 bits rounded once more; a parameter of
    another shape or type, on another device or with gaps is refused.  A step cannot be captured in a graph: its number, the rates and
    the gradients' addresses come from the host.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, max_grad_norm=None,
                 seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f'state_bits must be 8 or 32, not {state_bits}')
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise ValueError(f'max_grad_norm must be positive, not {max_grad_norm}')
        self.state_bits, self.max_grad_norm, self.seed = state_bits, max_grad_norm, int(seed)
        self._blank()
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def _blank(self):
        self.exp_avg = self.exp_avg_sq = self.scales = self.master = self.grad_norm = None
        self._params, self._numel, self._steps = [], None, np.zeros(0, np.int64)
        self._layouts = self._grad_layouts = None
        self._seen = [], []  # 16-bit parameters' versions and addresses when their masters were last as they are

    @staticmethod
    def _check_group(group):
        b1, b2 = group['betas']
        if not (group['lr'] >= 0 and group['eps'] >= 0 and group['weight_decay'] >= 0 and 0 <= b1 < 1 and 0 <= b2 < 1):
            raise ValueError('lr, eps and weight_decay must not be negative, betas must be in [0, 1): '
                             f"{ {k: group[k] for k in ('lr', 'betas', 'eps', 'weight_decay')} }")

    def add_param_group(self, group):
        super().add_param_group(group)
        group = self.param_groups[-1]
        try:
            self._check_group(group)
            self._check_params()
            for p in group['params']:
                N.require(p, 'parameter')
                like = self._params[0] if self._params else group['params'][0]
                if p.dtype != like.dtype or p.device != like.device:
                    raise TypeError(f'parameters must be of one type on one GPU: {p.dtype} on {p.device}, {like.dtype} on {like.device}')
                if not _dense(p):
                    raise ValueError('parameters must lie together in memory, without gaps or overlaps')
        except Exception:
            self.param_groups.pop()
            raise
        if self._params or group['params']:
            self._lay_out()

    def _check_params(self):
        """Refuses parameters that are no longer what their state was made for."""
        for p in self._params:
            was = self.state[p]['exp_avg'].shape
            if p.dtype != self._dtype or p.device != self.exp_avg.device or p.layout != ch.strided:
                raise TypeError(f'a parameter is {p.dtype} {p.layout} on {p.device} now; the state was made for {self._dtype} on {self.exp_avg.device}')
            if p.shape != was:
                raise ValueError(f'a parameter of shape {tuple(was)} is of shape {tuple(p.shape)} now: its state belongs to the values it had')
            if not _dense(p):
                raise ValueError('parameters must lie together in memory, without gaps or overlaps')

    @ch.no_grad()
    def _lay_out(self):
        """Flat state for all parameters of all groups, as they lie now; what there was keeps its values."""
        old = {p: (self.state[p], int(step)) for p, step in zip(self._params, self._steps)}
        seen = dict(zip(self._params, zip(*self._seen)))
        self._params = [p for group in self.param_groups for p in group['params']]
        n, device, dtype = len(self._params), self._params[0].device, self._params[0].dtype
        self._dtype = dtype
        self._numel = np.array([p.numel() for p in self._params], np.int64)
        self._start, sizes = np.zeros(n, np.int64), np.zeros(2, np.int64)
        total = N.lib.ffcvb_adamw_layout(n, self._numel.ctypes.data, self._start.ctypes.data, sizes.ctypes.data)
        zeros = lambda t: ch.zeros(total, dtype=t, device=device)  # noqa: E731
        eight = self.state_bits == 8
        self.exp_avg = zeros(ch.uint8).view(ch.float8_e4m3fn) if eight else zeros(ch.float32)
        self.exp_avg_sq = zeros(ch.uint8).view(ch.float8_e5m2) if eight else zeros(ch.float32)
        self.scales = ch.ones((total // _BLOCK, 2), device=device) if eight else None
        self.master = None if dtype == ch.float32 else zeros(ch.float32)
        self._table = ch.empty(int(sizes[0]), dtype=ch.uint8, device=device)
        self._workspace = ch.empty(max(16, int(sizes[1])), dtype=ch.uint8, device=device) if self.max_grad_norm else None
        self.grad_norm = ch.zeros((), device=device) if self.max_grad_norm else None
        self._table_size, self._at = int(sizes[0]), None
        self._layouts, self._grad_layouts = N.layouts(self._params), None
        self._group_of = np.repeat(np.arange(len(self.param_groups), dtype=np.int32), [len(g['params']) for g in self.param_groups])
        steps = np.zeros(n, np.int64)
        for i, p in enumerate(self._params):
            entry = dict(step=0, exp_avg=self._of(self.exp_avg, i), exp_avg_sq=self._of(self.exp_avg_sq, i))
            if eight:
                first = int(self._start[i]) // _BLOCK
                entry['scales'] = self.scales[first:first - (-p.numel() // _BLOCK)]
            if self.master is not None:
                entry['master'] = self._of(self.master, i)
            if p in old:
                was, steps[i] = old[p]
                entry['step'] = int(steps[i])
                self._take(entry, was)
            elif self.master is not None:
                entry['master'].copy_(p.detach())
            self.state[p] = entry
        self._steps = steps
        if self.master is not None:
            both = [seen.get(p, (p._version, p.data_ptr())) for p in self._params]
            self._seen = [version for version, _ in both], [place for _, place in both]
        self._host = self._numel.ctypes.data, self._steps.ctypes.data, self._group_of.ctypes.data

    def masters_from_parameters(self):
        """Makes masters follow 16-bit parameters that have been written to: where a value is not its master rounded, it becomes the
        master."""
        if self.master is not None:
            self._place()
            self._follow([1] * len(self._params))

    def _follow(self, which):
        n = len(self._params)
        N.check(N.lib.ffcvb_adamw_masters(self._args(), self._host[0], struct.pack(f'={n}Q', *which), N.raw_stream(self._params[0].get_device())))

    def _place(self):
        """Addresses of the parameters, which the table in device memory has too."""
        params = self._params
        if not self._layouts.check(*params):
            self._check_params()
            if any(_order(p) != _order(self.state[p]['exp_avg']) for p in params):
                self._lay_out()
            self._layouts = N.layouts(params)
        at = list(map(_address, params))
        if at != self._at:  # the first step, or parameters that have moved
            host = np.empty(max(1, self._table_size), np.uint8)
            where = np.array(at, np.uint64)
            N.check(N.lib.ffcvb_adamw_table(len(params), self._numel.ctypes.data, where.ctypes.data, host.ctypes.data))
            self._table.copy_(ch.from_numpy(host[:self._table_size]))
            self._at = at
        return at

    def _args(self):
        return N.ADAMW.pack(self._table.data_ptr(), self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(), N.ptr(self.scales),
                            N.ptr(self.master), N.ptr(self.grad_norm), N.ptr(self._workspace), self.seed, self._params[0].get_device(),
                            N.TYPES[self._dtype], self.state_bits, len(self._params), self.max_grad_norm or 0.0)

    def _take(self, own, was):
        """A parameter's state from another of the same shape, whatever order in memory either is in."""
        if 'master' in own:
            own['master'].copy_(was['master'])
        if self.state_bits == 8 and _order(own['exp_avg']) != _order(was['exp_avg']):
            for k, name in enumerate(('exp_avg', 'exp_avg_sq')):
                _in_eight(own[name], own['scales'][:, k], _from_eight(was[name], was['scales'][:, k]))
            return
        for name in ('exp_avg', 'exp_avg_sq', 'scales'):
            if name in own:
                own[name].copy_(was[name])

    def _of(self, flat, i):
        """Parameter i's part of a flat tensor, in the parameter's shape and order in memory."""
        p = self._params[i]
        return ch.as_strided(flat, p.shape, p.stride(), int(self._start[i]))

    def _as_parameter(self, p, g):
        """A gradient that is laid out as its parameter."""
        if g.layout != ch.strided or g.dtype != p.dtype or g.device != p.device:
            raise TypeError(f'gradients must be dense, of the parameters\' type and on their GPU, not {g.dtype} {g.layout} on {g.device}')
        if g.shape != p.shape:
            raise ValueError(f'a parameter of shape {tuple(p.shape)} has a gradient of shape {tuple(g.shape)}')
        return g if _order(g) == _order(p) else ch.empty_like(p, requires_grad=False).copy_(g.detach())

    def step(self, closure=None):
        if N.capturing():
            raise RuntimeError('a step of AdamW cannot be captured in a graph: a replay would repeat its number, rates and gradients\' addresses')
        loss = None
        if closure is not None:
            with ch.enable_grad():
                loss = closure()
        params, n = self._params, len(self._params)
        if not params:
            return loss
        at = self._place()
        if self.master is not None:
            seen = [p._version for p in params], at
            if seen != self._seen:
                self._follow([now != then for now, then in zip(zip(*seen), zip(*self._seen))])
        # addresses of gradients, 0 without one
        grads, kept = [p.grad for p in params], None
        if self._grad_layouts is not None and self._grad_layouts.check(*grads):
            grads_at = list(map(_address, grads))
        else:
            kept = [None if g is None else self._as_parameter(p, g) for p, g in zip(params, grads)]
            grads_at = [N.ptr(g) for g in kept]
            self._grad_layouts = N.layouts(kept) if all(g is not None and g is own for g, own in zip(kept, grads)) else None
        groups = b''
        for group in self.param_groups:
            self._check_group(group)
            groups += N.ADAMW_GROUP.pack(group['lr'], *group['betas'], group['eps'], group['weight_decay'])
        N.check(N.lib.ffcvb_adamw_step(self._args(), *self._host, struct.pack(f'={n}Q', *grads_at), groups, len(self.param_groups),
                                       N.raw_stream(params[0].get_device())))
        del kept
        # (a later backward pass that needs what they were says so)
        ch.autograd.graph.increment_version(params if all(grads_at) else [p for p, g in zip(params, grads_at) if g])
        if self.master is not None:
            self._seen = [p._version for p in params], at
        return loss

    def _count(self):
        """Brings the steps in ``state`` up to date."""
        for p, step in zip(self._params, self._steps):
            self.state[p]['step'] = int(step)

    def state_dict(self):
        self._count()
        saved = super().state_dict()
        saved['state_bits'] = self.state_bits
        return saved

    def __getstate__(self):
        self._count()
        saved = super().__getstate__()
        if self.state_bits == 8:  # (as whole numbers: pickle has no codes)
            saved['state'] = {p: {k: t.view(ch.uint8) if k.startswith('exp') else t for k, t in entry.items()} for p, entry in self.state.items()}
        return dict(saved, _own=(self.state_bits, self.max_grad_norm, self.seed))

    @ch.no_grad()
    def __setstate__(self, saved):
        """A copy (``copy.deepcopy``, ``pickle``) has flat state of its own."""
        saved = dict(saved)
        self.state_bits, self.max_grad_norm, self.seed = saved.pop('_own')
        was, saved['state'] = saved['state'], defaultdict(dict)
        super().__setstate__(saved)
        self._blank()
        if any(group['params'] for group in self.param_groups):
            self._lay_out()
        for i, p in enumerate(self._params):
            own, entry = self.state[p], was[p]
            self._take(own, {k: t.view(own[k].dtype) if k.startswith('exp') else t for k, t in entry.items()})
            self._steps[i] = own['step'] = entry['step']
        self._seen = [None] * len(self._params), [None] * len(self._params)

    @ch.no_grad()
    def load_state_dict(self, saved):
        """State as :meth:`state_dict` gives it, of the same parameters in the same groups; with ``state_bits=32`` also
        that of ``torch.optim.AdamW``.  Values are copied into the flat tensors; a parameter without saved state begins anew.  What
        does not fit is refused before anything is changed."""
        groups = saved['param_groups']
        if [len(g['params']) for g in groups] != [len(g['params']) for g in self.param_groups]:
            raise ValueError('the saved state has other parameter groups')
        if saved.get('state_bits', 32) != self.state_bits:
            raise ValueError(f"the saved state has {saved.get('state_bits', 32)}-bit moments, not {self.state_bits}-bit ones")
        options = [{key: theirs.get(key, value) for key, value in group.items() if key != 'params'}
                   for group, theirs in zip(self.param_groups, groups)]
        for group in options:
            self._check_group(group)
        entries = [saved['state'].get(i) for g in groups for i in g['params']]
        for p, entry in zip(self._params, entries):
            for name, view in self.state[p].items() if entry else ():
                if name == 'step' or (name == 'master' and name not in entry):
                    continue
                if entry[name].shape != view.shape or entry[name].dtype != view.dtype:
                    raise ValueError(f'saved {name}: {entry[name].dtype} {tuple(entry[name].shape)}, not {view.dtype} {tuple(view.shape)}')
                if self.state_bits == 8 and not _dense(entry[name]):
                    raise ValueError(f'saved {name}: values with gaps or overlaps have no blocks')
        for group, values in zip(self.param_groups, options):
            group.update(values)
        for i, (p, entry) in enumerate(zip(self._params, entries)):
            own = self.state[p]
            if entry:
                self._take(own, entry if 'master' in entry else dict(entry, master=p.detach()))
            else:
                for name in ('exp_avg', 'exp_avg_sq'):
                    _in_memory(own[name]).view(ch.uint8).zero_()
                if 'scales' in own:
                    own['scales'].fill_(1.0)
                if 'master' in own:
                    own['master'].copy_(p.detach())
            self._steps[i] = int(entry['step']) if entry else 0
        self._seen = [None] * len(self._params), [None] * len(self._params)  # (parameters may be others than those that the saved masters belong to)


def _dense(p):
    """Whether a tensor's values fill a stretch of memory, each once, in whatever order."""
    size = 1
    for stride, n in sorted((s, n) for s, n in zip(p.stride(), p.shape) if n != 1):
        if stride != size:
            return p.numel() == 0
        size *= n
    return True


def _order(t):
    """The order of a dense tensor's values in memory."""
    return [stride for stride, n in zip(t.stride(), t.shape) if n != 1]


def _in_memory(t):
    """A dense tensor's values in the order in which they lie in memory."""
    return ch.as_strided(t, (t.numel(),), (1,))


_TOP = {ch.float8_e4m3fn: 7, ch.float8_e5m2: 14}  # a block's largest value is 2^TOP .. 2^(TOP + 1) times its scale


def _from_eight(codes, scales):
    """A moment in 32 bits, in its codes' order in memory."""
    values = ch.empty_like(codes, dtype=ch.float32)
    _in_memory(values).copy_(_in_memory(codes).float() * scales.repeat_interleave(_BLOCK)[:codes.numel()])
    return values


def _in_eight(codes, scales, values):
    """Writes a moment as codes and scales, as the kernel does but rounded to the nearest."""
    if codes.numel() == 0:
        return
    own = ch.empty_like(codes, dtype=ch.float32).copy_(values)
    blocks = ch.nn.functional.pad(_in_memory(own), (0, -codes.numel() % _BLOCK)).view(-1, _BLOCK).double()
    top = _TOP[codes.dtype]
    power = (ch.frexp(blocks.abs().amax(1))[1] - 1).clamp(min=-126)
    finite = ch.isfinite(blocks).all(1)
    scales.copy_(ch.where(finite, ch.ldexp(ch.ones_like(power, dtype=ch.float64), power - top), ch.nan))
    scaled = ch.ldexp(blocks, (top - power)[:, None])
    if codes.dtype == ch.float8_e5m2:  # (above zero it stays above zero)
        scaled = ch.where(blocks > 0, scaled.clamp(min=2.0 ** -16), scaled)
    _in_memory(codes).copy_(scaled.view(-1)[:codes.numel()].float().to(codes.dtype))
