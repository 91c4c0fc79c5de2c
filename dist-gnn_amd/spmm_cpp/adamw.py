"""AdamW over many tensors at once (C ABI: dgnn_adamw, include/dgnn_train.h).

The reference's training loop steps ``torch.optim.Adam`` (light_dist_gnn/dist_train.py:32,45), a dozen passes over every
parameter. Here a step is one pass over parameter, gradient and moments, for up to 64 tensors a launch, with the moments
in 32 or in 8 bits.
"""
import math

import numpy as np
import torch

from . import _DTYPES, _ext

BLOCK = 256                       # elements that share a scale; a tensor starts at a multiple of it in the state buffers


def _kinds(bits, master):
    """{state name: (type, elements per scale or 1)} of one tensor."""
    if bits == 32:
        kinds = {'exp_avg': (torch.float32, 1), 'exp_avg_sq': (torch.float32, 1)}
    else:
        kinds = {'exp_avg': (torch.float8_e4m3fn, 1), 'exp_avg_scale': (torch.float32, BLOCK),
                 'exp_avg_rms': (torch.float8_e4m3fn, 1), 'exp_avg_rms_scale': (torch.float32, BLOCK)}
    if master:
        kinds['master'] = (torch.float32, 1)
    return kinds


class _Segment:
    """The parameters of one group that share a device and a type, and their state: one flat buffer per kind, every tensor's
    part starting at a multiple of 256 elements."""

    def __init__(self, params, bits, master, capturable):
        self.params, self.bits, self.has_master, self.capturable = params, bits, master, capturable
        self.device, self.dtype = params[0].device, params[0].dtype
        sizes = np.array([p.numel() for p in params], dtype=np.int64)
        blocks = -(-sizes // BLOCK)
        self.starts = (np.cumsum(blocks) - blocks) * BLOCK
        self.sizes, total = sizes, int(blocks.sum()) * BLOCK
        self.kinds = _kinds(bits, master)
        self.flat = {}
        for name, (dtype, per) in self.kinds.items():
            self.flat[name] = torch.zeros(max(total // per, 4), dtype=torch.uint8 if dtype.itemsize == 1 else dtype,
                                          device=self.device).view(dtype)[:total // per]
        if capturable:
            self.steps = torch.zeros(len(params), dtype=torch.int64, device=self.device)
            self.factors = torch.zeros(len(params), 4, dtype=torch.float32, device=self.device)
        else:
            self.steps = torch.zeros(len(params), dtype=torch.int64)
        f = self.flat
        self.table = _ext.AdamTable(params, self.starts.tolist(), bits, f['exp_avg'], f['exp_avg_sq' if bits == 32 else 'exp_avg_rms'],
                                    f.get('exp_avg_scale'), f.get('exp_avg_rms_scale'), f.get('master'), self.steps,
                                    self.factors if capturable else None)

    def views(self, i):
        """The state dict entry of parameter i: views of the flat buffers."""
        at, n = int(self.starts[i]), int(self.sizes[i])
        shape = self.params[i].shape
        one = {'step': self.steps[i]}
        for name, (_, per) in self.kinds.items():
            one[name] = self.flat[name][at:at + n].view(shape) if per == 1 else self.flat[name][at // per:at // per + -(-n // per)]
        return one


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) on the GPU, all tensors of a parameter group in one pass:

        m <- b1 m + (1 - b1) g,   v <- b2 v + (1 - b2) g^2
        p <- p (1 - lr weight_decay) - lr / (1 - b1^t)  m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    computed in fp32 whatever the parameters' type (fp32, bf16, fp16), p rounded once at the end.

    ``state_bits=8`` keeps m and sqrt(v) as e4m3 codes with one fp32 scale per 256 elements (2.03 bytes of state an element
    instead of 8). Codes are rounded with a dither that depends on the element and the step alone: plain rounding would hold
    a slow average where it is (v moves 0.1 % a step, a code's gap is 6 to 12 %); results are still reproducible to the bit.
    A gradient that is not finite spoils its block of 256 elements, not its element alone.

    ``master_weights=True`` (bf16 / fp16 parameters) keeps fp32 values that are updated and rounded into the parameters. An
    element of a parameter that is not its master rounded was written by somebody else since (a loaded checkpoint, a
    broadcast) and becomes its master's new value: the step reads the parameter for that (2 bytes of 18 an element).

    ``capturable=True`` keeps the step counts on the device, so that ``step()`` can be captured in a HIP graph and replayed;
    lr and weight_decay are those of the capture, and the gradients have to stay where they were. Take one step, or call
    ``init_state()``, before the capture. A counter belongs to a parameter: one without a gradient is left out and not counted.

    State tensors are views of flat buffers (``state_buffers()``): write into them or use ``load_state_dict``; putting
    other tensors in their place is not seen. Parameters must be contiguous and must not overlap, and stay in their group once
    they have state."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, master_weights=False,
                 capturable=False):
        for name, x in (('lr', lr), ('eps', eps), ('weight_decay', weight_decay)):
            if isinstance(x, torch.Tensor):
                raise ValueError(f'AdamW: {name} must be a number, got {x!r}')
        if state_bits not in (8, 32):
            raise ValueError(f'AdamW: state_bits must be 8 or 32, got {state_bits!r}')
        self._segments = None
        self.state_bits, self.master_weights, self.capturable = state_bits, bool(master_weights), bool(capturable)
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    # ------------------------------------------------------------------ state
    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        try:
            self._check_options(self.param_groups[-1])
            self._check_params()
        except Exception:
            self.param_groups.pop()                       # a group that is refused is not there
            raise

    @staticmethod
    def _check_options(group):
        for name in ('lr', 'eps', 'weight_decay'):
            x = float(group[name])
            if not x >= 0 or math.isinf(x):
                raise ValueError(f'AdamW: {name} must be a finite number >= 0, got {x!r}')
        betas = group['betas']
        if len(betas) != 2 or not all(0 <= b < 1 for b in betas):
            raise ValueError(f'AdamW: betas must lie in [0, 1), got {betas!r}')

    def _check_params(self):
        seen = set()
        for group in self.param_groups:
            for p in group['params']:
                if not p.is_cuda:
                    raise RuntimeError(f'AdamW: a parameter is on {p.device}; this optimiser has no CPU path')
                if p.dtype not in _DTYPES:
                    raise RuntimeError(f'AdamW: parameters must be fp32, bf16 or fp16, got {p.dtype}')
                if p.is_sparse or not p.is_contiguous():
                    raise RuntimeError('AdamW: parameters must be dense and contiguous')
                if self.master_weights and p.dtype == torch.float32:
                    raise RuntimeError('AdamW: master_weights is for bf16 and fp16 parameters')
                if id(p) in seen:
                    raise RuntimeError('AdamW: a parameter is given twice')
                seen.add(id(p))
        spans = sorted((p.device.index, p.data_ptr(), p.data_ptr() + p.numel() * p.element_size())
                       for g in self.param_groups for p in g['params'] if p.numel())
        for a, b in zip(spans, spans[1:]):
            if a[0] == b[0] and b[1] < a[2]:
                raise RuntimeError('AdamW: two parameters overlap in memory')

    def _current(self):
        """Whether param_groups hold the parameters that state was made for."""
        return (self._segments is not None and len(self._known) == len(self.param_groups)
                and all(_ext.same_objects(known, g['params']) for known, g in zip(self._known, self.param_groups)))

    @torch.no_grad()
    def init_state(self):
        """Allocates the state of parameters that have none yet (zeros; a master takes its parameter's value)."""
        if self._current():
            return
        self._check_params()
        if self._segments is None:
            self._segments, self._known = [], []
        for known, params in zip(self._known, [g['params'] for g in self.param_groups] + [()] * len(self._known)):
            if {id(p) for p in known} - {id(p) for p in params}:
                raise RuntimeError('AdamW: a parameter was taken out of param_groups or replaced after its state was made; make a new '
                                   'optimiser (load_state_dict brings the state along)')
        self._segments += [[] for _ in self.param_groups[len(self._segments):]]
        for group, segments in zip(self.param_groups, self._segments):
            known = {id(p) for s in segments for p in s.params}
            sorts = {}
            for p in group['params']:
                if id(p) not in known:
                    sorts.setdefault((p.device, p.dtype), []).append(p)
            for params in sorts.values():
                seg = _Segment(params, self.state_bits, self.master_weights, self.capturable)
                made = [seg.views(i) for i in range(len(params))]
                for one, p in zip(made, params):
                    if self.state.get(p):                 # a copy's
                        self._check(one, self.state[p])
                for one, p in zip(made, params):
                    if self.state.get(p):
                        self._take(one, self.state[p])
                    elif seg.has_master:
                        one['master'].copy_(p.detach())
                    self.state[p] = one
                segments.append(seg)
        self._known = [list(group['params']) for group in self.param_groups]

    def _check(self, to, given):
        """Refuses a state entry of a state dict (or of another copy of this optimiser) that does not fit the views ``to``."""
        if set(given) != set(to):
            raise ValueError(f'AdamW: a state with {sorted(given)} does not fit state_bits={self.state_bits}, '
                             f'master_weights={self.master_weights} (wanted: {sorted(to)})')
        for name, x in to.items():
            y = given[name]
            if name == 'step':
                int(y)
            elif not isinstance(y, torch.Tensor) or y.numel() != x.numel():
                raise ValueError(f'AdamW: state {name} does not have the parameter\'s size')
            elif x.dtype.itemsize == 1 and y.dtype != x.dtype:
                raise ValueError(f'AdamW: state {name} must be {x.dtype}, got {y.dtype}')

    def _take(self, to, given):
        """Copies a state entry that ``_check`` passed into the views ``to``."""
        for name, x in to.items():
            y = given[name]
            if name == 'step':
                x.fill_(int(y))
            elif x.dtype.itemsize == 1:
                x.view(torch.uint8).view(-1).copy_(y.contiguous().view(torch.uint8).view(-1))
            else:
                x.view(-1).copy_(y.reshape(-1))

    def state_buffers(self):
        """{name: flat tensor} of all state, in the order of the parameters, every tensor's part starting at a multiple of
        256 elements (of its 1 scale per 256): what a sharded or asynchronous checkpoint copies in a few pieces. Names of a
        second, third, ... set of parameters (another group, device or type) end in .1, .2, ..."""
        self.init_state()
        found = [s for segments in self._segments for s in segments]
        return {name + (f'.{i}' if i else ''): t for i, s in enumerate(found) for name, t in s.flat.items()}

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Writes the state into the buffers that are there (a captured step goes on with it); a parameter without an entry
        starts anew. A state that does not fit is refused with nothing written."""
        self.init_state()
        kept, found = (self._segments, self.state), {}
        own = {t.untyped_storage().data_ptr() for segments in self._segments for s in segments for t in (*s.flat.values(), s.steps)}

        def check(_, given):                              # behind the hooks that may change what is loaded
            ids = [i for g in given['param_groups'] for i in g['params']]
            for i, p in zip(ids, (p for g in self.param_groups for p in g['params'])):
                if given['state'].get(i):
                    self._check(self.state[p], given['state'][i])
                    found[p] = {n: y.clone() if isinstance(y, torch.Tensor) and y.untyped_storage().data_ptr() in own else y
                                for n, y in given['state'][i].items()}
            return {**given, 'state': {}}

        def fill(_):                                      # before the hooks that look at what was loaded
            self._segments, self.state = kept
            for group in self.param_groups:
                for p in group['params']:
                    to = self.state[p]
                    if p in found:
                        self._take(to, found[p])
                        continue
                    for name, x in to.items():
                        x.copy_(p) if name == 'master' else (x.view(torch.uint8) if x.dtype.itemsize == 1 else x).zero_()

        hooks = (self.register_load_state_dict_pre_hook(check), self.register_load_state_dict_post_hook(fill, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def __getstate__(self):
        return {**super().__getstate__(), 'state_bits': self.state_bits, 'master_weights': self.master_weights,
                'capturable': self.capturable}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._segments = None                             # a copy: flat buffers of its own, filled from the copied state
        if any(self.state.values()):
            self.init_state()

    # ------------------------------------------------------------------ step
    @torch.no_grad()
    def step(self, closure=None):
        """One step of every parameter that has a gradient; asynchronous on each device's current stream."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if not self._current():
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError('AdamW: take a step or call init_state() before capturing one in a graph')
            self.init_state()
        capturing = not self.capturable and torch.cuda.is_current_stream_capturing()
        ready = []
        for group, segments in zip(self.param_groups, self._segments):
            if capturing and any(p.grad is not None for p in group['params']):
                raise RuntimeError('AdamW: a step is captured in a graph, but the optimiser was made without capturable=True')
            self._check_options(group)
            b1, b2 = group['betas']
            for seg in segments:
                if seg.table.collect(float(group['lr']), b1, b2, float(group['eps']), float(group['weight_decay'])):
                    ready.append(seg.table)
        for table in ready:                               # every parameter has passed its checks: all are stepped or none
            table.launch()
        return loss
