"""AdamW on the HIP kernels (ops.adamw_step): all parameters of a group in one call, moments in float32 or in 8 bits.

The reference trains with torch's Adam, by name (trainer.py:43-45); config key 'optimizer': 'AdamW' takes this one instead."""
import torch

from . import _lib, ops


class AdamW(torch.optim.Optimizer):
    """Adam with decoupled weight decay.  state_bits 32: moments in float32 (state names and meaning of torch.optim.AdamW, whose
    state_dict it takes).  state_bits 8: exp_avg as float8_e4m3fn and exp_avg_sq as float8_e5m2 codes with two float32 scales a block
    of 128 elements ('scales') — 2.06 bytes a parameter instead of 8; a moment is codes.float() * its block's scale.
    max_grad_norm: clip by the norm over the gradients of ALL groups; the last step's norm is `grad_norm` (a tensor on the GPU, the same
    one at every step, captured or not: copy it to keep it).
    norm_reduce_fn: for parameters that are a rank's share of a model (dist.ShardedLightGCN, ColumnShardedLightGCN: their all_reduce;
    dist.column_shard_model: slice_reduce_fn, which the trainers pass): sums a tensor over the ranks, in place, so that every rank clips by
    the norm over all shares (parameters that dist marks as shares are refused without).  Called once a step on one float64 number, also
    where this rank has no gradient.
    seed: of the 8-bit moments' stochastic rounding.  The step count lives on the device and lr may be a one-element float32 tensor
    there: the step can sit in a HIP graph."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, max_grad_norm=None, seed=0,
                 norm_reduce_fn=None):
        if not isinstance(lr, torch.Tensor) and not lr >= 0.:
            raise ValueError('lr must not be negative')
        if not (0. <= betas[0] < 1. and 0. <= betas[1] < 1.) or not eps >= 0. or not weight_decay >= 0.:
            raise ValueError('betas must be in [0, 1), eps and weight_decay not negative')
        if state_bits not in (8, 32):
            raise ValueError('state_bits must be 8 or 32')
        if max_grad_norm is not None and not max_grad_norm > 0.:
            raise ValueError('max_grad_norm must be positive')
        self.max_grad_norm, self.seed, self.grad_norm, self.norm_reduce_fn = max_grad_norm, int(seed), None, norm_reduce_fn
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        if self.max_grad_norm is not None and self.norm_reduce_fn is None and \
                any(getattr(p, 'is_share', False) for p in self.param_groups[-1]['params']):
            self.param_groups.pop()
            raise ValueError('parameters that are a rank\'s share of a model are clipped by the norm over all ranks: norm_reduce_fn is missing')

    def _state_of(self, p, bits):
        state = self.state[p]
        if not state:
            state['step'] = torch.zeros((), dtype=torch.float32, device=p.device)
            for name, dtype in zip(('exp_avg', 'exp_avg_sq'), ops.MOMENT_DTYPES):
                state[name] = torch.zeros_like(p, dtype=torch.float32) if bits == 32 else torch.zeros_like(p, dtype=torch.uint8).view(dtype)
            if bits == 8:
                state['scales'] = torch.zeros(((p.numel() + ops.ADAMW_BLOCK - 1) // ops.ADAMW_BLOCK, 2), dtype=torch.float32, device=p.device)
        return state

    def _common_norm(self, grads):
        """self.grad_norm = the norm over the gradients of all groups, and of all ranks where they hold shares."""
        norm = ops.grad_norm(grads, out=self.grad_norm) if grads else self.grad_norm.zero_()
        if self.norm_reduce_fn is not None:
            square = norm.double().square()
            self.norm_reduce_fn(square)
            norm.copy_(square.sqrt())
        return norm

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls = []
        for gi, group in enumerate(self.param_groups):
            ps = [p for p in group['params'] if p.grad is not None]
            for p in ps:
                if not p.is_cuda or p.grad.is_sparse:
                    raise _lib.IgcnError('AdamW takes parameters on the GPU with dense gradients')
            gs = [p.grad if ops._same_order(p, p.grad) else torch.empty_like(p, dtype=p.grad.dtype).copy_(p.grad) for p in ps]
            if ps:
                calls.append((gi, group, ps, gs))
        norm = norm_out = None
        if self.max_grad_norm is not None:
            device = (calls[0][2] if calls else self.param_groups[0]['params'])[0].device
            if self.grad_norm is None or self.grad_norm.device != device:
                self.grad_norm = torch.zeros((), dtype=torch.float32, device=device)
            norm_out = self.grad_norm
            if len(calls) != 1 or self.norm_reduce_fn is not None:
                norm = self._common_norm([g for call in calls for g in call[3]])
        for gi, group, ps, gs in calls:
            states = [self._state_of(p, group['state_bits']) for p in ps]
            ops.adamw_step(ps, gs, [s['exp_avg'] for s in states], [s['exp_avg_sq'] for s in states], [s['step'] for s in states],
                           lr=group['lr'], betas=group['betas'], eps=group['eps'], weight_decay=group['weight_decay'],
                           max_grad_norm=self.max_grad_norm, scales=[s['scales'] for s in states] if group['state_bits'] == 8 else None,
                           seed=self.seed + (gi << 32), grad_norm=norm, norm_out=norm_out)
        return loss

    def __getstate__(self):                # (copies and pickles keep what torch's form of it does not know)
        return {**super().__getstate__(), 'max_grad_norm': self.max_grad_norm, 'seed': self.seed, 'grad_norm': self.grad_norm,
                'norm_reduce_fn': self.norm_reduce_fn}

    @staticmethod
    def _loaded(p, saved):
        """The state of p that a saved one stands for: float32 moments laid out like p, or codes and scales as they are."""
        if set(saved) & {'step', 'exp_avg', 'exp_avg_sq'} != {'step', 'exp_avg', 'exp_avg_sq'}:
            raise ValueError('a saved state holds step, exp_avg and exp_avg_sq')
        step = torch.as_tensor(saved['step'], dtype=torch.float32)
        moments = {name: saved[name] for name in ('exp_avg', 'exp_avg_sq')}
        if step.numel() != 1 or any(value.shape != p.shape for value in moments.values()):
            raise ValueError('a saved state has one step and moments of the parameter\'s shape (got %s and %s for %s)'
                             % (tuple(step.shape), [tuple(m.shape) for m in moments.values()], tuple(p.shape)))
        state = {'step': step.reshape(()).to(device=p.device, copy=True)}
        if 'scales' not in saved:
            if any(m.dtype not in (torch.float64, *ops._DTYPE_CODES) for m in moments.values()):
                raise ValueError('8-bit moments come with their scales')
            return {**state, **{name: torch.empty_like(p, dtype=torch.float32).copy_(m) for name, m in moments.items()}}
        if tuple(m.dtype for m in moments.values()) != ops.MOMENT_DTYPES or \
                saved['scales'].dtype != torch.float32 or saved['scales'].shape != ((p.numel() + ops.ADAMW_BLOCK - 1) // ops.ADAMW_BLOCK, 2):
            raise ValueError('8-bit moments are float8_e4m3fn and float8_e5m2 with float32 scales [ceil(numel / %d), 2]' % ops.ADAMW_BLOCK)
        if not all(ops._same_order(p, m) for m in moments.values()):
            raise ValueError('8-bit moments share scales in memory order: they must lie in memory as their parameter does')
        return {**state, **{name: m.to(device=p.device, copy=True) for name, m in moments.items()},
                'scales': saved['scales'].to(device=p.device, copy=True, memory_format=torch.contiguous_format)}

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """As torch's, but the moments keep the form they are saved in, 8-bit or not (torch's casts every floating state to its
        parameter's type), and what does not fit is refused before anything changes.  Takes the state of torch.optim.AdamW too, whose
        moments may be in the parameter's type; a group's state_bits then follow from what the state holds."""
        if any(g.get('amsgrad') or g.get('maximize') for g in state_dict['param_groups']):
            raise ValueError('a state with amsgrad or maximize is another optimizer\'s')
        saved = [i for g in state_dict['param_groups'] for i in g['params']]
        mine = [p for g in self.param_groups for p in g['params']]
        states = {i: self._loaded(p, state_dict['state'][i]) for i, p in zip(saved, mine) if state_dict['state'].get(i)}
        held = [{8 if 'scales' in states[i] else 32 for i in g['params'] if i in states} for g in state_dict['param_groups']]
        if any(len(bits) > 1 for bits in held):
            raise ValueError('a group holds its moments in one form')
        super().load_state_dict(state_dict)
        for bits, group in zip(held, self.param_groups):
            for name, value in self.defaults.items():
                group.setdefault(name, value)
            group['state_bits'] = bits.pop() if bits else group['state_bits']
        for i, p in zip(saved, mine):
            if i in states:
                self.state[p].update(states[i])
