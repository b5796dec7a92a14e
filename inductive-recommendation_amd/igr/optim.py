"""igr.optim - fused Adam on the HIP kernel (igr_adam_f32), and Muon for dense layers on top of it.

Adam: drop-in for the `Adam` the reference resolves by name (trainer.py:44-46):
same constructor (params, lr, betas, eps, weight_decay) and torch.optim.Adam
update rule, one pass over (param, grad, exp_avg, exp_avg_sq) per tensor
instead of torch's multi-kernel foreach sequence.

Muon: the weights of the dense layers (NGCF's gc / bi layers, AttIGCN's projections) take orthogonalised
momentum steps (ops.newton_schulz); embedding tables, biases and every other parameter take
Adam steps.  By name in a trainer config: 'optimizer': 'Muon' (for_model splits the parameters).
"""
import ctypes

import torch

from . import _lib as L
from . import ops

# tensors up to this many elements share one launch (igr_adam_multi_f32); larger ones take
# igr_adam_f32, whose non-temporal traffic pays on tables that do not fit the caches
SMALL_NUMEL = 1 << 18


class Adam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0):
        if lr < 0 or eps < 0 or not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError('invalid Adam hyper-parameters')
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.device_step = None  # (counter, base): step = state step + 1 + *counter, read on the device

    def set_device_step(self, counter):
        """hipGraph mode: the kernel adds *counter (device int64, the replays so far)
        to each tensor's step at the time of this call; the host counts stay put
        until advance_host_steps().  None returns to host-counted steps."""
        self.device_step = counter

    def advance_host_steps(self, n):
        for group in self.param_groups:
            for p in group['params']:
                st = self.state.get(p)
                if st:
                    st['step'] += n

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            self._step_group(group)
        return loss

    def _step_group(self, group):
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        ctr = self.device_step
        ctr_p = ctypes.c_void_p(0 if ctr is None else ctr.data_ptr())
        b1, b2 = group['betas']
        hyper = (float(group['lr']), float(b1), float(b2), float(group['eps']), float(group['weight_decay']))
        small = []  # (param, grad, state): tensors that share one launch (igr_adam_multi_f32)
        for p in group['params']:
            if p.grad is None:
                continue
            if p.grad.is_sparse:
                raise RuntimeError('igr Adam does not support sparse gradients')
            if not p.is_cuda:
                raise L.IgrError('igr Adam needs parameters on a ROCm device (no CPU fallback)')
            st = self.state[p]
            if not st:
                st['step'] = 0
                st['exp_avg'] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                st['exp_avg_sq'] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            if ctr is None:
                st['step'] += 1
            g = p.grad if p.grad.is_contiguous() else p.grad.contiguous()
            assert p.is_contiguous() and p.dtype == torch.float32
            step = st['step'] if ctr is None else st['step'] + 1
            if p.numel() <= SMALL_NUMEL and all(t.data_ptr() % 16 == 0 for t in (p, g, st['exp_avg'],
                                                                                  st['exp_avg_sq'])):
                small.append((p, g, st, step))
                continue
            L.call('igr_adam_f32', p.numel(), ctypes.c_void_p(p.data_ptr()), ctypes.c_void_p(g.data_ptr()),
                   ctypes.c_void_p(st['exp_avg'].data_ptr()), ctypes.c_void_p(st['exp_avg_sq'].data_ptr()),
                   *hyper, step, ctr_p, stream)
        for i in range(0, len(small), L.ADAM_MAX_SLOTS):
            chunk = small[i:i + L.ADAM_MAX_SLOTS]
            slots = (L.IgrAdamSlot * len(chunk))()
            for s, (p, g, st, step) in zip(slots, chunk):
                s.param, s.grad = p.data_ptr(), g.data_ptr()
                s.exp_avg, s.exp_avg_sq = st['exp_avg'].data_ptr(), st['exp_avg_sq'].data_ptr()
                s.n, s.step = p.numel(), step
            L.call('igr_adam_multi_f32', len(chunk), ctypes.cast(slots, ctypes.c_void_p), *hyper, ctr_p, stream)


class Muon(Adam):
    """Orthogonalised momentum for matrices, Adam for the rest.

    Parameter groups flagged 'orthogonal' (2-D float32 weights) step by
        m <- momentum * m + grad,   u = grad + momentum * m (nesterov) or m
        p <- (1 - lr * weight_decay) * p - lr * sqrt(max(1, rows / cols)) * newton_schulz(u)
    with the group's own lr; the other groups are Adam's.  Weights of one shape are orthogonalised in
    one batch.  Given plain parameters, every 2-D one is taken as orthogonal: pass embedding
    tables in a group with 'orthogonal': False, or use for_model, which takes the weights of
    nn.Linear layers only.  Steps can be captured in a hipGraph like Adam's."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, orthogonal_lr=0.02, momentum=0.95,
                 nesterov=True, ns_steps=5, ns_coeffs=ops.NEWTON_SCHULZ_COEFFS):
        if orthogonal_lr < 0 or not 0 <= momentum < 1 or ns_steps < 1 or len(ns_coeffs) != 3:
            raise ValueError('invalid Muon hyper-parameters')
        params = list(params)
        if params and not isinstance(params[0], dict):
            params = [{'params': [p for p in params if p.dim() == 2], 'orthogonal': True},
                      {'params': [p for p in params if p.dim() != 2], 'orthogonal': False}]
        self._orthogonal = dict(lr=orthogonal_lr, momentum=momentum, nesterov=nesterov, ns_steps=ns_steps,
                                ns_coeffs=tuple(ns_coeffs))
        groups = [dict(g, params=[g['params']] if isinstance(g['params'], torch.Tensor) else list(g['params'])) for g in params]
        super().__init__([g for g in groups if g['params']], lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)

    def add_param_group(self, param_group):
        """Also what the constructor adds each of its groups with: 'orthogonal' (False if not given) decides the rule, and
        with it which of the optimizer's settings the group takes where it names none."""
        g = dict(param_group)
        g['params'] = [g['params']] if isinstance(g['params'], torch.Tensor) else list(g['params'])
        g.setdefault('orthogonal', False)
        if g['orthogonal']:
            for p in g['params']:
                if p.dim() != 2 or p.dtype != torch.float32:
                    raise ValueError(f'Muon orthogonalises 2-D float32 weights, got {tuple(p.shape)} {p.dtype}')
            for k, v in self._orthogonal.items():
                g.setdefault(k, v)
        super().add_param_group(g)

    def load_state_dict(self, state_dict):
        """Groups have to follow the rule that they were saved under (an Adam's, which names none, is Adam's).  Settings
        that the saved groups lack stay this optimizer's."""
        saved = []
        for mine, group in zip(self.param_groups, state_dict['param_groups']):
            if bool(group.get('orthogonal', False)) != bool(mine['orthogonal']):
                raise ValueError('loaded state dict has a group under another rule (orthogonal: '
                                 f"{bool(group.get('orthogonal', False))}, here {bool(mine['orthogonal'])})")
            saved.append({**{k: v for k, v in mine.items() if k != 'params'}, **group})
        saved += state_dict['param_groups'][len(saved):]
        super().load_state_dict({**state_dict, 'param_groups': saved})

    @classmethod
    def for_model(cls, model, **kw):
        """Muon over a model's parameters: the weights of its nn.Linear layers orthogonalised, the rest Adam's."""
        dense = [m.weight for m in model.modules() if isinstance(m, torch.nn.Linear)]
        ids = {id(p) for p in dense}
        rest = [p for p in model.parameters() if id(p) not in ids]
        return cls([{'params': dense, 'orthogonal': True}, {'params': rest, 'orthogonal': False}], **kw)

    def advance_host_steps(self, n):
        for group in self.param_groups:
            for p in group['params']:
                st = self.state.get(p)
                if st and 'step' in st:  # orthogonalised weights count no steps
                    st['step'] += n

    def _step_group(self, group):
        if not group['orthogonal']:
            return super()._step_group(group)
        shapes = {}
        for p in group['params']:
            if p.grad is None:
                continue
            if p.grad.is_sparse:
                raise RuntimeError('igr Muon does not support sparse gradients')
            if not p.is_cuda:
                raise L.IgrError('igr Muon needs parameters on a ROCm device (no CPU fallback)')
            if p.numel() == 0:
                continue
            shapes.setdefault((p.device, tuple(p.shape)), []).append(p)
        for (device, (rows, cols)), ps in shapes.items():
            with torch.cuda.device(device):
                self._step_shape(group, device, rows, cols, ps)

    def _step_shape(self, group, device, rows, cols, ps):
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        direction = torch.empty(len(ps), rows, cols, dtype=torch.float32, device=device)
        grads = []
        slots = (L.IgrMuonSlot * len(ps))()
        for s, p, d in zip(slots, ps, direction):
            st = self.state[p]
            if not st:
                st['momentum'] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            assert p.is_contiguous() and p.dtype == torch.float32 and p.grad.dtype == torch.float32
            grads.append(p.grad if p.grad.is_contiguous() else p.grad.contiguous())
            s.param, s.grad, s.momentum = p.data_ptr(), grads[-1].data_ptr(), st['momentum'].data_ptr()
            s.direction, s.n = d.data_ptr(), p.numel()
        chunks = [(i, min(L.MUON_MAX_SLOTS, len(ps) - i)) for i in range(0, len(ps), L.MUON_MAX_SLOTS)]
        size = ctypes.sizeof(L.IgrMuonSlot)
        at = lambda i: ctypes.c_void_p(ctypes.addressof(slots) + i * size)  # noqa: E731
        for i, n in chunks:
            L.call('igr_muon_direction_f32', n, at(i), float(group['momentum']), int(bool(group['nesterov'])), stream)
        ortho = ops.newton_schulz(direction, steps=group['ns_steps'], coeffs=group['ns_coeffs'])
        for s, o in zip(slots, ortho):
            s.direction = o.data_ptr()
        scale = max(1.0, rows / cols) ** 0.5
        for i, n in chunks:
            L.call('igr_muon_apply_f32', n, at(i), float(group['lr']), float(group['weight_decay']), scale, stream)
