"""Gradient clipping and the AdamW step on the HIP kernels of csrc/optimizer.hip: what a training loop does between a
backward pass and the next forward pass.

`clip_grad_norm_` takes parameters and clips their gradients; `AdamW` is a `torch.optim.Optimizer` (learning-rate
schedulers, parameter groups, `state_dict` as torch's own AdamW, model.py:177-181) whose step takes the gradients' norm,
clips them while it reads them, and can be captured into a HIP graph.  It is two launches for up to 56 parameters of one
type in one group: the update is a launch per group, element type and 56 parameters, the norm ahead of it one
per element type and 120 parameters (without a norm: one launch per 256 parameters, which copies the step counters).
The tensor-level entry points are `nerf_amd.ops.grad_norm` and `nerf_amd.ops.clip_grad_norm_`.
"""
import ctypes

import torch

from . import ops
from ._lib import AdamwGroup, AdamwTensors, check, lib, lists


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Clip the gradients of `parameters` (an iterable, or one tensor) by their norm taken together, in place -> the norm
    before, a 0-d fp32 tensor.  Parameters without a gradient are passed over.  With `error_if_nonfinite` the norm is
    read back (one stream synchronisation) and a norm that is not finite raises with the gradients as they were."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if error_if_nonfinite:
        norm = ops.grad_norm(grads, norm_type)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f'clip_grad_norm_: the gradients\' norm of order {norm_type} is not finite')
    return ops.clip_grad_norm_(grads, max_norm, norm_type)


def own_max_norm(optimizer):
    """The norm that an optimizer clips at by itself (`AdamW` below with a max_norm), or None."""
    return optimizer.max_norm if isinstance(optimizer, AdamW) else None


# What torch.optim.AdamW keeps in its groups and has no say here.
_OTHER_SETTINGS = ('amsgrad', 'maximize', 'foreach', 'differentiable', 'fused', 'decoupled_weight_decay')


def _refuse_settings(settings):
    for k in ('amsgrad', 'maximize', 'differentiable'):
        if settings.get(k):
            raise ValueError(f'AdamW: {k} is not supported')


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay; arguments as torch.optim.AdamW's (`foreach`, `fused` and `capturable` choose among
    its ways to the same result and change nothing here; `amsgrad`, `maximize` and `differentiable` are refused where they
    are true), and, as the sixth to eighth,

    max_norm         the gradients are scaled by min(1, max_norm / (norm + 1e-6)) as they are read (`.grad` itself is not
                     written); the norm is taken over all parameter groups together.  None: no clipping.
    norm_type        2, 1 or inf.
    skip_nonfinite   a step whose gradient norm is infinite (in fp32) or NaN leaves parameters, moments and step counters as
                     they are.

    `grad_norm` holds the norm of the last step, replays of captured ones included (a 0-d fp32 tensor on the device; None
    before the first step, and without max_norm or skip_nonfinite).  Each step has a tensor of its own until one is captured:
    from then on it is one tensor, which every later step and every replay write (the first of them: a capture itself runs
    nothing), so that what is to be kept is cloned.

    Parameters are fp32, bf16 or fp16, on one HIP device, their gradients of the same type.  The moments are fp32 whatever
    the parameters are, and a 16-bit parameter has an fp32 master weight in the state ('master'), of which it is the
    rounding; a parameter that something else writes is taken as it is, and its master follows.  The step counters live on
    the device, so a captured step counts on with every replay; the learning rate of a group may be an fp32 device tensor,
    which a replay reads afresh.  Gradients are taken as they are: where the loss was scaled (fp16), they are divided by the
    scale ahead of the step.  The state is laid out by the first step, which therefore cannot be a captured one."""

    _graph_norm = None      # what grad_norm is from the first captured step on

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_norm=None, norm_type=2.0,
                 skip_nonfinite=False, *, amsgrad=False, maximize=False, foreach=None, capturable=True, differentiable=False,
                 fused=None):
        _refuse_settings(dict(amsgrad=amsgrad, maximize=maximize, differentiable=differentiable))
        if isinstance(max_norm, bool):          # (torch.optim.AdamW's sixth argument is amsgrad)
            raise ValueError(f'max_norm must be a number or None, got {max_norm}')
        if not torch.is_tensor(lr) and not lr >= 0.0:
            raise ValueError(f'invalid learning rate: {lr}')
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f'invalid betas: {betas}')
        if not eps >= 0.0:
            raise ValueError(f'invalid eps: {eps}')
        if not weight_decay >= 0.0:
            raise ValueError(f'invalid weight_decay: {weight_decay}')
        self.max_norm = None if max_norm is None else ops.check_max_norm(max_norm)
        self._kind = ops.norm_kind(norm_type)
        self.norm_type, self.skip_nonfinite = float(norm_type), bool(skip_nonfinite)
        self.grad_norm = None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, capturable=True))

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):       # (the base class says what else it takes)
            _refuse_settings(param_group)
        super().add_param_group(param_group)

    def __getstate__(self):         # (copies and pickles: the base class names what it keeps)
        return dict(super().__getstate__(), max_norm=self.max_norm, norm_type=self.norm_type,
                    skip_nonfinite=self.skip_nonfinite, _kind=self._kind, grad_norm=None, _graph_norm=None)

    def __setstate__(self, state):
        super().__setstate__(state)
        for g in self.param_groups:
            g['capturable'] = True

    def load_state_dict(self, state_dict):
        """A state dict of this class or of torch.optim.AdamW (without amsgrad / maximize), with the registered hooks as they
        are everywhere: the pre-hooks decide what is loaded, the post-hooks see it laid out."""
        loaded = {}

        def check_loaded(_, sd):                # behind the other pre-hooks, each of which may put another dict in its place
            for g in sd['param_groups']:
                _refuse_settings(dict(g, differentiable=False))
            loaded.update(sd)
        hooks = (self.register_load_state_dict_pre_hook(check_loaded),
                 self.register_load_state_dict_post_hook(lambda _: self._lay_out(loaded), prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for h in hooks:
                h.remove()

    def _lay_out(self, state_dict):
        """What the base class has loaded, as the kernels take it.  It gives floating-point state the parameter's type and may
        leave step counters on the host: the moments and masters are fp32 here, and the counters live beside them."""
        ids = [i for g in state_dict['param_groups'] for i in g['params']]
        for i, p in zip(ids, [p for g in self.param_groups for p in g['params']]):
            saved = state_dict['state'].get(i)
            if not saved:
                continue
            st = self.state[p]                  # (entries of other names stay as the base class loads them)
            for k in ('exp_avg', 'exp_avg_sq', 'master'):
                if k in saved:
                    st[k] = torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format).copy_(saved[k])
            if 'step' in saved:
                st['step'] = torch.as_tensor(saved['step'], dtype=torch.float32).to(p.device, copy=True).reshape(())
        for g in self.param_groups:             # (a scheduler's or a user's own options of a group stay)
            for k in _OTHER_SETTINGS:
                g.pop(k, None)
            g['capturable'] = True

    def _init_state(self, params):
        """Lay out the state of parameters that have none, or no master (the state of an optimizer that keeps none)."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError('AdamW: run one step ahead of a graph capture (it lays out the optimizer state; captured, '
                               'every replay would clear it)')
        steps = torch.zeros(len(params), dtype=torch.float32, device=params[0].device)
        for i, p in enumerate(params):
            st = self.state[p]
            like = dict(dtype=torch.float32, memory_format=torch.preserve_format)
            if not st:
                st['step'] = steps[i]
                st['exp_avg'] = torch.zeros_like(p, **like)
                st['exp_avg_sq'] = torch.zeros_like(p, **like)
            if p.dtype != torch.float32:
                st['master'] = p.detach().to(**like)

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lists_of = [g['params'] for g in self.param_groups]
        found = lists().optimizer(lists_of, self.state)     # (holds copies of reordered gradients: kept to the end)
        if type(found) is list:
            ops.list_call(found[0].get_device(), lambda _: self._init_state(found))
            found = lists().optimizer(lists_of, self.state)
        device, params, _, counts, *arrays = found
        if params:
            ops.list_call(device, lambda st: self._launch(device, len(params), memoryview(counts).cast('i'), arrays, st))
            torch.autograd.graph.increment_version(params)      # (the kernels write behind autograd's back)
        elif self.max_norm is not None or self.skip_nonfinite:
            self.grad_norm = (torch.zeros((), device=next((p.device for ps in lists_of for p in ps), None))
                              if self._graph_norm is None else self._graph_norm.zero_())
        return loss

    def _launch(self, device, n, counts, arrays, st):
        L = lib()
        groups = (AdamwGroup * len(counts))()
        for c, count, g in zip(groups, counts, self.param_groups):
            lr = g['lr']
            c.count = count
            if torch.is_tensor(lr):
                if lr.numel() != 1:
                    raise ValueError('AdamW: a tensor learning rate must have one element')
                if lr.is_cuda:
                    if lr.dtype != torch.float32 or lr.get_device() != device:
                        raise ValueError('AdamW: a tensor learning rate must be fp32 on the parameters\' device')
                    c.lr_device = lr.data_ptr()
                else:
                    c.lr = float(lr)
            else:
                c.lr = float(lr)
            c.beta1, c.beta2 = g['betas']
            c.eps, c.weight_decay = g['eps'], g['weight_decay']
        clips = self.max_norm is not None or self.skip_nonfinite
        nbytes = L.nerf_grad_workspace_bytes(n)
        ws = torch.empty(nbytes, dtype=torch.uint8, device='cuda')
        norm = None
        if clips:       # (a replay runs no Python: what it writes has to be what grad_norm names, whatever ran before it)
            norm = self._graph_norm
            if norm is None or norm.get_device() != device:
                norm = torch.empty((), dtype=torch.float32, device='cuda')
                if torch.cuda.is_current_stream_capturing():
                    self._graph_norm = norm
        check(L.nerf_adamw_step(ctypes.byref(AdamwTensors(n, *arrays)), groups, len(counts), self._kind if clips else 0,
                                float('inf') if self.max_norm is None else self.max_norm, int(self.skip_nonfinite),
                                ws.data_ptr(), nbytes, norm.data_ptr() if clips else None, st))
        if clips:
            self.grad_norm = norm
