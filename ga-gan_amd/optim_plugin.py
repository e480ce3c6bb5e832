"""Binding of `sg_adam_step` / `sg_lerp_multi` (include/sg_ops.h): the optimizer step of a
training phase and the generator's moving average, each as one launch per 64 tensors; and of
`sg_grad_norm` / `sg_scale_grads` / `sg_adam_step_list`: the global norm of a list of gradients, clipping
by it, and the step with the clip applied as the gradients are read.

`FusedAdam` stands in for the `torch.optim.Adam(params, lr, betas, eps)` the reference's
loop constructs (training/training_loop.py:303-312) together with the gradient
sanitising it applies before every step (`param.grad.nan_to_num(0, 1e5, -1e5)`, :509).
"""
import ctypes

import torch

from . import _lib

MAX_TENSORS = 64


class AdamTensor(ctypes.Structure):
    _fields_ = [('param', ctypes.c_void_p), ('grad', ctypes.c_void_p), ('exp_avg', ctypes.c_void_p),
                ('exp_avg_sq', ctypes.c_void_p), ('numel', ctypes.c_int64), ('step', ctypes.c_int32)]


class AdamParams(ctypes.Structure):
    _fields_ = [('tensors', ctypes.POINTER(AdamTensor)), ('count', ctypes.c_int32), ('lr', ctypes.c_float),
                ('beta1', ctypes.c_float), ('beta2', ctypes.c_float), ('eps', ctypes.c_float), ('grad_limit', ctypes.c_float)]


class LerpTensor(ctypes.Structure):
    _fields_ = [('dst', ctypes.c_void_p), ('src', ctypes.c_void_p), ('numel', ctypes.c_int64)]


class LerpParams(ctypes.Structure):
    _fields_ = [('tensors', ctypes.POINTER(LerpTensor)), ('count', ctypes.c_int32), ('beta', ctypes.c_float)]


def _check(t, what):
    if not t.is_cuda:
        raise RuntimeError(f'{what} must reside on CUDA device')
    if t.dtype != torch.float32 or not t.is_contiguous():
        raise RuntimeError(f'{what} must be a dense float32 tensor')


CLIP_EPS = 1e-6        # added to the norm a gradient is divided by, as torch.nn.utils.clip_grad_norm_ does


def _max_norm(value, what):
    value = float(value)
    if not value >= 0:
        raise RuntimeError(f'{what}: the largest norm must not be negative')
    return value


def grad_norm(grads, grad_limit=None):
    """sqrt(sum of squares over all elements of all tensors of `grads`) as a float32 scalar on their device (nothing waits for it).
    float32, float16 and bfloat16 tensors in any mixture and number, dense, on one device; squares are summed in double, in an
    order that depends on the sizes alone.  `grad_limit`: the norm of the gradients as `adam_step` sanitises them
    (NaN -> 0, +-Inf -> +-grad_limit); None: as they are.  An empty list has norm zero (a host scalar)."""
    grads = list(grads)
    if not grads:
        return torch.zeros([])
    if grad_limit is not None and not float(grad_limit) > 0:
        raise RuntimeError('grad_norm: grad_limit must be positive')
    return _lib.ext().grad_norm(grads, float(grad_limit or 0), 0.0, CLIP_EPS)[0]


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm):
    """Scale the gradients of `parameters` (a tensor or an iterable; those without one are skipped) in place by
    min(1, max_norm / (norm + 1e-6)) and return their global norm before that: torch.nn.utils.clip_grad_norm_ for the 2-norm, in
    a launch per 128 tensors and one more, then another pass over the gradients only if they are too long.  A norm that is not
    finite makes the gradients NaN or zero, as there.  No gradient may overlap another; one that is not dense costs a copy there
    and back, and one that overlaps itself (an expanded tensor) is replaced by a dense one.  `FusedAdam(max_grad_norm=...)` clips
    without the second pass."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    max_norm = _max_norm(max_norm, 'clip_grad_norm_')
    params = [p for p in parameters if p.grad is not None]
    if not params:
        return torch.zeros([])
    grads = [p.grad for p in params]
    if len({id(g) for g in grads}) < len(grads):
        raise RuntimeError('clip_grad_norm_: a tensor appears twice')
    dense = [g.contiguous() for g in grads]
    norm = _lib.ext().clip_grads(dense, max_norm, CLIP_EPS)
    for p, g, d in zip(params, grads, dense):
        if d is not g and torch._debug_has_internal_overlap(g) == 1:
            p.grad = d
        elif d is not g:
            g.copy_(d)
    return norm


def adam_step(params, grads, exp_avgs, exp_avg_sqs, steps, lr, beta1, beta2, eps, grad_limit=1e5, max_grad_norm=None):
    """In-place update of `params` (and of the moment estimates; `grads` are sanitised in place).  `steps[i]` is
    the number of updates tensor i has received including this one.  With `max_grad_norm` the update uses the sanitised
    gradients times min(1, max_grad_norm / (their global norm + 1e-6)) and returns that norm (a device scalar); `grads` keep
    the sanitised, unscaled values."""
    if not (len(params) == len(grads) == len(exp_avgs) == len(exp_avg_sqs) == len(steps)):
        raise RuntimeError('adam_step: lists differ in length')
    if max_grad_norm is not None:
        max_grad_norm = _max_norm(max_grad_norm, 'adam_step')
        if not params:
            return torch.zeros([])
        group = (params, grads, exp_avgs, exp_avg_sqs, [int(k) for k in steps], lr, beta1, beta2, eps, grad_limit)
        return _lib.ext().adam_step_clipped([group], max_grad_norm, CLIP_EPS)
    for i in range(0, len(params), MAX_TENSORS):
        chunk = range(i, min(i + MAX_TENSORS, len(params)))
        table = (AdamTensor * len(chunk))()
        nbytes = 0
        for k, j in enumerate(chunk):
            p, g, m, v = params[j], grads[j], exp_avgs[j], exp_avg_sqs[j]
            for t, what in ((p, 'param'), (g, 'grad'), (m, 'exp_avg'), (v, 'exp_avg_sq')):
                _check(t, what)
                if t.shape != p.shape or t.device != p.device:
                    raise RuntimeError(f'adam_step: {what} {tuple(t.shape)} does not match its parameter {tuple(p.shape)}')
            table[k] = AdamTensor(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), p.numel(), int(steps[j]))
            nbytes += 7 * 4 * p.numel()   # four reads, three writes (the gradient is rewritten too: + 1)
        args = AdamParams(table, len(chunk), lr, beta1, beta2, eps, grad_limit)
        _lib.launch('sg_adam_step', args, params[i], 'adam_kernel', nbytes)
    # the kernel wrote through raw pointers: tell autograd (and every cache keyed on tensor versions)
    torch.autograd.graph.increment_version(list(params) + list(grads) + list(exp_avgs) + list(exp_avg_sqs))


def ema_(dsts, srcs, beta):
    """dst = src.lerp(dst, beta) for every pair, in place (dst the moving average, src the live weights)."""
    if len(dsts) != len(srcs):
        raise RuntimeError('ema_: lists differ in length')
    for i in range(0, len(dsts), MAX_TENSORS):
        chunk = range(i, min(i + MAX_TENSORS, len(dsts)))
        table = (LerpTensor * len(chunk))()
        nbytes = 0
        for k, j in enumerate(chunk):
            d, s = dsts[j], srcs[j]
            _check(d, 'dst')
            _check(s, 'src')
            if d.shape != s.shape or d.device != s.device:
                raise RuntimeError(f'ema_: {tuple(d.shape)} vs {tuple(s.shape)}')
            table[k] = LerpTensor(d.data_ptr(), s.data_ptr(), d.numel())
            nbytes += 3 * 4 * d.numel()
        args = LerpParams(table, len(chunk), beta)
        _lib.launch('sg_lerp_multi', args, dsts[i], 'lerp_kernel', nbytes)
    torch.autograd.graph.increment_version(list(dsts))


class FusedAdam(torch.optim.Optimizer):
    """Adam without weight decay / amsgrad whose `step()` sanitises the gradients and updates every parameter
    that has one in a single launch per 64 tensors.  State layout (`step`, `exp_avg`, `exp_avg_sq` per parameter)
    and `state_dict()` follow torch.optim.Adam, so checkpoints of one load into the other.  A step whose tensors or settings are
    refused, in whichever group, changes no parameter, moment or count.

    `max_grad_norm` clips by the global norm of all the sanitised gradients of a step, over every parameter group: the norm
    costs one more read of the gradients, the scaling nothing (it happens as the update reads them; `.grad` keeps the
    sanitised values).  It is a property of the optimizer, not of its groups or its state dict, and may be changed between
    steps; `last_grad_norm` is the norm of the last step that clipped (a device scalar).  All parameters must then live on
    one device."""

    max_grad_norm = None           # (class attributes: a pickle or copy made without them steps unclipped)
    last_grad_norm = None

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, grad_limit=1e5, max_grad_norm=None):
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, grad_limit=grad_limit))
        self.max_grad_norm = None if max_grad_norm is None else _max_norm(max_grad_norm, 'FusedAdam')

    def __getstate__(self):
        return dict(super().__getstate__(), max_grad_norm=self.max_grad_norm)

    def load_state_dict(self, state_dict):
        """As torch.optim.Optimizer.load_state_dict; the step counts are brought back to the host afterwards (a
        snapshot read with map_location=<device> carries them as device tensors, and `step()` reads each count on
        the host: one blocking device read per parameter and step otherwise)."""
        super().load_state_dict(state_dict)
        for state in self.state.values():
            if isinstance(state.get('step'), torch.Tensor) and state['step'].device.type != 'cpu':
                state['step'] = state['step'].detach().to('cpu', torch.float32)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self.max_grad_norm is not None:
            _max_norm(self.max_grad_norm, 'FusedAdam')
            if len({group['grad_limit'] for group in self.param_groups}) > 1:
                raise RuntimeError('FusedAdam: parameter groups that are clipped together must share grad_limit')
        # A step that is refused changes nothing: everything is checked first, and counts and new moments enter the state behind the launches.
        work, states = [], []
        for group in self.param_groups:
            params, grads, ms, vs, steps = [], [], [], [], []
            for p in group['params']:
                if p.grad is None:
                    continue
                state = self.state.get(p)
                if not state:
                    state = dict(step=torch.tensor(0.0),          # (a host tensor, as torch.optim.Adam keeps it)
                                 exp_avg=torch.zeros_like(p, memory_format=torch.contiguous_format),
                                 exp_avg_sq=torch.zeros_like(p, memory_format=torch.contiguous_format))
                if not p.grad.is_contiguous():
                    p.grad = p.grad.contiguous()
                params.append(p)
                grads.append(p.grad)
                ms.append(state['exp_avg'])
                vs.append(state['exp_avg_sq'])
                steps.append(int(state['step']) + 1)
                states.append((p, state))
            if params:
                work.append((params, grads, ms, vs, steps, group['lr'], *group['betas'], group['eps'], group['grad_limit']))
        if work and self.max_grad_norm is not None:
            self.last_grad_norm = _lib.ext().adam_step_clipped(work, self.max_grad_norm, CLIP_EPS)
        elif work:
            _lib.ext().adam_check(work)
            for args in work:
                adam_step(*args)
        for p, state in states:
            state['step'] += 1
            self.state[p] = state
        return loss
