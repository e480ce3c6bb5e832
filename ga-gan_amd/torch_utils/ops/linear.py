"""Fully connected layer as one operator, with its gradients:

    y = act(x @ (w * w_gain).T + b * b_gain) * gain + residual          x [..., K], w [N, K], b [N], residual [..., N]

`FullyConnectedLayer.forward` of the reference (DissimilarDomains/training/networks.py:691-700: a product with the scaled
weight, then `bias_act`) in one kernel that applies the whole epilogue to the accumulators (`sg_linear`); the backward pass
is the activation's gradient with the bias's column sums in one pass and a product each for x and w (`sg_linear_backward`).
float32, float16 and bfloat16 with float32 sums and one rounding per output; activations, their default slopes and gains are
those of `bias_act`.

What the backward pass keeps besides x and w: nothing for 'linear'; for 'relu' and 'lrelu' the output itself, whose sign
is the pre-activation's, or - where a residual hides it - a byte per element; for the others the pre-activation values in
float32 (rounded to 16 bits they would cost the gradient more accuracy than rounding the gradient itself does).  A
backward pass that is asked for a graph of its own differentiates the same expression written with the op-by-op operators.

At a pre-activation of exactly zero the slope is that of the negative side, as in `bias_act`."""
import ctypes

import torch

from ... import _lib
from .. import misc
from . import bias_act
from . import conv2d_gradfix

i32, i64, f32, vp = _lib.i32, _lib.i64, _lib.f32, _lib.vp


class LinearParams(ctypes.Structure):
    _fields_ = [('x', vp), ('w', vp), ('b', vp), ('residual', vp), ('dtype', i32), ('act', i32),
                ('alpha', f32), ('gain', f32), ('w_gain', f32), ('b_gain', f32),
                ('m', i64), ('n', i64), ('k', i64), ('ldx', i64), ('ldw', i64), ('ldr', i64)]


_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _rows(t):
    """(t or a dense copy, elements between its rows): unit stride within a row, rows that do not overlap."""
    rows, cols = t.shape
    if (cols <= 1 or t.stride(1) == 1) and (rows <= 1 or t.stride(0) >= max(cols, 1)):
        return t, (t.stride(0) if rows > 1 else max(cols, 1))
    return t.contiguous(), max(cols, 1)


def _workspace(nbytes, device):
    return torch.empty([nbytes], dtype=torch.uint8, device=device) if nbytes else None


def _params(x, ldx, w, ldw, b, residual, ldr, cfg):
    act, alpha, gain, w_gain, b_gain = cfg
    return LinearParams(_lib.ptr(x), _lib.ptr(w), _lib.ptr(b), _lib.ptr(residual), _lib.DTYPES[x.dtype], act, alpha, gain, w_gain, b_gain,
                        x.shape[0], w.shape[0], x.shape[1], ldx, ldw, ldr)


def _forward(x, w, b, residual, cfg, want_z=False, want_positive=False):
    x, ldx = _rows(x)
    w, ldw = _rows(w)
    b = b.contiguous() if b is not None else None
    ldr = 0
    if residual is not None:
        residual, ldr = _rows(residual)
    m, n = x.shape[0], w.shape[0]
    y = torch.empty([m, n], dtype=x.dtype, device=x.device)
    z = torch.empty([m, n], dtype=torch.float32, device=x.device) if want_z else None
    positive = torch.empty([m, n], dtype=torch.uint8, device=x.device) if want_positive else None
    if y.numel():
        p = _params(x, ldx, w, ldw, b, residual, ldr, cfg)
        handle = _lib.lib()
        need = handle.sg_linear_workspace_bytes(ctypes.byref(p))
        work = _workspace(need, x.device)
        _lib.launch_raw(lambda stream: handle.sg_linear(ctypes.byref(p), _lib.ptr(y), _lib.ptr(z), _lib.ptr(positive), _lib.ptr(work), need, stream),
                        x, 'sg_linear', 'linear_gemm_kernel', _lib.nbytes(x, w, residual, y), 2.0 * m * n * x.shape[1])
    return y, z, positive


def reference(x, w, b, residual, act, alpha, gain, w_gain, b_gain):
    """The same from the op-by-op operators (differentiable to any order)."""
    z = x.matmul((w * w_gain if w_gain != 1 else w).t())
    y = bias_act.bias_act(z, b * b_gain if b is not None and b_gain != 1 else b, act=act, alpha=alpha, gain=gain)
    return y if residual is None else y + residual


class _Linear(torch.autograd.Function):
    """x [M, K]; cfg = (act name, alpha, gain, w_gain, b_gain)."""

    @staticmethod
    def forward(ctx, x, w, b, residual, cfg):
        act, alpha, gain = cfg[:3]
        spec = bias_act.activation_funcs[act]
        slopes = act != 'linear' and any(ctx.needs_input_grad[:3])
        by_sign = act in ('relu', 'lrelu')
        from_y = by_sign and residual is None and gain != 0 and (act == 'relu' or alpha >= 0)
        y, z, positive = _forward(x, w, b, residual, (spec.cuda_idx, *cfg[1:]), want_z=slopes and not by_sign,
                                  want_positive=slopes and by_sign and not from_y)
        ctx.cfg, ctx.has_residual, ctx.has_bias = cfg, residual is not None, b is not None
        ctx.save_for_backward(x, w, b, y if slopes and from_y else None, z, positive)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, b, y, z, positive = ctx.saved_tensors
        act, alpha, gain, w_gain, b_gain = ctx.cfg
        need = list(ctx.needs_input_grad)
        if conv2d_gradfix.parameter_gradients_disabled:      # (a first-order pass that differentiates with respect to inputs only)
            need[1] = need[2] = False
        dres = dy if need[3] else None
        if not any(need[:3]):
            return None, None, None, dres, None
        if torch.is_grad_enabled():       # a higher-order graph is wanted: differentiate the operators' version
            ins = [t.view_as(t) if t is not None else None for t in (x, w, b)]
            with torch.enable_grad():
                out = reference(*ins, None, act, alpha, gain, w_gain, b_gain)
                wanted = [i for i in range(3) if need[i]]
                grads = torch.autograd.grad([out], [ins[i] for i in wanted], [dy], create_graph=True)
            result = [None, None, None, dres, None]
            for i, g in zip(wanted, grads):
                result[i] = g
            return tuple(result)
        dy = dy.contiguous()
        xr, ldx = _rows(x)
        wr, ldw = _rows(w)
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
        dw = torch.empty(w.shape, dtype=x.dtype, device=x.device) if need[1] else None
        db = torch.empty(b.shape, dtype=x.dtype, device=x.device) if need[2] else None
        p = _params(xr, ldx, wr, ldw, None, None, 0, (bias_act.activation_funcs[act].cuda_idx, alpha, gain, w_gain, b_gain))
        handle = _lib.lib()
        nbytes = handle.sg_linear_backward_workspace_bytes(ctypes.byref(p))
        work = _workspace(nbytes, x.device)
        products = (dx is not None) + (dw is not None)
        _lib.launch_raw(lambda stream: handle.sg_linear_backward(ctypes.byref(p), _lib.ptr(dy), _lib.ptr(y), _lib.ptr(z), _lib.ptr(positive),
                                                                 _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), _lib.ptr(work), nbytes, stream),
                        x, 'sg_linear_backward', 'linear_gemm_kernel', _lib.nbytes(dy, x, w, dx, dw), 2.0 * products * p.m * p.n * p.k)
        return dx, dw, db, dres, None


def linear(x, w, b=None, residual=None, act='linear', alpha=None, gain=None, w_gain=1.0, b_gain=1.0):
    """x [..., K], w [N, K], b [N] or None, residual [..., N] (the output's shape) or None -> [..., N]; one dtype (float32,
    float16 or bfloat16) and one device.  Rows of x, w and residual may lie any distance apart; tensors whose last dimension
    is not contiguous are copied first.  `alpha` and `gain` default to the activation's."""
    assert isinstance(x, torch.Tensor) and isinstance(w, torch.Tensor)
    misc.require_gpu(x, 'linear')
    if x.dtype not in _DTYPES:
        raise RuntimeError(f'linear: unsupported dtype {x.dtype}')
    if x.dim() < 1 or w.dim() != 2 or w.shape[1] != x.shape[-1]:
        raise RuntimeError(f'linear: x {tuple(x.shape)} and w {tuple(w.shape)} do not match')
    out_shape = (*x.shape[:-1], w.shape[0])
    if b is not None and tuple(b.shape) != (w.shape[0],):
        raise RuntimeError(f'linear: b {tuple(b.shape)} must have one entry per row of w {tuple(w.shape)}')
    if residual is not None and tuple(residual.shape) != out_shape:
        raise RuntimeError(f'linear: residual {tuple(residual.shape)} must have the shape of the output {out_shape}')
    for name, t in (('w', w), ('b', b), ('residual', residual)):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise RuntimeError(f'linear: {name} must have the dtype and device of x')
    spec = bias_act.activation_funcs[act]
    cfg = (act, float(alpha if alpha is not None else spec.def_alpha), float(gain if gain is not None else spec.def_gain), float(w_gain), float(b_gain))
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1]) if x.numel() else x.reshape(x.shape[:-1].numel(), x.shape[-1])
    r2 = residual if residual is None or residual.dim() == 2 else residual.reshape(x2.shape[0], w.shape[0])
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or (b is not None and b.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        y = _Linear.apply(x2, w, b, r2, cfg)
    else:
        y = _forward(x2, w, b, r2, (spec.cuda_idx, *cfg[1:]))[0]
    return y if x.dim() == 2 else y.reshape(out_shape)
