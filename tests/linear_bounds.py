"""The fully connected layer in 64 bits, with elementwise error bounds for an evaluation in float32 sums and outputs of a given type.

u = 2^-24 (half a step of float32), h = eps / 2 of the output's type (half a step).  Written per element, with |.| elementwise:
  z   = w_gain x w^T + b_gain b            dz <= (K + 8) u (|w_gain| |x| |w|^T + |b_gain b|)   (any order of K products and sums, scale, bias)
  y   = gain act(z) + r                    dy <= |gain| L dz + 16 u (|gain act(z)| + |r|) + h |y|   L: largest slope
  s   = g act'(z)                          ds <= |g| (C dz + 16 u) + h |s|      C: largest curvature; at a corner of act closer than dz
                                                                          the slope may be the other side's: ds = |g| * jump there
  out = c s B (a product over P terms)     dout <= |c| (ds |B| + (P + 8) u |s| |B|) + h |out|
A float16 value below its normal range is off by up to 2^-25 more."""
import math

import torch

U = 2.0 ** -24
SELU_SCALE, SELU_ALPHA = 1.0507009873554804934193349852946, 1.6732632423543772848170429916717
LIPSCHITZ = dict(selu=SELU_SCALE * SELU_ALPHA, swish=1.1)        # largest |act'|, 1 elsewhere
CURVATURE = dict(selu=SELU_SCALE * SELU_ALPHA)                   # largest |act''| away from corners, 1 elsewhere
JUMP = dict(relu=1.0, lrelu=0.8, selu=SELU_SCALE * (SELU_ALPHA - 1))
GAINS = dict(relu=math.sqrt(2), lrelu=math.sqrt(2), swish=math.sqrt(2))


def act64(act, z, alpha=0.2):
    f = torch.nn.functional
    return dict(linear=lambda t: t, relu=f.relu, lrelu=lambda t: f.leaky_relu(t, alpha), tanh=torch.tanh, sigmoid=torch.sigmoid, elu=f.elu, selu=f.selu,
                softplus=lambda t: torch.logaddexp(t, torch.zeros_like(t)), swish=f.silu)[act](z)


def definition(x, w, b, r, act, gain=None, w_gain=1.0, b_gain=1.0, alpha=0.2):
    """y of float64 arguments."""
    z = x @ w.t() * w_gain
    if b is not None:
        z = z + b * b_gain
    y = act64(act, z, alpha) * (GAINS.get(act, 1.0) if gain is None else gain)
    return y if r is None else y + r


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _floor(dtype):
    return 2.0 ** -24 if dtype == torch.float16 else 1e-37


def bounds(x, w, b, r, act, dy=None, gain=None, w_gain=1.0, b_gain=1.0, alpha=0.2):
    """{name: (value, bound)} for y and, with dy, for the gradients dx, dw, db."""
    dtype = x.dtype
    h, low = _half(dtype), _floor(dtype)
    gain = GAINS.get(act, 1.0) if gain is None else gain
    leaves = [t.detach().double().requires_grad_(dy is not None) if t is not None else None for t in (x, w, b, r)]
    X, W, B, R = leaves
    M, K, N = X.shape[0], X.shape[1], W.shape[0]
    with torch.enable_grad():
        y = definition(X, W, B, R, act, gain, w_gain, b_gain, alpha)
    with torch.no_grad():
        z = X @ W.t() * w_gain + (B * b_gain if B is not None else 0)
        dz = (K + 8) * U * (X.abs() @ W.abs().t() * abs(w_gain) + (abs(b_gain) * B.abs() if B is not None else 0))
        a = act64(act, z, alpha) * gain
        out = dict(y=(y.detach(), abs(gain) * LIPSCHITZ.get(act, 1.0) * dz + 16 * U * (a.abs() + (R.abs() if R is not None else 0)) + h * y.detach().abs() + low))
    if dy is None:
        return out
    G = dy.double()
    grads = torch.autograd.grad(y, [t for t in (X, W, B) if t is not None], G)
    with torch.enable_grad():
        zz = z.clone().requires_grad_(True)
        slope, = torch.autograd.grad(act64(act, zz, alpha).sum(), zz)
    with torch.no_grad():
        s = G * slope
        curvature = CURVATURE.get(act, 0.0 if act in ('linear', 'relu', 'lrelu') else 1.0)
        ds = G.abs() * (curvature * dz + 16 * U) + h * s.abs() + low
        if act in JUMP:
            jump = abs(1 - alpha) if act == 'lrelu' else JUMP[act]
            ds = ds + G.abs() * jump * (z.abs() <= dz + low)
        c = abs(gain * w_gain)
        out['dx'] = grads[0], c * (ds @ W.abs() + (N + 8) * U * (s.abs() @ W.abs())) + h * grads[0].abs() + low
        out['dw'] = grads[1], c * (ds.t() @ X.abs() + (M + 8) * U * (s.abs().t() @ X.abs())) + h * grads[1].abs() + low
        if B is not None:
            c = abs(gain * b_gain)
            out['db'] = grads[2], c * (ds.sum(dim=0) + (M + 8) * U * s.abs().sum(dim=0)) + h * grads[2].abs() + low
    return {key: (v.detach(), e.detach()) for key, (v, e) in out.items()}


def check(got, want, what):
    value, bound = want
    off = (got.detach().double() - value).abs()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    worst = float((off / bound.clamp(min=1e-300)).max()) if off.numel() else 0.0
    assert bool((off <= bound).all()), f'{what}: {worst:.3g} times the bound'
