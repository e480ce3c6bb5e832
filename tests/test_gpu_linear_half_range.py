"""Gradients of float16 layers whose dy lies near either end of float16's range: s = dy act'(z) is held as float16 for the products,
times a power of two that brings the largest |dy| times the activation's largest slope to 2^14 .. 2^15, so that a slope above one
does not overflow and one far below one does not vanish.

Bounds as in tests/linear_bounds.py, but for s: scaled so, an element that falls below float16's normal range is off by at most
2^-25 / 2^14 of (largest slope * largest |dy|); allowed 2^-39 of it.  An output below the normal range: 2^-25."""
import math

import pytest
import torch

from linear_bounds import CURVATURE, JUMP, LIPSCHITZ, U, act64, check, definition

pytestmark = pytest.mark.gpu
DEV = 'cuda'
H = 2.0 ** -11


def bounds(x, w, b, act, dy, gain, w_gain, b_gain, alpha=0.2):
    X, W, B = (t.detach().double().requires_grad_(True) for t in (x, w, b))
    G = dy.double()
    with torch.enable_grad():
        grads = torch.autograd.grad(definition(X, W, B, None, act, gain, w_gain, b_gain, alpha), (X, W, B), G)
        z = (X @ W.t() * w_gain + B * b_gain).detach().requires_grad_(True)
        slope, = torch.autograd.grad(act64(act, z, alpha).sum(), z)
    X, W, B, z = (t.detach() for t in (X, W, B, z))
    dz = (X.shape[1] + 8) * U * (X.abs() @ W.abs().t() * abs(w_gain) + abs(b_gain) * B.abs())
    largest = abs(alpha) if act == 'lrelu' and abs(alpha) > 1 else max(1.0, LIPSCHITZ.get(act, 1.0))
    s = G * slope
    # (in float32; relative to the slope where the exponential carries it, absolute where it does not)
    ds = G.abs() * (CURVATURE.get(act, 0.0 if act in ('linear', 'relu', 'lrelu') else 1.0) * dz + 16 * U)
    if act == 'lrelu':
        ds = ds + G.abs() * abs(1 - alpha) * (z.abs() <= dz)
    elif act in JUMP:
        ds = ds + G.abs() * JUMP[act] * (z.abs() <= dz)
    held = ds + H * s.abs() + 2.0 ** -39 * largest * G.abs().max()
    c, out = abs(gain * w_gain), {}
    out['dx'] = grads[0], c * (held @ W.abs() + (W.shape[0] + 8) * U * (s.abs() @ W.abs())) + H * grads[0].abs() + 2.0 ** -25
    out['dw'] = grads[1], c * (held.t() @ X.abs() + (X.shape[0] + 8) * U * (s.abs().t() @ X.abs())) + H * grads[1].abs() + 2.0 ** -25
    c = abs(gain * b_gain)
    out['db'] = grads[2], c * (ds.sum(dim=0) + (X.shape[0] + 8) * U * s.abs().sum(dim=0)) + H * grads[2].abs() + 2.0 ** -25
    return out


def case(size, seed=0):
    m, k, n = size
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(s, device=DEV, generator=g) for s in ((m, k), (n, k), (n,), (m, n))]


def compare(x, w, b, act, dy, gain=1.0, w_gain=1.0, b_gain=1.0, **kw):
    from ga_gan_amd.torch_utils.ops import linear
    x, w, b, dy = (t.half() for t in (x, w, b, dy))
    assert all(bool(t.isfinite().all()) for t in (x, w, b, dy))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = linear.linear(x, w, b, act=act, gain=gain, w_gain=w_gain, b_gain=b_gain, **kw)
    got = torch.autograd.grad(y, leaves, dy)
    want = bounds(x, w, b, act, dy, gain, w_gain, b_gain, **kw)
    for name, v in zip(('dx', 'dw', 'db'), got):
        assert float(want[name][0].abs().max()) < 60000, name           # (the results themselves fit)
        check(v, want[name], name)
    return want


# few rows; slices; whole packets and not; 128 x 128 tiles; one element
SIZES = [(5, 24, 40), (64, 2048, 72), (33, 9, 257), (600, 771, 1200), (1, 1, 1)]


@pytest.mark.parametrize('size', SIZES)
@pytest.mark.parametrize('act, kw', [('selu', {}), ('swish', {}), ('lrelu', dict(alpha=1.5)), ('lrelu', dict(alpha=-4.0)), ('lrelu', {}), ('tanh', {})])
def test_large_dy(size, act, kw):
    x, w, b, dy = case(size)
    dy = dy.sign() * (61000 - 4000 * dy.abs().clamp(max=1))
    scale = 2.0 ** -8 / math.sqrt(max(size))
    compare(x, w / 8 / math.sqrt(size[1]) / scale, b / scale, act, dy, w_gain=scale, b_gain=scale, gain=2.0 ** -4, **kw)


@pytest.mark.parametrize('size', SIZES)
@pytest.mark.parametrize('act', ['sigmoid', 'tanh', 'swish', 'elu', 'lrelu'])
def test_small_dy_times_small_slopes(size, act):
    """dy around 2^-20 and, but for lrelu, slopes around 2^-11: products below the smallest float16, sums that are not."""
    x, w, b, dy = case(size, 1)
    dy = (dy.clamp(-2, 2) * 2.0 ** -20)
    shift = dict(sigmoid=7.5, tanh=4.2, swish=-10.0, elu=-7.5, lrelu=-1.0)[act]
    want = compare(x / 32 / math.sqrt(size[1]), w * 32, b / 8 + shift, act, dy, gain=256.0)
    if size[1] <= 24:                            # zeros would not pass (in long sums the bound of z alone is larger than these slopes)
        value, bound = want['dx']
        assert bool((value.abs() > bound).any())


@pytest.mark.parametrize('value', [math.nan, math.inf])
def test_values_that_are_not_finite_reach_their_row_alone(value):
    from ga_gan_amd.torch_utils.ops import linear
    x, w, b, dy = (t.half() for t in case((40, 24, 16), 2))
    x.requires_grad_(True)
    dy[3] = 0
    dy[3, 5] = value
    got, = torch.autograd.grad(linear.linear(x, w, b, act='swish'), x, dy)
    dy[3, 5] = 0
    want, = torch.autograd.grad(linear.linear(x, w, b, act='swish'), x, dy)
    assert not bool(got[3].isfinite().any())
    keep = torch.arange(40, device=DEV) != 3
    assert torch.equal(got[keep], want[keep]) and bool(want.isfinite().all())


def test_zeros():
    from ga_gan_amd.torch_utils.ops import linear
    x, w, b, dy = (t.half().requires_grad_(True) for t in case((40, 24, 16), 3))
    for g in torch.autograd.grad(linear.linear(x, w, b, act='sigmoid'), (x, w, b), torch.zeros_like(dy)):
        assert not bool(g.any())


def test_graph_replays_follow_dy():
    """The scale is found anew by every replay."""
    from ga_gan_amd.torch_utils.ops import linear
    x, w, b, dy = (t.half() for t in case((64, 48, 40), 4))
    x.requires_grad_(True), w.requires_grad_(True)
    step = lambda: torch.autograd.grad(linear.linear(x, w, b, act='selu', w_gain=2.0 ** -7), (x, w), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for size in (2.0 ** -22, 1.0, 2.0 ** 14, 2.0 ** -10):
        dy.normal_().clamp_(-3, 3).mul_(size)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(out, step()))
        assert all(bool(a.isfinite().all()) for a in out)
        torch.cuda.synchronize()
