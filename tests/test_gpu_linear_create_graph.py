"""Gradients of the fully connected layer that are themselves differentiable (create_graph=True): the first-order ones keep the bounds
of the others (tests/linear_bounds.py) in every type, and a penalty on them has the derivative its formula gives."""
import math

import pytest
import torch

from linear_bounds import LIPSCHITZ, act64, bounds, check

pytestmark = pytest.mark.gpu
DEV = 'cuda'
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(m, k, n, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(s, device=DEV, generator=g)
    return [t.to(dtype) for t in (r(m, k), r(n, k) / math.sqrt(k), r(n), r(m, n), r(m, n))]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('act', ['linear', 'relu', 'lrelu', 'tanh', 'sigmoid', 'elu', 'selu', 'softplus', 'swish'])
@pytest.mark.parametrize('residual', [False, True])
def test_first_order(act, dtype, residual):
    from ga_gan_amd.torch_utils.ops import linear
    x, w, b, r, dy = make(256, 512, 300, dtype)
    r = r if residual else None
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = linear.linear(x, w, b, residual=r, act=act)
    got = torch.autograd.grad(y, leaves, dy, create_graph=True)
    want = bounds(x, w, b, r, act, dy)
    for name, v in zip(('dx', 'dw', 'db'), got):
        assert v.dtype == dtype and (v.requires_grad or name == 'db')        # (without a bend db depends on dy alone)
        check(v, want[name], name)


@pytest.mark.parametrize('dtype', DTYPES)
def test_gains(dtype):
    from ga_gan_amd.torch_utils.ops import linear
    x, w, b, _, dy = make(33, 64, 40, dtype)
    for kw in (dict(act='lrelu', alpha=0.5, gain=-1.5), dict(act='lrelu', alpha=-0.3), dict(act='tanh', gain=3.0, w_gain=0.7, b_gain=0.25)):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        got = torch.autograd.grad(linear.linear(*leaves, **kw), leaves, dy, create_graph=True)
        want = bounds(x, w, b, None, dy=dy, **kw)
        for name, v in zip(('dx', 'dw', 'db'), got):
            check(v, want[name], name)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('act', ['relu', 'lrelu'])
def test_slopes_are_the_forward_pass_s(act, dtype):
    """Bit for bit where sums are exact: pre-activation values of whole numbers, some of them zero, and products of powers of two."""
    from ga_gan_amd.torch_utils.ops import linear
    g = torch.Generator(device=DEV).manual_seed(2)
    x, w, b = (torch.randint(-1, 2, s, device=DEV, generator=g).to(dtype).requires_grad_(True) for s in ((30, 16), (24, 16), (24,)))
    dy = torch.exp2(torch.randint(-2, 3, (30, 24), device=DEV, generator=g).float()).to(dtype)
    y = linear.linear(x, w, b, act=act, alpha=0.25, gain=1.0)
    assert bool((y == 0).any())
    for a, e in zip(torch.autograd.grad(y, (x, w, b), dy, retain_graph=True), torch.autograd.grad(y, (x, w, b), dy, create_graph=True)):
        assert torch.equal(a, e)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('act', ['lrelu', 'tanh', 'swish'])
def test_penalty(act, dtype):
    """P = sum g^2 with g = dP/dx: dP/dg = v = 2 g, exact in the type (g itself is off by at most its bound E, so v by 2 E).  With
    s = dy act'(z), c the default gain, a = v w^T c (what reaches s) and t = dy act''(z) a (what reaches z):
      dP/dw = c s^T v + t^T x,  dP/dx = t w.
    An error E2 = 2 E in v shows as c |s|^T E2 + (|dy act''| (c E2 |w|^T))^T |x|; everything else is float32 - sums of at most 100
    terms, 2^-17 of the absolute sums, and act', act'' at a z that is off by 60 u of |x| |w|^T, below 2^-16 - and one rounding, h:
    2^-14 of the absolute sums, with |act''| <= 2 for those, and h of the value."""
    from ga_gan_amd.torch_utils.ops import linear
    x, w, b, _, dy = make(20, 48, 33, dtype)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    g, = torch.autograd.grad(linear.linear(*leaves, act=act), leaves[0], dy, create_graph=True)
    got = torch.autograd.grad(g.float().square().sum(), leaves[:2], allow_unused=True)
    X, W, B = (t.detach().double().requires_grad_(True) for t in (x, w, b))
    G, c = dy.double(), math.sqrt(2) if act in ('lrelu', 'swish') else 1.0
    z = X @ W.t() + B
    if act == 'lrelu':
        assert float(z.abs().min()) > 1e-4                           # (nobody is in doubt about a sign)
    want_g, = torch.autograd.grad(act64(act, z) * c, X, G, create_graph=True)
    want = torch.autograd.grad(want_g.square().sum(), (X, W), allow_unused=True)
    with torch.no_grad():
        h, low = torch.finfo(dtype).eps / 2, 2.0 ** -24 if dtype == torch.float16 else 1e-37
        v, e2 = 2 * want_g.abs(), 2 * bounds(x, w, b, None, act, dy)['dx'][1]
        slope = LIPSCHITZ.get(act, 1.0)
        bend = 0.0 if act == 'lrelu' else 1.0
        ax, aw, ag = X.abs(), W.abs(), G.abs()
        t_of = lambda q: bend * ag * (c * q @ aw.t())                # (bend: largest |act''|: tanh 0.77, swish 0.5)
        slack = 2.0 ** -14
        bound_w = c * slope * (ag.t() @ e2) + t_of(e2).t() @ ax + slack * (c * slope * (ag.t() @ v) + 2 * t_of(v).t() @ ax)
        bound_x = (t_of(e2) + slack * 2 * t_of(v)) @ aw
    check(got[1], (want[1].detach(), bound_w + h * want[1].abs() + low), 'w')
    if act == 'lrelu':
        assert got[0] is None or not bool(got[0].any())
    else:
        check(got[0], (want[0].detach(), bound_x + h * want[0].abs() + low), 'x')
