"""The gradient of relu takes nothing from units that are off, whatever dy holds there: zero is selected, not multiplied (as `bias_act`
and torch do).  Bounds: tests/linear_bounds.py, of the same dy with zeros at those units."""
import math

import pytest
import torch

from linear_bounds import bounds, check

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('residual', [False, True])
@pytest.mark.parametrize('size', [(33, 64, 40), (70, 9, 33)])
def test_relu_ignores_dy_where_it_is_off(size, residual, dtype):
    from ga_gan_amd.torch_utils.ops import linear
    m, k, n = size
    g = torch.Generator(device=DEV).manual_seed(1)
    r = lambda *s: torch.randn(s, device=DEV, generator=g).to(dtype)
    x, w, b, dy, res = r(m, k), (r(n, k) / math.sqrt(k)).to(dtype), r(n), r(m, n), r(m, n) if residual else None
    off = (x.double() @ w.double().t() + b.double()) < -0.1              # (rounding does not turn these on)
    assert 0.2 < float(off.double().mean()) < 0.8
    wild = torch.tensor([math.nan, math.inf, -math.inf], device=DEV).to(dtype).repeat(dy.numel())[:dy.numel()].view_as(dy)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = linear.linear(x, w, b, residual=res, act='relu')
    got = torch.autograd.grad(y, leaves, torch.where(off, wild, dy))
    want = bounds(x, w, b, res, 'relu', torch.where(off, torch.zeros_like(dy), dy))
    for name, v in zip(('dx', 'dw', 'db'), got):
        check(v, want[name], name)
