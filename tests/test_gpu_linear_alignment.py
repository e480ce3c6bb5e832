"""A gradient dy that starts anywhere in memory gives the bits that an aligned one gives."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('act', ['linear', 'lrelu', 'swish'])
@pytest.mark.parametrize('size', [(1024, 1024, 1024), (2048, 776, 520), (40, 64, 24)])
def test_dy_at_an_odd_address(size, act, dtype):
    from ga_gan_amd.torch_utils.ops import linear
    m, k, n = size
    g = torch.Generator(device=DEV).manual_seed(0)
    x, w, b = (torch.randn(s, device=DEV, generator=g).to(dtype).requires_grad_(True) for s in ((m, k), (n, k), (n,)))
    flat = torch.randn(m * n + 1, device=DEV, generator=g).to(dtype)
    odd = flat[1:].view(m, n)
    assert odd.data_ptr() % 16 != 0
    y = linear.linear(x, w, b, act=act)
    got, want = (torch.autograd.grad(y, (x, w, b), dy, retain_graph=True) for dy in (odd, odd.clone()))
    assert all(torch.equal(a, e) for a, e in zip(got, want))
