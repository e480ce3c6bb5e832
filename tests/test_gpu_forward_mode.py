"""Forward-mode derivatives are not offered: a dual tensor is refused wherever it enters, with gradients wanted or not, rather than
having its tangent dropped."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.mark.parametrize('grad', [False, True])
@pytest.mark.parametrize('which', range(4))
def test_linear(which, grad):
    from ga_gan_amd.torch_utils.ops import linear
    args = [torch.randn(s, device=DEV) for s in ((4, 8), (6, 8), (6,), (4, 6))]
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match='jvp|forward'):
            linear.linear(*args[:3], residual=args[3], act='lrelu')


@pytest.mark.parametrize('grad', [False, True])
@pytest.mark.parametrize('which', range(2))
def test_embedding(which, grad):
    from ga_gan_amd.torch_utils.ops import embedding
    args = [torch.randn(9, 8, device=DEV), torch.randn(8, device=DEV)]
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match='jvp|forward'):
            embedding.embedding(torch.arange(5, device=DEV), *args)


def test_backward_of_a_dual_gradient():
    from ga_gan_amd.torch_utils.ops import embedding, linear
    x, w = torch.randn(4, 8, device=DEV, requires_grad=True), torch.randn(6, 8, device=DEV)
    table = torch.randn(9, 6, device=DEV, requires_grad=True)
    for leaf, y in ((x, linear.linear(x, w, act='lrelu')), (table, embedding.embedding(torch.arange(4, device=DEV), table))):
        with forward_ad.dual_level():
            dy = forward_ad.make_dual(torch.randn(4, 6, device=DEV), torch.ones(4, 6, device=DEV))
            with pytest.raises(RuntimeError, match='jvp|forward'):
                torch.autograd.grad(y, leaf, dy)


def test_networks_with_fused_layers():
    """A layer of a network: refused with the fused kernels, the library's derivative without."""
    from ga_gan_amd.training import networks
    layer = networks.FullyConnectedLayer(8, 6).to(DEV).requires_grad_(False)
    x, t = torch.randn(4, 8, device=DEV), torch.randn(4, 8, device=DEV)
    old = networks.FUSE_DENSE
    try:
        for networks.FUSE_DENSE in (False, True):
            with forward_ad.dual_level():
                if networks.FUSE_DENSE:
                    with pytest.raises(RuntimeError, match='jvp|forward'):
                        layer(forward_ad.make_dual(x, t))
                else:
                    tangent = forward_ad.unpack_dual(layer(forward_ad.make_dual(x, t))).tangent
                    torch.testing.assert_close(tangent, t @ (layer.weight * layer.weight_gain).t())
    finally:
        networks.FUSE_DENSE = old
