"""clip_grad_norm_ scales the gradient tensors themselves, however they lie in memory."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.mark.parametrize('max_norm', [0.5, 1e9])
def test_gradients_that_are_not_dense(max_norm):
    """Tolerance as in test_gpu_gradnorm.py: half a step and the scale's 2^-21."""
    from ga_gan_amd import optim_plugin
    g = torch.Generator(device=DEV).manual_seed(0)
    grads = [torch.randn(4, 6, 3, 3, device=DEV, generator=g).to(memory_format=torch.channels_last), torch.randn(9, 7, device=DEV, generator=g).t(),
             torch.randn(20, 8, device=DEV, generator=g)[::2, 1:6], torch.randn(5, device=DEV, generator=g)]
    params = [torch.nn.Parameter(torch.zeros(t.shape, device=DEV)) for t in grads]
    for p, t in zip(params, grads):
        p.grad = t
    before = [t.double() for t in grads]
    want = math.sqrt(sum(float(t.square().sum()) for t in before))
    versions = [t._version for t in grads]
    norm = optim_plugin.clip_grad_norm_(params, max_norm)
    assert abs(float(norm) - want) <= 2 ** -23 * want
    scale = min(1.0, max_norm / (want + 1e-6))
    for p, t, b, v in zip(params, grads, before, versions):
        assert p.grad is t and t._version > v
        assert bool(((t.double() - b * scale).abs() <= b.abs() * scale * (2.0 ** -24 + 2.0 ** -21)).all())


def test_a_gradient_that_overlaps_itself_is_replaced():
    from ga_gan_amd import optim_plugin
    p = torch.nn.Parameter(torch.zeros(6, 4, device=DEV))
    p.grad = torch.arange(4., device=DEV).expand(6, 4)
    before = p.grad.double()
    norm = optim_plugin.clip_grad_norm_(p, 0.5)
    want = float(before.norm())
    assert abs(float(norm) - want) <= 2 ** -23 * want
    want = before * (0.5 / (want + 1e-6))
    assert bool(((p.grad.double() - want).abs() <= want * (2.0 ** -24 + 2.0 ** -21)).all())


def test_one_gradient_of_two_parameters_is_refused():
    from ga_gan_amd import optim_plugin
    p, q = (torch.nn.Parameter(torch.zeros(4, 3, device=DEV)) for _ in range(2))
    p.grad = q.grad = torch.ones(3, 4, device=DEV).t()
    with pytest.raises(RuntimeError, match='twice'):
        optim_plugin.clip_grad_norm_([p, q], 1.0)
    assert bool((p.grad == 1).all())


def test_a_refused_call_leaves_them_alone():
    from ga_gan_amd import optim_plugin
    p, q = torch.nn.Parameter(torch.zeros(4, 4, device=DEV)), torch.nn.Parameter(torch.zeros(3))
    p.grad, q.grad = torch.ones(4, 4, device=DEV).t(), torch.ones(3)
    grad = p.grad
    with pytest.raises(RuntimeError):
        optim_plugin.clip_grad_norm_([p, q], 1.0)
    assert p.grad is grad and bool((grad == 1).all())
