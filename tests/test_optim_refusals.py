"""A step of the optimizer that is refused changes nothing: no count, no moment, no parameter, in any group."""
import pytest
import torch


def optimizer(params, **kw):
    from ga_gan_amd import optim_plugin
    return optim_plugin.FusedAdam(params, **kw)


@pytest.mark.parametrize('max_grad_norm', [None, 1.0])
def test_refused_for_its_device(max_grad_norm):
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    opt = optimizer([p], max_grad_norm=max_grad_norm)
    with pytest.raises(RuntimeError, match='CUDA'):
        opt.step()
    assert p not in opt.state or not opt.state[p]
    opt.state[p] = dict(step=torch.tensor(4.0), exp_avg=torch.zeros(3), exp_avg_sq=torch.zeros(3))
    with pytest.raises(RuntimeError, match='CUDA'):
        opt.step()
    assert int(opt.state[p]['step']) == 4


def two_groups(device, **second):
    p, q = (torch.nn.Parameter(torch.ones(n, device=device)) for n in (3, 5))
    return p, q, [dict(params=[p]), dict(params=[q], **second)]


def unchanged(opt, before):
    for p, (value, count) in before.items():
        assert torch.equal(p.detach(), value)
        assert (int(opt.state[p]['step']) if opt.state.get(p) else 0) == count
        if count == 0:
            assert not opt.state.get(p)


@pytest.mark.gpu
@pytest.mark.parametrize('max_grad_norm', [None, 1.0])
@pytest.mark.parametrize('stepped', [False, True])
@pytest.mark.parametrize('bad', ['betas', 'eps', 'strides'])
def test_refused_for_its_second_group(bad, stepped, max_grad_norm):
    p, q, groups = two_groups('cuda')
    opt = optimizer(groups, lr=0.1, max_grad_norm=max_grad_norm)
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    if stepped:
        opt.step()
    before = {t: (t.detach().clone(), int(stepped)) for t in (p, q)}
    if bad == 'betas':
        opt.param_groups[1]['betas'] = (0.9, 1.5)
    if bad == 'eps':
        opt.param_groups[1]['eps'] = -1.0
    if bad == 'strides':
        q.data = torch.ones(10, device='cuda')[::2]
        before[q] = (q.detach().clone(), int(stepped))
    with pytest.raises(RuntimeError):
        opt.step()
    unchanged(opt, before)


@pytest.mark.gpu
@pytest.mark.parametrize('stepped', [False, True])
def test_a_gradient_that_two_groups_share_is_refused_where_it_would_count_twice(stepped):
    p, q = (torch.nn.Parameter(torch.ones(4, device='cuda')) for _ in range(2))
    opt = optimizer([dict(params=[p]), dict(params=[q], lr=0.5)], lr=0.1, max_grad_norm=1.0)
    if stepped:
        p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
        opt.step()
    before = {t: (t.detach().clone(), int(stepped)) for t in (p, q)}
    p.grad = q.grad = torch.ones(4, device='cuda')
    with pytest.raises(RuntimeError, match='twice'):
        opt.step()
    unchanged(opt, before)


@pytest.mark.gpu
@pytest.mark.parametrize('max_grad_norm', [None, 1.0])
def test_a_step_after_a_refused_one_has_its_own_number(max_grad_norm):
    """Against torch's optimizer over the steps that took place (tolerance as in test_gpu_gradnorm.py)."""
    p = torch.nn.Parameter(torch.linspace(-1, 1, 8, device='cuda'))
    ref = torch.nn.Parameter(p.detach().clone())
    opt, adam = optimizer([p], lr=0.01, betas=(0.5, 0.9), max_grad_norm=max_grad_norm), torch.optim.Adam([ref], lr=0.01, betas=(0.5, 0.9), eps=1e-8)
    for step in range(3):
        p.grad = torch.linspace(0.1, 0.2, 8, device='cuda') * (step + 1)
        ref.grad = p.grad.clone()
        opt.param_groups[0]['eps'] = -1.0
        with pytest.raises(RuntimeError):
            opt.step()
        opt.param_groups[0]['eps'] = 1e-8
        opt.step()
        if max_grad_norm is not None:
            torch.nn.utils.clip_grad_norm_([ref], max_grad_norm)
        adam.step()
        torch.testing.assert_close(p, ref, rtol=2e-6, atol=1e-7)
    assert int(opt.state[p]['step']) == 3
