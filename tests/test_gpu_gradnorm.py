"""Global gradient norm, clipping and the clipped optimizer step (sg_grad_norm, sg_scale_grads, sg_adam_step_list) against
64-bit arithmetic.

Tolerances.  The norm: squares and sums are double (relative error below 1e-13 for 10^8 elements), then one rounding to float32,
2^-24; allowed 2^-23.  Clipped gradients: scale = max_norm / (norm + 1e-6) in float32 from the rounded norm (three roundings, 3 *
2^-24), the product rounded once to the gradient's type (half a step, eps / 2): allowed eps / 2 + 2^-21.  The step, with u = 2^-24 and the entry point's own float32 values of lr, betas and eps in the 64-bit
arithmetic (1 - beta is then exact for beta >= 1/2):  c = g scale is off by 4 u |c| (scale 3 u, product u);
  m' = m + (1 - beta1)(c - m), in either of lerp's forms: difference u (|c| + |m|), product, sum and c's own: 8 u (|m| + |c|)
  v' = beta2 v + (1 - beta2) c^2: terms are not negative; c^2 twice c's error and four roundings: 16 u v'
  p' = p - a m' / (sqrt(v') / b + eps): quotient of m' (8 u above) and a denominator off by 16 u relative, 4 roundings, one more
       for the difference: a / denominator * 8 u (|m| + |c|) + 24 u |update| + u (|p| + |update|).
A relative tolerance on p' or m' alone (as first written here, 2e-6) does not hold where the two terms cancel."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'

LISTS = {
    'one': [1],
    'odd': [1, 3, 5, 7, 9, 4097, 33, 0, 16384 * 3 + 5],
    'many': [(37 * i) % 1000 + 1 for i in range(300)],     # more than two tables of 128 tensors
    'large': [(1 << 23) + 3, 17, 1 << 22],
}


def _flat(sizes, dtype, seed, offset=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    flat = torch.randn([offset + sum(sizes)], device=DEV, generator=g).to(dtype)
    return flat, list(flat[offset:].split(sizes))


@pytest.mark.parametrize('name', list(LISTS))
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('offset', [0, 1])
def test_norm(name, dtype, offset):
    """Views of a flat buffer that start at any element."""
    from ga_gan_amd import optim_plugin
    _, grads = _flat(LISTS[name], dtype, 1, offset)
    want = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    got = optim_plugin.grad_norm(grads)
    assert got.shape == () and got.dtype == torch.float32 and got.is_cuda
    assert abs(float(got) - want) <= 2 ** -23 * want
    assert torch.equal(got, optim_plugin.grad_norm(grads))


def test_norm_of_mixed_types_and_extremes():
    from ga_gan_amd import optim_plugin
    grads = [torch.full([5], 3e38, device=DEV), torch.full([7], 60000., device=DEV, dtype=torch.float16), torch.full([9], 1e-30, device=DEV, dtype=torch.bfloat16)]
    want = math.sqrt(sum(float(g.double().square().sum()) for g in grads))     # 6.7e38: no float32
    assert float(optim_plugin.grad_norm(grads)) == math.inf and want > 3.5e38
    grads[0].fill_(1e20)                                                       # a square that float32 does not hold
    want = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    assert abs(float(optim_plugin.grad_norm(grads)) - want) <= 2 ** -23 * want
    tiny = [torch.full([1000], 1e-30, device=DEV)]                             # squares below float32's range
    assert abs(float(optim_plugin.grad_norm(tiny)) - 1e-30 * math.sqrt(1000)) <= 1e-6 * 1e-30 * math.sqrt(1000)
    wild = [torch.tensor([3., math.nan, math.inf, -math.inf, 4.], device=DEV)]
    assert math.isnan(float(optim_plugin.grad_norm(wild)))
    want = math.sqrt(25 + 2 * 1e10)
    assert abs(float(optim_plugin.grad_norm(wild, grad_limit=1e5)) - want) <= 2 ** -23 * want
    assert float(optim_plugin.grad_norm([])) == 0
    assert float(optim_plugin.grad_norm([torch.zeros([0], device=DEV)])) == 0


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('max_norm', [0.5, 1e6, 0.0])
def test_clip(dtype, max_norm):
    from ga_gan_amd import optim_plugin
    _, grads = _flat(LISTS['odd'] + LISTS['many'], dtype, 2, 3)
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads] + [torch.nn.Parameter(torch.zeros(3, device=DEV))]
    for p, g in zip(params, grads):
        p.grad = g
    before = [g.double().cpu() for g in grads]
    version = grads[0]._version
    want = math.sqrt(sum(float(g.square().sum()) for g in before))
    got = optim_plugin.clip_grad_norm_(params, max_norm)
    assert abs(float(got) - want) <= 2 ** -23 * want
    assert grads[0]._version > version and params[-1].grad is None
    scale = min(1.0, max_norm / (want + 1e-6))
    tiny = torch.finfo(dtype).tiny
    for g, b in zip(grads, before):
        bound = b.abs() * scale * (torch.finfo(dtype).eps / 2 + 2 ** -21) + (tiny if scale < 1 else 0)
        assert bool(((g.double().cpu() - b * scale).abs() <= bound).all())
        if scale == 1:
            assert torch.equal(g.double().cpu(), b)


def test_clip_of_a_norm_that_is_not_finite_follows_torch():
    from ga_gan_amd import optim_plugin
    for value in (math.nan, math.inf):
        ours = torch.nn.Parameter(torch.zeros(4, device=DEV))
        ours.grad = torch.tensor([1., value, -2., 3.], device=DEV)
        ref = torch.nn.Parameter(torch.zeros(4))
        ref.grad = torch.tensor([1., value, -2., 3.])
        a, b = optim_plugin.clip_grad_norm_(ours, 1.0), torch.nn.utils.clip_grad_norm_(ref, 1.0)
        np.testing.assert_array_equal(a.cpu().numpy(), b.numpy())
        np.testing.assert_array_equal(ours.grad.cpu().numpy(), ref.grad.numpy())


U = 2.0 ** -24


def _adam64(p, g, m, v, step, lr, b1, b2, eps, scale):
    """((p', bound), (m', bound), (v', bound))"""
    lr, b1, b2, eps = (float(np.float32(t)) for t in (lr, b1, b2, eps))
    c = g * scale
    m2 = b1 * m + (1 - b1) * c
    v2 = b2 * v + (1 - b2) * c * c
    a, denominator = lr / (1 - b1 ** step), v2.sqrt() / math.sqrt(1 - b2 ** step) + eps
    update = a * m2 / denominator
    dm = 8 * U * (m.abs() + c.abs())
    return ((p - update, a / denominator * dm + 24 * U * update.abs() + U * (p.abs() + update.abs()) + 1e-37), (m2, dm + 1e-37), (v2, 16 * U * v2 + 1e-37))


@pytest.mark.parametrize('offset', [0, 1])
@pytest.mark.parametrize('max_norm', [0.25, 1e9])
@pytest.mark.parametrize('beta1', [0.0, 0.9])
def test_clipped_step(offset, max_norm, beta1):
    from ga_gan_amd import optim_plugin
    sizes = [5, 1, 4096, 130, 4097 * 3] + [7] * 70                 # two tables of 64 tensors
    lists, flats = [], []
    for k in range(4):
        flat, views = _flat(sizes, torch.float32, 10 + k, offset if k != 2 else 0)     # (offset: the four tensors lie differently)
        flats.append(flat[offset if k != 2 else 0:])
        lists.append(views)
    flats[3].abs_()
    flats[1][2], flats[1][9], flats[1][-1] = math.nan, math.inf, -math.inf
    p, g, m, v = (f.double().cpu() for f in flats)
    clean = torch.nan_to_num(g, 0.0, 1e5, -1e5)
    norm = float(clean.norm())
    want = _adam64(p, clean, m, v, 3, 0.01, beta1, 0.99, 1e-8, min(1.0, max_norm / (norm + 1e-6)))
    got = optim_plugin.adam_step(*lists, [3] * len(sizes), 0.01, beta1, 0.99, 1e-8, max_grad_norm=max_norm)
    assert abs(float(got) - norm) <= 2 ** -23 * norm
    assert torch.equal(flats[1].cpu().double(), clean)             # what stays is the sanitised gradient, unscaled
    for name, a, (value, bound) in zip('pmv', (flats[0], flats[2], flats[3]), want):
        assert bool(((a.double().cpu() - value).abs() <= bound).all()), name


def test_optimizer_clips_over_its_groups_and_leaves_state_interchangeable():
    from ga_gan_amd import optim_plugin
    torch.manual_seed(0)
    a = [torch.nn.Parameter(torch.randn(33, 5, device=DEV)), torch.nn.Parameter(torch.randn(9, device=DEV)), torch.nn.Parameter(torch.randn(2, device=DEV))]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    groups = lambda q: [dict(params=q[:1], lr=0.01), dict(params=q[1:], lr=0.002)]
    fused = optim_plugin.FusedAdam(groups(a), betas=(0.5, 0.9), max_grad_norm=0.7)
    ref = torch.optim.Adam(groups(b), betas=(0.5, 0.9), eps=1e-8)
    for step in range(3):
        for p, q in zip(a[:2], b[:2]):                             # (the third never receives a gradient)
            p.grad = torch.randn_like(p) * 10 ** (step - 1)
            q.grad = p.grad.clone()
        norm = torch.nn.utils.clip_grad_norm_(b[:2], 0.7)
        ref.step()
        fused.step()
        assert abs(float(fused.last_grad_norm) - float(norm)) <= 1e-6 * float(norm)
    for p, q in zip(a, b):
        torch.testing.assert_close(p, q, rtol=2e-6, atol=1e-7)
    assert 'max_grad_norm' not in fused.state_dict()['param_groups'][0]
    fresh = torch.optim.Adam(groups(b), betas=(0.5, 0.9), eps=1e-8)
    fresh.load_state_dict(fused.state_dict())


def test_step_without_clipping_is_the_unclipped_step_bit_for_bit():
    from ga_gan_amd import optim_plugin
    sizes = [5, 4096, 130]
    a = [_flat(sizes, torch.float32, 20 + k)[1] for k in range(4)]
    a[3] = [t.abs() for t in a[3]]
    b = [[t.clone() for t in ts] for ts in a]
    optim_plugin.adam_step(*a, [2] * 3, 0.01, 0.5, 0.99, 1e-8)
    optim_plugin.adam_step(*b, [2] * 3, 0.01, 0.5, 0.99, 1e-8, max_grad_norm=1e9)
    for x, y in zip(a, b):
        for t, u in zip(x, y):
            assert torch.equal(t, u)


def test_step_issues_no_host_read():
    from ga_gan_amd import optim_plugin
    p = torch.nn.Parameter(torch.randn(100, device=DEV))
    opt = optim_plugin.FusedAdam([p], lr=0.01, max_grad_norm=1.0)
    p.grad = torch.randn_like(p)
    opt.step()
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode('error')
    try:
        opt.step()
        optim_plugin.clip_grad_norm_([p], 0.1)
    finally:
        torch.cuda.set_sync_debug_mode('default')


def test_graph_replays_follow_the_gradients():
    from ga_gan_amd import optim_plugin
    g = torch.Generator(device=DEV).manual_seed(3)
    params = [torch.nn.Parameter(torch.zeros(n, device=DEV)) for n in (5, 100000, 300)]
    for p in params:
        p.grad = torch.randn(p.shape, device=DEV, generator=g)
    optim_plugin.clip_grad_norm_(params, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = optim_plugin.clip_grad_norm_(params, 1.0)
    for trial in range(4):
        fresh = [torch.randn(p.shape, device=DEV, generator=g) * 10.0 ** (trial - 3) for p in params]
        for p, f in zip(params, fresh):
            p.grad.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        want = math.sqrt(sum(float(f.double().square().sum()) for f in fresh))
        assert abs(float(norm) - want) <= 2 ** -23 * want
        for p, f in zip(params, fresh):
            torch.testing.assert_close(p.grad, f * min(1.0, 1.0 / (want + 1e-6)), rtol=1e-6, atol=0)


def test_other_stream():
    from ga_gan_amd import optim_plugin
    x = torch.randn(1 << 22, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = x * 2
        norm = optim_plugin.grad_norm([y])
    side.synchronize()
    want = float(x.double().mul(2).square().sum().sqrt())
    assert abs(float(norm) - want) <= 2 ** -23 * want


def test_refusals():
    from ga_gan_amd import optim_plugin
    good = torch.zeros(4, device=DEV)
    for bad in (torch.zeros(4), torch.zeros(4, device=DEV, dtype=torch.float64), torch.zeros(4, 4, device=DEV).t()[:, :2]):
        with pytest.raises(RuntimeError):
            optim_plugin.grad_norm([good, bad])
    with pytest.raises(RuntimeError):
        optim_plugin.grad_norm([good], grad_limit=-1.0)
    p, q = torch.nn.Parameter(torch.zeros(4, device=DEV)), torch.nn.Parameter(torch.zeros(4, device=DEV))
    p.grad = q.grad = torch.ones(4, device=DEV)
    with pytest.raises(RuntimeError, match='twice'):
        optim_plugin.clip_grad_norm_([p, q], 1.0)
    with pytest.raises(RuntimeError, match='negative'):
        optim_plugin.clip_grad_norm_([p], -1.0)
    with pytest.raises(RuntimeError, match='negative'):
        optim_plugin.clip_grad_norm_([p], float('nan'))
    t = lambda: torch.zeros(4, device=DEV)
    with pytest.raises(RuntimeError, match='twice'):
        optim_plugin.adam_step([good], [t()], [good], [t()], [1], 1e-3, 0.9, 0.99, 1e-8, max_grad_norm=1.0)
    with pytest.raises(RuntimeError):
        optim_plugin.adam_step([good], [t()], [t()], [torch.zeros(5, device=DEV)], [1], 1e-3, 0.9, 0.99, 1e-8, max_grad_norm=1.0)
    with pytest.raises(RuntimeError):
        optim_plugin.adam_step([good], [t()], [t()], [t()], [0], 1e-3, 0.9, 0.99, 1e-8, max_grad_norm=1.0)
