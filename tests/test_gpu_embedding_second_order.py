"""The table's gradient differentiated where some indices lie outside the table: those tokens add to no row, so nothing of the table's
second-order gradient reaches their dy, and the bias's does."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.mark.parametrize('bias', [False, True])
@pytest.mark.parametrize('tokens', [40, 600])
def test_indices_outside_the_table(tokens, bias):
    """Tolerance: the lookup and its product by two, 2^-22 of the values' size; the row sums' own error, tokens * 2^-24 of theirs."""
    from ga_gan_amd.torch_utils.ops import embedding
    g = torch.Generator(device=DEV).manual_seed(0)
    table, b = torch.randn(9, 16, device=DEV, generator=g).requires_grad_(True), torch.randn(16, device=DEV, generator=g).requires_grad_(True)
    dy = torch.randn(tokens, 16, device=DEV, generator=g).requires_grad_(True)
    index = torch.randint(0, 9, [tokens], device=DEV, generator=g)
    outside = torch.arange(tokens, device=DEV) % 4 == 1
    bad = torch.where(outside, torch.where(index % 2 == 0, -1 - index, 9 + index), index)
    leaves = [table, b] if bias else [table]
    grads = torch.autograd.grad(embedding.embedding(bad, table, b if bias else None, w_gain=0.5, b_gain=2.0), leaves, dy, create_graph=True)
    got, = torch.autograd.grad(sum(t.square().sum() for t in grads), dy)
    d = dy.detach().double().requires_grad_(True)
    want = torch.zeros(9, 16, device=DEV, dtype=torch.float64).index_add(0, index[~outside], d[~outside]).mul(0.5).square().sum()
    if bias:
        want = want + (d.sum(dim=0) * 2).square().sum()
    want, = torch.autograd.grad(want, d)
    size = float(d.detach().abs().sum(dim=0).max()) * 8
    assert bool(got.isfinite().all())
    assert float((got.double() - want).abs().max()) <= (tokens + 8) * 2.0 ** -24 * size + 2.0 ** -22 * float(want.abs().max())
    assert bool((got[outside] == 0).all()) or bias
