"""Table lookup and its gradient (sg_embedding, sg_embedding_backward) against 64-bit arithmetic.

Bounds, u = 2^-24, h = eps / 2 of the type: the lookup is a product and a sum in float32 and one rounding: 3 u (|product| + |bias|)
+ h |y|.  A gradient row is a sum of c rows in float32 in any order, times the gain, rounded: (c + 3) u (sum of |dy|) |gain| + h |value|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24


def op():
    from ga_gan_amd.torch_utils.ops import embedding
    return embedding.embedding


def indices(kind, tokens, v, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if kind == 'one':
        return torch.full([tokens], v // 2, device=DEV)
    if kind == 'ascending':
        return torch.arange(tokens, device=DEV) * v // max(tokens, 1)
    u = torch.rand(tokens, device=DEV, generator=g, dtype=torch.float64)
    return (float(v) ** u - 1 if kind == 'skewed' else u * v).long().clamp(0, v - 1)


def compare(index, table, b, dy, w_gain=0.5, b_gain=2.0):
    dtype = table.dtype
    h = torch.finfo(dtype).eps / 2
    low = 2.0 ** -24 if dtype == torch.float16 else 1e-37
    t = table.detach().requires_grad_(True)
    bb = b.detach().requires_grad_(True) if b is not None else None
    y = op()(index, t, bb, w_gain=w_gain, b_gain=b_gain)
    leaves = [t] if b is None else [t, bb]
    grads = torch.autograd.grad(y, leaves, dy)
    again = torch.autograd.grad(op()(index, t, bb, w_gain=w_gain, b_gain=b_gain), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))
    product = table.double()[index] * w_gain
    bias = b.double() * b_gain if b is not None else torch.zeros(table.shape[1], device=DEV).double()
    want = product + bias
    assert y.shape == want.shape and y.dtype == dtype
    assert bool(((y.double() - want).abs() <= 3 * U * (product.abs() + bias.abs()) + h * want.abs() + low).all())
    flat, d = index.reshape(-1), dy.double().reshape(-1, table.shape[1])
    zeros = torch.zeros(table.shape, device=DEV, dtype=torch.float64)
    want, size = zeros.index_add(0, flat, d) * w_gain, zeros.index_add(0, flat, d.abs()) * abs(w_gain)
    count = torch.bincount(flat, minlength=table.shape[0]).double()[:, None]
    assert grads[0].shape == table.shape
    off = (grads[0].double() - want).abs()
    assert bool((off <= (count + 3) * U * size + h * want.abs() + low * (count > 0)).all())       # rows without tokens: exactly zero
    if b is not None:
        want, size = d.sum(dim=0) * b_gain, d.abs().sum(dim=0) * abs(b_gain)
        assert bool(((grads[1].double() - want).abs() <= (len(d) + 3) * U * size + h * want.abs() + low).all())


def make(tokens, v, f, dtype, kind='uniform', columns=False, bias=True, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    table = (torch.randn([f, v], device=DEV, generator=g).t() if columns else torch.randn([v, f], device=DEV, generator=g)).to(dtype)
    b = torch.randn([f], device=DEV, generator=g).to(dtype) if bias else None
    return indices(kind, tokens, v, seed), table, b, torch.randn([tokens, f], device=DEV, generator=g).to(dtype)


# the three ways a gradient is formed: up to 256 tokens, up to 4096 (one workgroup sorts), beyond
SIZES = [(1, 1, 1), (1, 5, 512), (0, 4, 8), (64, 1000, 512), (255, 3, 65), (256, 257, 64), (257, 256, 64), (300, 255, 7), (1000, 65536, 24), (4096, 70, 130),
         (4097, 70000, 40), (20000, 300, 96), (5000, 1, 33),
         (200, 20000, 1100), (20, 60000, 72)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('columns', [False, True])
@pytest.mark.parametrize('size', SIZES)
def test_sizes(size, columns, dtype):
    compare(*make(*size, dtype, columns=columns))


@pytest.mark.parametrize('kind', ['one', 'ascending', 'skewed'])
@pytest.mark.parametrize('tokens', [200, 3000, 30000])
@pytest.mark.parametrize('f', [64, 513])
def test_distributions(kind, tokens, f):
    """One index for all, sorted ones, natural frequencies: runs inside one wave's positions and across many."""
    compare(*make(tokens, 500, f, torch.float32, kind))
    compare(*make(tokens, 500, f, torch.bfloat16, kind, bias=False))


def test_long_run():
    """More spans than one round of 64 probes finds."""
    index, table, b, dy = make(300000, 7, 8, torch.float32, 'one')
    index[:100], index[-5:] = 0, 6
    compare(index, table, b, dy)


@pytest.mark.parametrize('v', [255, 256, 65535, 65536])
@pytest.mark.parametrize('tokens', [2000, 9000])
def test_table_sizes_at_a_digit_border(v, tokens):
    index, table, b, dy = make(tokens, v, 16, torch.float32)
    index[::3] = v - 1
    compare(index, table, b, dy)


def test_indices_of_four_digits():
    index, table, b, dy = make(5000, (1 << 24) + 5, 2, torch.float32)
    index[:2], index[-1] = (1 << 24) + 4, 1 << 24
    compare(index, table, b, dy)


def test_more_than_32_bits_of_offset():
    """A table and outputs beyond 2^32 bytes: rows on both sides of the border, exactly (gains of one, no bias, indices once)."""
    v, f = (1 << 20) + 3, 2056
    table = torch.empty([v, f], dtype=torch.bfloat16, device=DEV)
    ramp = torch.arange(f, device=DEV)
    number = torch.arange(v, device=DEV)
    for i in range(0, v, 1 << 18):
        part = number[i:i + (1 << 18), None] * 31 + ramp
        table[i:i + (1 << 18)] = (part % 251).bfloat16()          # (whole numbers below 256 are bfloat16's)
    index = torch.randperm(v, device=DEV)
    table.requires_grad_(True)
    y = op()(index, table)
    for i in (0, 1 << 19, (1 << 20) - 2045, v - 3000):
        assert torch.equal(y[i:i + 3000], table[index[i:i + 3000]])
    grad, = torch.autograd.grad(y, table, y.detach())
    for i in (0, 1 << 19, (1 << 20) - 2045, v - 3000):
        assert torch.equal(grad[i:i + 3000], table[i:i + 3000])


def test_strides_and_index_types():
    g = torch.Generator(device=DEV).manual_seed(1)
    big = torch.randn([60, 90], device=DEV, generator=g)
    index = indices('uniform', 77, 20)
    dy = torch.randn([64, 77], device=DEV, generator=g).t()
    for table in (big[:20, 3:67], big[::3, 8:72], big[:, ::3].t()[:20].repeat(1, 2)[:, :64], big[:1, :64].expand(20, 64)):
        compare(index, table, big[5, 10:74], dy)
    compare(index.int(), big[:20, 3:67], big[:, 4].repeat(2)[:64], dy)
    compare(indices('uniform', 154, 20)[::2], big[:20, 3:67], None, dy)
    compare(index[:72].view(2, 3, 12), big[:20, 3:67], None, dy[:72].reshape(2, 3, 12, 64))


@pytest.mark.parametrize('tokens', [100, 1000, 10000])
def test_indices_outside_the_table(tokens):
    index, table, b, dy = make(tokens, 50, 32, torch.float32)
    outside = torch.arange(tokens, device=DEV) % 3 == 0
    index[outside] = torch.tensor([-1, 50, 2 ** 40, -2 ** 50, 51], device=DEV).repeat(tokens)[:int(outside.sum())]
    t = table.requires_grad_(True)
    y = op()(index, t, b)
    assert bool(y[outside].isnan().all()) and bool(y[~outside].isfinite().all())
    got, = torch.autograd.grad(y, t, dy)
    want, = torch.autograd.grad(op()(index[~outside], t, b), t, dy[~outside].contiguous())
    torch.testing.assert_close(got, want, rtol=0, atol=tokens * U * float(dy.abs().sum(dim=0).max()))


def test_equals_the_product_with_one_hot_rows():
    """Bit for bit: what a conditional network computes from one-hot labels."""
    index, table, b, _ = make(37, 11, 64, torch.float32, columns=True)
    weight = table.t()
    onehot = torch.nn.functional.one_hot(index, 11).float()
    want = torch.addmm((b * 0.5).unsqueeze(0), onehot, (weight * 0.3).t())
    assert torch.equal(op()(index, weight.t(), b, w_gain=0.3, b_gain=0.5), want)


def test_second_order():
    index, table, b, dy = make(40, 9, 16, torch.float32)
    def penalty(f, t, bb, d):
        y = f(t, bb)
        gt, gb = torch.autograd.grad(y, (t, bb), d, create_graph=True)
        return torch.autograd.grad(gt.square().sum() + gb.square().sum(), d)[0]
    leaf = lambda v: v.clone().requires_grad_(True)
    got = penalty(lambda t, bb: op()(index, t, bb, w_gain=0.5, b_gain=2.0), leaf(table), leaf(b), leaf(dy))
    want = penalty(lambda t, bb: t[index] * 0.5 + bb * 2.0, leaf(table.double()), leaf(b.double()), leaf(dy.double()))
    assert float((got.double() - want).abs().max()) <= 1e-5 * float(want.abs().max())


@pytest.mark.parametrize('tokens', [100, 1000, 10000])
def test_graph_replays(tokens):
    index, table, b, dy = make(tokens, 300, 32, torch.float32)
    t, bb = table.clone().requires_grad_(True), b.clone().requires_grad_(True)
    step = lambda: torch.autograd.grad(op()(index, t, bb), (t, bb), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        index.copy_(indices('skewed', tokens, 300, seed))
        dy.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step()))
        torch.cuda.synchronize()


def test_refusals():
    index, table, b, _ = make(4, 8, 6, torch.float32)
    f = op()
    for args in [(index.float(), table), (index, table.double()), (index.cpu(), table), (index, table, b[:5]), (index, table, b.half()), (index, table[0]),
                 (index, table[:0])]:
        with pytest.raises(RuntimeError):
            f(*args)
