"""The large tiles of the fully connected layer's 16-bit products: which sizes reach them (asked of the rule itself, so that a rule that
moves says so here), and their results against 64 bits within the bounds of tests/linear_bounds.py."""
import ctypes
import re

import pytest
import torch

from linear_bounds import bounds, check
from test_cabi_operators import handle, linear_params

DTYPES = [torch.float16, torch.bfloat16]
CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
STEP = 64                                    # 16-bit elements along the sum

# m, k, n, and for one of the three products (0: y, 1: dx, 2: dw) the tile, whether it is cut into slices, and whether an operand's rows
# are copied into whole packets: at least six whole steps in every slice, and a last step that is cut
CASES = [(337, 408, 5616, 0, 128, False, False), (275, 399, 6536, 0, 128, False, True), (654, 5152, 480, 0, 128, True, False),
         (278, 5146, 1134, 0, 128, True, True), (5778, 1048, 2072, 0, 256, False, False), (1170, 1034, 9762, 0, 256, False, True),
         (1362, 4568, 2976, 0, 256, True, False), (387, 5635, 8500, 0, 256, True, True), (7094, 280, 392, 1, 128, False, False),
         (258, 6552, 406, 1, 128, False, True), (1091, 272, 4496, 1, 128, True, False), (515, 581, 5012, 1, 128, True, True),
         (7114, 1696, 1056, 1, 256, False, False), (1673, 7081, 1044, 1, 256, False, True), (399, 9512, 4392, 1, 256, True, False),
         (8817, 389, 4892, 1, 256, True, True), (387, 6672, 288, 2, 128, False, False), (390, 5832, 325, 2, 128, False, True),
         (5159, 392, 776, 2, 128, True, False), (5129, 1093, 269, 2, 128, True, True), (780, 3720, 3240, 2, 256, False, False),
         (776, 1182, 9850, 2, 256, False, True), (3911, 4960, 840, 2, 256, True, False), (4278, 8210, 389, 2, 256, True, True)]


def kernel(m, k, n, product, dtype, **kw):
    p = linear_params(m=m, k=k, n=n, ldx=k, ldw=k, dtype=CODES[dtype], **kw)
    return handle().sg_linear_kernel(ctypes.byref(p), product).decode()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('m, k, n, product, tile, sliced, padded', CASES)
def test_sizes_reach_their_tiles(m, k, n, product, tile, sliced, padded, dtype):
    found = re.fullmatch(r'linear_gemm_kernel<(\d+), direct> (\d+) x (\d+)', kernel(m, k, n, product, dtype))
    assert found and int(found[1]) == tile and (int(found[2]) > 1) == sliced, found
    length = (k, n, m)[product]
    last = length - (int(found[2]) - 1) * int(found[3]) * STEP          # of the last slice
    assert length % STEP != 0 and last >= 6 * STEP
    assert ((k if product == 0 else n) % 8 != 0 or k % 8 != 0) == padded
    rows, cols = ((m, n), (m, k), (n, k))[product]
    assert rows % tile != 0 or cols % tile != 0                          # edge tiles


def test_small_products_and_refusals():
    assert kernel(1, 512, 512, 0, torch.float32) == 'linear_thin_kernel'
    assert kernel(10000, 512, 512, 0, torch.float32).startswith('linear_gemm_kernel<64, direct> 1 x ')
    assert kernel(70, 3, 70, 0, torch.bfloat16).startswith('linear_gemm_kernel<64, short>')
    assert kernel(70, 33, 70, 0, torch.bfloat16).startswith('linear_gemm_kernel<64, loose>')
    for kw in (dict(act=0), dict(m=-1)):
        p = linear_params(**kw)
        assert handle().sg_linear_kernel(ctypes.byref(p), 0) == b''
    assert handle().sg_linear_kernel(ctypes.byref(linear_params()), 3) == b'' and handle().sg_linear_kernel(None, 0) == b''


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('m, k, n, product, tile, sliced, padded', CASES)
def test_results(m, k, n, product, tile, sliced, padded, dtype):
    """All three products, with bias and residual; twice for the same bits."""
    from ga_gan_amd.torch_utils.ops import linear
    g = torch.Generator(device='cuda').manual_seed(m)
    r = lambda *s: torch.randn(s, device='cuda', generator=g)
    x, w, b, res, dy = (t.to(dtype) for t in (r(m, k), r(n, k) / k ** 0.5, r(n), r(m, n), r(m, n)))
    leaves = [t.requires_grad_(True) for t in (x, w, b, res)]
    y = linear.linear(x, w, b, residual=res, act='lrelu')
    grads = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    want = bounds(x, w, b, res, 'lrelu', dy)
    for name, v in zip(('y', 'dx', 'dw', 'db'), (y, *grads)):
        check(v, want[name], name)
    assert torch.equal(linear.linear(x, w, b, residual=res, act='lrelu'), y)
    assert all(torch.equal(p, q) for p, q in zip(grads, torch.autograd.grad(y, leaves, dy)))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('act', ['swish', 'linear'])
@pytest.mark.parametrize('m, k, n', [(1170, 1034, 9762), (4278, 8210, 389), (5778, 1048, 2072)])
def test_other_epilogues(m, k, n, act, dtype):
    """Pre-activation values kept for the backward pass; no activation, where dy itself is an operand; no bias, no residual."""
    from ga_gan_amd.torch_utils.ops import linear
    g = torch.Generator(device='cuda').manual_seed(m)
    r = lambda *s: torch.randn(s, device='cuda', generator=g)
    x, w, dy = (t.to(dtype) for t in (r(m, k), r(n, k) / k ** 0.5, r(m, n)))
    leaves = [t.requires_grad_(True) for t in (x, w)]
    y = linear.linear(x, w, act=act)
    want = bounds(x, w, None, None, act, dy)
    for name, v in zip(('y', 'dx', 'dw'), (y, *torch.autograd.grad(y, leaves, dy))):
        check(v, want[name], name)
