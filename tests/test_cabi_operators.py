"""CPU-side checks of the fully connected layer's, the table lookup's and the gradient norm's entry points: bad arguments are
refused by name before anything is launched (no GPU needed), and workspace queries answer."""
import ctypes

import pytest
import torch

i32, i64, f32, vp = ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p
ONE = vp(16)        # a pointer that is never followed


class LinearParams(ctypes.Structure):
    _fields_ = [('x', vp), ('w', vp), ('b', vp), ('residual', vp), ('dtype', i32), ('act', i32), ('alpha', f32), ('gain', f32), ('w_gain', f32),
                ('b_gain', f32), ('m', i64), ('n', i64), ('k', i64), ('ldx', i64), ('ldw', i64), ('ldr', i64)]


class EmbeddingParams(ctypes.Structure):
    _fields_ = [('index', vp), ('table', vp), ('bias', vp), ('dtype', i32), ('index_bytes', i32), ('tokens', i64), ('v', i64), ('f', i64),
                ('stride_v', i64), ('stride_f', i64), ('w_gain', f32), ('b_gain', f32)]


class GradList(ctypes.Structure):
    _fields_ = [('grads', vp), ('numel', vp), ('dtype', vp), ('count', i32)]


class AdamList(ctypes.Structure):
    _fields_ = [('param', vp), ('grad', vp), ('exp_avg', vp), ('exp_avg_sq', vp), ('numel', vp), ('step', vp), ('count', i32), ('lr', f32), ('beta1', f32),
                ('beta2', f32), ('eps', f32), ('grad_limit', f32), ('grad_scale', vp)]


def handle():
    from ga_gan_amd import _lib
    return _lib.lib()


def linear_params(**kw):
    return LinearParams(**{**dict(x=ONE, w=ONE, dtype=0, act=3, alpha=0.2, gain=1.0, w_gain=1.0, b_gain=1.0, m=4, n=8, k=16, ldx=16, ldw=16), **kw})


@pytest.mark.parametrize('kw, code, text', [(dict(dtype=3), -2, b'dtype'), (dict(act=0), -1, b'activation'), (dict(act=10), -1, b'activation'),
                                            (dict(m=-1), -1, b'sizes'), (dict(k=1 << 40, ldx=1 << 40, ldw=1 << 40), -1, b'sizes'), (dict(ldx=15), -1, b'strides'),
                                            (dict(ldw=3), -1, b'strides'), (dict(x=None), -3, b'NULL'), (dict(w=None), -3, b'NULL'),
                                            (dict(residual=ONE, ldr=7), -1, b'residual')])
def test_linear_refuses(kw, code, text):
    h = handle()
    p = linear_params(**kw)
    assert h.sg_linear(ctypes.byref(p), ONE, None, None, None, 0, None) == code
    assert text in h.sg_last_error()
    if 'residual' not in kw:
        assert h.sg_linear_backward(ctypes.byref(p), ONE, ONE, None, None, None, None, None, ONE, 1 << 20, None) == code


def test_linear_refuses_missing_outputs_and_workspace():
    h = handle()
    p = linear_params()
    assert h.sg_linear(None, ONE, None, None, None, 0, None) == -3
    assert h.sg_linear(ctypes.byref(p), None, None, None, None, 0, None) == -3
    big = linear_params(m=64, n=64, k=8192, ldx=8192, ldw=8192)               # one tile: cut into slices
    need = h.sg_linear_workspace_bytes(ctypes.byref(big))
    assert need > 0
    assert h.sg_linear(ctypes.byref(big), ONE, None, None, ONE, need - 1, None) == -1 and b'workspace' in h.sg_last_error()
    assert h.sg_linear(ctypes.byref(big), ONE, None, None, vp(8), need, None) == -1
    assert h.sg_linear(ctypes.byref(linear_params(m=0)), None, None, None, None, 0, None) == 0       # nothing to do, nothing launched
    long_rows = linear_params(ldx=1 << 24)
    assert h.sg_linear(ctypes.byref(long_rows), ONE, None, None, ONE, 1 << 30, None) == -2 and b'too long' in h.sg_last_error()


def test_linear_backward_wants_one_source_of_the_slope():
    h = handle()
    call = lambda p, y, z, positive: h.sg_linear_backward(ctypes.byref(p), ONE, y, z, positive, ONE, None, None, ONE, 1 << 30, None)
    assert call(linear_params(act=3), None, None, None) == -1
    assert call(linear_params(act=3), ONE, None, ONE) == -1
    assert call(linear_params(act=3), None, ONE, None) == -1 and b'y or positive' in h.sg_last_error()
    assert call(linear_params(act=4), ONE, None, None) == -1 and b'z' in h.sg_last_error()
    assert call(linear_params(act=1), ONE, None, None) == -1 and b'none' in h.sg_last_error()
    p = linear_params(act=3)
    need = h.sg_linear_backward_workspace_bytes(ctypes.byref(p))
    assert h.sg_linear_backward(ctypes.byref(p), ONE, ONE, None, None, ONE, None, None, ONE, need - 1, None) == -1 and b'workspace' in h.sg_last_error()
    assert h.sg_linear_backward(ctypes.byref(p), None, ONE, None, None, ONE, None, None, ONE, need, None) == -3


def test_embedding_refuses():
    h = handle()
    good = dict(index=ONE, table=ONE, dtype=0, index_bytes=8, tokens=300, v=10, f=8, stride_v=8, stride_f=1, w_gain=1.0, b_gain=1.0)
    for kw, code, text in [(dict(dtype=3), -2, b'dtype'), (dict(index_bytes=2), -1, b'indices'), (dict(tokens=-1), -1, b'tokens'), (dict(v=0), -1, b'table'),
                           (dict(v=1 << 40), -1, b'table'), (dict(stride_v=-8), -1, b'stride'), (dict(table=None), -3, b'NULL')]:
        p = EmbeddingParams(**{**good, **kw})
        assert h.sg_embedding(ctypes.byref(p), ONE, None) == code and text in h.sg_last_error()
        assert h.sg_embedding_backward(ctypes.byref(p), ONE, None, ONE, 1 << 30, None) == code
    p = EmbeddingParams(**good)
    assert h.sg_embedding(ctypes.byref(p), None, None) == -3
    need = h.sg_embedding_backward_workspace_bytes(ctypes.byref(p))
    assert need > 0
    assert h.sg_embedding_backward(ctypes.byref(p), ONE, None, None, 0, None) == -1 and b'workspace' in h.sg_last_error()
    strided = EmbeddingParams(**{**good, 'stride_v': 9})
    assert h.sg_embedding_backward(ctypes.byref(strided), ONE, None, ONE, 1 << 30, None) == -1 and b'dense' in h.sg_last_error()


def grad_list(pointers=(16, 32), numel=(4, 5), dtype=(0, 2)):
    keep = [(vp * len(pointers))(*pointers), (i64 * len(numel))(*numel), (i32 * len(dtype))(*dtype)]
    return GradList(*[ctypes.cast(a, vp) for a in keep], len(pointers)), keep


def test_gradient_norm_refuses():
    h = handle()
    p, keep = grad_list()
    need = h.sg_grad_norm_workspace_bytes(ctypes.byref(p))
    assert need == 2 * 8                                                       # one partial sum per small tensor
    norm = lambda q, limit=0.0, most=1.0, eps=1e-6, out=ONE, work=ONE, n=need: h.sg_grad_norm(ctypes.byref(q), limit, most, eps, out, work, n, None)
    assert norm(p, most=-1.0) == -1 and norm(p, eps=-1.0) == -1
    assert norm(p, out=None) == -3
    assert norm(p, work=None) == -1 and b'workspace' in h.sg_last_error()
    assert norm(p, n=need - 1) == -1
    for kw, code in [(dict(dtype=(0, 3)), -2), (dict(numel=(4, -1)), -1), (dict(pointers=(16, 0)), -3), (dict(pointers=(16, 33)), -1)]:
        q, keep2 = grad_list(**kw)
        assert norm(q) == code
        assert h.sg_scale_grads(ctypes.byref(q), ONE, None) == code
    assert h.sg_scale_grads(ctypes.byref(p), None, None) == -3


def test_adam_list_refuses_whole_lists():
    h = handle()
    def call(numel=(4, 4), step=(1, 1), pointers=(16, 32), **kw):
        arrays = [(vp * 2)(*pointers) for _ in range(4)] + [(i64 * 2)(*numel), (i32 * 2)(*step)]
        p = AdamList(*[ctypes.cast(a, vp) for a in arrays], 2, **{**dict(lr=1e-3, beta1=0.5, beta2=0.9, eps=1e-8, grad_limit=1e5), **kw})
        return h.sg_adam_step_list(ctypes.byref(p), None)
    assert call(step=(1, 0)) == -1 and b'step 0' in h.sg_last_error()
    assert call(numel=(4, -4)) == -1
    assert call(pointers=(16, 0)) == -3
    assert call(beta1=1.0) == -1 and call(beta2=-0.1) == -1 and call(grad_limit=0.0) == -1 and call(eps=-1.0) == -1


def test_python_entry_points_refuse_host_tensors():
    from ga_gan_amd import optim_plugin
    from ga_gan_amd.torch_utils.ops import embedding, linear
    with pytest.raises(RuntimeError, match='GPU'):
        linear.linear(torch.zeros(2, 3), torch.zeros(4, 3))
    with pytest.raises(RuntimeError, match='GPU'):
        embedding.embedding(torch.zeros(2, dtype=torch.int64), torch.zeros(4, 3))
    with pytest.raises(RuntimeError, match='CUDA'):
        optim_plugin.grad_norm([torch.zeros(3)])
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    with pytest.raises(RuntimeError, match='CUDA'):
        optim_plugin.clip_grad_norm_(p, 1.0)
    with pytest.raises(RuntimeError, match='CUDA'):
        optim_plugin.FusedAdam([p], max_grad_norm=1.0).step()
    with pytest.raises(RuntimeError, match='negative'):
        optim_plugin.FusedAdam([p], max_grad_norm=-1.0)
    assert float(optim_plugin.grad_norm([])) == 0


def test_copies_of_the_optimizer_clip_as_it_does():
    """Copies and pickles keep max_grad_norm; a state from before it existed steps unclipped."""
    import copy
    import pickle
    from ga_gan_amd import optim_plugin
    opt = optim_plugin.FusedAdam([torch.nn.Parameter(torch.zeros(3))], max_grad_norm=0.5)
    for twin in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert twin.max_grad_norm == 0.5 and twin.last_grad_norm is None
    old = opt.__getstate__()
    del old['max_grad_norm']
    twin = optim_plugin.FusedAdam.__new__(optim_plugin.FusedAdam)
    twin.__setstate__(old)
    assert twin.max_grad_norm is None


def test_a_step_that_is_refused_counts_for_nothing():
    from ga_gan_amd import optim_plugin
    p, q = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(2))
    opt = optim_plugin.FusedAdam([dict(params=[p]), dict(params=[q], grad_limit=7.0)], max_grad_norm=1.0)
    p.grad, q.grad = torch.ones(3), torch.ones(2)
    with pytest.raises(RuntimeError, match='grad_limit'):
        opt.step()
    assert not opt.state[p] and not opt.state[q]
    opt = optim_plugin.FusedAdam([p])
    opt.max_grad_norm = -1.0
    with pytest.raises(RuntimeError, match='negative'):
        opt.step()
    assert not opt.state[p]
