"""A recording of launches that ends while a backward pass is on its way in another thread."""
import sys
import threading
import time

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.mark.parametrize('begins', [False, True])
def test_a_recording_ends_during_a_backward_pass(begins):
    """The interpreter is held here until the pass waits for it, then the recording ends (or ends and another begins)."""
    from ga_gan_amd import _lib
    from ga_gan_amd.torch_utils.ops import linear
    x, w, dy = torch.randn(8, 64, device=DEV), torch.randn(32, 64, device=DEV, requires_grad=True), torch.randn(8, 32, device=DEV)
    want, = torch.autograd.grad(linear.linear(x, w, act='tanh'), w, dy)
    got = []
    for _ in range(3):
        y = linear.linear(x, w, act='tanh')
        _lib.profile_begin()
        interval = sys.getswitchinterval()
        sys.setswitchinterval(10)
        try:
            thread = threading.Thread(target=lambda: got.append(torch.autograd.grad(y, w, dy)[0]))
            thread.start()
            until = time.perf_counter() + 0.05
            while time.perf_counter() < until:
                pass
            _lib.profile_end()
            if begins:
                _lib.profile_begin()
        finally:
            sys.setswitchinterval(interval)
        thread.join()
        if begins:
            _lib.profile_end()
    torch.cuda.synchronize()
    assert len(got) == 3 and all(torch.equal(g, want) for g in got)
