"""Fully connected layer as one operator, with its gradients:

    y = act(x @ (w * w_gain).T + b * b_gain) * gain + residual          x [..., K], w [N, K], b [N], residual [..., N]

`FullyConnectedLayer.forward` of the reference (DissimilarDomains/training/networks.py:691-704: a product with the scaled
weight, then `bias_act`) in one kernel that applies the whole epilogue to the accumulators (`sg_linear`); the backward pass
is the activation's gradient with the bias's column sums in one pass and a product each for x and w (`sg_linear_backward`).
float32, float16 and bfloat16 with float32 sums and one rounding per output; activations, their default slopes and gains are
those of `bias_act`.

What the backward pass keeps besides x and w: nothing for 'linear'; for 'relu' and 'lrelu' the output itself, whose sign
is the pre-activation's, or - where a residual or float16's short range hides it - a byte per element; for the others the
pre-activation values in float32 (rounded to 16 bits they would cost the gradient more accuracy than rounding the gradient itself
does).  A backward pass that is asked for a graph of its own (create_graph=True) differentiates the same expression written with the
framework's operators, in float32 with one rounding per gradient, and with the slopes of the forward pass for 'relu' and 'lrelu'.

At a pre-activation of exactly zero the slope is that of the negative side, as in `bias_act`."""
import torch

from ... import _lib
from . import bias_act


def linear(x, w, b=None, residual=None, act='linear', alpha=None, gain=None, w_gain=1.0, b_gain=1.0):
    """x [..., K], w [N, K], b [N] or None, residual [..., N] (the output's shape) or None -> [..., N]; one dtype (float32,
    float16 or bfloat16) and one device.  Rows of x, w and residual may lie any distance apart; tensors whose last dimension
    is not contiguous, or whose rows are 2^23 bytes or more apart, are copied first, and rows of that length are refused (the
    output's by the backward pass).  `alpha` and `gain` default to the activation's.  Forward-mode tangents are refused."""
    assert isinstance(x, torch.Tensor) and isinstance(w, torch.Tensor)
    spec = bias_act.activation_funcs[act]
    return _lib.ext().linear(x, w, b, residual, spec.cuda_idx, spec.def_alpha if alpha is None else alpha, spec.def_gain if gain is None else gain,
                             w_gain, b_gain)
