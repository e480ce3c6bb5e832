"""Rows of a table by index, scaled, plus a bias, with the table's gradient summed over equal indices:

    y[..., :] = table[index[...]] * w_gain + b * b_gain                index [...] int32 / int64, table [V, F], b [F]

The label embedding of a conditional network: what `self.embed(one_hot)` of the reference's mapping network
(DissimilarDomains/training/networks.py:765-842) computes with a product over all classes - bit for bit in float32 - given
the class numbers themselves; `table` is then the layer's weight transposed (a view: no copy is made, and its gradient comes
in the same layout).  The gradient sums the rows of dy that share an index in the order of the tokens, in float32 and without
atomics, so that the same inputs give the same bits (`sg_embedding`, `sg_embedding_backward`).  The pair of functions is
closed under differentiation: the gradient's own gradient is a lookup again.

Indices outside the table are not checked on the host (that would wait for the device): they read as rows of NaN and add to
no row of the table's gradient (the bias's sums every token).  Forward-mode tangents are refused."""
import torch

from ... import _lib


def embedding(index, table, b=None, w_gain=1.0, b_gain=1.0):
    """index [...] int32 or int64, table [V, F] in any layout, b [F] or None -> [..., F] of the table's dtype (float32, float16 or
    bfloat16); one device."""
    assert isinstance(index, torch.Tensor) and isinstance(table, torch.Tensor)
    return _lib.ext().embedding(index, table, b, w_gain, b_gain)
