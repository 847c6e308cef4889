"""The last linear layer of a classifier with its softmax cross entropy, without keeping the logits:

    z = input @ weight.T + bias
    loss = logsumexp(z) - (1 - label_smoothing) * z[target] - label_smoothing * mean(z)

as ``torch.nn.functional.cross_entropy(linear(input, weight, bias), target, ...)`` defines it, ``input`` [..., features],
``weight`` [classes, features], ``target`` [...] int64.  The logits are never stored: the backward computes them again, and their
gradient exists for one piece of the call, of up to 256 MB or 256 rows or classes, cut along the longer of rows and classes (the whole
call, where it is no larger).  The loss is float32 (float64 for float64 inputs).  Weights and biases that differ in dtype from the features
follow them.  There is no second derivative: what is made of gradients taken with ``create_graph=True`` cannot be differentiated.

Logits, statistics and losses are fp32 for 16-bit and fp32 inputs (fp64 for fp64).  For 16-bit inputs the gradient of the logits is rounded
to 16 bits for the two products, as it would be as a tensor of its own; the bias gradient is the sum of unrounded values.  Sums are those
of the tensor cores, whose additions cut where others round; no more than 256 cuts meet in a 16-bit logit, 4096 in a
16-bit gradient and 16 in anything of fp32 before the sum goes on in ordinary fp32.  The same call gives the same bits.

Rows whose target is ``ignore_index`` have no loss and no gradient whatever their features hold.  A target that is no class makes the loss
NaN.  Features that are not finite make the loss of their row NaN.  So do weights that are not finite, except where the logit is -inf:
that takes the class out of the row, as a bias of -inf does (fp32: or makes its loss NaN).
"""
from ...._native import native

__all__ = ['linear_cross_entropy']


def linear_cross_entropy(input, weight, target, bias=None, ignore_index=-100, reduction='mean', label_smoothing=0.0):
    return native.linear_cross_entropy(input, weight, target, bias, ignore_index, reduction, label_smoothing)
