"""The last linear layer of a classifier with its softmax cross entropy, without keeping the logits:

    z = input @ weight.T + bias
    loss = logsumexp(z) - (1 - label_smoothing) * z[target] - label_smoothing * mean(z)

as ``torch.nn.functional.cross_entropy(linear(input, weight, bias), target, ...)`` defines it, ``input`` [..., features],
``weight`` [classes, features], ``target`` [...] int64.  The backward computes the logits again, a piece of the vocabulary at a
time; neither they nor their gradient ever exist as a whole.  The loss is float32 (float64 for float64 inputs).  Weights and biases
that differ in dtype from the features follow them.

Logits, sums and statistics are fp32 for 16-bit and fp32 inputs (fp64 for fp64); for 16-bit inputs the gradient of the logits is rounded
to 16 bits between the products, as it would be as a tensor of its own.  The same call gives the same bits.

Rows whose target is ``ignore_index`` have no loss and no gradient whatever their features hold.  A target that is no class makes the loss
NaN.  Features or weights that are not finite make the losses of the rows they reach NaN; a bias of -inf takes a class out.
"""
from ...._native import native

__all__ = ['linear_cross_entropy']


def linear_cross_entropy(input, weight, target, bias=None, ignore_index=-100, reduction='mean', label_smoothing=0.0):
    return native.linear_cross_entropy(input, weight, target, bias, ignore_index, reduction, label_smoothing)
