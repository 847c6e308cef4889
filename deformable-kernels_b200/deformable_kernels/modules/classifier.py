"""The head of a classification network: dropout and the last linear layer with its loss.

The reference ships no classifier; networks built from its layers end in ``nn.Dropout``, ``nn.Linear`` and
``nn.CrossEntropyLoss``.  These modules stand in their place on CUDA: ``Dropout`` keeps no mask, ``LinearCrossEntropy`` (an
``nn.Linear`` with the same parameters and state dict) goes from features and targets to the loss without storing logits.
"""
import torch
from torch import nn

from ..ops.deform_kernel.functions import dropout, linear_cross_entropy

__all__ = ['Dropout', 'LinearCrossEntropy']


class Dropout(nn.Module):
    """``nn.Dropout`` without a stored mask.  Each call in training mode draws its generator's seed and offset on the device
    from torch's default CUDA generator: ``torch.manual_seed`` repeats the masks, activation checkpointing makes the same
    one again, and a captured call draws anew at every replay.  The result has the input's memory format.  ``shared_dims``: the
    elements of that many trailing dimensions are dropped together (2: whole feature planes)."""

    def __init__(self, p=0.5, shared_dims=0):
        super().__init__()
        if not 0 <= p <= 1:
            raise ValueError('dropout probability has to be between 0 and 1, but got {}'.format(p))
        self.p = p
        self.shared_dims = shared_dims

    def forward(self, input):
        if not self.training or self.p == 0:
            return input
        state = torch.randint(0, 2 ** 63 - 1, (2,), device=input.device)
        if input.is_contiguous():
            return dropout(input, self.p, state, shared_dims=self.shared_dims)
        # dense in another order (channels last): the draws are independent, so they can follow the memory, except that the
        # elements which share one have to be neighbours there
        order = sorted(range(input.dim()), key=input.stride, reverse=True)
        back = sorted(range(input.dim()), key=order.__getitem__)
        moved = input.permute(order)
        if not moved.is_contiguous():
            return dropout(input, self.p, state, shared_dims=self.shared_dims)
        if min(order[input.dim() - self.shared_dims:], default=input.dim()) >= input.dim() - self.shared_dims:
            return dropout(moved, self.p, state, shared_dims=self.shared_dims).permute(back)
        return dropout(input, self.p, state, shared_dims=self.shared_dims).permute(order).contiguous().permute(back)

    def extra_repr(self):
        return 'p={}, shared_dims={}'.format(self.p, self.shared_dims)


class LinearCrossEntropy(nn.Linear):
    """Dropout, linear layer and softmax cross entropy: ``head(features, target)`` is the loss, ``head(features)`` the logits.

    ``features`` [..., in_features], ``target`` [...] int64.  Parameters, initialisation and state dict are those of
    ``nn.Linear(in_features, num_classes, bias)``; ``ignore_index``, ``reduction`` and ``label_smoothing`` those of
    ``nn.CrossEntropyLoss``.  Under autocast the features are taken in its dtype, but for float64, which autocast leaves alone."""

    def __init__(self, in_features, num_classes, bias=True, dropout=0.0, ignore_index=-100, reduction='mean', label_smoothing=0.0,
                 device=None, dtype=None):
        super().__init__(in_features, num_classes, bias, device=device, dtype=dtype)
        self.dropout = Dropout(dropout)
        self.ignore_index = ignore_index
        self.reduction = reduction
        self.label_smoothing = label_smoothing

    def forward(self, input, target=None):
        input = self.dropout(input)
        if target is None:
            return nn.functional.linear(input, self.weight, self.bias)
        if input.is_cuda and torch.is_autocast_enabled() and input.dtype != torch.float64:
            input = input.to(torch.get_autocast_dtype('cuda'))
        return linear_cross_entropy(input, self.weight, target, self.bias, self.ignore_index, self.reduction, self.label_smoothing)

    def extra_repr(self):
        return '{}, ignore_index={}, reduction={}, label_smoothing={}'.format(super().extra_repr(), self.ignore_index, self.reduction,
                                                                             self.label_smoothing)
