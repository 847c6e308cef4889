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
    """``nn.Dropout`` without a stored mask.  Each call in training mode draws from the next offset of the module's own
    generator state ``[seed, offset]``, which lives on the device and advances there: a captured call draws anew at every
    replay.  ``seed=None`` takes one from torch's default generator when the module is built.  ``shared_dims``: the
    elements of that many trailing dimensions are dropped together (2: whole feature planes)."""

    def __init__(self, p=0.5, shared_dims=0, seed=None):
        super().__init__()
        if not 0 <= p <= 1:
            raise ValueError('dropout probability has to be between 0 and 1, but got {}'.format(p))
        self.p = p
        self.shared_dims = shared_dims
        self.seed = int(torch.randint(0, 2 ** 62, ())) if seed is None else seed
        # not a buffer: data-parallel wrappers would make every rank's state that of rank 0
        self._state = self._step = None

    def rng_state(self):
        """[seed, offset of the next call]: what set_rng_state takes to go on from here."""
        return [self.seed, 0] if self._state is None else self._state.tolist()

    def set_rng_state(self, state):
        self.seed, offset = state
        if self._state is not None:
            self._state.copy_(torch.tensor([self.seed, offset]))
        else:
            self._start = offset

    _start = 0

    def _state_on(self, device):
        if self._state is None or self._state.device != device:
            offset = self._start if self._state is None else int(self._state[1])
            self._state = torch.tensor([self.seed, offset], device=device)
            self._step = torch.tensor([0, 1], device=device)
        return self._state

    def forward(self, input):
        if not self.training or self.p == 0:
            return input
        state = self._state_on(input.device)
        out = dropout(input, self.p, state, shared_dims=self.shared_dims)
        state.add_(self._step)
        return out

    def extra_repr(self):
        return 'p={}, shared_dims={}'.format(self.p, self.shared_dims)


class LinearCrossEntropy(nn.Linear):
    """Dropout, linear layer and softmax cross entropy: ``head(features, target)`` is the loss, ``head(features)`` the logits.

    ``features`` [..., in_features], ``target`` [...] int64.  Parameters, initialisation and state dict are those of
    ``nn.Linear(in_features, num_classes, bias)``; ``ignore_index``, ``reduction`` and ``label_smoothing`` those of
    ``nn.CrossEntropyLoss``.  Under autocast the features are taken in its dtype."""

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
        if input.is_cuda and torch.is_autocast_enabled():
            input = input.to(torch.get_autocast_dtype('cuda'))
        return linear_cross_entropy(input, self.weight, target, self.bias, self.ignore_index, self.reduction, self.label_smoothing)

    def extra_repr(self):
        return '{}, ignore_index={}, reduction={}, label_smoothing={}'.format(super().extra_repr(), self.ignore_index, self.reduction,
                                                                             self.label_smoothing)
