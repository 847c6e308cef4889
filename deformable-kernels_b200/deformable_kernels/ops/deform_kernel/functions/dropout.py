"""Dropout whose mask is never stored (the reference's classifiers use torch's, which keeps one):

    y = x / (1 - p) where draw >= round(p * 2^32), else 0

The draws come from a counter-based generator (Philox4x32-10) under ``(seed, offset)``; the backward makes them again.
``seed`` is an integer, or an int64 CUDA tensor ``[seed, offset]`` that the kernel reads (a captured call draws anew when
the caller advances it; the argument ``offset`` is added to its second value).  The same pair gives the same mask, whatever
the dtype: calls that leave both at their defaults, or repeat a pair, drop the SAME elements, so every layer and every step
needs a pair of its own (``modules.Dropout`` draws one from torch's generator for each call).  ``shared_dims``: the elements of
that many trailing dimensions share a draw (0: every element has its own, 2: whole planes of [N, C, H, W], 3: whole samples).
Takes float16, bfloat16, float32 and float64; dropped elements are zero whatever the input holds there.  Elements are counted
in the order of the dimensions, whatever the strides, and the result is contiguous.
"""
from ...._native import native

__all__ = ['dropout']


def dropout(input, p=0.5, seed=0, offset=0, shared_dims=0):
    return native.dropout(input, p, seed, offset, shared_dims)
