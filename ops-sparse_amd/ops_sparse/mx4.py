"""Microscaled 4-bit floating point on torch tensors: rows laid out in it, and the experts' products of such rows.

A row is blocks of 32 values that share a power of two (the format of OCP's Microscaling specification with elements
e2m1).  A layer of experts whose weights were laid out once is served by::

    hidden = grouped_mm_mx4(mx4_quantize(x), w_in, plan, gather=True)
    y = combine(grouped_mm_mx4(mx4_quantize(act(hidden)), w_out, plan), plan, weights)

at a quarter of the 16-bit weights' bytes.  Everything runs on the current torch stream; nothing waits for the device
and there is no CPU path.  The products are for serving: they have no gradient.  Arguments that do not fit raise
ValueError, types that are not supported TypeError.  The reference has no counterpart.
"""
from typing import NamedTuple

import torch

from . import experts
from .experts import _module


class MX4(NamedTuple):
    """Rows in microscaled 4 bits, B blocks of 32 values each (uint8 tensors on the device).

    codes [..., 16 * B]: a value's sign and three bits, which stand for 0, 0.5, 1, 1.5, 2, 3, 4 and 6, two to a byte with
    the first in the low half; zero past the row's last value.  scales [..., B]: e stands for 2^(e - 127), 255 for NaN.
    Parts of the rows, and of the blocks, are parts of both tensors.
    """
    codes: torch.Tensor
    scales: torch.Tensor


def mx4_quantize(x):
    """x [..., K] (fp32, fp16 or bf16) as :class:`MX4`, ceil(K / 32) blocks a row.

    A block's scale has the exponent of its largest value less 2; each value over it is rounded to the nearest of the
    format, ties to the even code, and at most 6 (up to 8 the largest may be over its scale).  A block that holds
    infinity or NaN becomes NaN.  The result has no gradient.
    """
    return MX4(*(experts._MODULE or _module()).mx4_quantize(x))


def mx4_dequantize(q, width=None, dtype=torch.float32):
    """The values [..., width] of :class:`MX4` rows in fp32, fp16 or bf16; width: of the rows' last block, all of it
    unless it is given."""
    return (experts._MODULE or _module()).mx4_dequantize(q.codes, q.scales, width, dtype)


def grouped_mm_mx4(a, w, plan=None, gather=False, out_dtype=torch.bfloat16):
    """:func:`ops_sparse.grouped_mm` of :class:`MX4` rows: y[r] = w[e] @ a[r] for the rows r of each expert e, rows of no
    expert zero; w [E, N, K], a [R, K] in the plan's row order or, with ``gather``, [T, K] in token order.  With no plan
    one dense product, w [N, K].  Both have the same number of blocks; sums are in fp32, rounded once to out_dtype
    (fp32, fp16 or bf16).  Codes whose rows are not aligned to 16 bytes are copied.  No gradient.
    """
    offsets, tokens, places = plan if plan is not None else (None, None, None)
    return (experts._MODULE or _module()).grouped_mm_mx4(a.codes, a.scales, w.codes, w.scales, offsets, tokens, places,
                                                         gather, out_dtype)
