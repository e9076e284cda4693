"""The experts' operators on torch tensors: routing, ragged products grouped by expert, their combination.

T tokens each choose k of E experts.  The choice is a CSR matrix of k entries per row; :class:`ExpertPlan` is its
pattern by columns, which the products read.  One layer is::

    weights, ids, plan = route(x @ gate.T, k)               # the router
    h = grouped_mm(x, w_in, plan, gather=True)              # row r: w_in[e] @ x[token of r], e the expert of row r
    y = combine(grouped_mm(act(h), w_out, plan), plan, weights)

``weights``, the products and the combination are differentiable (once).  Everything runs on the current torch stream
through the C entry points of libaclsparse_hip.so; nothing waits for the device.  There is no CPU path.  Arguments
that do not fit raise ValueError, types that are not supported TypeError.  The reference has no counterpart.

The checks, outputs and autograd nodes are C++ (csrc/experts_torch.cpp): in Python they took longer than the kernels
of a small layer.
"""
import importlib.util
import os
from typing import NamedTuple, Optional

import torch

from . import _lib

MODULE_PATH = os.path.join(_lib.LIB_DIR, "_ops_sparse_experts.so")


class ExpertPlan(NamedTuple):
    """The assignments of tokens to experts, sorted by expert (int32 tensors on the device).

    offsets [E + 1]: rows offsets[e] to offsets[e + 1] are expert e's; tokens [T * k]: the token of each row (-1
    past offsets[E]); places [T, k]: the row of each assignment, -1 for a dropped one.  ``tokens`` and ``places``
    may be None where rows are grouped by other means: such a plan serves products that do not gather.  Some of the
    experts, a part of ``offsets`` with the ``w`` of those, have the others' rows as rows of no expert.  The gradient
    of a gathered operand goes by places: an assignment whose place is set to -1 afterwards has no part in it.
    """
    offsets: torch.Tensor
    tokens: Optional[torch.Tensor] = None
    places: Optional[torch.Tensor] = None


_MODULE = None


def _module():
    """The C++ module, loaded once; raises if it is missing or was built from other sources."""
    global _MODULE
    if _MODULE is None:
        _lib.lib()  # raises if the library that the module calls is missing or stale
        if not os.path.exists(MODULE_PATH):
            raise RuntimeError(f"{MODULE_PATH} is missing: build it with "
                               "`python -c 'import __graft_entry__ as g; g.build()'` (there is no CPU fallback)")
        spec = importlib.util.spec_from_file_location("_ops_sparse_experts", MODULE_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        from .build import CSRC, source_hash

        if os.path.isdir(CSRC) and "ACLSPARSE_HIP_LIB" not in os.environ and module.build_id != source_hash():
            raise RuntimeError(f"{MODULE_PATH} is stale: rebuild it with "
                               "`python -c 'import __graft_entry__ as g; g.build()'`")
        module.bind(_lib.LIB_PATH)
        _MODULE = module
    return _MODULE


def route(logits, k, normalize=True):
    """(weights, ids, plan) of router logits [T, E] (fp32, fp16 or bf16; E <= 1024, k <= 64): the k largest of each
    row, ties to the lowest index, never -inf (such a choice has id -1, weight 0 and place -1; NaN counts as the
    largest).

    weights [T, k] fp32 (differentiable): exp(l_j - max) / sum, the sum over the chosen or, with ``normalize`` false,
    over the row; ids [T, k] int32, largest first; plan: the assignments sorted by expert.
    """
    weights, ids, offsets, tokens, places = (_MODULE or _module()).route(logits, k, normalize)
    return weights, ids, ExpertPlan(offsets, tokens, places)


def expert_plan(ids, experts):
    """The plan of a given choice: ids [T, k] int32, those outside [0, experts) dropped."""
    return ExpertPlan(*(_MODULE or _module()).expert_plan(ids, experts))


def grouped_mm(a, w, plan, gather=False):
    """y [R, N]: y[r] = w[e] @ a[r] for the rows r of each expert e, rows of no expert zero (differentiable).

    w [E, N, K], fp16 or bf16 (any strides whose last is 1 avoid a copy); a of its type: [R, K] in the plan's row
    order or, with ``gather``, [T, K] in token order: row r then reads a[plan.tokens[r]].  An a of fewer rows than the
    plan's tokens (with ``gather``, places) is refused, more are no expert's; a plan of offsets alone takes any R.
    Sums are in fp32.
    """
    return (_MODULE or _module()).grouped_mm(a, w, plan.offsets, plan.tokens, plan.places, gather)


def grouped_mm_scaled(a, a_scale, w, w_scale, plan=None, gather=False, out_dtype=torch.bfloat16):
    """:func:`grouped_mm` of 8-bit integers: y[r, n] = a_scale[i] * w_scale[e, n] * (the exact integer product), i the
    row of a that row r reads.  a int8, a_scale [rows of a] fp32, w [E, N, K] int8, w_scale [E, N] fp32; with no plan
    one dense product, w [N, K] and w_scale [N].  K <= 131071, so that the sum stays within 32 bits.  No gradient:
    one asked for through the scales raises RuntimeError.
    """
    offsets, tokens, places = plan if plan is not None else (None, None, None)
    return (_MODULE or _module()).grouped_mm_scaled(a, a_scale, w, w_scale, offsets, tokens, places, gather, out_dtype)


def combine(y, plan, weights=None):
    """out [T, H]: out[t] = sum over j of weights[t, j] * y[plan.places[t, j]], summed in fp32 (differentiable).

    y [R, H] fp16 or bf16 in the plan's row order; weights [T, k] fp32, None for ones.  Dropped assignments (places
    outside [0, R)) add nothing.  Any places will do, -1 set afterwards among them: the gradient of a row of y that no
    place names is zero, that of one that several name the sum of their parts.
    """
    return (_MODULE or _module()).combine(y, plan.offsets, plan.places, weights)
