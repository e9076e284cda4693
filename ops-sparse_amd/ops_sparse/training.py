"""What a model is trained with, on torch tensors: the log probabilities of given tokens and the AdamW step.

One step is::

    r = token_logprobs(logits, targets, entropy=True)      # [T], differentiable
    loss = -(r.logprobs.sum() + 0.01 * r.entropy.sum()) / count
    grads = torch.autograd.grad(loss, params)
    adamw_step(params, grads, state, lr=3e-4)              # state = adamw_state(params, bits=8)

and an answer's tokens are reported with ``token_logprobs(logits, tokens, top=20)``.  Everything runs on the current
torch stream through the C entry points of libaclsparse_hip.so; nothing waits for the device, so a step can be captured
in a HIP graph.  There is no CPU path.  Arguments that do not fit raise ValueError, types that are not supported
TypeError.  The reference has no counterpart.
"""
from typing import List, NamedTuple, Optional, Tuple

import torch

from . import experts
from .experts import _module


class TokenLogprobs(NamedTuple):
    """logprobs [...]; entropy [...], top_logprobs and top_ids [..., top], None where not asked for."""
    logprobs: torch.Tensor
    entropy: Optional[torch.Tensor] = None
    top_logprobs: Optional[torch.Tensor] = None
    top_ids: Optional[torch.Tensor] = None


def token_logprobs(logits, targets, top=0, entropy=False):
    """:class:`TokenLogprobs` of rows of logits [..., V] (fp32, fp16 or bf16) at targets [...] (int32 or int64).

    logprobs: log softmax at the target, 0 (and no gradient) for a target outside [0, V), as padding has; entropy: of
    each row's distribution; with ``top`` (up to 64) the largest logits' ids in int32, largest first, ties to the lowest
    id, never -inf (such a place has id -1), and their log probabilities.  Results are fp32, statistics too.  The log
    probabilities, the entropy and the alternatives' log probabilities are differentiable (once) with respect to the
    logits.  Logits of -inf have probability 0; a row of nothing else has log probabilities of -inf, entropy 0 and the
    gradient 0.  A NaN in a row makes its results NaN and counts as its largest.
    """
    return TokenLogprobs(*(experts._MODULE or _module()).token_logprobs(logits, targets, top, entropy))


class AdamWState(NamedTuple):
    """What AdamW keeps of a list of tensors, one entry of each list per tensor of n values.

    moments: [2, P] with P = n rounded up to 32, the first moment and the second one, fp32 or uint8 codes; exponents:
    [2, P / 32] uint8 for the codes, None for fp32; masters: the values in fp32, None where the parameters themselves
    are kept; step: int32 [1] or longer, the steps taken in its first place, others are not used; seed: of the rounding of
    8-bit moments (32 bits); factors: two odd numbers of 32 bits that the rounding's random numbers are made with, where
    8-bit moments are to be another program's bit by bit (include/cann_ops_sparse.h says how), None for the library's own.
    """
    moments: List[torch.Tensor]
    exponents: Optional[List[torch.Tensor]]
    masters: Optional[List[torch.Tensor]]
    step: torch.Tensor
    seed: int = 0
    factors: Optional[Tuple[int, int]] = None


def adamw_state(params, bits=32, masters=True, seed=0):
    """The state before the first step.  bits: 32, or 8 for moments in 8-bit floating point whose blocks of 32 values
    share a power of two, rounded at random so that slow changes add up; masters: keep values in fp32 where any of the
    parameters is of 16 bits (without them a change under half a step of the parameter's type is lost)."""
    params = list(params)
    if bits not in (8, 32):
        raise ValueError(f"bits must be 8 or 32, got {bits}")
    if not params:
        raise ValueError("there must be a parameter")
    device = params[0].device
    padded = [(p.numel() + 31) // 32 * 32 for p in params]
    moments = [torch.zeros(2, n, dtype=torch.float32 if bits == 32 else torch.uint8, device=device) for n in padded]
    exponents = [torch.zeros(2, n // 32, dtype=torch.uint8, device=device) for n in padded] if bits == 8 else None
    with torch.no_grad():
        kept = [p.float().clone() if p.dtype == torch.float32 else p.float() for p in params] if (
            masters and any(p.dtype != torch.float32 for p in params)) else None
    return AdamWState(moments, exponents, kept, torch.zeros(2, dtype=torch.int32, device=device), int(seed))


def adamw_step(params, grads, state, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, grad_scale=None):
    """One step over all tensors, in place: m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2, p = p (1 - lr weight_decay)
    - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps).

    params: contiguous, fp32, fp16 or bf16; grads: of their shapes and any of these types, None for a tensor that is left
    as it is; lr: a number, or a tensor of one fp32 on the device; grad_scale: a tensor of one fp32 on the device that all
    gradients are multiplied by (clipping by a norm).  The steps are counted on the device, so that a captured step counts
    with each replay.  With masters in the state the step goes by them and the parameters get them rounded.  Tensors that
    a step writes share no memory (but a parameter in fp32 may be its own master).
    """
    tensor = lr if isinstance(lr, torch.Tensor) else None
    (experts._MODULE or _module()).adamw_step(list(params), list(grads), state.moments, state.exponents, state.masters,
                                              state.step, state.seed, 0.0 if tensor is not None else lr, tensor,
                                              betas[0], betas[1], eps, weight_decay, grad_scale, state.factors)


def adamw_moments(state):
    """The moments' values in fp32, [2, P] for each tensor (the state's own for 32 bits; zero past a tensor's end)."""
    if state.exponents is None:
        return state.moments
    return (experts._MODULE or _module()).adamw_moments(state.moments, state.exponents)
