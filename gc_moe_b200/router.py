"""The router in front of the layer: its product (``router_logits_for_gc_moe``)
and the choice of experts (``route_for_gc_moe``).

The reference takes ``topk_idx`` and ``topk_weights`` as inputs (README.md:234-252)
and routes in its tests with a softmax over the k largest logits
(tests/test_gc_moe.py:130-168).  Inference only: the results carry no gradient.
"""

from __future__ import annotations

from operator import index
from typing import Optional, Tuple

import torch

from . import _native

_WEIGHT_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_SCORINGS = ('softmax', 'sigmoid')
_GROUP_SCORES = ('top2', 'max')


def transform_router_weight_for_gc_moe(weight: torch.Tensor) -> torch.Tensor:
    """Router weight [E, H] -> the BF16 planes [P, E, H] that
    ``router_logits_for_gc_moe`` reads; their sum is the weight.

    A BF16 weight is its own single plane (no copy when it is contiguous; it then
    has to start on 16 bytes).  The 24 significant bits of an FP32 weight are three
    planes of 8: the nearest BF16, the BF16 nearest to what is left, and the rest.
    The product takes one plane or three: a weight of BF16 values stored in FP32
    is one, FP16's 11 bits are three, the last of them zero.  Call once per
    weight, outside graph capture.
    """
    if weight.dim() != 2 or weight.dtype not in _WEIGHT_TYPES:
        raise ValueError('router weight must be 2-D bfloat16, float16 or float32')
    weight = weight.detach()
    if weight.dtype == torch.bfloat16:
        return weight.contiguous().unsqueeze(0)
    if weight.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError('transform weights outside CUDA Graph capture')
    rest = weight.float()
    planes = []
    for _ in range(3):
        planes.append(rest.to(torch.bfloat16))
        rest = rest - planes[-1].float()
    planes = torch.stack(planes)
    if not bool(torch.isfinite(planes).all()):
        raise ValueError('router weight has values that are not finite in bfloat16')
    return planes if bool((planes[1:] != 0).any()) else planes[:1].contiguous()


def check_router_weight(router_weight, hidden, device) -> None:
    if (router_weight.dim() != 3 or router_weight.dtype != torch.bfloat16 or router_weight.shape[0] not in (1, 3)
            or not 0 < router_weight.shape[1] <= 2048 or router_weight.shape[2] != hidden
            or router_weight.get_device() != device or not router_weight.is_contiguous() or router_weight.data_ptr() % 16):
        raise ValueError(f'router_weight must be contiguous, 16-byte aligned bfloat16 [1 or 3, E <= 2048, {hidden}] on '
                         'the device of x; call transform_router_weight_for_gc_moe first')


def router_logits_for_gc_moe(x: torch.Tensor, router_weight: torch.Tensor,
                             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """FP32 ``x @ W.T`` [T, E] of BF16 ``x`` [T, H] (rows may have a stride, their
    starts are 16-byte aligned, H is a multiple of 8 up to 2^30, T at most 262140)
    and the planes of ``transform_router_weight_for_gc_moe`` [P, E, H]: exact
    products, FP32 sums in an order that depends on the sizes alone.  An infinity
    in ``x`` gives what it gives times the weight itself, whatever the planes.
    ``out``: the tensor to write, contiguous; it may start anywhere in its storage.

    Runs on the current stream and can be captured.  A launch whose bounded wait
    gives up leaves NaN, which routing takes as masked: only
    ``GCSymmBuffer.raise_on_device_error`` tells it from a row without routes.
    """
    return _native.binding().router_logits(x, router_weight, out)


def check_routing(experts, topk, scoring, bias, num_groups, topk_groups, group_score, scale, device) -> None:
    """Raise for options that ``route_for_gc_moe`` would refuse, for callers that
    enqueue something before it."""
    for count in (topk, num_groups, topk_groups):
        index(count)                                     # TypeError for what is not a whole number, 2.0 among them
    if scoring not in _SCORINGS:
        raise ValueError(f'scoring must be one of {_SCORINGS}, got {scoring!r}')
    if group_score not in _GROUP_SCORES:
        raise ValueError(f'group_score must be one of {_GROUP_SCORES}, got {group_score!r}')
    if not (0 < topk <= 32 and 0 < num_groups <= 32 and 0 < topk_groups <= num_groups and 0 < experts <= 2048
            and experts % num_groups == 0 and topk <= experts // num_groups * topk_groups):
        raise ValueError(f'invalid routing: top {topk} of {experts} experts in {topk_groups} of {num_groups} groups')
    lanes = 1 << (32 // num_groups).bit_length() - 1     # of the warp, per group; 64 experts each
    if experts > 64 * lanes * num_groups:
        raise NotImplementedError(f'{num_groups} groups of {experts // num_groups} experts are too large: '
                                  f'at most {64 * lanes} each')
    if not -3.0e38 <= scale <= 3.0e38:
        raise ValueError('scale must be finite')
    if bias is not None and (bias.shape != (experts,) or bias.dtype != torch.float32 or bias.get_device() != device
                             or not bias.is_contiguous()):
        raise ValueError(f'bias must be contiguous float32 [{experts}] on the device of the logits')


def route_for_gc_moe(logits: torch.Tensor, topk: int, *, scoring: str = 'softmax',
                     bias: Optional[torch.Tensor] = None, num_groups: int = 1, topk_groups: Optional[int] = None,
                     group_score: str = 'top2', renormalize: bool = True, scale: float = 1.0,
                     out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``topk_idx`` int64 [T, k] and ``topk_weights`` FP32 [T, k] of router
    ``logits`` [T, E] (FP32, BF16 or FP16; rows may have a stride).

    * score: ``sigmoid`` of the logit, or ``softmax`` over all experts of the row;
    * choice: the k largest ``score + bias`` (``bias`` FP32 [E]), without a bias
      the k largest logits, descending, ties to the lower expert.  The order is
      that of the sums in 64 bits;
    * groups: of ``num_groups`` groups of consecutive experts the ``topk_groups``
      best are eligible; a group's value is the sum of its two largest
      ``score + bias`` (``'top2'``; of as many as it has) or the largest of what
      the choice goes by (``'max'``); ties to the lower group;
    * weight: the score without the bias, divided by the sum of the row's k if
      ``renormalize``, times ``scale``.

    An expert whose logit (or bias) is -inf or NaN is never chosen and has no part
    in the softmax: rows that pad a batch are masked that way.  Where no expert is
    left the index is -1, which the layer takes as no route, and the weight 0.  A
    logit of +inf counts as the largest finite float.

    ``out``: the two tensors to write, contiguous, such as the first T rows of
    the workspace's ``topk_idx`` and ``topk_weights``.  Runs on the current stream
    and can be captured.
    """
    if scoring not in _SCORINGS or group_score not in _GROUP_SCORES:
        raise ValueError(f'scoring must be one of {_SCORINGS} and group_score one of {_GROUP_SCORES}, got {scoring!r} and '
                         f'{group_score!r}')
    idx, weights = (None, None) if out is None else out
    return _native.binding().route(logits, topk, scoring == 'sigmoid', bias, num_groups,
                                   num_groups if topk_groups is None else topk_groups, group_score == 'max',
                                   bool(renormalize), scale, idx, weights)
