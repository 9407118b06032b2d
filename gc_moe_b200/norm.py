"""``rms_norm_for_gc_moe``: residual addition, RMS norm and the layer's 8-bit
input format in one kernel.

The reference's operator starts from rows that are already normed and quantised
(README.md:234-252); this is the step in front of it.  Inference only: the
results carry no gradient.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from . import _native
from .heuristics import get_block_m_for_gc_moe


class NormedInputs(NamedTuple):
    """Results of ``rms_norm_for_gc_moe``."""
    x: torch.Tensor                      # e4m3 [T, H]
    x_sf: torch.Tensor                   # int32 [T, ceil(H / 128)], four scale bytes per word
    normed: Optional[torch.Tensor]       # bf16 [T, H], or None
    residual: Optional[torch.Tensor]     # x + residual, type of the residual; None without one


_result = NormedInputs._make


def rms_norm_for_gc_moe(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                        eps: float = 1e-6, *, normed: Union[bool, torch.Tensor] = True,
                        residual_out: Optional[torch.Tensor] = None, sym_buffer=None) -> NormedInputs:
    """``h = x + residual``; ``v = h / sqrt(mean(h * h) + eps) * weight``, all in
    FP32, from BF16 ``x`` [T, H], ``residual`` [T, H] and ``weight`` [H] (BF16 or
    FP32 each; H a multiple of 32 up to 32768; the weight 16-byte aligned).

    Returns ``v`` as e4m3 rows with one UE8M0 scale ``2^ceil(log2(amax / 448))``
    per 32 channels (the layer's input format; rows and words of the workspace
    when ``sym_buffer`` is given, the rows of ``shared_l1_acts_sf`` included,
    else new tensors), ``v`` in BF16 when ``normed`` is true (or the tensor to
    write it to), and ``h`` in the type of ``residual``: in ``residual_out``,
    which may be ``residual`` itself, or a new tensor.  Rows may have a stride;
    their starts are 16-byte aligned.  Apart from ``residual_out`` being
    ``residual``, outputs overlap no input.  The squares are summed in FP32: rows
    whose sum overflows it (entries beyond 1e17) do not come out as the formula says.
    A row's result does not depend on the other rows or their number.

    Runs on the current stream and can be captured.
    """
    if sym_buffer is None:
        return _result(_native.binding().rms_norm(x, weight, residual, eps, normed, residual_out, None, None, None, 0))
    if sym_buffer.buffer is None:
        raise ValueError('symmetric buffer has been destroyed')
    if x.dim() != 2 or x.shape[1] != sym_buffer.x.shape[1]:
        raise ValueError(f'x is {list(x.shape)}, the workspace has hidden {sym_buffer.x.shape[1]}')
    tokens = x.shape[0]
    if tokens > sym_buffer.num_max_tokens_per_rank:
        raise ValueError(f'{tokens} tokens exceed the workspace capacity {sym_buffer.num_max_tokens_per_rank}')
    shared_sf, block_m = getattr(sym_buffer, 'shared_l1_acts_sf', None), 0
    if shared_sf is not None:
        block_m = get_block_m_for_gc_moe(sym_buffer.group.size(), sym_buffer.num_experts,
                                         sym_buffer.num_max_tokens_per_rank, tokens, sym_buffer.num_topk)
    return _result(_native.binding().rms_norm(x, weight, residual, eps, normed, residual_out, sym_buffer.x[:tokens],
                                              sym_buffer.x_sf[:tokens], shared_sf, block_m))
