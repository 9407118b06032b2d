"""``rms_norm_for_gc_moe``: residual addition, RMS norm and the layer's 8-bit
input format in one kernel.

The reference's operator starts from rows that are already normed and quantised
(README.md:234-252); this is the step in front of it.  Inference only: the
results carry no gradient.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Union

import torch

from . import _native
from .heuristics import get_block_m_for_gc_moe

_BF16 = (torch.bfloat16,)
_FLOATS = (torch.bfloat16, torch.float32)


class NormedInputs(NamedTuple):
    """Results of ``rms_norm_for_gc_moe``."""
    x: torch.Tensor                      # e4m3 [T, H]
    x_sf: torch.Tensor                   # int32 [T, ceil(H / 128)], four scale bytes per word
    normed: Optional[torch.Tensor]       # bf16 [T, H], or None
    residual: Optional[torch.Tensor]     # x + residual, type of the residual; None without one


def _check_rows(t, name: str, shape, dtypes, device: int) -> int:
    """Elements between the rows of ``t``; raise if it is not such rows."""
    tokens, hidden = shape
    if t.dtype not in dtypes or t.shape != shape or t.get_device() != device:
        raise ValueError(f'{name} must be {" or ".join(str(d)[6:] for d in dtypes)} {list(shape)} on the device of x')
    stride, one = t.stride()
    if one != 1:
        raise ValueError(f'{name} must be contiguous in its last dimension')
    return stride if tokens > 1 else hidden          # a single row has no stride of its own


def _rows_like(t: torch.Tensor, stride: int) -> torch.Tensor:
    """New contiguous tensor of the shape and type of ``t``, whose rows are ``stride`` apart."""
    return torch.empty_like(t) if stride == t.shape[1] else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def rms_norm_for_gc_moe(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                        eps: float = 1e-6, *, normed: Union[bool, torch.Tensor] = True,
                        residual_out: Optional[torch.Tensor] = None, sym_buffer=None) -> NormedInputs:
    """``h = x + residual``; ``v = h / sqrt(mean(h * h) + eps) * weight``, all in
    FP32, from BF16 ``x`` [T, H], ``residual`` [T, H] and ``weight`` [H] (BF16 or
    FP32 each; H a multiple of 32).

    Returns ``v`` as e4m3 rows with one UE8M0 scale ``2^ceil(log2(amax / 448))``
    per 32 channels (the layer's input format; rows and words of the workspace
    when ``sym_buffer`` is given, the rows of ``shared_l1_acts_sf`` included,
    else new tensors), ``v`` in BF16 when ``normed`` is true (or the tensor to
    write it to), and ``h`` in the type of ``residual``: in ``residual_out``,
    which may be ``residual`` itself, or a new tensor.  Rows may have a stride;
    their starts are 16-byte aligned.  Apart from ``residual_out`` being
    ``residual``, outputs overlap no input.

    Runs on the current stream and can be captured.
    """
    if x.dim() != 2 or not x.is_cuda:
        raise ValueError('x must be a 2-D CUDA bfloat16 tensor, contiguous in its last dimension')
    tokens, hidden = shape = x.shape
    device = x.get_device()
    x_stride = _check_rows(x, 'x', shape, _BF16, device)
    if hidden == 0 or hidden % 32:
        raise ValueError(f'hidden {hidden} must be a positive multiple of 32')
    if (weight.dtype not in _FLOATS or weight.shape != (hidden,) or weight.get_device() != device
            or not weight.is_contiguous()):
        raise ValueError(f'weight must be contiguous bfloat16 or float32 [{hidden}] on the device of x')
    residual_ptr = residual_stride = residual_out_ptr = residual_out_stride = residual_f32 = 0
    if residual is not None:
        residual_stride = residual_out_stride = _check_rows(residual, 'residual', shape, _FLOATS, device)
        if residual_out is None:
            residual_out, residual_out_stride = _rows_like(residual, residual_stride), hidden
        elif residual_out is not residual:
            residual_out_stride = _check_rows(residual_out, 'residual_out', shape, (residual.dtype,), device)
        residual_ptr, residual_out_ptr = residual.data_ptr(), residual_out.data_ptr()
        residual_f32 = int(residual.dtype is torch.float32)
    elif residual_out is not None:
        raise ValueError('residual_out needs a residual')
    normed_ptr, normed_stride = 0, hidden
    if normed is True:
        normed = _rows_like(x, x_stride)
        normed_ptr = normed.data_ptr()
    elif normed is False or normed is None:
        normed = None
    else:
        normed_stride = _check_rows(normed, 'normed', shape, _BF16, device)
        normed_ptr = normed.data_ptr()
    shared_sf, shared_rows, block_m = None, 0, 0
    if sym_buffer is None:
        words = (hidden + 127) // 128
        x_q = torch.empty_strided(shape, (hidden, 1), dtype=torch.float8_e4m3fn, device=x.device)
        x_sf = torch.empty_strided((tokens, words), (words, 1), dtype=torch.int32, device=x.device)
    else:
        if sym_buffer.buffer is None:
            raise ValueError('symmetric buffer has been destroyed')
        if hidden != sym_buffer.x.shape[1]:
            raise ValueError(f'x has hidden {hidden}, the workspace {sym_buffer.x.shape[1]}')
        if tokens > sym_buffer.num_max_tokens_per_rank:
            raise ValueError(f'{tokens} tokens exceed the workspace capacity {sym_buffer.num_max_tokens_per_rank}')
        if sym_buffer.x.get_device() != device:
            raise ValueError('the workspace is on another device than x')
        x_q, x_sf = sym_buffer.x[:tokens], sym_buffer.x_sf[:tokens]
        shared_sf = getattr(sym_buffer, 'shared_l1_acts_sf', None)
        if shared_sf is not None:
            shared_rows = shared_sf.shape[0]
            block_m = get_block_m_for_gc_moe(sym_buffer.group.size(), sym_buffer.num_experts,
                                             sym_buffer.num_max_tokens_per_rank, tokens, sym_buffer.num_topk)
    args = _native.NormArgs(
        x.data_ptr(), residual_ptr, weight.data_ptr(), x_q.data_ptr(), x_sf.data_ptr(), normed_ptr, residual_out_ptr,
        0 if shared_sf is None else shared_sf.data_ptr(), x_stride, residual_stride, normed_stride, residual_out_stride,
        shared_rows, block_m, tokens, hidden, residual_f32, int(weight.dtype is torch.float32), float(eps), device)
    code = _native.library().gcmoe_rms_norm(ctypes.byref(args), _native.current_stream(device))
    if code:
        _native.raise_for(code)
    return NormedInputs(x_q, x_sf, normed, residual_out)
