"""One token per row of logits (``sample_tokens``): temperature, top-k, top-p and min-p in one launch.

The random number is an argument, so a draw is a function of its inputs: the same on every run and at every batch size.
The reference samples through ``generate`` (main_lossless_comp.py, ``--do_sample``), which sorts the vocabulary and draws with
``torch.multinomial``; ``FusedSampler`` puts this draw into ``generate``.
"""
from __future__ import annotations

import numbers
from typing import Optional, Union

import torch

from . import _lib
from .codec import _scratch_for
from .rows import increment_version, on_device, stream_ptr

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16, torch.float32: _lib.FP32}
Setting = Union[float, int, torch.Tensor]


def _setting(name: str, value: Optional[Setting], off, B: int, dtype: torch.dtype, device: torch.device) -> Optional[torch.Tensor]:
    """A setting as one entry per row, or None where it is off for all."""
    if value is None:
        return None
    if isinstance(value, numbers.Real):
        if value != value:
            raise ValueError(f'{name} is not a number')
        if off is not None and off(value):
            return None
        return torch.full((B,), value, dtype=dtype, device=device)
    if value.shape != (B,) or value.dtype != dtype or value.device != device:
        raise ValueError(f'{name} must be a number or {dtype} [{B}] on {device}: got {value.dtype} {list(value.shape)} on {value.device}')
    return value.contiguous()


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, temperature: Setting = 1.0, top_k: Optional[Setting] = 0,
                  top_p: Optional[Setting] = 1.0, min_p: Optional[Setting] = 0.0, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Draw one token of every row of ``logits`` ``[B, V]`` (bf16, fp16 or fp32) with the row's entry of ``uniforms``, fp32 ``[B]`` in [0, 1).

    Tokens are ordered by descending logit, the lower token first among equals.  The first ``top_k`` stay (0: all); of those, each whose
    predecessors' softmax weights at ``temperature`` add up to less than ``top_p`` of all (1: all; the first always stays); of those, each
    whose weight is at least ``min_p`` times the largest.  The draw is the first token, in the order of the vocabulary, at which
    the running sum of the weights that stay exceeds the uniform number times their total.  ``temperature`` 0 takes the first token of the
    largest logit.  Minus infinity and NaN are never drawn; a row of nothing else gives -1.

    The settings are numbers for all rows or tensors of one entry per row (fp32, ``top_k`` int32).  Returns int64 ``[B]``, ``out`` if given.
    """
    if logits.dim() != 2 or logits.dtype not in _DTYPES or logits.shape[1] == 0 or logits.shape[1] >= 2 ** 31:
        raise ValueError(f'logits must be bf16, fp16 or fp32 [B, V]: got {logits.dtype} {list(logits.shape)}')
    B, V = logits.shape
    dev = logits.device
    if uniforms.dtype != torch.float32 or uniforms.shape != (B,) or uniforms.device != dev:
        raise ValueError(f'uniforms must be fp32 [{B}] on {dev}: got {uniforms.dtype} {list(uniforms.shape)} on {uniforms.device}')
    temperature = _setting('temperature', temperature, None, B, torch.float32, dev)
    if temperature is None:
        raise ValueError('temperature must be given (0: the largest logit)')
    top_k = _setting('top_k', top_k, lambda v: v <= 0 or v >= V, B, torch.int32, dev)
    top_p = _setting('top_p', top_p, lambda v: v >= 1, B, torch.float32, dev)
    min_p = _setting('min_p', min_p, lambda v: v <= 0, B, torch.float32, dev)
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=dev)
    elif out.dtype != torch.int64 or out.shape != (B,) or not out.is_contiguous() or out.device != dev:
        raise ValueError(f'out must be contiguous int64 [{B}] on {dev}')
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    uniforms = uniforms.contiguous()
    _scratch_for(dev)
    with on_device(dev):
        rc = _lib.lib().adacode_sample_tokens(
            logits.data_ptr(), logits.stride(0), _DTYPES[logits.dtype], B, V, uniforms.data_ptr(), temperature.data_ptr(),
            None if top_k is None else top_k.data_ptr(), None if top_p is None else top_p.data_ptr(),
            None if min_p is None else min_p.data_ptr(), out.data_ptr(), stream_ptr(dev))
    _lib.check(rc, 'adacode_sample_tokens')
    increment_version([out])
    return out
