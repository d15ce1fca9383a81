"""One token per row of logits (``sample_tokens``): temperature, top-k, top-p and min-p in one launch.

The random number is an argument, so a draw is a function of its inputs, the same on every run.  How many CTAs have a row follows
from the batch, and with it the order in which weights are added up in 64 bits: at another batch size a draw can only differ
where the aim lies within that rounding (a relative 3e-11 for 2**18 tokens) of the border between two outcomes.
The reference samples through ``generate`` (main_lossless_comp.py, ``--do_sample``), which sorts the vocabulary and draws with
``torch.multinomial``; ``FusedSampler`` puts this draw into ``generate``.
"""
from __future__ import annotations

import numbers
from typing import Optional, Union

import torch

from . import _lib
from .codec import _scratch_for
from .paged import refuse_autograd
from .rows import on_device, stream_ptr, written

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16, torch.float32: _lib.FP32}
Setting = Union[float, int, torch.Tensor]
_MOST_TOKENS = 1 << 30


def _setting(name: str, value: Setting, B: int, dtype: torch.dtype, device: torch.device) -> tuple:
    """A setting as (tensor of one entry per row or None, number for all rows)."""
    if isinstance(value, numbers.Real):
        if value != value:
            raise ValueError(f'{name} is not a number')
        return None, value
    if not isinstance(value, torch.Tensor) or value.shape != (B,) or value.dtype != dtype or value.device != device:
        raise ValueError(f'{name} must be a number or {dtype} [{B}] on {device}: got {value!r}')
    return value.contiguous(), 0


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0,
                  top_p: Setting = 1.0, min_p: Setting = 0.0, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Draw one token of every row of ``logits`` ``[B, V]`` (bf16, fp16 or fp32) with the row's entry of ``uniforms``, fp32 ``[B]`` in [0, 1).

    Tokens are ordered by descending logit, the lower token first among equals.  The first ``top_k`` stay (0: all); of those, each whose
    predecessors' softmax weights at ``temperature`` add up to less than ``top_p`` of all (1: all; the first always stays); of those, each
    whose weight is at least ``min_p`` times the largest.  The draw is the first token, in the order of the vocabulary, at which
    the running sum of the weights that stay exceeds the uniform number times their total.  ``temperature`` 0 takes the first token of the
    largest logit.  Minus infinity and NaN are never drawn; a row of nothing else gives -1.

    The settings are numbers for all rows or tensors of one entry per row (fp32, ``top_k`` int32).  Returns int64 ``[B]``, ``out`` if given.
    """
    if logits.is_cuda:
        got = _lib.native().sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p, out)
        if got is not False:
            return got
    # (what is left: a call to refuse, or one whose tensors have to be laid out first)
    if logits.dim() != 2 or logits.dtype not in _DTYPES or logits.shape[1] == 0 or logits.shape[1] > _MOST_TOKENS:
        raise ValueError(f'logits must be bf16, fp16 or fp32 [B, V], V at most {_MOST_TOKENS}: got {logits.dtype} {list(logits.shape)}')
    B, V = logits.shape
    dev = logits.device
    if uniforms.dtype != torch.float32 or uniforms.shape != (B,) or uniforms.device != dev:
        raise ValueError(f'uniforms must be fp32 [{B}] on {dev}: got {uniforms.dtype} {list(uniforms.shape)} on {uniforms.device}')
    settings = [_setting(name, value, B, dtype, dev) for name, value, dtype in (
        ('temperature', temperature, torch.float32), ('top_k', top_k, torch.int32), ('top_p', top_p, torch.float32),
        ('min_p', min_p, torch.float32))]
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=dev)
    elif out.dtype != torch.int64 or out.shape != (B,) or not out.is_contiguous() or out.device != dev:
        raise ValueError(f'out must be contiguous int64 [{B}] on {dev}')
    refuse_autograd('sample_tokens', (), (out,))
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    uniforms = uniforms.contiguous()
    _scratch_for(dev)
    (t, t_all), (k, k_all), (p, p_all), (m, m_all) = settings
    with on_device(dev):
        rc = _lib.lib().adacode_sample_tokens(
            logits.data_ptr(), logits.stride(0), _DTYPES[logits.dtype], B, V, uniforms.data_ptr(), None if t is None else t.data_ptr(), t_all,
            None if k is None else k.data_ptr(), max(-1, min(int(k_all), 2 ** 31 - 1)), None if p is None else p.data_ptr(), p_all,
            None if m is None else m.data_ptr(), m_all, out.data_ptr(), stream_ptr(dev))
    _lib.check(rc, 'adacode_sample_tokens')
    written(out)
    return out


class FusedSampler:
    """``sample_tokens`` inside ``model.generate``: a logits processor that leaves every row one token, which greedy decoding then takes.

        model.generate(**inputs, do_sample=False, logits_processor=LogitsProcessorList([FusedSampler(0.7, top_k=50, seed=0)]))

    It has to be the last processor.  The uniform numbers come from a generator of its own on the logits' device.
    """

    def __init__(self, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0, seed: int = 0):
        self.settings = (float(temperature), int(top_k), float(top_p), float(min_p))
        self.seed, self.generator = int(seed), None

    def __call__(self, input_ids: torch.Tensor, scores: torch.Tensor) -> torch.Tensor:
        if self.generator is None or self.generator.device != scores.device:
            self.generator = torch.Generator(scores.device).manual_seed(self.seed)
        uniforms = torch.rand(scores.shape[0], generator=self.generator, device=scores.device)
        tokens = sample_tokens(scores, uniforms, *self.settings)
        return torch.full_like(scores, -torch.inf).scatter_(1, tokens.clamp(min=0)[:, None], 0.0)
