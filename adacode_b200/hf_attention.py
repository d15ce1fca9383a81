"""Decode steps of a HF-transformers model served by the fused attention kernel.

The reference's caches hand dense K/V back from ``update`` and the model's own attention reads
them (``decode_impl: 'materialize_dense'``, float_cache_utils.py:1342).  This module wires the
other route: inside ``fused_decode(cache)`` a single-token ``update`` only appends (same packing
schedule, same adjuster steps) and returns the new token's K/V, and the attention function
registered here as ``'float11_fused'`` computes the step with ``adacode_decode_attn`` straight
from the packed planes.  Prefill and everything outside the context manager go through SDPA on
the dense tensors, as before.

    model.config._attn_implementation = 'float11_fused'     # after register()
    cache = Float11Cache(model.config, ...)
    with fused_decode(cache):
        out = model.generate(ids, past_key_values=cache, ...)

With ``fused_decode(cache, model, chunks=True)`` updates of several tokens behind the prefill (the next turn of a conversation, a chunk of a
prompt) go the same way: the chunk's attention is computed by ``paged_attention`` over the dense view.  Left-padded batches are served too, in
chunks and single steps.  For a chunk behind a prefill transformers makes a mask (``[B, 1, T, S]``), which the kernel does not read; it is compared once
per forward pass, and waited for, with the causal one behind each sequence's padding, and has to be that.  Assisted generation is not served: the cache
cannot take rejected tokens back (``crop``).  Keys that are not what the cache's last update of the layer returned, as those of a model that
runs with another cache or with none inside the context, are refused.

Limits: every cached token is attended to, head_dim 64 or 128.  A step whose attention mask hides
any cached position (left-padded batches) or whose layer uses a sliding window cannot be served by
the kernel; such a step raises instead of attending to the wrong tokens, attention sinks (``s_aux``), soft-capped
scores, additive biases and chunks that are not causal raise too, and ``fused_decode``
refuses a model whose attention implementation is not the one registered here (its SDPA would see
one token only).  Results are close to, not bit-identical with, the materialising path
(different summation order), so generated tokens can differ where two logits are nearly tied.
"""
from __future__ import annotations

import contextlib
from typing import Optional

import torch

ATTENTION_NAME = 'float11_fused'
# what models hand over that changes the scores or their sum, and that neither the kernels nor SDPA take
_NOT_SERVED = ('s_aux', 'softcap', 'position_bias')
_active_cache = None


def float11_fused_attention(module, query, key, value, attention_mask, dropout: float = 0.0,
                            scaling: Optional[float] = None, **kwargs):
    """Attention function with the ``AttentionInterface`` signature."""
    cache = _active_cache
    chunks = cache is not None and getattr(cache, '_fused_chunks', False)
    if cache is not None and getattr(cache, '_fused_decode', False):
        for name in _NOT_SERVED:
            if kwargs.get(name) is not None:
                raise NotImplementedError(f'float11_fused attention has no {name}; use another attention implementation')
    if cache is not None and (query.shape[2] == 1 or (chunks and key.shape[2] == query.shape[2] and _behind_prefill(cache, module, query))) and \
            getattr(cache, '_fused_decode', False):
        layer = cache.layers[module.layer_idx]
        if chunks:
            updated = getattr(cache, '_fused_keys', {}).get(module.layer_idx)
            if updated is not None and updated() is not key:
                raise NotImplementedError('float11_fused attention: these keys are not what the last update of the cache in fused_decode returned '
                                          '(a model with another cache, or with none?)')
            is_causal = kwargs.get('is_causal')
            if query.shape[2] > 1 and attention_mask is None and not (getattr(module, 'is_causal', True) if is_causal is None else is_causal):
                raise NotImplementedError('float11_fused attention of several tokens is causal; use the materialising path')
            # (some models' modules know their window, others hand the config's over; one that hides nothing is none)
            window, total = kwargs.get('sliding_window') or getattr(module, 'sliding_window', None) or 0, layer.get_seq_length()
            if window >= total:
                window = 0
            if attention_mask is not None and attention_mask.shape[2] != query.shape[2]:
                raise NotImplementedError(f'float11_fused attention: a mask of {attention_mask.shape[2]} rows for {query.shape[2]} queries')
            starts = None if attention_mask is None else _left_padding(cache, module.layer_idx, attention_mask, query.shape[0], total, window)
            if query.shape[2] > 1 or starts is not None or window:
                return layer.chunk_attention(query, scale=scaling, seq_starts=starts, window=window).transpose(1, 2).contiguous(), None
            return layer.decode_attention(query, scale=scaling).transpose(1, 2).contiguous(), None
        if getattr(module, 'sliding_window', None):
            raise NotImplementedError('float11_fused attention has no sliding window; use the materialising path')
        if attention_mask is not None and not _mask_shows_everything(cache, attention_mask):
            raise NotImplementedError('float11_fused attention attends to every cached token, but this step\'s '
                                      'attention mask hides some (left padding?); use the materialising path')
        out = layer.decode_attention(query, scale=scaling)           # [B, Hq, 1, D]
        return out.transpose(1, 2).contiguous(), None               # [B, 1, Hq, D]
    from transformers.integrations.sdpa_attention import sdpa_attention_forward
    return sdpa_attention_forward(module, query, key, value, attention_mask, dropout=dropout, scaling=scaling,
                                  **kwargs)


def _mask_shows_everything(cache, mask: torch.Tensor) -> bool:
    """True when a boolean mask is all True or an additive mask is all zero.  All layers of a
    forward pass get the same mask object, so the (synchronising) check runs once per step."""
    seen = getattr(cache, '_fused_mask_seen', None)
    if seen is not None and seen[0] is mask:
        return seen[1]
    ok = bool(mask.all()) if mask.dtype == torch.bool else bool((mask == 0).all())
    cache._fused_mask_seen = (mask, ok)
    return ok


def _behind_prefill(cache, module, query: torch.Tensor) -> bool:
    """Whether the layer held tokens before this chunk (its first update is attended to by SDPA on the model's own tensors)."""
    return cache.layers[module.layer_idx].get_seq_length() > query.shape[2]


def _left_padding(cache, layer_idx: int, mask: torch.Tensor, batch: int, total: int, window: int) -> Optional[torch.Tensor]:
    """First visible position of every sequence (int32 [B]) of a mask that is causal, with the layer's sliding window, behind left padding;
    None where nothing is padded.  All layers of a kind get the same mask object in a forward pass, so the (synchronising) check runs
    once per pass and kind, and again where the mask has been written to since (which a tensor of inference mode does not tell: there, for
    every layer); a layer that is not behind the last one asked for begins another pass."""
    seen_layer, known = getattr(cache, '_fused_masks_known', (-1, ()))
    known = [k for k in known if layer_idx > seen_layer]
    cache._fused_masks_known = layer_idx, known
    as_now = None if mask.is_inference() else (mask._version, window, total)
    for k in known:
        if as_now is not None and k[0] is mask and k[1] == as_now:
            return k[2]
    visible = mask if mask.dtype == torch.bool else mask == 0
    T = visible.shape[2]
    if visible.shape[3] != total:
        raise NotImplementedError(f'float11_fused attention: a mask of {visible.shape[3]} positions for {total} cached tokens')
    j = torch.arange(total, device=mask.device)
    at = torch.arange(total - T, total, device=mask.device)[:, None]
    # (with a window, the last query does not see where its sequence begins: the first one may)
    starts = visible[:, 0].any(1).to(torch.int8).argmax(-1)
    causal = (j >= starts[:, None, None]) & (j <= at)
    if window:
        causal &= j > at - window
    is_causal, padded = torch.stack([(visible == causal[:, None]).all(), (starts > 0).any()]).tolist()
    if not is_causal:
        raise NotImplementedError('float11_fused attention takes masks that are causal behind left padding; use the materialising path')
    out = starts.to(torch.int32).expand(batch).contiguous() if padded else None
    if as_now is not None:
        known.append((mask, as_now, out))
    return out


def register() -> str:
    """Register the attention function with transformers, and SDPA's masks for it (without them a padded batch would come without
    any); returns its name."""
    from transformers import AttentionInterface
    from transformers.masking_utils import AttentionMaskInterface, sdpa_mask
    AttentionMaskInterface.register(ATTENTION_NAME, sdpa_mask)
    AttentionInterface.register(ATTENTION_NAME, float11_fused_attention)
    return ATTENTION_NAME


@contextlib.contextmanager
def fused_decode(cache, model=None, chunks: bool = False):
    """Single-token updates of ``cache`` skip the dense rebuild while this context is active, with ``chunks`` all updates behind the prefill.
    Pass the model (or its config) to have its attention implementation checked: with any other
    implementation the model's own attention would run on the one token ``update`` returns."""
    global _active_cache
    if model is not None:
        cfg = getattr(model, 'config', model)
        impl = getattr(cfg, '_attn_implementation', None)
        if impl != ATTENTION_NAME:
            raise RuntimeError(f"fused_decode needs config._attn_implementation == '{ATTENTION_NAME}' "
                               f'(call hf_attention.register() and set it); found {impl!r}')
    previous = _active_cache
    _active_cache = cache
    cache._fused_decode, cache._fused_chunks = True, bool(chunks)
    try:
        yield cache
    finally:
        cache._fused_decode = cache._fused_chunks = False
        cache._fused_mask_seen = None
        cache._fused_masks_known = -1, []
        cache._fused_keys = {}
        _active_cache = previous
