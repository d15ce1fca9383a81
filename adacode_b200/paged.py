"""New tokens of a serving step and a paged cache of dense keys and values: ``append_rotary`` and ``paged_attention``.

A paged cache is two tensors of pages ``[P, Hkv, page_size, D]`` (any strides, unit stride along D) and a ``block_table``
int32 ``[B, W]`` of page numbers: position ``p`` of sequence ``b`` is slot ``p % page_size`` of page ``block_table[b, p // page_size]``.
A page of 128 tokens is what ``compress_tiled_tensor`` packs, and a dense cache ``[B, H, T, D]`` is one page per sequence with the table
``arange(B)[:, None]``: that is how the caches of this package use these functions (``Float11Cache.update_rotary``,
``Float11Cache.chunk_attention``).

``seq_lens`` int32 ``[B]`` counts the tokens of every sequence with the new ones of the call.  New tokens lie one sequence
after the other along the first dimension; ``cu_seqlens`` int32 ``[B + 1]`` says where each sequence begins (without it all have equally
many), and tokens before ``cu_seqlens[0]`` or from ``cu_seqlens[B]`` on are padding, which is left alone.  Tables and lengths stay on the device: a call
never waits for them, and a captured call may be replayed with others.  What only they can show to be wrong, a position without a page
of the pool, is never followed: nothing is written there, zeros are read, and the device's
status word says so (``codec.check_device_status``).  Pages of which no new token sees anything (before all windows, inside
the left padding) need no entry for ``paged_attention``.

The reference has neither: its caches concatenate (float_cache_utils.py:860-881) what the model has rotated with torch
operations, and rebuild dense keys and values for the model's own attention (:1342).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch
from torch.autograd import forward_ad

from . import _lib
from .codec import _scratch_for, device_status
from .rows import on_device, stream_ptr, written

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}
_ANGLES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16, torch.float32: _lib.FP32}
_MAX_AXES = 4
_INT32 = torch.int32
_MOST = 2 ** 31 - 1
_MOST_SCALE = torch.finfo(torch.float32).max


def _describe_cache(N: int, key_pages: torch.Tensor, value_pages: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    cu_seqlens: Optional[torch.Tensor]) -> _lib.PagedCache:
    """The checked cache of a call with N new tokens."""
    if key_pages.dim() != 4 or key_pages.shape != value_pages.shape:
        raise ValueError(f'key_pages and value_pages must both be [pages, heads, page_size, D]: got {tuple(key_pages.shape)} and '
                         f'{tuple(value_pages.shape)}')
    if key_pages.dtype not in _DTYPES or value_pages.dtype != key_pages.dtype:
        raise ValueError(f'pages must be bf16 or fp16, keys and values alike: got {key_pages.dtype} and {value_pages.dtype}')
    P, H, page, D = key_pages.shape
    kp, kh, ks, ku = key_pages.stride()
    vp, vh, vs, vu = value_pages.stride()
    if D > 1 and (ku != 1 or vu != 1):
        raise ValueError('pages must have unit stride along D')
    if block_table.dim() != 2 or block_table.dtype is not _INT32 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError('block_table must be int32 [B, W] with unit stride along W')
    B, W = block_table.shape
    if seq_lens.dtype is not _INT32 or seq_lens.shape != (B,) or not seq_lens.is_contiguous():
        raise ValueError('seq_lens must be contiguous int32 [B]')
    if B == 0 or W == 0 or key_pages.numel() == 0:
        raise ValueError('the cache has no pages or no sequences')
    if max(N, B, W, H, page) > _MOST or P >= _MOST:
        raise ValueError('sizes must fit in 31 bits')
    if cu_seqlens is None:
        if N % B != 0:
            raise ValueError(f'without cu_seqlens the {N} new tokens must divide evenly among {B} sequences')
    elif cu_seqlens.dtype is not _INT32 or cu_seqlens.shape != (B + 1,) or not cu_seqlens.is_contiguous():
        raise ValueError('cu_seqlens must be contiguous int32 [B + 1]')
    return _lib.PagedCache(key_pages.data_ptr(), value_pages.data_ptr(), kp, kh, ks, vp, vh, vs, block_table.data_ptr(), block_table.stride(0),
                           seq_lens.data_ptr(), None if cu_seqlens is None else cu_seqlens.data_ptr(), W, B, P, page, H, D,
                           _DTYPES[key_pages.dtype], N)


def _same_device(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f'{name} is on {t.device}, the pages are on {device}')


def _states(name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype) -> torch.Tensor:
    if tuple(t.shape) != shape or t.dtype != dtype:
        raise ValueError(f'{name} must be {dtype} {list(shape)}: got {t.dtype} {list(t.shape)}')
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _refuse_overlap(**written_to) -> None:
    for name, t in written_to.items():
        if t is not None and any(stride == 0 and n > 1 for stride, n in zip(t.stride(), t.shape)):
            raise ValueError(f'{name} is written to and must not overlap itself: strides {list(t.stride())}')


def refuse_autograd(what: str, read: tuple, written_to: tuple) -> None:
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (*read, *written_to)):
        raise RuntimeError(f'{what} has no forward-mode derivative: hand over the primal tensors')
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (*read, *written_to)):
        raise RuntimeError(f'{what} has no backward pass: call it under torch.no_grad()')
    if not torch.is_inference_mode_enabled() and any(t is not None and t.is_inference() for t in written_to):
        raise RuntimeError(f'{what}: inference tensors are written to in inference mode only')


def append_rotary(key: torch.Tensor, value: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, key_pages: torch.Tensor,
                  value_pages: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, *, query: Optional[torch.Tensor] = None,
                  cu_seqlens: Optional[torch.Tensor] = None, sections: Optional[Sequence[int]] = None, interleaved: bool = False,
                  out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Rotate new tokens by their positions and append them to a paged cache, in one launch.

    ``key`` and ``value`` ``[N, Hkv, D]`` (and ``query`` ``[N, Hq, D]``) are what the projections give.  ``cos`` and ``sin`` ``[N, R / 2]``
    (or ``[1, N, R / 2]``), fp32 or of the keys' type, are the angles of every token's position; the first R columns of every head
    are rotated: columns ``f`` and ``f + R / 2`` against each other, or ``2 f`` and ``2 f + 1`` if ``interleaved``.  (A HF model's
    ``position_embeddings`` hold every angle twice: hand over ``cos[..., :R // 2]``.)  Positions of several axes (time,
    height, width) have ``cos`` and ``sin`` ``[A, N, R / 2]``, A at most four, and ``sections``: how many consecutive
    frequencies are taken from each axis.

    Keys (rotated, in 32 bits and rounded once) and values are written to the last tokens of their sequences.  Returns the rotated
    queries, in ``out`` if given (which may be ``query``, and must not overlap any other argument), or None without ``query``.
    """
    if key_pages.is_cuda:
        got = _lib.native().append_rotary(key, value, cos, sin, key_pages, value_pages, block_table, seq_lens, query, cu_seqlens,
                                          None if sections is None else tuple(sections),
                                          bool(interleaved), out, device_status(key_pages.device))
        if got is not False:
            return got
    # (what is left: a call to refuse, or one whose tensors have to be laid out first)
    if key.dim() != 3 or key_pages.dim() != 4:
        raise ValueError('key must be [N, Hkv, D] and the pages [pages, Hkv, page_size, D]')
    N, dtype = key.shape[0], key_pages.dtype
    cache = _describe_cache(N, key_pages, value_pages, block_table, seq_lens, cu_seqlens)
    H, D = cache.Hkv, cache.D
    key, value = _states('key', key, (N, H, D), dtype), _states('value', value, (N, H, D), dtype)
    if D % 2 != 0 or D > 512:
        raise ValueError(f'the head size must be even and at most 512, got {D}')
    if cos.shape != sin.shape or cos.dtype != sin.dtype or cos.dtype not in _ANGLES or (cos.dtype != torch.float32 and cos.dtype != dtype):
        raise ValueError(f'cos and sin must be alike, fp32 or {dtype}: got {cos.dtype} {list(cos.shape)} and {sin.dtype} {list(sin.shape)}')
    if cos.dim() == 2:
        cos, sin = cos[None], sin[None]
    if cos.dim() != 3 or cos.shape[1] != N or 2 * cos.shape[2] > D:
        raise ValueError(f'cos and sin must be [N, R / 2] or [axes, N, R / 2] for {N} tokens and R <= {D}: got {list(cos.shape)}')
    axes, _, half = cos.shape
    if sections is None:
        if axes != 1:
            raise ValueError('angles of several axes need sections')
        sections = (half,)
    sections = [int(n) for n in sections]
    if len(sections) != axes or axes > _MAX_AXES or min(sections) < 0 or sum(sections) != half:
        raise ValueError(f'sections must say how many of the {half} frequencies each of the {axes} axes (at most {_MAX_AXES}) has: got {sections}')
    if half > 1 and cos.stride(2) != 1:
        cos = cos.contiguous()
    if sin.stride() != cos.stride():
        cos, sin = cos.contiguous(), sin.contiguous()
    Hq = 0
    if query is not None:
        if query.dim() != 3:
            raise ValueError('query must be [N, Hq, D]')
        Hq = query.shape[1]
        query = _states('query', query, (N, Hq, D), dtype)
        if out is None:
            out = torch.empty((N, Hq, D), dtype=dtype, device=query.device)
        elif tuple(out.shape) != (N, Hq, D) or out.dtype != dtype or (D > 1 and out.stride(2) != 1):
            raise ValueError(f'out must be {dtype} {[N, Hq, D]} with unit stride along D')
    elif out is not None:
        raise ValueError('out without query')
    _refuse_overlap(key_pages=key_pages, value_pages=value_pages, out=out)
    refuse_autograd('append_rotary', (key, value, cos, sin, query), (key_pages, value_pages, out))
    dev = key_pages.device
    sc = _scratch_for(dev)
    _same_device(dev, key=key, value=value, cos=cos, sin=sin, value_pages=value_pages, block_table=block_table, seq_lens=seq_lens, query=query,
                 cu_seqlens=cu_seqlens, out=out)
    rotary = _lib.Rotary(cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.stride(1), axes,
                         (ctypes.c_int32 * _MAX_AXES)(*sections), half, int(bool(interleaved)), _ANGLES[cos.dtype])
    with on_device(dev):
        rc = _lib.lib().adacode_append_rotary(
            ctypes.byref(cache), ctypes.byref(rotary), query.data_ptr() if Hq else None, *(query.stride()[:2] if Hq else (0, 0)), Hq,
            out.data_ptr() if Hq else None, *(out.stride()[:2] if Hq else (0, 0)), key.data_ptr(), *key.stride()[:2],
            value.data_ptr(), *value.stride()[:2], sc.status.data_ptr(), stream_ptr(dev))
    _lib.check(rc, 'adacode_append_rotary')
    written(key_pages, value_pages, out)
    return out


def paged_attention(query: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, *, cu_seqlens: Optional[torch.Tensor] = None, max_query_len: Optional[int] = None,
                    scale: Optional[float] = None, causal: bool = True, window: int = 0, seq_starts: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of a chunk of new tokens of every sequence over the sequence's pages, which hold the chunk too.

    ``query`` ``[N, Hq, D]``, D 64 or 128, in the pages' type; ``Hq`` a multiple of the pages' heads.  The token at
    position ``p`` of sequence ``b`` attends to the positions ``j`` with ``seq_starts[b] <= j < seq_lens[b]`` (int32 ``[B]``:
    what is before is left padding), ``j <= p`` if ``causal``, and ``j > p - window`` if ``window`` is positive.  A token that
    sees nothing gets 0; what hidden positions hold never matters.  ``max_query_len``, the most new tokens of one sequence, chooses the
    kernel; without it the call assumes that one sequence may have nearly all.  Pages hold 16, 32, 64 or a multiple of 128 tokens;
    with one page per sequence (``block_table`` ``[B, 1]``) any number.

    Scores and sums are of 32 bits; the softmax weights are rounded to the pages' type for their product with the values.
    Returns ``[N, Hq, D]``, ``out`` if given, which must not overlap the queries.
    """
    if key_pages.is_cuda:
        got = _lib.native().paged_attention(query, key_pages, value_pages, block_table, seq_lens, cu_seqlens, max_query_len, scale, bool(causal),
                                            window, seq_starts, out, device_status(key_pages.device))
        if got is not False:
            return got
    # (what is left: a call to refuse, or one whose tensors have to be laid out first)
    if query.dim() != 3:
        raise ValueError('query must be [N, Hq, D]')
    N, Hq, D = query.shape
    cache = _describe_cache(N, key_pages, value_pages, block_table, seq_lens, cu_seqlens)
    if D not in (64, 128):
        raise ValueError(f'the head size must be 64 or 128, got {D}')
    query = _states('query', query, (N, Hq, cache.D), key_pages.dtype)
    if Hq == 0 or Hq % cache.Hkv != 0:
        raise ValueError(f'{Hq} query heads are not a multiple of {cache.Hkv} cached ones')
    page = cache.page_size
    if cache.table_width > 1 and page % 128 != 0 and page not in (16, 32, 64):
        raise ValueError(f'pages of several per sequence must hold 16, 32, 64 or a multiple of 128 tokens, got {page}')
    if window < 0:
        raise ValueError('window must be positive, or 0 for none')
    if scale is None:
        scale = D ** -0.5
    if not abs(scale) <= _MOST_SCALE:
        raise ValueError(f'scale must be finite in 32 bits, got {scale}')
    if seq_starts is not None and (seq_starts.dtype is not _INT32 or seq_starts.shape != seq_lens.shape or not seq_starts.is_contiguous()):
        raise ValueError('seq_starts must be contiguous int32 [B]')
    if out is None:
        out = torch.empty((N, Hq, D), dtype=query.dtype, device=query.device)
    elif tuple(out.shape) != (N, Hq, D) or out.dtype != query.dtype or out.stride(2) != 1:
        raise ValueError(f'out must be {query.dtype} {[N, Hq, D]} with unit stride along D')
    elif N > 0 and out.data_ptr() == query.data_ptr():
        raise ValueError('out must not be the queries, which are read again where a numerator is not finite')
    if max_query_len is None:
        max_query_len = N // cache.B if cu_seqlens is None else N
    elif max_query_len < 0:
        raise ValueError('max_query_len must not be negative')
    _refuse_overlap(out=out)
    refuse_autograd('paged_attention', (query, key_pages, value_pages), (out,))
    dev = key_pages.device
    sc = _scratch_for(dev)
    _same_device(dev, query=query, value_pages=value_pages, block_table=block_table, seq_lens=seq_lens, cu_seqlens=cu_seqlens,
                 seq_starts=seq_starts, out=out)
    if any((t.data_ptr() & 15) or any(s & 7 for s, n in zip(t.stride()[:-1], t.shape) if n > 1) for t in (query, key_pages, value_pages, out)):
        raise ValueError('queries, pages and out must lie on 16-byte boundaries, with strides that are multiples of 8')
    with on_device(dev):
        # (memory of every call's own: calls of other streams, and graphs that were captured, share nothing)
        most = min(int(max_query_len), _MOST)
        ws = torch.empty(int(_lib.lib().adacode_paged_attn_workspace_bytes(most, Hq, cache.Hkv, D)), dtype=torch.uint8, device=dev)
        rc = _lib.lib().adacode_paged_attn(
            ctypes.byref(cache), query.data_ptr(), *query.stride()[:2], Hq, out.data_ptr(), *out.stride()[:2],
            None if seq_starts is None else seq_starts.data_ptr(), most, float(scale), int(bool(causal)), min(int(window), _MOST),
            ws.data_ptr(), ws.numel(), sc.status.data_ptr(), stream_ptr(dev))
    _lib.check(rc, 'adacode_paged_attn')
    written(out)
    return out
