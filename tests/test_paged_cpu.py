"""What the paged operators and the sampler refuse, found out before anything is launched."""
import pytest
import torch

from adacode_b200 import append_rotary, paged_attention, sample_tokens

BF, I32 = torch.bfloat16, torch.int32


def cache(P=5, H=2, page=16, D=64, B=2, W=2, dtype=BF):
    return (torch.zeros(P, H, page, D, dtype=dtype), torch.zeros(P, H, page, D, dtype=dtype), torch.zeros(B, W, dtype=I32),
            torch.full((B,), 4, dtype=I32))


def test_attention_refuses():
    k, v, table, lens = cache()
    q = torch.zeros(4, 4, 64, dtype=BF)
    bad = [
        ((q[0], k, v, table, lens), {}),                                             # rank
        ((q[:, :3], k, v, table, lens), {}),                                         # heads
        ((q.half(), k, v, table, lens), {}),                                         # another type
        ((q, k, v[:, :, :8], table, lens), {}),                                      # other shapes of keys and values
        ((q, k.float(), v.float(), table, lens), {}),
        ((q, k, v, table.long(), lens), {}),
        ((q, k, v, table, lens.long()), {}),
        ((q, k, v, table, lens[:1]), {}),
        ((q[:3], k, v, table, lens), {}),                                            # 3 tokens among 2 sequences
        ((q, k, v, table, lens), {'cu_seqlens': torch.zeros(2, dtype=I32)}),
        ((q, k, v, table, lens), {'cu_seqlens': torch.zeros(3)}),
        ((q, k, v, table, lens), {'seq_starts': torch.zeros(3, dtype=I32)}),
        ((q, k, v, table, lens), {'window': -1}),
        ((q, k, v, table, lens), {'max_query_len': -1}),
        ((q, k, v, table, lens), {'out': torch.zeros(4, 4, 64)}),
        ((q, k.transpose(2, 3).contiguous().transpose(2, 3), v, table, lens), {}),   # no unit stride
        ((q[..., :32], k[..., :32], v[..., :32], table, lens), {}),                  # head size
        ((q, *cache(page=24)), {}),                                                  # page size
    ]
    for args, more in bad:
        with pytest.raises(ValueError):
            paged_attention(*args, **more)


def test_append_refuses():
    k, v, table, lens = cache()
    x, c = torch.zeros(4, 2, 64, dtype=BF), torch.zeros(4, 32)
    bad = [
        ((x[0], x, c, c, k, v, table, lens), {}),
        ((x, x[:, :1], c, c, k, v, table, lens), {}),
        ((x, x.half(), c, c, k, v, table, lens), {}),
        ((x, x, c, c[:, :16], k, v, table, lens), {}),
        ((x, x, c.double(), c.double(), k, v, table, lens), {}),
        ((x, x, c.half(), c.half(), k, v, table, lens), {}),
        ((x, x, c[:3], c[:3], k, v, table, lens), {}),
        ((x, x, torch.zeros(4, 33), torch.zeros(4, 33), k, v, table, lens), {}),     # more columns than a head has
        ((x, x, torch.zeros(2, 4, 32), torch.zeros(2, 4, 32), k, v, table, lens), {}),
        ((x, x, torch.zeros(2, 4, 32), torch.zeros(2, 4, 32), k, v, table, lens), {'sections': (16, 8)}),
        ((x, x, torch.zeros(5, 4, 32), torch.zeros(5, 4, 32), k, v, table, lens), {'sections': (16, 4, 4, 4, 4)}),
        ((x, x, c, c, k, v, table, lens), {'out': x}),
        ((x, x, c, c, k, v, table, lens), {'query': x, 'out': x[:2]}),
        ((x, x, c, c, k, v, table, lens), {'query': x[0]}),
    ]
    for args, more in bad:
        with pytest.raises(ValueError):
            append_rotary(*args, **more)


def test_sampling_refuses():
    x, u = torch.zeros(3, 10), torch.zeros(3)
    for args, more in (((x[0], u), {}), ((x.double(), u), {}), ((x, u[:2]), {}), ((x, u.double()), {}), ((x[:, :0], u), {}),
                       ((x, u), {'temperature': None}), ((x, u), {'top_k': torch.zeros(3)}), ((x, u), {'top_p': torch.zeros(2)}),
                       ((x, u), {'min_p': float('nan')}), ((x, u), {'out': torch.zeros(3)})):
        with pytest.raises(ValueError):
            sample_tokens(*args, **more)


def test_no_gradients_and_no_cpu():
    from adacode_b200 import _lib
    k, v, table, lens = cache()
    q = torch.zeros(4, 4, 64, dtype=BF, requires_grad=True)
    with pytest.raises(RuntimeError, match='backward'):
        paged_attention(q, k, v, table, lens)
    with pytest.raises(_lib.AdacodeError, match='CUDA'):
        paged_attention(q.detach(), k, v, table, lens)
    with pytest.raises(_lib.AdacodeError, match='CUDA'):
        sample_tokens(torch.zeros(3, 10), torch.zeros(3), temperature=0.0)


def test_entry_points_refuse_without_a_gpu():
    """The C entry points answer bad arguments by a code."""
    import ctypes
    from adacode_b200 import _lib
    L = _lib.lib()
    one = ctypes.create_string_buffer(64)
    at = ctypes.addressof(one)
    fine = dict(key_pages=at, value_pages=at, key_page=8, key_head=8, key_slot=8, value_page=8, value_head=8, value_slot=8, block_table=at,
                table_stride=1, seq_lens=at, cu_seqlens=None, table_width=1, B=1, n_pages=1, page_size=16, Hkv=1, D=64, dtype=0, N=1)

    def attend(ws=0, **more):
        c = _lib.PagedCache(**{**fine, **more})
        return L.adacode_paged_attn(ctypes.byref(c), at, 64, 64, 1, at, 64, 64, None, 1, 0.1, 1, 0, at, ws, at, None)
    for more in (dict(key_pages=None), dict(B=0), dict(D=96), dict(dtype=2), dict(N=-1), dict(page_size=0), dict(key_slot=4), dict(Hkv=2),
                 dict(table_width=2, page_size=24), dict(seq_lens=None)):
        assert attend(**more) == _lib.ERR_INVALID_ARG, more
    assert attend(N=0) == _lib.OK
    c, r = _lib.PagedCache(**fine), _lib.Rotary(at, at, 0, 32, 1, (ctypes.c_int32 * 4)(31), 32, 0, 2)
    assert L.adacode_append_rotary(ctypes.byref(c), ctypes.byref(r), None, 0, 0, 0, None, 0, 0, at, 64, 64, at, 64, 64, at, None) == _lib.ERR_INVALID_ARG
    assert L.adacode_sample_tokens(at, 4, 7, 1, 4, at, at, 1.0, None, 0, None, 1.0, None, 0.0, at, None) == _lib.ERR_INVALID_ARG
    assert L.adacode_sample_tokens(at, 4, 0, 1, 0, at, at, 1.0, None, 0, None, 1.0, None, 0.0, at, None) == _lib.ERR_INVALID_ARG
    assert L.adacode_sample_tokens(at, 4, 0, 0, 4, at, at, 1.0, None, 0, None, 1.0, None, 0.0, at, None) == _lib.OK


def test_attention_refuses_scales_and_outputs():
    k, v, table, lens = cache()
    q = torch.zeros(4, 4, 64, dtype=BF)
    for more in ({'scale': float('nan')}, {'scale': float('inf')}, {'scale': -1e39}, {'out': q}):
        with pytest.raises(ValueError, match='scale|out'):
            paged_attention(q, k, v, table, lens, **more)


def test_no_forward_derivatives():
    """A tangent that a call would drop is refused; primal tensors inside a dual level are not."""
    from torch.autograd import forward_ad
    from adacode_b200 import _lib
    k, v, table, lens = cache()
    q, x, c = torch.zeros(4, 4, 64, dtype=BF), torch.zeros(4, 2, 64, dtype=BF), torch.zeros(4, 32)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))            # noqa: E731
        with torch.no_grad():
            for args in ((dual(q), k, v, table, lens), (q, dual(k), v, table, lens), (q, k, dual(v), table, lens)):
                with pytest.raises(RuntimeError, match='derivative'):
                    paged_attention(*args)
            with pytest.raises(RuntimeError, match='derivative'):
                paged_attention(q, k, v, table, lens, out=dual(torch.zeros_like(q)))
            for i in range(6):
                args = [x, x, c, c, k, v]
                args[i] = dual(args[i])
                with pytest.raises(RuntimeError, match='derivative'):
                    append_rotary(*args, table, lens)
            with pytest.raises(RuntimeError, match='derivative'):
                append_rotary(x, x, c, c, k, v, table, lens, query=dual(q))
        with pytest.raises(_lib.AdacodeError, match='CUDA'):                    # (as outside: they are on the CPU)
            paged_attention(q, k, v, table, lens)


def test_no_forward_derivatives_through_the_cache():
    from torch.autograd import forward_ad
    from adacode_b200.float_cache_utils import _Rotary
    q, x, c = torch.zeros(1, 4, 3, 64, dtype=BF), torch.zeros(1, 2, 3, 64, dtype=BF), torch.zeros(1, 3, 64)
    with forward_ad.dual_level(), torch.no_grad():
        for i in range(5):
            args = [q, x, x, c, c]
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError, match='derivative'):
                _Rotary(*args, None, False)
        _Rotary(q, x, x, c, c, None, False)


def test_outputs_that_overlap_themselves_are_refused():
    """As copy_ refuses them: every element of what is written to has a place of its own."""
    k, v, table, lens = cache()
    q, x, c = torch.zeros(4, 4, 64, dtype=BF), torch.zeros(4, 2, 64, dtype=BF), torch.zeros(4, 32)
    for out in (torch.zeros(1, 4, 64, dtype=BF).expand(4, 4, 64), torch.zeros(4, 1, 64, dtype=BF).expand(4, 4, 64)):
        with pytest.raises(ValueError, match='overlap'):
            paged_attention(q, k, v, table, lens, out=out)
        with pytest.raises(ValueError, match='overlap'):
            append_rotary(x, x, c, c, k, v, table, lens, query=q, out=out)
    for n in range(3):
        shape = list(k.shape)
        shape[n] = 1
        flat = torch.zeros(shape, dtype=BF).expand(k.shape)
        for pages in ((flat, v), (k, flat)):
            with pytest.raises(ValueError, match='overlap'):
                append_rotary(x, x, c, c, *pages, table, lens)
    one = torch.zeros(1, 1, 64, dtype=BF)                                       # (a dimension of one entry may have any stride)
    from adacode_b200 import _lib
    with pytest.raises(_lib.AdacodeError, match='CUDA'):
        paged_attention(one, k[:, :1], v[:, :1], table[:1], lens[:1], out=torch.zeros(64, dtype=BF).as_strided((1, 1, 64), (0, 0, 1)))


def test_sampling_writes_to_inference_tensors_in_inference_mode_only():
    from adacode_b200 import _lib
    x, u = torch.zeros(3, 10), torch.zeros(3)
    with torch.inference_mode():
        out = torch.zeros(3, dtype=torch.int64)
        with pytest.raises(_lib.AdacodeError, match='CUDA'):
            sample_tokens(x, u, out=out)
    with pytest.raises(RuntimeError, match='inference'):
        sample_tokens(x, u, out=out)
