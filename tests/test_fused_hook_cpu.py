"""The attention function of a HF model on the CPU: which calls reach the layers' own attention, with what, and which are refused."""
from types import SimpleNamespace

import pytest
import torch

from adacode_b200 import hf_attention

B, HQ, T, D, TOTAL = 2, 4, 5, 64, 200


class Layer:
    """A cached layer that notes how it is asked."""

    def __init__(self, total=TOTAL):
        self.total, self.asked = total, []

    def get_seq_length(self):
        return self.total

    def chunk_attention(self, query, scale=None, seq_starts=None, window=0):
        self.asked.append(('chunk', None if seq_starts is None else seq_starts.tolist(), window))
        return torch.zeros_like(query)

    def decode_attention(self, query, scale=None):
        self.asked.append(('decode',))
        return torch.zeros_like(query)


def hook(monkeypatch, chunks=True, total=TOTAL):
    layer = Layer(total)
    cache = SimpleNamespace(layers=[layer], _fused_decode=True, _fused_chunks=chunks)
    monkeypatch.setattr(hf_attention, '_active_cache', cache)

    def call(T=T, mask=None, module=None, **more):
        x = torch.zeros(B, HQ, T, D, dtype=torch.bfloat16)
        out, weights = hf_attention.float11_fused_attention(module or SimpleNamespace(layer_idx=0), x, x[:, :2], x[:, :2], mask, scaling=D ** -0.5, **more)
        assert out.shape == (B, T, HQ, D) and weights is None
        return layer.asked[-1]
    return call


def causal(T, total=TOTAL, window=0, starts=(0, 0)):
    j, at = torch.arange(total), torch.arange(total - T, total)[:, None]
    seen = (j <= at) & (j >= torch.tensor(starts)[:, None, None])
    return (seen & (j > at - window) if window else seen)[:, None]


@pytest.mark.parametrize('chunks', [False, True])
@pytest.mark.parametrize('T', [1, T])
@pytest.mark.parametrize('name', ['s_aux', 'softcap', 'position_bias'])
def test_what_the_kernels_leave_out_is_refused(monkeypatch, name, T, chunks):
    """Sinks, soft-capped scores and additive biases: an attention without them is another one, from the first update on."""
    call = hook(monkeypatch, chunks)
    value = 30.0 if name == 'softcap' else torch.zeros(HQ)
    for total in (TOTAL, T):
        hf_attention._active_cache.layers[0].total = total
        with pytest.raises(NotImplementedError, match=name):
            call(T, **{name: value})
    hf_attention._active_cache.layers[0].total = TOTAL
    if chunks or T == 1:
        assert call(T, **{name: None})[0] == ('decode' if T == 1 else 'chunk')


def test_attention_that_is_not_causal_is_refused(monkeypatch):
    call = hook(monkeypatch)
    for more in (dict(is_causal=False), dict(module=SimpleNamespace(layer_idx=0, is_causal=False))):
        with pytest.raises(NotImplementedError, match='causal'):
            call(**more)
        assert call(1, **more) == ('decode',)                                   # the last token sees everything either way
        assert call(mask=causal(T, starts=(0, 7)), **more) == ('chunk', [0, 7], 0)      # a mask says what is seen
    assert call(is_causal=True) == call(is_causal=None) == ('chunk', None, 0)
    # what the call says goes before what the module says
    assert call(is_causal=True, module=SimpleNamespace(layer_idx=0, is_causal=False)) == ('chunk', None, 0)


@pytest.mark.parametrize('as_argument', [False, True])
def test_windows(monkeypatch, as_argument):
    """A window is the module's, or handed over with every call; one that hides nothing is none, and single tokens then stay with the packed planes."""
    call = hook(monkeypatch)
    more = (lambda w: dict(sliding_window=w)) if as_argument else (lambda w: dict(module=SimpleNamespace(layer_idx=0, sliding_window=w)))
    assert call(**more(50), mask=causal(T, window=50)) == ('chunk', [TOTAL - T - 49] * B, 50)
    assert call(**more(50)) == ('chunk', None, 50)
    assert call(1, **more(50)) == ('chunk', None, 50)
    assert call(**more(50), mask=causal(T, window=50, starts=(0, 170))) == ('chunk', [TOTAL - T - 49, 170], 50)
    with pytest.raises(NotImplementedError, match='masks'):
        call(**more(50), mask=causal(T))
    with pytest.raises(NotImplementedError, match='masks'):
        call(**more(None), mask=causal(T, window=50))
    for w in (TOTAL, TOTAL + 1, None):
        assert call(1, **more(w)) == ('decode',)
        assert call(1, mask=causal(1), **more(w)) == ('decode',)
        assert call(**more(w), mask=causal(T, window=w or 0)) == ('chunk', None, 0)
        assert call(**more(w)) == ('chunk', None, 0)
    assert call(1, **more(TOTAL - 1)) == ('chunk', None, TOTAL - 1)


def test_masks_with_one_row_for_all_queries(monkeypatch):
    """A mask that hides padding alone, the same for all queries, is not a causal one."""
    call = hook(monkeypatch)
    with pytest.raises(NotImplementedError, match='mask'):
        call(mask=causal(1, starts=(0, 9)))
    assert call(1, mask=causal(1, starts=(0, 9))) == ('chunk', [0, 9], 0)
    assert call(mask=causal(T, starts=(0, 9))) == ('chunk', [0, 9], 0)


def test_keys_of_another_cache_are_refused(monkeypatch):
    """Inside fused_decode(chunks=True), attention of a model that runs without the cache, or with another one, is not answered from the cache."""
    import adacode_b200.float_cache_utils as fc
    from adacode_b200 import Float11Cache
    from tests.scenarios import StubConfig
    from tests.test_state_machine_cpu import oracle_codec
    monkeypatch.setattr(fc, 'codec', oracle_codec)
    caches = [Float11Cache(StubConfig(1), right=129, exp_bits=4, need_adjust=False, update_steps=0, block_size=128, layout='segmented_tiled') for _ in range(2)]
    x = torch.randn((B, 2, 150, D)).to(torch.bfloat16)
    asked = []

    def answer(name):
        def attend(self, query, **more):
            asked.append((name, self))
            return torch.zeros_like(query)
        return attend
    monkeypatch.setattr(fc.float11Layer, 'chunk_attention', answer('chunk'))
    monkeypatch.setattr(fc.float11Layer, 'decode_attention', answer('decode'))
    module = SimpleNamespace(layer_idx=0)
    attend = lambda key: hf_attention.float11_fused_attention(module, torch.zeros(B, HQ, key.shape[2], D, dtype=torch.bfloat16), key, key, None)     # noqa: E731
    with hf_attention.fused_decode(caches[0], chunks=True):
        for _ in range(2):
            for n in (100, 5, 1):
                key, _ = caches[0].update(x[:, :, :n], x[:, :, :n], 0)
                if caches[0].get_seq_length() > 100:
                    attend(key)
                    assert asked.pop() == ('decode' if n == 1 else 'chunk', caches[0].layers[0])
                    other, _ = caches[1].update(x[:, :, :n], x[:, :, :n], 0)
                    for foreign in (other[:, :, -n:], x[:, :, :n].clone()):
                        with pytest.raises(NotImplementedError, match='another'):
                            attend(foreign)
        assert not asked
        import pickle
        assert pickle.loads(pickle.dumps(caches[0])).get_seq_length() == caches[0].get_seq_length()
    # outside, and inside a context of single tokens, chunks are SDPA's
    key = x[:, :, :5].repeat(1, 2, 1, 1)
    out, _ = hf_attention.float11_fused_attention(SimpleNamespace(layer_idx=0), key, key, key, None)
    assert out.shape == (B, 5, HQ, D) and not asked


@pytest.mark.parametrize('inference', [False, True])
def test_masks_that_change_between_layers(monkeypatch, inference):
    """One tensor, written anew between two layers of a pass: each layer has what it holds then; unchanged, it is looked at once."""
    cache = SimpleNamespace(layers=[Layer() for _ in range(3)], _fused_decode=True, _fused_chunks=True)
    monkeypatch.setattr(hf_attention, '_active_cache', cache)
    x = torch.zeros(B, HQ, T, D, dtype=torch.bfloat16)
    with torch.inference_mode(inference):
        mask = causal(T, starts=(0, 9)).clone()
        for i in (0, 1):
            hf_attention.float11_fused_attention(SimpleNamespace(layer_idx=i), x, x, x, mask)
        mask.copy_(causal(T, starts=(5, 0)))
        hf_attention.float11_fused_attention(SimpleNamespace(layer_idx=2), x, x, x, mask)
        assert [layer.asked for layer in cache.layers] == [[('chunk', [0, 9], 0)], [('chunk', [0, 9], 0)], [('chunk', [5, 0], 0)]]
        mask.zero_()
        with pytest.raises(NotImplementedError, match='mask'):
            hf_attention.float11_fused_attention(SimpleNamespace(layer_idx=2), x, x, x, mask)
