"""Cached tokens cannot be taken back: crop says so, and leaves alone what it need not touch."""
import pytest
import torch

from adacode_b200 import Float11Cache
from tests.scenarios import StubConfig


def test_crop(monkeypatch):
    import adacode_b200.float_cache_utils as fc
    from tests.test_state_machine_cpu import oracle_codec
    monkeypatch.setattr(fc, 'codec', oracle_codec)
    cache = Float11Cache(StubConfig(2), right=129, exp_bits=4, need_adjust=False, update_steps=0, block_size=128, layout='segmented_tiled')
    cache.crop(10)                                                                           # nothing is cached yet
    x = torch.randn((1, 2, 140, 64)).to(torch.bfloat16)
    for i in (0, 1):
        cache.update(x, x, i)
    for keep in (140, 200):
        cache.crop(keep)
    for keep in (139, 0, -1, -140):
        with pytest.raises(NotImplementedError, match='crop'):
            cache.crop(keep)
    assert cache.get_seq_length() == 140
    assert torch.equal(cache.materialize_layer(1)[0], x)
