"""Flags of the runner that would have no effect are refused before anything is loaded."""
import pytest

from adacode_b200 import main_lossless_comp as runner

BASE = ['--model_config_name', 'llama_3p1_8B_config', '--random_init', '--kv_cache_impl', 'float11', '--use_synthetic_data']


@pytest.mark.parametrize('more', [['--temperature', '0.7'], ['--do_sample', '--temperature', '0.7'], ['--do_sample', '--top_k', '5'], ['--do_sample', '--top_p', '0.9'],
                                  ['--do_sample', '--min_p', '0.1'], ['--do_sample', '--sample_seed', '3'], ['--fused_sample'], ['--fused_chunks'],
                                  ['--fused_chunks', '--fused_decode', '--kv_cache_impl', 'dynamic']], ids=' '.join)
def test_flags_without_effect(more):
    with pytest.raises(ValueError, match='needs'):
        runner.run(runner.get_parse().parse_args(BASE + more))


def test_settings_of_the_sampler():
    parse = lambda more: runner.sampler_settings(runner.get_parse().parse_args(BASE + more))                     # noqa: E731
    assert parse([]) is None and parse(['--do_sample']) is None
    assert parse(['--do_sample', '--fused_sample']) == (1.0, 50, 1.0, 0.0, 0)
    assert parse(['--do_sample', '--fused_sample', '--temperature', '0', '--top_k', '0', '--top_p', '0.9', '--min_p', '0.1', '--sample_seed', '4']) == (0.0, 0, 0.9, 0.1, 4)
