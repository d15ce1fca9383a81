"""The operators of a serving step together, and through the caches, a HF model and the runner."""
import json

import pytest
import torch

from tests import scenarios, serving_oracle as oracle, synth

pytestmark = pytest.mark.gpu
BF, I32 = torch.bfloat16, torch.int32


def near(got, want, size):
    """One rounding of the weights over sums of |values|, one of the result, and an fp32 dot product's error (tests of paged_attention)."""
    h = 2.0 ** -8
    assert bool(((got.double() - want).abs() <= h * want.abs() + (h + 2.0 ** -12) * (1 + h) * size + 1e-30).all())


def test_steps_over_a_paged_cache():
    """Prompts, then decode steps: rotated and appended, attended to, sampled; every step against dense 64-bit tensors of what was appended."""
    from adacode_b200 import append_rotary, paged_attention, sample_tokens
    from adacode_b200 import codec
    Hq, Hkv, D, page, V = 8, 2, 64, 16, 500
    g = torch.Generator('cpu').manual_seed(0)
    prompts, steps = [70, 5, 33], 20
    B = len(prompts)
    pool_k, pool_v = (torch.full((40, Hkv, page, D), float('nan'), dtype=BF, device='cuda') for _ in range(2))
    table = torch.randperm(40, generator=g).to(I32)[:B * 8].view(B, 8).cuda()
    unembed = (torch.randn((Hq * D, V), generator=g) * 0.2).cuda()
    lens = [0] * B
    keys, values = [torch.zeros((0, Hkv, D), device='cuda') for _ in prompts], [torch.zeros((0, Hkv, D), device='cuda') for _ in prompts]
    for step in range(steps):
        new = prompts if step == 0 else [1] * B
        lens = [a + n for a, n in zip(lens, new)]
        N = sum(new)
        q, k, v = ((torch.randn((N, h, D), generator=g)).to(BF).cuda() for h in (Hq, Hkv, Hkv))
        at = torch.cat([torch.arange(t - n, t) for n, t in zip(new, lens)])
        cos, sin = (x.float().cuda() for x in oracle.angles(at, D // 2))
        seq, cu = torch.tensor(lens, dtype=I32, device='cuda'), oracle.cumulative(new)
        rq = append_rotary(k, v, cos, sin, pool_k, pool_v, table, seq, query=q, cu_seqlens=cu)
        out = paged_attention(rq, pool_k, pool_v, table, seq, cu_seqlens=cu, max_query_len=max(new))
        rk = oracle.rotate(k, cos, sin)
        i = 0
        for b, n in enumerate(new):
            keys[b], values[b] = torch.cat([keys[b], rk[i:i + n].to(BF).float()]), torch.cat([values[b], v[i:i + n].float()])
            got = torch.cat([pool_k[int(p), :].transpose(0, 1) for p in table[b, :-(-lens[b] // page)]])[:lens[b]]
            assert bool(((got.double() - keys[b].double()).abs() <= 2.0 ** -7 * keys[b].double().abs() + 1e-6).all())     # (ties of the rounding)
            keys[b] = got.float()
            i += n
        want, size = oracle.attention(rq, pool_k, pool_v, table, lens, new)
        near(out, want, size)
        last = cu[1:].long() - 1
        logits = out[last].flatten(1).float() @ unembed
        u = torch.rand(B, generator=g).cuda()
        tokens = sample_tokens(logits, u, 0.8, 40, 0.95)
        for b in range(B):
            token, border = oracle.sample(logits[b].cpu(), u[b].item(), float(torch.tensor(0.8)), 40, float(torch.tensor(0.95)))
            assert int(tokens[b]) == token or border < 1e-10
    codec.check_device_status(torch.device('cuda', 0))


def test_full_pages_are_packed_and_attended_to():
    """Pages of 128 tokens are segments: packed, the decode step from the planes agrees with the one over the pages."""
    from adacode_b200 import append_rotary, compress_tiled_tensor, decode_attention, paged_attention
    T, Hq, Hkv, D = 300, 8, 2, 128
    table = torch.tensor([[4, 1, 3]], dtype=I32, device='cuda')
    pool = torch.zeros((2, 5, Hkv, 128, D), dtype=BF, device='cuda')
    k, v = (synth.kv_tensor((1, Hkv, T, D), seed=s)[0].transpose(0, 1).contiguous().to('cuda') for s in (1, 2))
    cos, sin = (x.float().cuda() for x in oracle.angles(torch.arange(T), D // 2))
    seq = torch.tensor([T], dtype=I32, device='cuda')
    append_rotary(k, v, cos, sin, pool[0], pool[1], table, seq)
    q = torch.randn((1, Hq, D), device='cuda').to(BF)
    want, size = oracle.attention(q, pool[0], pool[1], table, [T], [1])
    near(paged_attention(q, pool[0], pool[1], table, seq), want, size)
    segments = [[compress_tiled_tensor(pool[i][int(p)][None], 130, nbits=3)[0] for p in (4, 1)] for i in (0, 1)]
    tails = [pool[i][3][None, :, :T - 256] for i in (0, 1)]
    got = decode_attention(q, segments[0], segments[1], tails[0], tails[1])
    near(got, want, size)


def cache_of(layers=1, **more):
    from adacode_b200 import Float11Cache
    return Float11Cache(scenarios.StubConfig(layers), right=[(130, 129)] * layers, exp_bits=[(3, 3)] * layers, need_adjust=True, update_steps=128,
                        block_size=128, layout='segmented_tiled', **more)


@pytest.mark.parametrize('workspace', ['shared', 'layer'])
@pytest.mark.parametrize('D', [64, 128])
def test_chunks_through_the_cache(D, workspace):
    """Prefill, then chunks of many sizes across block and adjust borders; with padding and windows."""
    B, Hq, Hkv = 2, 8, 2
    sizes = [290, 1, 5, 130, 17, 1, 256, 40]
    total = sum(sizes)
    k, v = (synth.kv_tensor((B, Hkv, total, D), seed=s).to('cuda') for s in (3, 4))
    cache = cache_of(dense_workspace=workspace)
    at = sizes[0]
    cache.update(k[:, :, :at], v[:, :, :at], 0)
    starts = [0, 37]
    for n, T in enumerate(sizes[1:]):
        q = torch.randn((B, T, Hq, D), device='cuda').to(BF).transpose(1, 2)
        more = {} if n % 3 == 0 else {'seq_starts': torch.tensor(starts, dtype=I32, device='cuda')} if n % 3 == 1 else {'window': 50}
        got = cache.chunk_attention(q, k[:, :, at:at + T], v[:, :, at:at + T], 0, **more)
        at += T
        table = torch.arange(B, dtype=I32)[:, None]
        want, size = oracle.attention(q.transpose(1, 2).reshape(B * T, Hq, D), k[:, :, :at], v[:, :, :at], table, [at] * B, [T] * B,
                                      starts=starts if 'seq_starts' in more else None, window=more.get('window', 0))
        near(got.transpose(1, 2).reshape(B * T, Hq, D), want, size)
    dense_k, dense_v = cache.materialize_layer(0)
    assert torch.equal(dense_k, k) and torch.equal(dense_v, v)
    with pytest.raises(ValueError):
        cache.layers[0].chunk_attention(torch.zeros((B, Hq, total + 1, D), dtype=BF, device='cuda'))


@pytest.mark.parametrize('interleaved', [False, True])
def test_rotary_updates_are_updates_of_rotated_states(interleaved):
    """The same cache contents as update() of keys that append_rotary rotated beforehand, whatever the schedule."""
    B, Hq, Hkv, D, R = 2, 4, 2, 64, 32
    sizes = [200, 1, 1, 60, 1, 130]
    k, v = (synth.kv_tensor((B, Hkv, sum(sizes), D), seed=s).to('cuda') for s in (5, 6))
    q = torch.randn((B, Hq, sum(sizes), D), device='cuda').to(BF)
    c, s = oracle.angles(torch.arange(sum(sizes)), R // 2)
    double = (lambda x: x.repeat_interleave(2, -1)) if interleaved else (lambda x: torch.cat([x, x], -1))
    cos, sin = (double(x).float().cuda()[None] for x in (c, s))
    one, two = cache_of(), cache_of()
    at = 0
    for T in sizes:
        now = slice(at, at + T)
        rq, keys, values = one.update_rotary(q[:, :, now], k[:, :, now], v[:, :, now], cos[:, now], sin[:, now], 0, interleaved=interleaved)
        rk = torch.stack([oracle.rotate(k[b, :, now].transpose(0, 1), c[now].float().cuda(), s[now].float().cuda(), interleaved).transpose(0, 1) for b in range(B)])
        want_q = torch.stack([oracle.rotate(q[b, :, now].transpose(0, 1), c[now].float().cuda(), s[now].float().cuda(), interleaved).transpose(0, 1) for b in range(B)])
        at += T
        assert keys.shape[2] == at and torch.equal(values, v[:, :, :at])
        assert bool(((keys[:, :, -T:].double() - rk).abs() <= 2.0 ** -8 * rk.abs() + 1e-4).all())
        assert bool(((rq.double() - want_q).abs() <= 2.0 ** -8 * want_q.abs() + 1e-5).all())
        two.update(keys[:, :, -T:].clone(), v[:, :, now], 0)
    assert one.layers[0].segment_params() == two.layers[0].segment_params()
    a, b = [t.clone() for t in one.materialize_layer(0)], [t.clone() for t in two.materialize_layer(0)]
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and one.layers[0].segment_params()
    with pytest.raises(ValueError):
        one.update_rotary(q[:, :, :2], k[:, :, :2], v[:, :, :2], cos[:, :3], sin[:, :3], 0)


def test_rotary_updates_with_three_axes():
    B, Hq, Hkv, D = 1, 2, 2, 64
    T, sections = 9, (16, 8, 8)
    k, v = (synth.kv_tensor((B, Hkv, T, D), seed=s).to('cuda') for s in (7, 8))
    q = torch.randn((B, Hq, T, D), device='cuda').to(BF)
    positions = torch.stack([torch.arange(T), torch.arange(T) % 3, torch.arange(T) // 3])
    c, s = oracle.angles(positions, D // 2)
    cos, sin = (torch.cat([x, x], -1).float().cuda()[:, None] for x in (c, s))
    cache = cache_of()
    _, keys, _ = cache.update_rotary(q, k, v, cos, sin, 0, sections=sections)
    want = oracle.rotate(k[0].transpose(0, 1), oracle.select_axes(c.float(), sections).cuda(), oracle.select_axes(s.float(), sections).cuda()).transpose(0, 1)
    assert bool(((keys[0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4).all())


def tiny_model(impl=None):
    import transformers
    cfg = transformers.LlamaConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                                   vocab_size=320, max_position_embeddings=2048)
    torch.manual_seed(0)
    model = transformers.AutoModelForCausalLM.from_config(cfg).to(torch.bfloat16).cuda().eval()
    if impl:
        model.config._attn_implementation = impl
    return model


@pytest.mark.parametrize('padded', [False, True])
def test_hf_chunks(padded):
    """A conversation in turns: logits of every chunk within bf16 noise of a DynamicCache's."""
    from transformers import DynamicCache
    from adacode_b200 import hf_attention
    stock, fused = tiny_model(), tiny_model(hf_attention.register())
    g = torch.Generator('cpu').manual_seed(1)
    turns = [150, 9, 1, 140, 1]
    ids = torch.randint(3, 320, (2, sum(turns)), generator=g).cuda()
    mask = torch.ones_like(ids)
    if padded:
        mask[1, :21] = 0
    reference, cache = DynamicCache(config=stock.config), cache_of(2)
    with torch.no_grad(), hf_attention.fused_decode(cache, fused, chunks=True):
        at = 0
        for T in turns:
            position = (mask[:, :at + T].cumsum(1) - 1).clamp(min=0)[:, at:]
            a = stock(ids[:, at:at + T], attention_mask=mask[:, :at + T], position_ids=position, past_key_values=reference, use_cache=True).logits
            b = fused(ids[:, at:at + T], attention_mask=mask[:, :at + T], position_ids=position, past_key_values=cache, use_cache=True).logits
            at += T
            real = mask[:, at - T:at].bool()
            # (two layers in bf16: a handful of roundings of 2**-8 on the way to logits of size one)
            assert float((a - b)[real].float().abs().max()) <= 16 * 2.0 ** -8 * float(a[real].float().abs().max())
    assert cache.layers[0].materialize_calls <= 2 * len(turns)


def test_hf_generate_with_the_fused_sampler():
    from transformers import LogitsProcessorList
    from adacode_b200 import FusedSampler, sample_tokens
    model = tiny_model()
    ids = torch.randint(3, 320, (3, 12), generator=torch.Generator('cpu').manual_seed(2)).cuda()

    class Recorder(FusedSampler):
        def __call__(self, input_ids, scores):
            got = super().__call__(input_ids, scores)
            self.seen.append((scores.clone(), got.argmax(-1)))
            return got
    runs = []
    for _ in range(2):
        sampler = Recorder(0.9, top_k=30, top_p=0.95, seed=7)
        sampler.seen = []
        out = model.generate(ids, do_sample=False, max_new_tokens=10, min_new_tokens=10, logits_processor=LogitsProcessorList([sampler]), pad_token_id=0)
        runs.append(out)
        generator = torch.Generator('cuda').manual_seed(7)
        for step, (scores, picked) in enumerate(sampler.seen):
            assert torch.equal(out[:, 12 + step], picked)
            assert torch.equal(picked, sample_tokens(scores, torch.rand(3, generator=generator, device='cuda'), 0.9, 30, 0.95))
    assert torch.equal(*runs)


def test_runner_samples_and_attends_in_chunks(tmp_path, monkeypatch):
    from adacode_b200 import main_lossless_comp as runner
    monkeypatch.chdir(tmp_path)
    args = ['--model_config_name', 'llama_3p1_8B_config', '--random_init', '--random_init_layers', '1', '--kv_cache_impl', 'float11', '--use_synthetic_data',
            '--synthetic_seq_length', '140', '--batch_size', '2', '--num_seqence', '2', '--max_new_tokens', '4', '--min_new_tokens', '4', '--do_sample',
            '--fused_sample', '--top_k', '20', '--temperature', '0.7', '--fused_decode', '--fused_chunks', '--output_path', 'out.json']
    runner.run(runner.get_parse().parse_args(args))
    record = json.loads((tmp_path / 'out.json').read_text())['synthetic'][0]
    assert record['fused_sample'] == {'temperature': 0.7, 'top_k': 20, 'top_p': 1.0, 'min_p': 0.0} and record['total_new_tokens'] == 8.0
    with pytest.raises(ValueError):
        runner.run(runner.get_parse().parse_args([a for a in args if a != '--do_sample']))


def test_refused_rotary_updates_leave_the_cache_alone():
    B, Hq, Hkv, D, T = 1, 2, 2, 64, 3
    k, v = (synth.kv_tensor((B, Hkv, 40, D), seed=s).to('cuda') for s in (7, 8))
    q = torch.randn((B, Hq, T, D), device='cuda').to(BF)
    cos, sin = torch.ones((1, T, D), device='cuda'), torch.zeros((1, T, D), device='cuda')
    cache = cache_of()
    cache.update(k, v, 0)
    good = (q, k[:, :, :T], v[:, :, :T], cos, sin, 0)
    for i, x in ((0, q[:, :, :2]), (0, q[0]), (0, q.cpu()), (1, k[:, :, :2]), (2, v[:, :1, :T]), (3, cos[..., :63]), (4, sin[:, :2]), (3, cos.cpu())):
        with pytest.raises(ValueError):
            cache.update_rotary(*good[:i], x, *good[i + 1:])
    for sections in ((16, 15), (33, -1), ()):
        with pytest.raises(ValueError):
            cache.update_rotary(*good, sections=sections)
    with pytest.raises(ValueError):
        cache.update_rotary(q, *good[1:3], *(torch.cat([x, x])[:, None] for x in (cos, sin)), 0)              # two axes without sections
    with pytest.raises(RuntimeError):
        cache.update_rotary(q.clone().requires_grad_(), *good[1:])
    assert cache.get_seq_length() == 40
    # no tokens at all, and then some
    rotated, keys, _ = cache.update_rotary(q[:, :, :0], k[:, :, :0], v[:, :, :0], cos[:, :0], sin[:, :0], 0)
    assert rotated.shape == (B, Hq, 0, D) and torch.equal(keys, k)
    rotated, keys, values = cache.update_rotary(*good)
    assert torch.equal(rotated, q) and torch.equal(keys, torch.cat([k, k[:, :, :T]], 2)) and torch.equal(values, torch.cat([v, v[:, :, :T]], 2))


def test_masks_are_read_again_in_every_pass():
    """A mask tensor that is written anew between passes, and one row for all sequences."""
    from types import SimpleNamespace
    from adacode_b200 import hf_attention
    B, Hq, Hkv, D, T = 2, 4, 2, 64, 5
    k, v = (synth.kv_tensor((B, Hkv, 90, D), seed=s).to('cuda') for s in (9, 10))
    q = torch.randn((B, Hq, T, D), device='cuda').to(BF)
    layers = [SimpleNamespace(layer_idx=i, sliding_window=None) for i in (0, 1)]
    causal = torch.arange(90, device='cuda') <= torch.arange(85, 90, device='cuda')[:, None]
    mask = causal.expand(1, 1, T, 90).clone()
    cache = cache_of(2)
    for i in (0, 1):
        cache.update(k, v, i)
    table = torch.arange(B, dtype=I32)[:, None]
    with torch.no_grad(), hf_attention.fused_decode(cache, chunks=True):
        for start in (0, 30, 7):
            mask.copy_(causal & (torch.arange(90, device='cuda') >= start))
            want, size = oracle.attention(q.transpose(1, 2).reshape(B * T, Hq, D), k, v, table, [90] * B, [T] * B, starts=[start] * B)
            for layer in layers:
                got, _ = hf_attention.float11_fused_attention(layer, q, k[:, :, -T:], v[:, :, -T:], mask)
                near(got.reshape(B * T, Hq, D), want, size)


def windowed_model(kind, impl=None):
    """Layers with a sliding window: all of them, which their attention modules hand over with every call, or the second of two."""
    import transformers
    common = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64, vocab_size=320,
                  max_position_embeddings=2048, sliding_window=100)
    cfg = transformers.MistralConfig(**common) if kind == 'all' else transformers.Qwen3Config(**common, use_sliding_window=True, max_window_layers=1)
    torch.manual_seed(0)
    model = transformers.AutoModelForCausalLM.from_config(cfg).to(torch.bfloat16).cuda().eval()
    if impl:
        model.config._attn_implementation = impl
    return model


@pytest.mark.parametrize('padded', [False, True])
@pytest.mark.parametrize('kind', ['all', 'second'])
def test_hf_chunks_with_sliding_windows(kind, padded):
    from transformers import DynamicCache
    from adacode_b200 import hf_attention
    stock, fused = windowed_model(kind), windowed_model(kind, hf_attention.register())
    g = torch.Generator('cpu').manual_seed(3)
    turns = [50, 9, 1, 60, 1, 40, 1, 150]                                                # below the window, across and above it
    ids = torch.randint(3, 320, (2, sum(turns)), generator=g).cuda()
    mask = torch.ones_like(ids)
    if padded:
        mask[1, :21] = 0
    reference, cache = DynamicCache(config=stock.config), cache_of(2)
    with torch.no_grad(), hf_attention.fused_decode(cache, fused, chunks=True):
        at = 0
        for T in turns:
            position = (mask[:, :at + T].cumsum(1) - 1).clamp(min=0)[:, at:]
            a = stock(ids[:, at:at + T], attention_mask=mask[:, :at + T], position_ids=position, past_key_values=reference, use_cache=True).logits
            b = fused(ids[:, at:at + T], attention_mask=mask[:, :at + T], position_ids=position, past_key_values=cache, use_cache=True).logits
            at += T
            real = mask[:, at - T:at].bool()
            # (two layers in bf16, as in test_hf_chunks)
            assert float((a - b)[real].float().abs().max()) <= 16 * 2.0 ** -8 * float(a[real].float().abs().max())


def test_rotary_updates_that_do_not_fit_the_cache_leave_it_alone():
    """Heads, sequences or head sizes other than the cached ones, and buffers that may only be written to in inference mode."""
    D, T = 64, 3
    k, v = (synth.kv_tensor((2, 2, 40, D), seed=s).to('cuda') for s in (7, 8))
    cos, sin = torch.ones((1, T, D), device='cuda'), torch.zeros((1, T, D), device='cuda')
    q = torch.randn((2, 2, T, D), device='cuda').to(BF)
    cache = cache_of()
    cache.update(k, v, 0)
    good = (q, k[:, :, :T], v[:, :, :T], cos, sin, 0)
    for wrong in ((q, k[:, :1, :T], v[:, :1, :T], cos, sin, 0), (q[:1], k[:1, :, :T], v[:1, :, :T], cos, sin, 0),
                  (q[..., :32], k[:, :, :T, :32], v[:, :, :T, :32], cos[..., :32], sin[..., :32], 0)):
        with pytest.raises(ValueError):
            cache.update_rotary(*wrong)
        assert cache.get_seq_length() == 40 and cache.layers[0]._res_k.length == cache.layers[0]._res_v.length == 40
        packed = cache_of()                                                              # (nothing but packed blocks)
        packed.update(*(x.repeat(1, 1, 4, 1)[:, :, :128] for x in (k, v)), 0)
        with pytest.raises(ValueError):
            packed.update_rotary(*wrong)
        assert packed.get_seq_length() == 128
    _, keys, _ = cache.update_rotary(*good)
    assert torch.equal(keys, torch.cat([k, k[:, :, :T]], 2))
    with torch.inference_mode():
        inner = cache_of()
        inner.update(k, v, 0)
    with pytest.raises(RuntimeError, match='inference'):
        inner.update_rotary(*good)
    assert inner.get_seq_length() == 40 and inner.layers[0]._res_k.length == 40
    with torch.inference_mode():
        _, keys, _ = inner.update_rotary(*good)
    assert torch.equal(keys, torch.cat([k, k[:, :, :T]], 2))


@pytest.mark.parametrize('dtype', [torch.float16, torch.float32, BF])
def test_other_types_through_the_cache(dtype):
    """Queries of a model in another type come back in it; they are rounded to bf16, as keys and values are, on their way."""
    B, Hq, Hkv, D, T = 1, 4, 2, 64, 5
    k, v = (synth.kv_tensor((B, Hkv, 70, D), seed=s).to('cuda') for s in (9, 10))
    q = torch.randn((B, Hq, T, D), device='cuda').to(dtype)
    c, s = oracle.angles(torch.arange(70 - T, 70), D // 2)
    cos, sin = (torch.cat([x, x], -1).float().cuda()[None] for x in (c, s))
    cache, same = cache_of(), cache_of()
    for x in (cache, same):
        x.update(k[:, :, :-T], v[:, :, :-T], 0)
    rq, _, _ = cache.update_rotary(q, k[:, :, -T:].to(dtype), v[:, :, -T:].to(dtype), cos, sin, 0)
    want, _, _ = same.update_rotary(q.to(BF), k[:, :, -T:], v[:, :, -T:], cos, sin, 0)
    assert rq.dtype == dtype and torch.equal(rq, want.to(dtype))
    got = cache.layers[0].chunk_attention(rq)
    assert got.dtype == dtype and torch.equal(got, same.layers[0].chunk_attention(want).to(dtype))
    with pytest.raises(ValueError, match='floating'):
        cache.layers[0].chunk_attention(rq.int())
