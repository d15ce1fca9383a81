"""Rotated appends to a paged cache and attention over it, against 64 bits."""
import math

import pytest
import torch

from tests import serving_oracle as oracle

pytestmark = pytest.mark.gpu
I32 = torch.int32
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def close(got, want, size, dtype, length):
    """Weights are rounded to the type once (half a step each, over sums of |values| with weights 1), the result once; scores carry an
    fp32 dot product's error (128 products near 10 in all: 2**-24 x 128 x 10, below 2**-12 as a weight's relative error with that of exp2).
    fp16 weights below 2**-14 have fixed steps: half of 2**-24 each."""
    h = HALF[dtype]
    bound = h * want.abs() + (h + 2.0 ** -12) * (1 + h) * size + 1e-30
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25 * (length * size.amax(-1, keepdim=True) + 1)
    err = (got.double() - want).abs()
    worst = float((err / bound).max())
    assert worst <= 1.0, f'error {worst:.2f} times what rounding explains'


CASES = [
    # new tokens, cached tokens, Hq, Hkv, D, page, dtype, more
    ([1], [1], 1, 1, 64, 16, 'bf16', {}),
    ([1], [2051], 32, 8, 128, 16, 'bf16', {}),
    ([1, 1, 1], [17, 128, 129], 8, 2, 128, 16, 'bf16', {}),
    ([1] * 40, [3 * i + 1 for i in range(40)], 4, 4, 64, 32, 'fp16', {}),
    ([5, 3, 0, 1], [300, 3, 40, 1000], 32, 8, 128, 16, 'bf16', {}),
    ([16], [16], 16, 1, 128, 64, 'bf16', {}),
    ([9, 33], [200, 129], 7, 1, 128, 128, 'fp16', {}),
    ([33, 64], [40, 700], 20, 4, 128, 64, 'bf16', {}),
    ([130, 1, 77], [1500, 900, 77], 8, 2, 64, 32, 'bf16', {}),
    ([257], [2000], 8, 8, 128, 256, 'bf16', {}),
    ([300, 511], [300, 640], 12, 4, 128, 128, 'bf16', {}),
    ([509], [1021], 32, 8, 128, 128, 'bf16', {}),
    ([97, 60, 50], [700, 333, 999], 16, 4, 64, 32, 'fp16', {'window': 128}),
    ([40, 1], [900, 600], 8, 2, 128, 16, 'bf16', {'window': 1}),
    ([1, 1], [900, 60], 8, 2, 128, 16, 'bf16', {'window': 129}),
    ([64, 200], [400, 260], 8, 2, 128, 64, 'bf16', {'starts': [390, 0]}),
    ([64, 200], [64, 260], 8, 2, 64, 64, 'bf16', {'starts': [60, 260]}),
    ([1, 4], [500, 40], 8, 2, 128, 64, 'bf16', {'starts': [130, 37]}),
    ([64, 3], [400, 260], 8, 2, 128, 64, 'bf16', {'causal': False}),
    ([200], [333], 4, 2, 64, 64, 'fp16', {'causal': False, 'window': 50, 'starts': [100]}),
    ([70], [333], 4, 2, 64, 64, 'bf16', {'scale': 0.5}),
]
TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16}


def run_case(new, lens, Hq, Hkv, D, page, dtype, layout='phsd', fill=math.nan, seed=0, hint=True, **more):
    from adacode_b200 import paged_attention
    dtype = TYPES[dtype]
    k, v, table, seq = oracle.make_cache(lens, Hkv, D, page, dtype, seed=seed, fill=fill, layout=layout)
    q = torch.randn((sum(new), Hq, D), generator=torch.Generator('cpu').manual_seed(seed + 1)).to(dtype).cuda()
    want, size = oracle.attention(q, k, v, table, lens, new, **more)
    args = dict(more)
    if 'starts' in args:
        args['seq_starts'] = torch.tensor(args.pop('starts'), dtype=I32, device='cuda')
    if hint:
        args['max_query_len'] = max(new)
    got = paged_attention(q, k, v, table, seq, cu_seqlens=oracle.cumulative(new), **args)
    close(got, want, size, dtype, max(lens))
    return got


@pytest.mark.parametrize('case', CASES, ids=lambda c: f'{c[0][:3]}x{c[1][:3]}-{c[2]}/{c[3]}x{c[4]}-p{c[5]}-{c[6]}-{"-".join(c[7])}')
def test_attention(case):
    *shape, more = case
    run_case(*shape, **more)


@pytest.mark.parametrize('layout', ['phsd', 'pshd'])
@pytest.mark.parametrize('page', [16, 32, 64, 128, 384])
@pytest.mark.parametrize('T', [1, 70])
def test_attention_pages(page, layout, T):
    run_case([T, T, T], [T + 500, T, T + 129], 8, 2, 128, page, 'bf16', layout=layout, seed=page)


def test_attention_without_hint_and_lengths():
    """Without max_query_len and cu_seqlens the result is the same."""
    from adacode_b200 import paged_attention
    lens = [100, 30, 555]
    k, v, table, seq = oracle.make_cache(lens, 2, 128, 32, torch.bfloat16)
    q = torch.randn((12, 8, 128), device='cuda').bfloat16()
    want, size = oracle.attention(q, k, v, table, lens, [4, 4, 4])
    close(paged_attention(q, k, v, table, seq), want, size, torch.bfloat16, 555)
    close(paged_attention(q, k, v, table, seq, cu_seqlens=oracle.cumulative([4, 4, 4])), want, size, torch.bfloat16, 555)


@pytest.mark.parametrize('T', [1, 3, 150])
@pytest.mark.parametrize('cap', [37, 200, 1000])
def test_attention_one_page_per_sequence(T, cap):
    """A dense cache [B, H, cap, D] is one page per sequence; what lies behind a sequence has no influence."""
    from adacode_b200 import paged_attention
    T = min(T, cap)
    lens = [cap, max(T, cap // 2), T]
    dense = [torch.full((3, 2, cap, 64), math.nan, dtype=torch.bfloat16, device='cuda') for _ in range(2)]
    for x in dense:
        for b, n in enumerate(lens):
            x[b, :, :n] = torch.randn((2, n, 64), device='cuda').bfloat16()
    table = torch.arange(3, dtype=I32, device='cuda')[:, None]
    q = torch.randn((3 * T, 4, 64), device='cuda').bfloat16()
    want, size = oracle.attention(q, *dense, table, lens, [T] * 3)
    close(paged_attention(q, *dense, table, torch.tensor(lens, dtype=I32, device='cuda')), want, size, torch.bfloat16, cap)


@pytest.mark.parametrize('T', [1, 200])
def test_query_strides_and_out(T):
    from adacode_b200 import paged_attention
    lens = [T + 90, T + 300]
    k, v, table, seq = oracle.make_cache(lens, 2, 64, 64, torch.bfloat16)
    wide = torch.randn((2 * T, 3 * 8 * 64), device='cuda').bfloat16()          # queries inside a fused projection
    q = wide[:, 512:1024].view(2 * T, 8, 64)
    room = torch.full((2 * T, 16, 64), 7.0, dtype=torch.bfloat16, device='cuda')
    out = room[:, 4:12]
    want, size = oracle.attention(q, k, v, table, lens, [T, T])
    got = paged_attention(q, k, v, table, seq, out=out)
    assert got is out
    close(out, want, size, torch.bfloat16, max(lens))
    assert (room[:, :4] == 7).all() and (room[:, 12:] == 7).all()


@pytest.mark.parametrize('new', [[1, 1], [3, 40], [150, 1]])
def test_padding_behind_the_last_sequence_is_left_alone(new):
    from adacode_b200 import append_rotary, paged_attention
    lens = [n + 70 for n in new]
    k, v, table, seq = oracle.make_cache(lens, 2, 64, 16, torch.bfloat16)
    N = sum(new) + 5
    q = torch.randn((N, 4, 64), device='cuda').bfloat16()
    q[sum(new):] = math.nan
    out = torch.full_like(q, 7.0)
    paged_attention(q, k, v, table, seq, cu_seqlens=oracle.cumulative(new), out=out)
    want, size = oracle.attention(q, k, v, table, lens, new)
    close(out[:sum(new)], want[:sum(new)], size[:sum(new)], torch.bfloat16, max(lens))
    assert (out[sum(new):] == 7).all()
    rotated = torch.full_like(q, 7.0)
    kept = k.clone(), v.clone()
    c = torch.ones((N, 32), device='cuda')
    append_rotary(q[:, :2].contiguous(), q[:, 2:].contiguous(), c, 0 * c, k, v, table, seq, query=q, cu_seqlens=oracle.cumulative(new), out=rotated)
    assert (rotated[sum(new):] == 7).all()
    assert not torch.isnan(k).any() and not torch.equal(k, kept[0])


@pytest.mark.parametrize('T,G', [(1, 4), (5, 4), (140, 2)])
@pytest.mark.parametrize('bad', [math.inf, -math.inf, math.nan])
def test_hidden_infinities(T, G, bad):
    """Keys and values that nobody sees, or that only later tokens of the chunk see, have no influence on the others."""
    from adacode_b200 import paged_attention
    lens, starts = [T + 333], [150]
    k, v, table, seq = oracle.make_cache(lens, 2, 128, 64, torch.bfloat16, fill=bad)
    page = lambda at: (int(table[0, at // 64]), slice(None), at % 64)                    # noqa: E731
    for at in (0, 64, 149):                                                              # left padding, inside the first tile that counts too
        k[page(at)] = bad
        v[page(at)] = bad
    q = torch.randn((T, 2 * G, 128), device='cuda').bfloat16()
    args = dict(seq_starts=torch.tensor(starts, dtype=I32, device='cuda'))
    want, size = oracle.attention(q, k, v, table, lens, [T], starts=starts)
    assert torch.isfinite(want).all()
    close(paged_attention(q, k, v, table, seq, **args), want, size, torch.bfloat16, lens[0])
    if T > 1:                                                                            # the last token's value: seen by the last row alone
        at = lens[0] - 1
        v[page(at)[0], 0, page(at)[2], 5] = bad
        want, size = oracle.attention(q, k, v, table, lens, [T], starts=starts)
        got = paged_attention(q, k, v, table, seq, **args)
        odd = ~torch.isfinite(want)
        assert int(odd.sum()) == G and bool(odd[-1, :G, 5].all())
        assert torch.equal(got.double()[odd].nan_to_num(3.0), want[odd].nan_to_num(3.0))
        close(torch.where(odd, 0, got), torch.where(odd, 0.0, want), torch.where(odd, 1.0, size), torch.bfloat16, lens[0])


@pytest.mark.parametrize('T', [1, 150])
def test_seen_infinities(T):
    from adacode_b200 import paged_attention
    lens = [T + 200]
    k, v, table, seq = oracle.make_cache(lens, 1, 64, 64, torch.bfloat16)
    q = torch.randn((T, 2, 64), device='cuda').bfloat16()
    v[int(table[0, 0]), 0, 3, 7] = math.inf
    v[int(table[0, 1]), 0, 3, 9] = -math.inf
    v[int(table[0, 0]), 0, 3, 11] = math.nan
    v[int(table[0, 0]), 0, 4, 13], v[int(table[0, 0]), 0, 5, 13] = math.inf, -math.inf
    want, size = oracle.attention(q, k, v, table, lens, [T])
    got = paged_attention(q, k, v, table, seq).double()
    odd = ~torch.isfinite(want)
    assert int(odd.sum()) == 4 * 2 * T
    assert torch.equal(got[odd].nan_to_num(3.0), want[odd].nan_to_num(3.0))
    close(torch.where(odd, 0, got), torch.where(odd, 0.0, want), size, torch.bfloat16, lens[0])
    # a score that is NaN makes its row NaN, one that is minus infinity has no weight
    q[0, 0, 0] = math.nan
    got = paged_attention(q, k, v, table, seq)
    assert torch.isnan(got[0, 0]).all() and torch.isfinite(got[0, 1, 0])
    q = torch.zeros_like(q) + 1
    k[int(table[0, 0]), 0, :, 0] = -math.inf
    v = torch.randn_like(v)
    want, size = oracle.attention(q, k, v, table, lens, [T])
    close(paged_attention(q, k, v, table, seq), want, size, torch.bfloat16, lens[0])
    k[..., 0] = -math.inf
    assert (paged_attention(q, k, v, table, seq) == 0).all()


@pytest.mark.parametrize('T', [1, 140])
def test_large_values_do_not_overflow(T):
    """Sums of weights times values near the type's largest stay what their mean is."""
    from adacode_b200 import paged_attention
    lens = [T + 500]
    k, v, table, seq = oracle.make_cache(lens, 1, 128, 128, torch.bfloat16)
    v.fill_(3e38)
    q = torch.randn((T, 2, 128), device='cuda').bfloat16()
    want, size = oracle.attention(q, k, v, table, lens, [T])
    close(paged_attention(q, k, v, table, seq), want, size, torch.bfloat16, lens[0])


@pytest.mark.parametrize('T', [1, 200])
def test_growing_scores(T):
    """Running maxima that rise by much from tile to tile, and fall."""
    from adacode_b200 import paged_attention
    lens = [T + 1000]
    for order in (1, -1):
        k, v, table, seq = oracle.make_cache(lens, 1, 64, 128, torch.bfloat16)
        for n in range(lens[0] // 128 + 1):
            k[int(table[0, n])] *= 0.1
            k[int(table[0, n]), :, :, 0] = (2.0 if order > 0 else 18.0) + order * 2.0 * n
        q = torch.randn((T, 2, 64), device='cuda').bfloat16()
        q[:, 0, 0], q[:, 1, 0] = 30.0, -30.0
        want, size = oracle.attention(q, k, v, table, lens, [T])
        got = paged_attention(q, k, v, table, seq)
        # (scores reach 70: an fp32 dot product's error and log2(e)'s rounding are up to 2**-23 x 70 x 3 of a weight)
        err = (got.double() - want).abs() / (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12 + 2.0 ** -14) * size + 1e-30)
        assert float(err.max()) <= 1.0


def test_bad_pages_are_left_out_and_reported():
    from adacode_b200 import _lib, append_rotary, codec, paged_attention
    dev = torch.device('cuda', torch.cuda.current_device())
    codec.check_device_status(dev)
    lens = [100, 40]
    k, v, table, seq = oracle.make_cache(lens, 2, 64, 16, torch.bfloat16)
    q = torch.randn((4, 4, 64), device='cuda').bfloat16()
    good = paged_attention(q, k, v, table, seq)
    for wrong in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        broken = table.clone()
        broken[0, 2] = wrong
        got = paged_attention(q, k, v, broken, seq)
        assert torch.equal(got[2:], good[2:])
        with pytest.raises(_lib.AdacodeError, match='no page'):
            codec.check_device_status(dev)
    x, c = torch.randn((4, 2, 64), device='cuda').bfloat16(), torch.ones((4, 32), device='cuda')
    broken = table.clone()
    broken[0, 6] = -1                                                                    # tokens 98 and 99 lie there
    before = k.clone(), v.clone()
    append_rotary(x, x, c, 0 * c, k, v, broken, seq)
    changed = (k != before[0]).flatten(1).any(1).nonzero().flatten().tolist()
    assert changed == [int(table[1, 2])]
    with pytest.raises(_lib.AdacodeError, match='no page'):
        codec.check_device_status(dev)
    long = seq.clone()
    long[0] = 500                                                                        # behind the table
    paged_attention(q, k, v, table, long)
    append_rotary(x, x, c, 0 * c, k, v, table, long)
    with pytest.raises(_lib.AdacodeError, match='no page'):
        codec.check_device_status(dev)
    short = seq.clone()
    short[0] = 1                                                                         # fewer cached than new tokens
    assert (paged_attention(q, k, v, table, short)[0] == 0).all()
    short[0] = 0
    assert (paged_attention(q, k, v, table, short)[:2] == 0).all()
    assert torch.equal(paged_attention(q, k, v, table, short)[2:], paged_attention(q, k, v, table, seq)[2:])
    codec.check_device_status(dev)


def test_long_cache_offsets():
    """Pages beyond 2**31 elements from the pool's begin."""
    from adacode_b200 import append_rotary, paged_attention
    P = (1 << 31) // (8 * 128 * 128) + 40
    pool = torch.empty((2, P, 8, 128, 128), dtype=torch.bfloat16, device='cuda')         # 8.8 GB
    k, v = pool[0], pool[1]
    lens, new = [300, 140], [3, 140]
    table = torch.tensor([[P - 1, 3, P - 7], [P - 2, P - 3, 0]], dtype=I32, device='cuda')
    for p in (P - 1, 3, P - 7, P - 2, P - 3):
        k[p], v[p] = torch.randn((8, 128, 128), device='cuda').bfloat16(), torch.randn((8, 128, 128), device='cuda').bfloat16()
    q = torch.randn((143, 16, 128), device='cuda').bfloat16()
    seq, cu = torch.tensor(lens, dtype=I32, device='cuda'), oracle.cumulative(new)
    x = torch.randn((143, 8, 128), device='cuda').bfloat16()
    cos, sin = (t.float().cuda() for t in oracle.angles(torch.arange(143), 64))
    append_rotary(x, x, cos, sin, k, v, table, seq, cu_seqlens=cu)
    assert torch.equal(v[P - 2, :, :128].transpose(0, 1), x[3:131]) and torch.equal(v[P - 7, :, 41:44].transpose(0, 1), x[:3])
    want, size = oracle.attention(q, k, v, table, lens, new)
    close(paged_attention(q, k, v, table, seq, cu_seqlens=cu), want, size, torch.bfloat16, 300)


# ---------------------------------------------------------------------------------------- append

APPENDS = [
    # new, lens, Hq, Hkv, D, page, R, interleaved, axes, dtype, angles
    ([1], [1], 1, 1, 64, 16, 64, False, 1, 'bf16', torch.float32),
    ([1] * 33, [7 * i + 1 for i in range(33)], 32, 8, 128, 16, 128, False, 1, 'bf16', torch.bfloat16),
    ([3, 0, 50], [20, 9, 50], 8, 2, 128, 16, 96, False, 3, 'bf16', torch.float32),
    ([40, 7], [140, 7], 5, 1, 64, 37, 32, True, 1, 'fp16', torch.float16),
    ([40, 7], [140, 70], 6, 3, 64, 64, 48, True, 3, 'fp16', torch.float32),
    ([9], [30], 2, 2, 80, 16, 20, False, 1, 'bf16', torch.float32),              # ten angles: column by column
    ([9], [30], 2, 2, 66, 8, 66, True, 2, 'bf16', torch.float32),
    ([9], [30], 2, 2, 72, 8, 0, False, 1, 'bf16', torch.float32),                # nothing to rotate
    ([200], [1000], 0, 4, 256, 128, 256, False, 1, 'bf16', torch.float32),       # keys and values only
    ([11], [1000], 4, 4, 512, 128, 512, True, 4, 'bf16', torch.bfloat16),
]


@pytest.mark.parametrize('layout', ['phsd', 'pshd'])
@pytest.mark.parametrize('case', APPENDS, ids=lambda c: f'{c[0][:3]}-{c[2]}/{c[3]}x{c[4]}-p{c[5]}-r{c[6]}-{c[7]}-{c[8]}-{c[9]}')
def test_append(case, layout):
    from adacode_b200 import append_rotary
    new, lens, Hq, Hkv, D, page, R, interleaved, axes, dtype, angle_type = case
    dtype, N, half = TYPES[dtype], sum(new), R // 2
    k, v, table, seq = oracle.make_cache(lens, Hkv, D, page, dtype, layout=layout)
    g = torch.Generator('cpu').manual_seed(5)
    q, key, value = (torch.randn((N, h, D), generator=g).to(dtype).cuda() for h in (max(Hq, 1), Hkv, Hkv))
    at = torch.cat([torch.arange(n - m, n) for m, n in zip(new, lens)])
    positions = at if axes == 1 else torch.stack([(at * (a + 3)) % 97 for a in range(axes)])
    sections = None if axes == 1 else [half - (axes - 1) * (half // (axes + 1))] + [half // (axes + 1)] * (axes - 1)
    cos, sin = (t.to(angle_type).cuda() for t in oracle.angles(positions, half))
    want_k, want_v = k.double(), v.double()
    cs, sn = (cos, sin) if axes == 1 else (oracle.select_axes(t, sections) for t in (cos, sin))
    rk, rq = (oracle.rotate(t, cs, sn, interleaved) for t in (key, q))
    i = 0
    for b, (m, n) in enumerate(zip(new, lens)):
        for t in range(n - m, n):
            want_k[int(table[b, t // page]), :, t % page] = rk[i]
            want_v[int(table[b, t // page]), :, t % page] = value[i].double()
            i += 1
    got = append_rotary(key, value, cos, sin, k, v, table, seq, query=q if Hq else None, cu_seqlens=oracle.cumulative(new), sections=sections,
                        interleaved=interleaved)
    assert torch.equal(v.double(), want_v)

    def near(x, want, source):
        # one rounding of the result, and of each of two products and their sum in 32 bits
        top = source.double().abs().amax()
        assert bool(((x.double() - want).abs() <= HALF[dtype] * want.abs() + 3 * 2.0 ** -24 * top * (1 + HALF[dtype]) * 2 + 2.0 ** -25).all())
    near(k, want_k, key)
    if Hq:
        near(got, rq, q)
    else:
        assert got is None


def test_append_in_place_strided_and_hf_angles():
    """Queries and keys inside one projection, rotated in place; angles as a HF model hands them on, every one twice."""
    from adacode_b200 import append_rotary
    lens = [130, 140]
    k, v, table, seq = oracle.make_cache(lens, 2, 128, 64, torch.bfloat16)
    wide = torch.randn((6, 12, 128), device='cuda').bfloat16()
    q, key, value = wide[:, :8], wide[:, 8:10], wide[:, 10:]
    cos, sin = (torch.cat([t, t], -1).bfloat16().cuda().view(2, 3, 128) for t in oracle.angles(torch.tensor([127, 128, 129, 137, 138, 139]), 64))
    rq, rk = (oracle.rotate(t, cos.view(6, 128)[:, :64], sin.view(6, 128)[:, :64]) for t in (q, key))
    tail = wide[:, 8:].clone()
    got = append_rotary(key, value, cos.view(6, 128)[:, :64], sin.view(6, 128)[:, :64], k, v, table, seq, query=q, out=q)
    assert got is q and torch.equal(wide[:, 8:], tail)
    assert bool(((q.double() - rq).abs() <= 2.0 ** -8 * rq.abs() + 1e-5).all())
    at = k[int(table[1, 2]), :, 9:12].transpose(0, 1).double()
    assert bool(((at - rk[3:]).abs() <= 2.0 ** -8 * rk[3:].abs() + 1e-5).all())


# ---------------------------------------------------------------------------------------- streams, graphs, devices

def test_streams_and_replayed_graphs():
    """Calls on two streams at once, and two captured graphs replayed with other lengths, tables and contents."""
    from adacode_b200 import paged_attention
    shapes = [([1, 1, 1], [2000, 800, 90]), ([150, 33], [1500, 700])]
    states = []
    for n, (new, lens) in enumerate(shapes):
        k, v, table, seq = oracle.make_cache(lens, 4, 128, 64, torch.bfloat16, seed=n)
        q = torch.randn((sum(new), 16, 128), device='cuda').bfloat16()
        out = torch.zeros_like(q)
        states.append((q, k, v, table, seq, oracle.cumulative(new), max(new), out, new, lens))

    def call(s):
        return paged_attention(s[0], s[1], s[2], s[3], s[4], cu_seqlens=s[5], max_query_len=s[6], out=s[7])
    wants = [call(s).clone() for s in states]
    graphs = []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(s)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    for _ in range(20):
        for s in states:
            s[7].zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s[7], w) for s, w in zip(states, wants))
        for s in states:
            s[7].zero_()
        torch.cuda.synchronize()
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                call(s)
        torch.cuda.synchronize()
        assert all(torch.equal(s[7], w) for s, w in zip(states, wants))
    # other lengths under the same graph
    s = states[0]
    s[4].copy_(torch.tensor([700, 90, 33], dtype=I32))
    s[1].normal_()
    want, size = oracle.attention(s[0], s[1], s[2], s[3], [700, 90, 33], s[8])
    graphs[0].replay()
    close(s[7], want, size, torch.bfloat16, 700)


def test_repeated_calls_give_the_same_bits():
    from adacode_b200 import paged_attention
    lens = [3000, 100, 1700]
    k, v, table, seq = oracle.make_cache(lens, 2, 128, 16, torch.bfloat16)
    for T in (1, 50):
        q = torch.randn((3 * T, 8, 128), device='cuda').bfloat16()
        first = paged_attention(q, k, v, table, seq)
        for _ in range(5):
            assert torch.equal(paged_attention(q, k, v, table, seq), first)


def test_strides_of_single_entries_do_not_matter():
    """Dimensions of one entry with strides that no alignment allows."""
    from adacode_b200 import append_rotary, paged_attention
    storage = torch.randn(1 << 16, device='cuda').bfloat16()
    k, v = (storage[o:].as_strided((1, 1, 128, 64), (7, 13, 64, 1)) for o in (0, 1 << 14))
    q = storage[1 << 15:].as_strided((1, 1, 64), (5, 3, 1))
    table, seq = torch.zeros((1, 1), dtype=I32, device='cuda'), torch.tensor([100], dtype=I32, device='cuda')
    want, size = oracle.attention(q, k, v, table, [100], [1])
    close(paged_attention(q, k, v, table, seq), want, size, torch.bfloat16, 100)
    x, c = q.clone(), torch.ones((1, 32), device='cuda')
    append_rotary(x, x, c, 0 * c, k, v, table, seq)
    assert torch.equal(v[0, 0, 99], x[0, 0]) and torch.equal(k[0, 0, 99], x[0, 0])


def test_inference_mode_and_grad_mode():
    from adacode_b200 import append_rotary, paged_attention
    k, v, table, seq = oracle.make_cache([20], 2, 64, 16, torch.bfloat16)
    x, c = torch.randn((1, 2, 64), device='cuda').bfloat16(), torch.ones((1, 32), device='cuda')
    with torch.inference_mode():
        ki, vi = k.clone(), v.clone()
        append_rotary(x, x, c, 0 * c, ki, vi, table, seq, query=x)
        got = paged_attention(x, ki, vi, table, seq)
    with pytest.raises(RuntimeError, match='inference'):
        append_rotary(x, x, c, 0 * c, ki, vi, table, seq)
    append_rotary(x, x, c, 0 * c, k, v, table, seq)
    assert torch.equal(paged_attention(x, k, v, table, seq), got)
    with pytest.raises(RuntimeError, match='backward'):
        append_rotary(x.clone().requires_grad_(), x, c, 0 * c, k, v, table, seq)
    with pytest.raises(ValueError, match='is on cpu'):
        paged_attention(x, k, v, table, seq.cpu())


def test_many_sequences_and_heads_per_group():
    """More sequences than a warp has lanes, some without new tokens; many query heads on one cached head."""
    g = torch.Generator('cpu').manual_seed(4)
    new = [int(n) for n in torch.randint(0, 4, (200,), generator=g)]
    lens = [n + int(m) for n, m in zip(new, torch.randint(0, 300, (200,), generator=g))]
    run_case(new, [max(n, 1) for n in lens], 4, 2, 64, 32, 'bf16')
    run_case([3, 1], [500, 200], 96, 1, 128, 64, 'bf16')
    run_case([1, 1], [300, 200], 300, 1, 64, 64, 'fp16')


def test_versions_are_counted():
    from adacode_b200 import append_rotary
    k, v, table, seq = oracle.make_cache([20], 2, 64, 16, torch.bfloat16)
    x, c = torch.randn((1, 2, 64), device='cuda').bfloat16(), torch.ones((1, 32), device='cuda')
    before = k._version, v._version
    append_rotary(x, x, c, c, k, v, table, seq)
    assert k._version > before[0] and v._version > before[1]


@pytest.mark.parametrize('T', [1, 140])
def test_scale_zero(T):
    """All that is seen has the same weight, and what is hidden still has none."""
    run_case([T, T], [T + 70, T + 301], 8, 2, 128, 64, 'bf16', scale=0.0, starts=[3, 0])
    run_case([T], [T + 301], 8, 2, 64, 64, 'fp16', scale=0.0, window=40)
    run_case([T], [T + 301], 8, 2, 64, 64, 'bf16', scale=-0.3)


@pytest.mark.parametrize('T', [1, 140])
def test_windows_and_lengths_beyond_32_bits(T):
    from adacode_b200 import codec, paged_attention
    lens = [T + 200]
    k, v, table, seq = oracle.make_cache(lens, 2, 64, 64, torch.bfloat16)
    q = torch.randn((T, 4, 64), device='cuda').bfloat16()
    want = paged_attention(q, k, v, table, seq, max_query_len=T)
    for window in (2 ** 31 - 1, 2 ** 32 + 5):
        assert torch.equal(paged_attention(q, k, v, table, seq, max_query_len=T, window=window), want)
    close(paged_attention(q, k, v, table, seq, max_query_len=2 ** 32 + T), *oracle.attention(q, k, v, table, lens, [T]), torch.bfloat16, lens[0])
    # fewer cached than new tokens, and everything left padding: nothing is seen
    few, starts = torch.zeros_like(seq), torch.full_like(seq, 2 ** 31 - 1)
    for window in (0, 3, 2 ** 31 - 1):
        assert (paged_attention(q, k, v, table, few, seq_starts=starts, window=window, causal=False) == 0).all()
        assert (paged_attention(q, k, v, table, seq, seq_starts=starts, window=window) == 0).all()
    codec.check_device_status(q.device)


@pytest.mark.parametrize('first', [1, 4, 70])
def test_tokens_before_the_first_sequence_are_left_alone(first):
    """cu_seqlens[0] above 0: what is before it is of no sequence, like what is behind the last."""
    from adacode_b200 import append_rotary, paged_attention
    new, lens = [3, 40], [90, 75]
    k, v, table, seq = oracle.make_cache(lens, 2, 64, 16, torch.bfloat16)
    N = first + sum(new) + 2
    q = torch.randn((N, 4, 64), device='cuda').bfloat16()
    cu = oracle.cumulative(new) + first
    out = torch.full_like(q, 7.0)
    paged_attention(q, k, v, table, seq, cu_seqlens=cu, out=out)
    mine = slice(first, first + sum(new))
    want, size = oracle.attention(q[mine], k, v, table, lens, new)
    close(out[mine], want, size, torch.bfloat16, max(lens))
    rotated, c = torch.full_like(q, 7.0), torch.ones((N, 32), device='cuda')
    want_k, want_v = k.clone(), v.clone()
    append_rotary(q[mine, :2], q[mine, 2:], c[mine], 0 * c[mine], want_k, want_v, table, seq, cu_seqlens=oracle.cumulative(new))
    append_rotary(q[:, :2], q[:, 2:], c, 0 * c, k, v, table, seq, query=q, cu_seqlens=cu, out=rotated)
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    assert torch.equal(rotated[mine], q[mine])
    for x in (out, rotated):
        assert (x[:first] == 7).all() and (x[mine.stop:] == 7).all()


def test_threads_share_a_stream_and_a_workspace():
    """C callers of different kernels (types, head sizes, steps and chunks) from four threads: no call's launches come between another's two."""
    import ctypes
    import threading
    from adacode_b200 import _lib, codec, paged_attention
    L = _lib.lib()
    shapes = [([1, 1], [3000, 900], 128, 'bf16'), ([150, 33], [1500, 700], 128, 'fp16'), ([150, 9], [1700, 400], 64, 'bf16'), ([1, 2], [2000, 1100], 64, 'fp16')]
    workspace = torch.empty(max(L.adacode_paged_attn_workspace_bytes(256, 16, 4, 128), L.adacode_paged_attn_workspace_bytes(1, 16, 4, 128)), dtype=torch.uint8,
                            device='cuda')
    status, stream = codec.device_status(workspace.device), torch.cuda.current_stream().cuda_stream
    calls = []
    for n, (new, lens, D, dtype) in enumerate(shapes):
        k, v, table, seq = oracle.make_cache(lens, 4, D, 64, TYPES[dtype], seed=n)
        q, cu = torch.randn((sum(new), 16, D), device='cuda').to(TYPES[dtype]), oracle.cumulative(new)
        want, outs = paged_attention(q, k, v, table, seq, cu_seqlens=cu, max_query_len=max(new)), [torch.zeros_like(q) for _ in range(50)]
        c = _lib.PagedCache(k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3], table.data_ptr(), table.stride(0), seq.data_ptr(), cu.data_ptr(),
                            table.shape[1], 2, k.shape[0], 64, 4, D, {'bf16': _lib.BF16, 'fp16': _lib.FP16}[dtype], sum(new))
        calls.append((c, q, max(new), D ** -0.5, want, outs, (k, v, table, seq, cu)))
    torch.cuda.synchronize()
    codes, start = [], threading.Barrier(4)

    def work(c, q, longest, scale, want, outs, held):
        torch.cuda.set_device(workspace.device)
        start.wait()
        for out in outs:
            codes.append(L.adacode_paged_attn(ctypes.byref(c), q.data_ptr(), *q.stride()[:2], 16, out.data_ptr(), *out.stride()[:2], None, longest, scale, 1, 0,
                                              workspace.data_ptr(), workspace.numel(), status.data_ptr(), stream))
    threads = [threading.Thread(target=work, args=x) for x in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert codes == [_lib.OK] * 200
    assert all(torch.equal(out, x[4]) for x in calls for out in x[5])
    codec.check_device_status(workspace.device)


@pytest.mark.parametrize('page', [16, 128])
@pytest.mark.parametrize('T', [1, 3, 140])
def test_hidden_pages_need_no_entry(T, page):
    """Pages before the window and inside the left padding may have been given back: their entries are no pages, and nothing is reported."""
    from adacode_b200 import _lib, codec, paged_attention
    lens = [T + 700, T + 390]
    k, v, table, seq = oracle.make_cache(lens, 2, 64, page, torch.bfloat16, fill=math.nan)
    q = torch.randn((2 * T, 8, 64), device='cuda').bfloat16()
    starts = torch.tensor([0, 300], dtype=I32, device='cuda')
    codec.check_device_status(q.device)
    for more, hidden in ((dict(window=60), [700 - 59, 390 - 59]), (dict(starts=[0, 300]), [0, 300]), (dict(window=150, starts=[0, 300]), [700 - 149, 300])):
        args = {('seq_starts' if n == 'starts' else n): (starts if n == 'starts' else x) for n, x in more.items()}
        want, size = oracle.attention(q, k, v, table, lens, [T, T], **more)
        for gone in (-1, k.shape[0]):
            partly = table.clone()
            for b, n in enumerate(hidden):
                partly[b, :n // page] = gone
            close(paged_attention(q, k, v, partly, seq, max_query_len=T, **args), want, size, torch.bfloat16, max(lens))
            codec.check_device_status(q.device)
            partly[0, hidden[0] // page] = gone                                          # one more: a page that is seen
            paged_attention(q, k, v, partly, seq, max_query_len=T, **args)
            with pytest.raises(_lib.AdacodeError, match='no page'):
                codec.check_device_status(q.device)


def milliseconds(call, times=5):
    """The least of some times on the device."""
    call()
    taken = []
    for _ in range(times):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        b.synchronize()
        taken.append(a.elapsed_time(b))
    return min(taken)


@pytest.mark.parametrize('T', [1, 5, 200])
def test_infinities_in_left_padding_cost_nothing(T):
    """What every row of a sequence's new tokens is kept from seeing (padding, what lies before all windows) is out of the way before it is multiplied:
    a model's padding may hold NaN in every layer.  (The bound is far above what a call's time varies by: computed again row by row such a
    call took 80 to 500 times as long.)"""
    from adacode_b200 import codec, paged_attention
    B, L = 2, 4000
    k, v = (torch.randn((B, 8, L, 128), device='cuda').bfloat16() for _ in range(2))
    table, seq = torch.arange(B, dtype=I32, device='cuda')[:, None], torch.full((B,), L, dtype=I32, device='cuda')
    q = torch.randn((B * T, 32, 128), device='cuda').bfloat16()
    for more in (dict(seq_starts=torch.tensor([100, 1000], dtype=I32, device='cuda')), dict(window=1500)):
        call = lambda: paged_attention(q, k, v, table, seq, max_query_len=T, **more)     # noqa: E731, B023
        want, plain = call(), milliseconds(call)
        odd = v.clone()
        for b, n in enumerate([100, 1000] if 'window' not in more else [L - T - 1500 + 1] * B):
            odd[b, :, :n] = math.nan
        v, kept = odd, v
        assert torch.equal(call(), want)
        spoilt = milliseconds(call)
        v = kept
        assert spoilt < 5 * plain + 0.05, (spoilt, plain)
    codec.check_device_status(q.device)


@pytest.mark.parametrize('T', [1, 200])
def test_scaled_scores_beyond_32_bits(T):
    """A score that is finite but whose product with the scale is not counts as an infinite one: no number where it is the largest, no weight
    where it is negative."""
    from adacode_b200 import paged_attention
    lens = [T + 300]
    k, v, table, seq = oracle.make_cache(lens, 1, 64, 64, torch.bfloat16)
    q = torch.zeros((T, 2, 64), dtype=torch.bfloat16, device='cuda')
    q[:, 0, 0], q[:, 1, 0] = 1.0, -1.0
    at = (int(table[0, 1]), 0, 3)
    k[..., 0] = 0.0
    k[at[0], at[1], at[2], 0] = 2.0 ** 120
    for sign in (1.0, -1.0):
        got = paged_attention(q, k, v, table, seq, scale=sign * 2.0 ** 10)
        up, down = (0, 1) if sign > 0 else (1, 0)
        assert torch.isnan(got[:, up]).all()
        hidden = k.clone()
        hidden[at] = 0.0
        hidden[at[0], at[1], at[2], 0] = math.inf                                        # whose score of `down`, in 64 bits too, is minus infinity
        want, size = oracle.attention(q[:, down:down + 1], hidden, v, table, lens, [T], scale=sign * 2.0 ** 10)
        close(got[:, down:down + 1], want, size, torch.bfloat16, lens[0])
    k[..., 0] = 2.0 ** 120
    got = paged_attention(q, k, v, table, seq, scale=2.0 ** 10)
    assert torch.isnan(got[:, 0]).all() and (got[:, 1] == 0).all()


def test_outputs_that_overlap_themselves_are_refused():
    from adacode_b200 import append_rotary, paged_attention
    k, v, table, seq = oracle.make_cache([20, 9], 2, 64, 16, torch.bfloat16)
    q, x, c = torch.randn((4, 4, 64), device='cuda').bfloat16(), torch.randn((4, 2, 64), device='cuda').bfloat16(), torch.ones((4, 32), device='cuda')
    out = torch.zeros((1, 4, 64), dtype=torch.bfloat16, device='cuda').expand(4, 4, 64)
    with pytest.raises(ValueError, match='overlap'):
        paged_attention(q, k, v, table, seq, out=out)
    with pytest.raises(ValueError, match='overlap'):
        append_rotary(x, x, c, c, k, v, table, seq, query=q, out=out)
    with pytest.raises(ValueError, match='overlap'):
        append_rotary(x, x, c, c, k, v[:, :1].expand(v.shape), table, seq)
    assert (out == 0).all()
    # pages that are only read may
    got = paged_attention(q, k, v, table, seq)
    assert torch.isfinite(got).all()
