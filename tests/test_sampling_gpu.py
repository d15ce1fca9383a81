"""The sampler against one row after the other in 64 bits."""
import math

import pytest
import torch

from tests import serving_oracle as oracle

pytestmark = pytest.mark.gpu
TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def check(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, **more):
    """Every row equal, but for rows whose draw lies within 1e-10 of the border of another outcome (64-bit sums of up to 2**18 weights:
    2**18 x 2**-53 = 3e-11 at worst)."""
    from adacode_b200 import sample_tokens
    got = sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p, **more).tolist()
    f = lambda x, b: x[b].item() if isinstance(x, torch.Tensor) else float(torch.tensor(x, dtype=torch.float32))   # noqa: E731
    for b in range(logits.shape[0]):
        want, near = oracle.sample(logits[b].cpu(), f(uniforms, b), f(temperature, b), int(f(top_k, b)), f(top_p, b), f(min_p, b))
        assert got[b] == want or near < 1e-10, (b, got[b], want, near)
    return got


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.3), dict(top_k=1), dict(top_k=7), dict(top_k=50, top_p=0.9), dict(top_p=0.5),
            dict(top_p=0.0), dict(top_p=0.95, min_p=0.01, temperature=1.7), dict(min_p=0.2), dict(min_p=1.0), dict(top_k=100000, top_p=0.999),
            dict(top_k=900, temperature=3.0), dict(top_k=3000, top_p=0.7, temperature=5.0)]


@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('V', [1, 2, 31, 257, 5000, 32000, 151936])
def test_sampling(V, dtype):
    g = torch.Generator('cpu').manual_seed(V)
    B = 7 if V < 10000 else 3
    for n, s in enumerate(SETTINGS):
        logits = (torch.randn((B, V), generator=g) * 2.5).to(TYPES[dtype]).cuda()
        check(logits, torch.rand(B, generator=g).cuda(), **s)


def test_settings_per_row():
    g = torch.Generator('cpu').manual_seed(3)
    B, V = 64, 3001
    logits = (torch.randn((B, V), generator=g) * 3).cuda()
    check(logits, torch.rand(B, generator=g).cuda(), temperature=torch.tensor([0.0, 0.5, 1.0, 2.0] * 16, device='cuda'),
          top_k=torch.tensor([0, 5, 40, 4000, -1, 1, 3001, 77] * 8, dtype=torch.int32, device='cuda'),
          top_p=torch.tensor([1.0, 0.9, 0.3, 0.0, 1.5, 0.99, 0.5, 0.8] * 8, device='cuda').roll(3),
          min_p=torch.tensor([0.0, 0.1, 0.0, 0.01] * 16, device='cuda').roll(1))


@pytest.mark.parametrize('s', [dict(top_k=3), dict(top_k=40), dict(top_p=0.5), dict(top_p=0.31, top_k=60), dict(min_p=0.9), dict()],
                         ids=lambda s: '-'.join(f'{k}{v}' for k, v in s.items()))
@pytest.mark.parametrize('V', [64, 1000, 40000])
def test_ties(V, s):
    """Rows of few different values: the lower tokens of a value stay."""
    g = torch.Generator('cpu').manual_seed(V)
    for values in (1, 2, 5):
        logits = torch.randint(0, values, (4, V), generator=g).float().cuda()
        u = torch.tensor([0.0, 0.25, 0.6, 1 - 2.0 ** -24], device='cuda')
        check(logits, u, **s)
        check((logits * 0.5 - 0.5).bfloat16(), u, **s)                              # minus zero and zero are one value
    signed = torch.zeros((1, V), device='cuda')
    signed[0, ::2] = -0.0
    assert check(signed, torch.zeros(1, device='cuda'), **s) == [0]


def test_forbidden_tokens_and_empty_rows():
    V = 1000
    logits = torch.randn((6, V), generator=torch.Generator('cpu').manual_seed(1)).cuda()
    logits[0] = -math.inf
    logits[1] = math.nan
    logits[2, :900] = -math.inf
    logits[3, 3:] = math.nan
    logits[4, 17], logits[4, 400] = math.inf, math.inf
    logits[5, 1:] = -math.inf
    for s in (dict(), dict(top_k=300), dict(top_p=0.99), dict(top_k=2000, top_p=0.9), dict(min_p=0.001), dict(temperature=0.0)):
        for u in (0.0, 0.3, 0.7, 1 - 2.0 ** -24):
            got = check(logits, torch.full((6,), u, device='cuda'), **s)
            assert got[0] == got[1] == -1 and got[2] >= 900 and 0 <= got[3] < 3 and got[4] in (17, 400) and got[5] == 0


def test_tiny_and_huge_temperatures():
    """Temperatures at which only the largest logits count, and at which all count alike."""
    g = torch.Generator('cpu').manual_seed(12)
    logits = torch.randn((4, 900), generator=g).cuda()
    logits[:, 100], logits[:, 700] = 9.0, 9.0
    logits[3] *= -1e30
    u = torch.tensor([0.0, 0.4, 0.6, 0.9], device='cuda')
    for t in (1e-45, 1e-38, 1e-20, 1e-6, 1e-3):
        for s in (dict(), dict(top_k=5), dict(top_p=0.9), dict(min_p=1.0)):
            got = check(logits, u, temperature=t, **s)
            assert got[:3] == [100, 100, 700]
    for s in (dict(), dict(top_k=100), dict(top_p=0.5)):
        check(logits[:3], u[:3], temperature=3e38, **s)


def test_distribution():
    """Even steps of the uniform number give every token its share, to within one step."""
    from adacode_b200 import sample_tokens
    n = 4096
    row = torch.tensor([0.3, -1.0, 2.0, 0.0, 1.0, -3.0, 0.5], device='cuda')
    u = (torch.arange(n, device='cuda') + 0.5) / n
    got = torch.bincount(sample_tokens(row.expand(n, 7), u, temperature=0.8), minlength=7).double().cpu() / n
    assert bool(((got - torch.softmax(row.double().cpu() / 0.8, 0)).abs() <= 1.0 / n).all())


def test_strides_out_streams_and_graphs():
    from adacode_b200 import sample_tokens
    g = torch.Generator('cpu').manual_seed(9)
    wide = torch.randn((5, 3, 777), generator=g).cuda()
    u = torch.rand(5, generator=g).cuda()
    check(wide[:, 1], u, top_k=20)                                                   # rows of a larger tensor
    check(wide[:, :, 5].t().contiguous().t(), u)                                     # no unit stride
    check(wide[:, 1, 3:], u, top_p=0.9)                                              # rows off every boundary
    check(wide[:, 1].bfloat16()[:, 1:], u, top_p=0.9)
    out = torch.zeros(5, dtype=torch.int64, device='cuda')
    want = check(wide[:, 1], u, top_k=20, out=out)
    assert out.tolist() == want
    logits, side = wide[:, 1].contiguous(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    k = torch.full((5,), 20, dtype=torch.int32, device='cuda')
    t = torch.ones(5, device='cuda')
    with torch.cuda.graph(graph):
        sample_tokens(logits, u, t, k, out=out)
    logits.copy_(wide[:, 2])
    u.copy_(torch.rand(5, generator=g))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph.replay()
    side.synchronize()
    assert out.tolist() == check(wide[:, 2], u, t, k)
    assert sample_tokens(logits[:0], u[:0]).shape == (0,)


def test_many_rows():
    g = torch.Generator('cpu').manual_seed(11)
    logits = (torch.randn((600, 513), generator=g) * 2).bfloat16().cuda()
    check(logits, torch.rand(600, generator=g).cuda(), top_k=40, top_p=0.9)


@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('scale', [0.01, 3.0, 9.0])
def test_nuclei_of_many_rows(scale, dtype):
    """Nuclei of a few tokens to most of the vocabulary; logits with a step that is coarse against the nucleus' end, and single heavy tokens."""
    g = torch.Generator('cpu').manual_seed(5)
    logits = torch.randn((12, 70001), generator=g) * scale
    logits[::3, 17] = logits[::3].amax(1) + 2.3
    logits = logits.to(TYPES[dtype]).cuda()
    for s in (dict(top_p=0.95, temperature=0.8), dict(top_p=0.6), dict(top_p=0.999, min_p=1e-4, temperature=1.5), dict(top_p=1e-6)):
        check(logits, torch.rand(12, generator=g).cuda(), **s)


@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
def test_masks_of_the_lowest_value(dtype):
    """Tokens masked by a type's lowest number instead of minus infinity: whole regions, and nearly all of the vocabulary."""
    g = torch.Generator('cpu').manual_seed(6)
    logits = (torch.randn((8, 50000), generator=g) * 3).to(TYPES[dtype]).cuda()
    lowest = torch.finfo(TYPES[dtype]).min
    logits[:3, 9000:48000] = lowest
    logits[3:6, torch.randperm(50000, generator=g)[:49970].cuda()] = lowest
    logits[6, 1:] = lowest
    logits[7] = lowest
    for s in (dict(top_k=50), dict(top_k=50, temperature=0.01), dict(top_k=400, top_p=0.9), dict(top_p=0.95), dict(min_p=0.01), dict(),
              dict(top_k=20, temperature=1e3)):
        check(logits, torch.rand(8, generator=g).cuda(), **s)


@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('V', [5000, 32000, 151936])
def test_few_neighbours_among_the_lowest_value(V, dtype):
    """Fewer tokens than top_k that are not masked by the type's lowest number, next to each other: inside one group of tokens that a thread takes
    at a time, across two, at the row's ends; their logits up to 20 apart, rising and falling."""
    g = torch.Generator('cpu').manual_seed(V)
    rows = []
    for n in (2, 3, 5, 10):
        for first in (0, 2, 1027, V - n):
            gap = (0.5, 2.0, 20.0)[len(rows) % 3]
            line = 10 - gap * torch.arange(n)
            row = torch.full((V,), torch.finfo(TYPES[dtype]).min)
            row[first:first + n] = line if len(rows) % 2 else line.flip(0)
            rows.append(row)
    logits = torch.stack(rows).to(TYPES[dtype]).cuda()
    for s in (dict(top_k=50), dict(top_k=400, temperature=4.0), dict(top_k=50, top_p=0.95), dict(top_k=50, temperature=0.05)):
        for u in (torch.rand(len(rows), generator=g), torch.full((len(rows),), 1 - 2.0 ** -24)):
            check(logits, u.cuda(), **s)


def test_draws_at_every_batch_size():
    """A row's token is what 64 bits give, whatever stands beside it: how many CTAs have a row changes the order of the sums alone."""
    from adacode_b200 import sample_tokens
    g = torch.Generator('cpu').manual_seed(13)
    row = (torch.randn((1, 40000), generator=g) * 3).cuda()
    u = torch.rand(1, generator=g).cuda()
    for s in (dict(), dict(top_p=0.9), dict(top_k=50, top_p=0.9), dict(min_p=0.01)):
        for B in (1, 40, 100, 400):
            f32 = {k: float(torch.tensor(v)) if isinstance(v, float) else v for k, v in s.items()}
            want, near = oracle.sample(row[0].cpu(), u.item(), **f32)
            assert near > 1e-10 and sample_tokens(row.expand(B, -1), u.expand(B).contiguous(), **s).tolist() == [want] * B
