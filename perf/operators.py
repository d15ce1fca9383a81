"""The operators of a serving step as measurable cases: new tokens are rotated and appended to a paged cache, attend to
it, and the logits that come of it are sampled.

Kinds of work (``case['kind']``):

``append``  ``adacode_b200.append_rotary``: queries and keys of new tokens are rotated by their positions (one axis, or three for
            images and video), keys and values go to the pages that hold their positions.
``attend``  ``adacode_b200.paged_attention``: a chunk of new tokens of each sequence attends to the sequence's pages, itself
            included; one token per sequence is a decode step.
``sample``  ``adacode_b200.sample_tokens``: one token per row of logits from a given uniform number, after temperature, top-k,
            top-p and min-p.

A paged cache here is ``pages [P, Hkv, page, D]`` for keys and for values, and ``block_table [B, W]`` of page numbers; sequences
have different lengths, their pages lie in any order.  ``run`` computes a case by elementary torch operations, or through the package
where ``own`` is set.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def listed() -> list:
    return [
        # a decode step of one conversation: the smallest call, launches and latency count
        {'name': 'attend_step', 'kind': 'attend', 'B': 1, 'T': 1, 'S': 2051, 'Hq': 32, 'Hkv': 8, 'D': 128, 'page': 16, 'window': 0,
         'padded': False, 'dtype': 'bf16'},
        # a decode step of a serving batch of all lengths: bound by reading the cache
        {'name': 'attend_step_batch', 'kind': 'attend', 'B': 64, 'T': 1, 'S': 8192, 'Hq': 32, 'Hkv': 8, 'D': 128, 'page': 64, 'window': 0,
         'padded': False, 'dtype': 'bf16'},
        # five drafted tokens of each of sixteen sequences are verified
        {'name': 'attend_verify', 'kind': 'attend', 'B': 16, 'T': 5, 'S': 4523, 'Hq': 32, 'Hkv': 8, 'D': 128, 'page': 16, 'window': 0,
         'padded': False, 'dtype': 'bf16'},
        # the next turn of a conversation behind a long prompt
        {'name': 'attend_turn', 'kind': 'attend', 'B': 1, 'T': 509, 'S': 20557, 'Hq': 32, 'Hkv': 8, 'D': 128, 'page': 128, 'window': 0,
         'padded': False, 'dtype': 'bf16'},
        # a chunk of two long prompts: the largest, bound by the products
        {'name': 'attend_prefill', 'kind': 'attend', 'B': 2, 'T': 2048, 'S': 16384, 'Hq': 32, 'Hkv': 8, 'D': 128, 'page': 128, 'window': 0,
         'padded': False, 'dtype': 'bf16'},
        # a small model's heads, left-padded prompts, a sliding window
        {'name': 'attend_heads64', 'kind': 'attend', 'B': 8, 'T': 97, 'S': 1664, 'Hq': 16, 'Hkv': 4, 'D': 64, 'page': 32, 'window': 512,
         'padded': True, 'dtype': 'fp16'},
        # the tokens of one decode step of a batch: latency
        {'name': 'append_step', 'kind': 'append', 'B': 32, 'T': 1, 'S': 4146, 'Hq': 32, 'Hkv': 8, 'D': 128, 'page': 16, 'rotary': 128,
         'axes': 1, 'interleaved': False, 'dtype': 'bf16', 'angles': 'bf16'},
        # chunks of prompts with images: positions of three axes, a quarter of the columns not rotated
        {'name': 'append_images', 'kind': 'append', 'B': 3, 'T': 1201, 'S': 2901, 'Hq': 16, 'Hkv': 2, 'D': 128, 'page': 64, 'rotary': 96,
         'axes': 3, 'interleaved': False, 'dtype': 'bf16', 'angles': 'fp32'},
        # two long prompts at once: bound by memory
        {'name': 'append_prompt', 'kind': 'append', 'B': 2, 'T': 8192, 'S': 8192, 'Hq': 32, 'Hkv': 8, 'D': 128, 'page': 128, 'rotary': 128,
         'axes': 1, 'interleaved': True, 'dtype': 'bf16', 'angles': 'fp32'},
        # one conversation's next token
        {'name': 'sample_one', 'kind': 'sample', 'B': 1, 'V': 32000, 'top_k': 50, 'top_p': 1.0, 'min_p': 0.0, 'temperature': 1.0, 'dtype': 'bf16'},
        # a serving batch with the usual settings
        {'name': 'sample_batch', 'kind': 'sample', 'B': 64, 'V': 128256, 'top_k': 50, 'top_p': 0.9, 'min_p': 0.0, 'temperature': 0.7, 'dtype': 'fp32'},
        # many samples of a warm distribution: the nucleus holds most of the vocabulary
        {'name': 'sample_warm', 'kind': 'sample', 'B': 192, 'V': 151936, 'top_k': 0, 'top_p': 0.95, 'min_p': 0.001, 'temperature': 1.3, 'dtype': 'bf16'},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(('attend', 'attend', 'append', 'sample'))
    if kind == 'sample':
        V = _log_int(rng, 100, 262144)
        return {'kind': kind, 'B': _log_int(rng, 1, max(1, min(512, 25_000_000 // V))), 'V': V, 'top_k': rng.choice((0, 0, 1, 20, 50, 400)),
                'top_p': rng.choice((1.0, 0.5, 0.8, 0.95)), 'min_p': rng.choice((0.0, 0.0, 0.05, 0.001)),
                'temperature': rng.choice((0.0, 0.3, 0.7, 1.0, 1.5)), 'dtype': rng.choice(('bf16', 'fp16', 'fp32'))}
    Hkv = rng.choice((1, 2, 4, 8))
    Hq = Hkv * rng.choice((1, 2, 4, 5, 7, 8))
    page = rng.choice((16, 32, 64, 128, 256))
    dtype = rng.choice(('bf16', 'bf16', 'fp16'))
    if kind == 'append':
        D = rng.choice((64, 128))
        N = _log_int(rng, 1, 400_000 // Hq)
        B = min(N, _log_int(rng, 1, 64))
        T = max(1, N // B)
        return {'kind': kind, 'B': B, 'T': T, 'S': T + rng.randrange(0, 2000), 'Hq': Hq, 'Hkv': Hkv, 'D': D, 'page': page,
                'rotary': D * rng.choice((2, 3, 4, 4)) // 4, 'axes': rng.choice((1, 1, 3)), 'interleaved': rng.random() < 0.4, 'dtype': dtype,
                'angles': rng.choice(('fp32', dtype))}
    T = rng.choice((1, 1, _log_int(rng, 2, 16), _log_int(rng, 16, 2048)))
    B = _log_int(rng, 1, max(1, min(96, 60_000 // (T * Hq))))
    # (a pass keeps the plain form's scores below two billion values, and its gathered cache below half a billion)
    S = T + _log_int(rng, 1, max(2, min(32768, 2_000_000_000 // (B * T * Hq) - T, 4_000_000 // (B * Hkv))))
    return {'kind': kind, 'B': B, 'T': T, 'S': S, 'Hq': Hq, 'Hkv': Hkv, 'D': rng.choice((64, 128, 128)), 'page': page,
            'window': rng.choice((0, 0, 0, 1 + S // 3)), 'padded': rng.random() < 0.3, 'dtype': dtype}


def _spread(n: int, lo: float) -> list:
    """n shares of 1 between ``lo`` and 1, the first of them 1, in no order."""
    return [1.0 - (1.0 - lo) * math.fmod(0.618033988749895 * i, 1.0) for i in range(n)]


def _lengths(case: dict) -> tuple:
    """(new tokens, cached tokens with the new ones) of every sequence."""
    T, S = case['T'], case['S']
    new = [max(1, round(T * f)) for f in _spread(case['B'], 0.5)]
    return new, [n + round((S - T) * f) for n, f in zip(new, _spread(case['B'], 0.25))]


def _starts(case: dict) -> list:
    """Hidden tokens at the front of every sequence: left padding of a batch."""
    return [round((1.0 - f) * 2 * (s - 1)) if f > 0.5 else 0 for s, f in zip(_lengths(case)[1], _spread(case['B'], 0.3))]


def _randn(shape, g: torch.Generator, dtype: torch.dtype) -> torch.Tensor:
    return torch.randn(shape, generator=g, device='cuda', dtype=torch.float32).to(dtype)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator('cuda').manual_seed(seed)
    state = {'case': case}
    B = case['B']
    if case['kind'] == 'sample':
        # a model's logits: a bulk of unlikely tokens and some that stand out, other temperatures in other rows
        V = case['V']
        logits = torch.randn((B, V), generator=g, device='cuda') * 1.5
        logits += 6.0 * (torch.rand((B, V), generator=g, device='cuda') < 40.0 / V) * torch.rand((B, V), generator=g, device='cuda')
        state['logits'] = logits.to(_DTYPES[case['dtype']])
        state['uniforms'] = torch.rand(B, generator=g, device='cuda')
        state['temperature'] = case['temperature'] * (0.8 + 0.4 * torch.rand(B, generator=g, device='cuda'))
        state['top_k'] = torch.full((B,), case['top_k'], dtype=torch.int32, device='cuda')
        state['top_p'] = torch.full((B,), case['top_p'], device='cuda')
        state['min_p'] = torch.full((B,), case['min_p'], device='cuda')
        return state
    dtype, page, Hq, Hkv, D = _DTYPES[case['dtype']], case['page'], case['Hq'], case['Hkv'], case['D']
    new, total = _lengths(case)
    width = -(-max(total) // page)
    held = torch.tensor([-(-t // page) for t in total])
    n_pages = int(held.sum()) + 3                                       # (the pool has pages of other sequences too)
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed), dtype=torch.int32)[:n_pages - 3]
    table = torch.full((B, width), -1, dtype=torch.int32)
    table[torch.arange(width) < held[:, None]] = order
    N = sum(new)
    state.update(block_table=table.cuda(), seq_lens=torch.tensor(total, dtype=torch.int32).cuda(),
                 cu_seqlens=torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda())
    # keys have an offset and some loud channels, as projections do
    loud = 1.0 + 3.0 * (torch.rand((Hkv, 1, D), generator=g, device='cuda') < 0.03)
    state['key_pages'] = (_randn((n_pages, Hkv, page, D), g, torch.float32) * loud + 0.5 * _randn((Hkv, 1, D), g, torch.float32)).to(dtype)
    state['value_pages'] = _randn((n_pages, Hkv, page, D), g, dtype)
    state['query'] = _randn((N, Hq, D), g, dtype)
    if case['kind'] == 'attend':
        state['max_query_len'] = max(new)
        state['seq_starts'] = torch.tensor(_starts(case), dtype=torch.int32).cuda() if case['padded'] else None
        return state
    state['key'] = _randn((N, Hkv, D), g, dtype)
    state['value'] = _randn((N, Hkv, D), g, dtype)
    # angles of the tokens' positions, as a model's rotary embedding hands them on: one table for all layers
    half, axes = case['rotary'] // 2, case['axes']
    at = torch.cat([torch.arange(t - n, t, dtype=torch.float64) for n, t in zip(new, total)]).cuda()
    if axes == 3:                                                       # time, height and width of patches in a grid 30 wide
        at = torch.stack([at // 900, at // 30 % 30, at % 30]) + at // 1000
        angle = at[..., None] * 1000000.0 ** (-torch.arange(half, dtype=torch.float64, device='cuda') / half)
    else:
        angle = at[..., None] * 500000.0 ** (-torch.arange(half, dtype=torch.float64, device='cuda') / half)
    state['cos'], state['sin'] = (f(angle).to(_DTYPES[case['angles']]) for f in (torch.cos, torch.sin))
    return state


def _sections(case: dict):
    """Columns of the angles that each axis has."""
    half = case['rotary'] // 2
    side = half * 3 // 8
    return (half - 2 * side, side, side) if case['axes'] == 3 else None


def run(state: dict):
    case = state['case']
    if own:
        import adacode_b200
        if case['kind'] == 'sample':
            return adacode_b200.sample_tokens(state['logits'], state['uniforms'], temperature=state['temperature'], top_k=state['top_k'],
                                              top_p=state['top_p'], min_p=state['min_p'])
        if case['kind'] == 'append':
            rotated = adacode_b200.append_rotary(
                state['key'], state['value'], state['cos'], state['sin'], state['key_pages'], state['value_pages'], state['block_table'],
                state['seq_lens'], query=state['query'], cu_seqlens=state['cu_seqlens'], sections=_sections(case),
                interleaved=case['interleaved'])
            return rotated, state['key_pages'], state['value_pages']
        return adacode_b200.paged_attention(
            state['query'], state['key_pages'], state['value_pages'], state['block_table'], state['seq_lens'], cu_seqlens=state['cu_seqlens'],
            max_query_len=state['max_query_len'], window=case['window'], seq_starts=state['seq_starts'])
    return {'sample': _plain_sample, 'append': _plain_append, 'attend': _plain_attend}[case['kind']](state)


def _tokens(state: dict) -> tuple:
    """Sequence and position of every new token."""
    cu, lens = state['cu_seqlens'].long(), state['seq_lens'].long()
    i = torch.arange(state['query'].shape[0], device=cu.device)
    b = torch.searchsorted(cu[1:], i, right=True)
    return b, lens[b] - cu[b + 1] + i


def _plain_append(state: dict):
    case = state['case']
    cos, sin = state['cos'].float(), state['sin'].float()
    if case['axes'] > 1:
        axis = torch.repeat_interleave(torch.arange(case['axes'], device=cos.device), torch.tensor(_sections(case), device=cos.device))
        cos, sin = (x.gather(0, axis.expand(1, x.shape[1], -1))[0] for x in (cos, sin))
    cos, sin = cos[:, None], sin[:, None]
    R = case['rotary']

    def rotate(x):
        y = x.float()
        if case['interleaved']:
            a, b = y[..., 0:R:2], y[..., 1:R:2]
            front = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., :R // 2], y[..., R // 2:R]
            front = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([front, y[..., R:]], -1).to(x.dtype)

    b, at = _tokens(state)
    page = state['block_table'][b, at // case['page']].long()
    state['key_pages'][page, :, at % case['page']] = rotate(state['key'])
    state['value_pages'][page, :, at % case['page']] = state['value']
    return rotate(state['query']), state['key_pages'], state['value_pages']


def _plain_attend(state: dict):
    case = state['case']
    query, table = state['query'], state['block_table'].long().clamp(min=0)
    B, Hq, Hkv, D = case['B'], case['Hq'], case['Hkv'], case['D']
    T, S = state['max_query_len'], table.shape[1] * case['page']
    cu, lens = state['cu_seqlens'].long(), state['seq_lens'].long()
    keys, values = (p[table].transpose(1, 2).reshape(B, Hkv, S, D).float() for p in (state['key_pages'], state['value_pages']))
    # queries of all sequences, filled up to the longest chunk
    t = torch.arange(T, device=query.device)
    index = (cu[:-1, None] + t).clamp(max=query.shape[0] - 1)
    q = query[index].float().transpose(1, 2).reshape(B, Hkv, Hq // Hkv * T, D)
    at = lens[:, None] - (cu[1:] - cu[:-1])[:, None] + t
    j = torch.arange(S, device=query.device)
    seen = (j <= at[..., None]) & (j < lens[:, None, None])
    if case['window']:
        seen &= j > at[..., None] - case['window']
    if state['seq_starts'] is not None:
        seen &= j >= state['seq_starts'][:, None, None]
    scores = (q @ keys.transpose(2, 3)).view(B, Hq, T, S).mul_(D ** -0.5).masked_fill_(~seen[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = weights.sum(-1, keepdim=True)
    out = (weights.view(B, Hkv, Hq // Hkv * T, S) @ values).view(B, Hq, T, D) / torch.where(total == 0, 1.0, total)
    b, at = _tokens(state)
    return out[b, :, at - lens[b] + (cu[b + 1] - cu[b])].to(query.dtype)


def _plain_sample(state: dict):
    # (64 bits: the sums are long, and a token's neighbours on the line of sums are borders)
    x, T = state['logits'].double(), state['temperature'].double()[:, None]
    V = x.shape[1]
    value, token = torch.sort(x, dim=1, descending=True, stable=True)
    weight = torch.where(T > 0, ((value - value[:, :1]) / T).exp(), (torch.arange(V, device=x.device) == 0).double())
    rank = torch.arange(V, device=x.device)
    k = state['top_k'].long()[:, None]
    weight = torch.where((k <= 0) | (rank < k), weight, 0.0)
    before = weight.cumsum(1) - weight
    nucleus = (before < state['top_p'].double()[:, None] * weight.sum(1, keepdim=True)) | (rank == 0) | (state['top_p'][:, None] >= 1)
    weight = torch.where(nucleus & (weight >= state['min_p'].double()[:, None]), weight, 0.0)
    weight = torch.zeros_like(weight).scatter_(1, token, weight)           # back in the order of the vocabulary
    line = weight.cumsum(1)
    aim = state['uniforms'].double()[:, None] * line[:, -1:]
    return ((line > aim) & (weight > 0)).long().argmax(1)


def work(case: dict) -> dict:
    if case['kind'] == 'sample':
        n = case['B'] * case['V']
        return {'bytes': n * (4 if case['dtype'] == 'fp32' else 2) + case['B'] * 28, 'flops': 4 * n}
    new, total = _lengths(case)
    N, Hq, Hkv, D = sum(new), case['Hq'], case['Hkv'], case['D']
    if case['kind'] == 'append':
        angles = N * case['rotary'] // 2 * 2 * (4 if case['angles'] == 'fp32' else 2)   # (of three axes, each column's own)
        return {'bytes': 2 * 2 * N * (Hq + 2 * Hkv) * D + angles, 'flops': 3 * N * (Hq + Hkv) * case['rotary']}
    starts = _starts(case) if case['padded'] else [0] * case['B']
    pairs = read = 0
    for n, t, s in zip(new, total, starts):
        w = case['window'] or t
        first, last = t - n, t - 1                                          # positions of the chunk
        # (position p sees min(p + 1 - s, w) tokens if that is positive)
        lo, hi = max(first, s), last
        full = max(lo, s + w - 1)                                           # from here on whole windows
        if lo <= hi:
            edge = min(full, hi + 1)
            pairs += (edge - lo) * (lo + edge - 1 - 2 * (s - 1)) // 2 + max(0, hi + 1 - edge) * w
            read += t - max(s, lo - w + 1)
    return {'bytes': 2 * (2 * N * Hq * D + 2 * read * Hkv * D), 'flops': 4 * pairs * Hq * D}


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case['kind'] == 'sample':
        return _exact_sample(state)
    new, total = _lengths(case)
    page, R = case['page'], case.get('rotary')
    if case['kind'] == 'append':
        cos, sin = state['cos'].double(), state['sin'].double()
        if case['axes'] > 1:
            parts = [[x[a][:, sum(_sections(case)[:a]):sum(_sections(case)[:a + 1])] for a in range(3)] for x in (cos, sin)]
            cos, sin = (torch.cat(p, 1) for p in parts)
        turn = torch.complex(cos, sin)[:, None]

        def rotate(x):
            y = x.double().clone()
            pairs = y[..., :R].unflatten(-1, (R // 2, 2) if case['interleaved'] else (2, R // 2))
            pairs = pairs if case['interleaved'] else pairs.transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            y[..., :R] = (z if case['interleaved'] else z.transpose(-1, -2)).flatten(-2)
            return y

        key, keys, values, i = rotate(state['key']), state['key_pages'].double(), state['value_pages'].double(), 0
        for b, (n, t) in enumerate(zip(new, total)):
            for first in range((t - n) // page * page, t, page):           # page by page
                lo, hi = max(first, t - n), min(first + page, t)
                p, at = int(state['block_table'][b, first // page]), i + lo - (t - n)
                keys[p, :, lo - first:hi - first] = key[at:at + hi - lo].transpose(0, 1)
                values[p, :, lo - first:hi - first] = state['value'][at:at + hi - lo].transpose(0, 1).double()
            i += n
        return rotate(state['query']), keys, values
    if work(case)['flops'] > 2e13:
        return None
    out = torch.zeros(state['query'].shape, dtype=torch.float64, device='cuda')
    G, i = case['Hq'] // case['Hkv'], 0
    starts = _starts(case) if case['padded'] else [0] * case['B']
    for b, (n, t) in enumerate(zip(new, total)):
        pages = state['block_table'][b, :-(-t // page)].long()
        for h in range(case['Hkv']):
            k, v = (state[name][pages, h].reshape(-1, case['D'])[:t].double() for name in ('key_pages', 'value_pages'))
            for lo in range(0, n, 512):
                hi = min(n, lo + 512)
                q = state['query'][i + lo:i + hi, h * G:(h + 1) * G].double()
                s = torch.einsum('tgd,jd->tgj', q, k) / math.sqrt(case['D'])
                at = torch.arange(t - n + lo, t - n + hi, device='cuda')[:, None, None]
                j = torch.arange(t, device='cuda')
                hidden = (j > at) | (j < starts[b]) | ((j <= at - case['window']) if case['window'] else False)
                p = torch.softmax(s.masked_fill_(hidden, -math.inf), -1).nan_to_num_(0.0)
                out[i + lo:i + hi, h * G:(h + 1) * G] = torch.einsum('tgj,jd->tgd', p, v)
        i += n
    return out


def _exact_sample(state: dict):
    picked = []
    for b in range(state['case']['B']):
        x, T = state['logits'][b].double(), float(state['temperature'][b])
        if T <= 0:
            picked.append((x == x.max()).nonzero()[0, 0])
            continue
        order = torch.argsort(x, descending=True, stable=True)
        if int(state['top_k'][b]) > 0:
            order = order[:int(state['top_k'][b])]
        p = torch.softmax(x[order] / T, 0)
        if float(state['top_p'][b]) < 1:
            reached = int(torch.searchsorted(p.cumsum(0), torch.tensor(float(state['top_p'][b]), dtype=torch.float64, device='cuda')))
            order, p = order[:reached + 1], p[:reached + 1]
        kept = p >= float(state['min_p'][b]) * p[0]
        order, by_token = order[kept].sort()
        line = p[kept][by_token].cumsum(0)
        picked.append(order[torch.searchsorted(line, state['uniforms'][b].double() * line[-1], right=True).clamp(max=len(order) - 1)])
    return torch.stack(picked)
