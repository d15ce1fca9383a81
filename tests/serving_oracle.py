"""64-bit oracles of rotated appends, attention over pages and sampling, one sequence, head or row after the other, on the CPU
or wherever the inputs lie; and random cases for them."""
import math

import torch


def make_cache(lens, Hkv, D, page, dtype, seed=0, spare=3, layout='phsd', fill=None, device='cuda'):
    """Pages, table and lengths of sequences of ``lens`` tokens.  Slots that hold no token, and spare pages, hold ``fill`` (random values
    without); table entries behind a sequence's pages are -1."""
    g = torch.Generator('cpu').manual_seed(seed)
    width = max(1, -(-max(lens) // page))
    used = [-(-n // page) for n in lens]
    P = sum(used) + spare
    order = torch.randperm(P, generator=g).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    n = 0
    for b, u in enumerate(used):
        table[b, :u] = order[n:n + u]
        n += u
    pages = []
    for _ in range(2):
        x = torch.randn((P, Hkv, page, D), generator=g).to(dtype)
        if fill is not None:
            held = torch.zeros((P, page), dtype=torch.bool)
            for b, length in enumerate(lens):
                for p in range(used[b]):
                    held[table[b, p], :max(0, min(page, length - p * page))] = True
            x = torch.where(held[:, None, :, None], x, torch.tensor(fill, dtype=dtype))
        x = x.to(device)
        if layout == 'pshd':                                # slots outside heads, as [P, page, H, D] lies in memory
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        pages.append(x)
    return pages[0], pages[1], table.to(device), torch.tensor(lens, dtype=torch.int32, device=device)


def cumulative(new, device='cuda'):
    return torch.tensor([0, *new], dtype=torch.int64).cumsum(0).to(torch.int32).to(device)


def gather(pages, table_row, length, page):
    """[H, length, D] of one sequence in 64 bits."""
    n = -(-length // page)
    ids = table_row[:n].long()
    x = pages[ids].double()                                 # [n, H, page, D]
    return x.transpose(0, 1).reshape(x.shape[1], n * page, x.shape[3])[:, :length]


def attention(query, key_pages, value_pages, table, lens, new, scale=None, causal=True, window=0, starts=None):
    """(result, the same with |values|) in 64 bits; rows behind the last sequence stay 0."""
    N, Hq, D = query.shape
    H, page = key_pages.shape[1], key_pages.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out, size = (torch.zeros((N, Hq, D), dtype=torch.float64, device=query.device) for _ in range(2))
    i = 0
    for b, (n, length) in enumerate(zip(new, lens)):
        if n:
            k, v = (gather(p, table[b], length, page) for p in (key_pages, value_pages))
            q = query[i:i + n].double().transpose(0, 1).reshape(H, Hq // H, n, D)
            s = torch.einsum('hgnd,hjd->hgnj', q, k) * scale
            at = torch.arange(length - n, length, device=query.device)[:, None]
            j = torch.arange(length, device=query.device)
            seen = (j >= (0 if starts is None else starts[b])) & (j < length) & ((j <= at) | (not causal))
            if window:
                seen = seen & (j > at - window)
            s = torch.where(seen, s, -math.inf)
            top = s.amax(-1, keepdim=True) if length else s.sum(-1, keepdim=True)
            p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            total = p.sum(-1, keepdim=True)
            p = torch.where(total == 0, 0.0, p / total)
            # (a hidden value has no weight, not the weight 0: 0 x inf is NaN)
            odd = ~torch.isfinite(v)
            r = torch.einsum('hgnj,hjd->hgnd', p, torch.where(odd, 0.0, v))
            if bool(odd.any()):
                w = seen.to(torch.float64) * (p > 0)
                count = [torch.einsum('hgnj,hjd->hgnd', w, (v == math.inf).double()), torch.einsum('hgnj,hjd->hgnd', w, (v == -math.inf).double()),
                         torch.einsum('hgnj,hjd->hgnd', w, torch.isnan(v).double())]
                r = torch.where(count[0] > 0, math.inf, r)
                r = torch.where(count[1] > 0, -math.inf, r)
                r = torch.where((count[2] > 0) | ((count[0] > 0) & (count[1] > 0)), math.nan, r)
            out[i:i + n] = r.reshape(Hq, n, D).transpose(0, 1)
            size[i:i + n] = torch.einsum('hgnj,hjd->hgnd', p, torch.where(odd, 0.0, v).abs()).reshape(Hq, n, D).transpose(0, 1)
        i += n
    return out, size


def rotate(x, cos, sin, interleaved=False):
    """Columns of [N, H, D] in 64 bits; cos and sin [N, half]."""
    y = x.double().clone()
    half = cos.shape[1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    p, q = y[..., a].clone(), y[..., b].clone()
    y[..., a] = p * c - q * s
    y[..., b] = q * c + p * s
    return y


def angles(positions, half, base=10000.0, sections=None):
    """cos and sin, 64 bits: [N, half], or [A, N, half] for positions [A, N]."""
    freq = base ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    angle = positions.double()[..., None].cpu() * freq
    return torch.cos(angle), torch.sin(angle)


def select_axes(x, sections):
    """[N, half] from [A, N, half]."""
    ends = [sum(sections[:a + 1]) for a in range(len(sections))]
    return torch.cat([x[a][:, e - n:e] for a, (n, e) in enumerate(zip(sections, ends))], dim=1)


def sample(row, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row (list of floats as fp64 tensor on the CPU): the token, and how near the draw came to the border of another outcome,
    relative to the total."""
    x = row.double()
    x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
    order = torch.argsort(x, descending=True, stable=True)
    order = order[x[order] > -math.inf]
    if len(order) == 0:
        return -1, 1.0
    if temperature <= 0:
        return int(order[0]), 1.0
    if top_k > 0:
        order = order[:top_k]
    w = torch.exp((x[order] - x[order[0]]) / temperature)
    near = 1.0
    if top_p < 1:
        before = w.cumsum(0) - w
        gaps = (before / w.sum() - top_p).abs()
        near = min(near, float(gaps.min()))
        kept = before < top_p * w.sum()
        kept[0] = True
        order, w = order[kept], w[kept]
    kept = (w >= min_p) & (w > 0)
    if min_p > 0:
        near = min(near, float((w / min_p - 1).abs().min()))
    order, w = order[kept], w[kept]
    order, by_token = order.sort()
    line = w[by_token].cumsum(0)
    aim = uniform * float(line[-1])
    near = min(near, float(((line - aim).abs() / line[-1])[:-1].min()) if len(line) > 1 else 1.0)
    return int(order[min(int(torch.searchsorted(line, torch.tensor(aim, dtype=torch.float64), right=True)), len(order) - 1)]), near
