"""Paged caches for the tests, and the operators on them in plain 64-bit arithmetic (CPU)."""
import math

import torch


def make_cache(seed, lengths, hk, d, page, dtype, spare=3, layout="nhd"):
    """(k_cache, v_cache, block_table) on the GPU: pages in random order, NaN wherever no token lies, -1 behind a sequence's pages."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    total = sum(counts) + spare
    order = torch.randperm(total, generator=g).tolist()
    table = torch.full((len(lengths), max(1, max(counts))), -1, dtype=torch.int32)
    k = torch.full((total, page, hk, d), math.nan, dtype=dtype)
    v = k.clone()
    at = 0
    for b, n in enumerate(lengths):
        for i in range(counts[b]):
            p, rows = order[at], min(page, n - i * page)
            at += 1
            table[b, i] = p
            k[p, :rows] = torch.randn(rows, hk, d, generator=g).to(dtype)
            v[p, :rows] = torch.randn(rows, hk, d, generator=g).to(dtype)
    if layout == "hnd":
        k, v = (t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in (k, v))
    elif layout == "fused":
        both = torch.stack([k, v], 2).cuda()
        k, v = both[:, :, 0], both[:, :, 1]
    else:
        k, v = k.cuda(), v.cuda()
    return k, v, table.cuda()


def rows_of(cache, table, b, n):
    """The n rows of sequence b, [n, Hk, D] in fp64 on the CPU."""
    page = cache.shape[1]
    t = torch.arange(n)
    return cache.cpu()[table.cpu()[b].long()[t // page], t % page].double()


def attend(q, k_cache, v_cache, table, lengths, scale=None, window=-1, softcap=0.0):
    """(out, lse, weights per sequence [Hk, n], a bound on the scores' errors in fp32) in fp64."""
    b, s, h, d = q.shape
    hk = k_cache.shape[2]
    group = h // hk
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(b, s, h, d, dtype=torch.float64)
    lse = torch.full((b, h, s), math.inf, dtype=torch.float64)
    weights, worst = [], 0.0
    for i, n in enumerate(lengths):
        k, v = rows_of(k_cache, table, i, n), rows_of(v_cache, table, i, n)
        w = torch.zeros(hk, n, dtype=torch.float64)
        for t in range(s):
            hi = n - s + t + 1
            lo = max(0, hi - 1 - window) if window >= 0 else 0
            if hi <= lo:
                continue
            qt = q[i, t].cpu().double().view(hk, group, d)
            x = torch.einsum("hgd,nhd->hgn", qt, k[lo:hi]) * scale
            worst = max(worst, (torch.einsum("hgd,nhd->hgn", qt.abs(), k[lo:hi].abs()) * abs(scale)).nan_to_num(0, 0, 0).max().item())
            if softcap > 0:
                x = softcap * torch.tanh(x / softcap)
            z = torch.logsumexp(x, -1)
            p = torch.exp(x - z[..., None])
            lse[i, :, t] = z.flatten()
            out[i, t] = torch.einsum("hgn,nhd->hgd", p, v[lo:hi]).flatten(0, 1)
            w[:, lo:hi] += p.sum(1)
        weights.append(w)
    # d products and sums, each off by 2^-23 of the sum of the magnitudes at most, some roundings around them, exp2's 2^-22.
    return out, lse, weights, (d + 16) * 2.0 ** -23 * worst + 2.0 ** -20


def turn(x, positions, inv_freq, sections, interleaved_axes=False, interleaved_pairs=False, inverse=False):
    """x [B, S, H, D] turned, in fp64; positions [axes, B, S]."""
    n, axes = sum(sections), len(sections)
    if interleaved_axes:
        axis = [i % axes if i < axes * sections[i % axes] else 0 for i in range(n)]
    else:
        axis = [a for a, s in enumerate(sections) for _ in range(s)]
    angle = torch.stack([positions[a].double() * f for a, f in zip(axis, inv_freq.double().tolist())], -1)[:, :, None]
    cos, sin = angle.cos(), angle.sin() * (-1 if inverse else 1)
    x = x.double()
    out = x.clone()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved_pairs else (slice(0, n), slice(n, 2 * n))
    out[..., first] = x[..., first] * cos - x[..., second] * sin
    out[..., second] = x[..., second] * cos + x[..., first] * sin
    return out


def turn_tolerance(x, dtype):
    """One rounding of the result, products and cosines in fp32 (2^-24 each), angles to 1e-6 rad, of a pair as large as any."""
    return dict(rtol=torch.finfo(dtype).eps / 2 * 1.001, atol=float(x.abs().max()) * 4e-6 + torch.finfo(dtype).tiny)


def choose(mass, n, budget, recent):
    """Which of n tokens a head keeps, by a stable sort."""
    if n <= budget:
        return list(range(n))
    worth = [math.inf if math.isnan(x) else x for x in mass[: n - recent].double().tolist()]
    nan = [math.isnan(x) for x in mass[: n - recent].tolist()]
    first = sorted(range(n - recent), key=lambda i: (not nan[i], -worth[i], i))[: budget - recent]
    return sorted(first) + list(range(n - recent, n))
