"""The frame-attention operators in 64 bits on the host, loop by loop from their definition, and the
error bounds that follow from the operators' arithmetic.

u is half a step of the type (torch.finfo(t).eps / 2, the largest relative error of one rounding),
w = 2^-24 that of fp32.
"""
import math

import torch

W = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def spans(starts, streams, tokens):
    """(first, count) of the new tokens of every stream."""
    if starts is None:
        return [(b * (tokens // streams), tokens // streams) for b in range(streams)]
    s = starts.tolist()
    return [(s[b], s[b + 1] - s[b]) for b in range(streams)]


def place(table, slot, page):
    return int(table[slot // page]), slot % page


def rotary(x, positions, frequencies, sections, interleaved, inverse=False):
    """The turned tensor, and the bound of its error.

    fp32 parts: the fraction of a turn is rounded to fp32 (at most 2^-26 of a turn, 1.6 w rad), sine and
    cosine are good to 2 steps of fp32 (4 w for values up to 1), so each factor is off by at most 6 w; the
    product and the fused sum add one rounding each (w times the magnitudes): 7 w (|a| + |b|), and the
    final rounding u |result|."""
    x64 = x.double().cpu()
    pairs = sum(sections) // 2
    axis = [a for a, n in enumerate(sections) for _ in range(n // 2)]
    angle = positions.cpu().double()[:, axis] * frequencies.cpu()
    if inverse:
        angle = -angle
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    ia = torch.arange(pairs) * 2 if interleaved else torch.arange(pairs)
    ib = ia + 1 if interleaved else ia + pairs
    out, mag = x64.clone(), torch.zeros_like(x64)
    a, b = x64[..., ia], x64[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return out, 7 * W * mag + half_step(x.dtype) * out.abs()


def gather(pool, table, length, h, page):
    rows = [place(table, s, page) for s in range(length)]
    at = torch.tensor([r[0] for r in rows], dtype=torch.long)
    off = torch.tensor([r[1] for r in rows], dtype=torch.long)
    return pool[at, h, off].double()


def attention(q, keys, values, page_table, lens, starts=None, scale=None, causal_block=0, weights=None, decay=1.0):
    """out, lse, weights and their bounds (all float64 on the host).

    Scores: a sum of D exact products in fp32 is off by at most D w sum |q k|, its scaling and the
    subtraction in the exponent by 3 w |s|; the maximum subtracted cancels.  So an exponential is off by a
    factor 1 + d with d <= scale D w max sum |q k| + 4 w max |s| + 4 w (the exponential itself).  Each
    probability that multiplies a value is rounded to the type (u, the 16-bit types), n of them are
    summed in fp32 (n w), twice (numerator and normaliser).  In all, relative to sum p |v|:
    u + 2 d + 2 n w + 8 w; and the result's own rounding u |out|."""
    q, keys, values = q.cpu(), keys.cpu(), values.cpu()
    table, lens = page_table.cpu(), lens.cpu()
    tokens, heads, dim = q.shape
    pages, kv, page, _ = keys.shape
    group = heads // kv
    scale = dim ** -0.5 if scale is None else scale
    u = half_step(q.dtype) if q.dtype != torch.float32 else 0.0
    out, out_tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    lse, lse_tol = torch.full((tokens, heads), math.nan, dtype=torch.float64), torch.zeros(tokens, heads, dtype=torch.float64)
    new_w = weights.double().cpu().clone() if weights is not None else None
    w_tol = torch.zeros_like(new_w) if weights is not None else None
    for b, (first, count) in enumerate(spans(starts, table.shape[0], tokens)):
        length = int(lens[b])
        for h in range(kv):
            k, v = gather(keys, table[b], length, h, page), gather(values, table[b], length, h, page)
            received, r_tol = torch.zeros(length, dtype=torch.float64), torch.zeros(length, dtype=torch.float64)
            for i in range(count):
                n = length if causal_block == 0 else max(0, min(length, length - count + (i // causal_block + 1) * causal_block))
                for g in range(h * group, (h + 1) * group):
                    t = first + i
                    if n == 0:
                        lse[t, g] = -math.inf
                        continue
                    qq = q[t, g].double()
                    s = (k[:n] @ qq) * scale
                    top = s.max()
                    p = (s - top).exp()
                    total = p.sum()
                    p = p / total
                    sabs = abs(scale) * (k[:n].abs() @ qq.abs()).max()
                    d = dim * W * sabs + 4 * W * s.abs().max() + 4 * W
                    out[t, g] = p @ v[:n]
                    out_tol[t, g] = (u + 2 * d + 2 * n * W + 8 * W) * (p @ v[:n].abs()) + half_step(q.dtype) * out[t, g].abs()
                    lse[t, g] = top + total.log()
                    lse_tol[t, g] = d + n * W + 4 * W * (lse[t, g].abs() + top.abs() + 1)
                    received[:n] += p
                    # the log-sum's own error enters the exponent once more
                    r_tol[:n] += p * (2 * d + n * W + 8 * W * (lse[t, g].abs() + top.abs() + 2))
            if weights is not None:
                for s in range(length):
                    pg, off = place(table[b], s, page)
                    old = 0.0 if decay == 0 else decay * float(new_w[pg, h, off])
                    new_w[pg, h, off] = old + received[s]
                    w_tol[pg, h, off] = r_tol[s] + (count * group + 2) * W * (received[s] + abs(old))
    return out, out_tol, lse, lse_tol, new_w, w_tol


def slots(weights, page_table, lens, tokens, budget, starts=None, stamps=None, keep_from=None):
    weights, table, lens = weights.cpu(), page_table.cpu(), lens.cpu()
    pages, kv, page = weights.shape
    out, new = torch.full((kv, tokens), -99, dtype=torch.int32), torch.zeros(table.shape[0], dtype=torch.int32)
    for b, (first, count) in enumerate(spans(starts, table.shape[0], tokens)):
        n = int(lens[b])
        e = min(max(n + count - budget, 0), n, count)
        most = max(budget, n)
        new[b] = min(n + count - e, most)
        for h in range(kv):
            ranked = []
            for s in range(n):
                pg, off = place(table[b], s, page)
                if not 0 <= pg < pages:
                    ranked.append((-1, 0, 0.0, s))
                    continue
                w = float(weights[pg, h, off])
                kept = stamps is not None and int(stamps[pg, h, off]) >= int(keep_from[b])
                ranked.append((int(kept), int(w != w), 0.0 if w != w else w, s))
            ranked.sort()
            given = sorted(r[3] for r in ranked[:e])
            given += [s if s < most else -1 for s in range(n, n + count - e)]
            out[h, first:first + count] = torch.tensor(given, dtype=torch.int32)
    return out, new


def assert_within(got, want, tol, what=""):
    g = got.double().cpu()
    assert torch.equal(g.isnan(), want.isnan()), f"{what}: NaN in other places"
    same = (g == want) | want.isnan()
    over = ((g - want).abs() - tol).masked_fill(same, -math.inf)
    assert bool((over <= 0).all()), (f"{what}: {int((over > 0).sum())} of {g.numel()} values off, worst "
                                     f"{float((g - want).abs().masked_fill(same, 0).max()):.3g}")
