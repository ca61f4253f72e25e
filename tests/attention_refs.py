"""Attention and the cache's bookkeeping from their definitions, in float64 and plain Python on the CPU."""
import torch

from serving_refs import EPS32, f64


def attention(q, k, v, causal=True, scale=None):
    """(o, mag, size) of one sequence: q [n,H,D] over k, v [t,G,D] in float64, row i of q seeing keys up to i (causal).
    mag is the weighted mean of |v|; size the largest scale * sum |q||k| of a row."""
    n, H, D = q.shape
    t, G = k.shape[0], k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    o, mag, size = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(n, H, 1, dtype=torch.float64)
    for h in range(H if n and t else 0):
        g = h // (H // G)
        score, mass = scale * (q[:, h] @ k[:, g].t()), scale * (q[:, h].abs() @ k[:, g].abs().t())
        if causal:
            ahead = torch.arange(t)[None] > torch.arange(n)[:, None]
            score, mass = score.masked_fill(ahead, -float("inf")), mass.masked_fill(ahead, 0)
        p = torch.softmax(score, -1)
        o[:, h], mag[:, h], size[:, h, 0] = p @ v[:, g], p @ v[:, g].abs(), mass.amax(-1)
    return o, mag, size


def tolerance(o, mag, size, D, n, dtype):
    """Roundings of 2^-24: a score is a sum of D products (D + 1 of its terms' size, at most ``size``), times the scale in two
    roundings, minus a bound of its own size in one, and exponentiated with an error of two; a weight and the sum of weights it
    is divided by are each off by that (so it counts twice); sums over n keys and the carried scale-downs add n and 8.  With bfloat16
    operands a weight is rounded once more (2^-8), and so is the output, by as much again where 32-bit error moves it across
    a rounding boundary."""
    rel = EPS32 * (2 * ((D + 8) * size + 8) + n + 8)
    if dtype == torch.bfloat16:
        return (rel + 2.0 ** -8) * mag + 2.0 ** -7 * o.abs() + 1e-30
    return rel * mag + 2 * EPS32 * o.abs() + 1e-30


def check(got, o, mag, size, n, what):
    tol = tolerance(o, mag, size, o.shape[-1], n, got.dtype)
    got = f64(got)
    assert got.shape == o.shape, (what, got.shape, o.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - o).abs() - tol
    worst = over.max().item() if over.numel() else -1.0
    assert worst <= 0, f"{what}: {int((over > 0).sum())} of {over.numel()} values off, worst by {worst:.3e} past its tolerance"


def pages_of(n, page):
    return (n + page - 1) // page


def assign(tables, lengths, tokens, free, taken, page, capacity, slots=None):
    """(rows, cu, lengths, taken, tables) as lists, request by request."""
    tables, lengths = [list(r) for r in tables], list(lengths)
    S, M, F = len(tables), len(tables[0]) if tables else 0, len(free)
    rows, cu, after, at, want_so_far, lacking = [-1] * capacity, [0], [], taken, 0, False
    for b, (c, n) in enumerate(zip(lengths, tokens)):
        start, end = cu[-1], cu[-1] + n
        cu.append(end)
        s = b if slots is None else slots[b]
        need = pages_of(c + n, page) - pages_of(c, page)
        if not 0 <= s < S or c + n > M * page or end > capacity:
            after.append(c)
            continue
        want_so_far += need
        if need and (lacking or taken + want_so_far > F):
            lacking = True
            after.append(c)
            continue
        have = pages_of(c, page)
        tables[s][have:have + need] = free[at:at + need]
        at += need
        after.append(c + n)
        for i in range(n):
            x = c + i
            p = tables[s][x // page]
            rows[start + i] = p * page + x % page if p >= 0 else -1
    return rows, [min(x, capacity) for x in cu], after, at, tables


def release(tables, lengths, free, taken, page, slots=None):
    """(free, taken): the pages back, downwards from taken."""
    free, at, before = list(free), taken, 0
    for b, n in enumerate(lengths):
        s = b if slots is None else slots[b]
        own = tables[s][:pages_of(n, page)] if 0 <= s < len(tables) else []
        if before + len(own) <= taken:
            for p in own:
                at -= 1
                free[at] = p
        before += len(own)
    return free, at
