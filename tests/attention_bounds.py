"""Bounds of attention's error that a lost or doubled key, or a weight rounded once too often, does not pass; all in float64.

u is half a step of the output's type relative to a value, 2^-8 for bfloat16, and w what a weight is off by for entering the product
with v in bfloat16: 2^-8 once rounded (prompts), 2^-16 in two terms (single tokens), 0 with float32 operands.
"""
import torch

from serving_refs import EPS32, f64

ONE_TERM, TWO_TERMS = 2.0 ** -8, 2.0 ** -16


def parts(q, k, v, causal=True, scale=None):
    """Of one sequence, q [n,H,D] over k, v [t,G,D]: o, mag = sum p|v|, root = sqrt(sum p^2 v^2), all [n,H,D], and size [n,H,1],
    the largest scale * sum |q||k| of a row."""
    n, H, D = q.shape
    t, share = k.shape[0], H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    o, mag, root, size = (torch.zeros(n, H, d, dtype=torch.float64) for d in (D, D, D, 1))
    ahead = torch.ones(n, t, dtype=torch.bool).triu(1) if causal else torch.zeros(n, t, dtype=torch.bool)
    for h in range(H):
        g = h // share
        p = torch.softmax((scale * (q[:, h] @ k[:, g].t())).masked_fill(ahead, -float("inf")), -1)
        o[:, h], mag[:, h], root[:, h] = p @ v[:, g], p @ v[:, g].abs(), (p ** 2 @ v[:, g] ** 2).sqrt()
        size[:, h, 0] = (scale * (q[:, h].abs() @ k[:, g].abs().t())).masked_fill(ahead, 0).amax(-1)
    return o, mag, root, size


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def each(o, mag, size, t, dtype, w):
    """What a value may be off by, whatever the signs of the roundings: 32-bit roundings of a score (D + 8 of at most ``size``), of a
    weight and of the sum it is divided by, and of sums over t keys; w of every weight; the output's own of what came of them."""
    e = (EPS32 * (2 * ((o.shape[-1] + 8) * size + 8) + t + 8) + (w if dtype == torch.bfloat16 else 0)) * mag
    return e + half_step(dtype) * (o.abs() + e) + 1e-30


BLOCK = 32


def _norm(x):
    """The 2-norms of x [n,H,D] over D and 32 rows: [blocks,H]."""
    n, H, D = x.shape
    x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, -n % BLOCK))
    return x.view(-1, BLOCK, H, D).permute(0, 2, 1, 3).flatten(2).norm(dim=-1)


def norms(o, mag, root, size, t, dtype, w):
    """What 32 rows of a head may be off by in the 2-norm, [blocks,H]: roundings of one key and another are independent, so their
    sum grows as the root of the sum of squares.  A weight's are those of its score (a sum of D products: sqrt(D), and four of its
    size) and its exponential (two), 32-bit, and w; sums over t keys sqrt(t).  Four times that, which is rms; the output's own
    rounding at its most.  Once rounded to bfloat16 a weight is off by less than w, of which the rms is under a half: once that."""
    D, top = o.shape[-1], size.amax(0)[:, 0]
    weight = EPS32 * (D ** 0.5 + 4) * (top + 2) + (w if dtype == torch.bfloat16 else 0) / (4 if w == ONE_TERM else 1)
    return half_step(dtype) * _norm(o) + 4 * weight * _norm(root) + 4 * EPS32 * t ** 0.5 * _norm(mag) + 1e-30


def over(got, o, mag, root, size, t, w, dtype=None):
    """How far the worst value, and the worst rows of a head, pass their bound (up to 1: within)."""
    dtype = dtype or got.dtype
    err = f64(got) - o
    if not torch.isfinite(err).all():
        return float("inf"), float("inf")
    rows = _norm(err) / norms(o, mag, root, size, t, dtype, w)
    return (err.abs() / each(o, mag, size, t, dtype, w)).max().item(), rows.max().item()


def within(got, want, t, w, what):
    value, rows = over(got, *want, t, w)
    assert value <= 1 and rows <= 1, f"{what}: a value {value:.3f}, rows of a head {rows:.3f} times their bound"


# ------------------------------------------------------------------------------------------
#  Inputs at which a mistake shows
# ------------------------------------------------------------------------------------------
def balanced(q, k, v, dtype):
    """v of one sequence and head of keys, less its weighted mean over the first query head's weights: the output is nearly 0, so
    that its own rounding hides nothing of the weights'."""
    p = torch.softmax(q.shape[-1] ** -0.5 * (f64(q)[0, 0] @ f64(k)[:, 0].t()), -1)
    x = f64(v)[:, 0]
    return (x - (p @ x) * torch.ones_like(x)).to(dtype)[:, None]


def pointed(gen, n, H, G, D, at, dtype):
    """q [n,H,D], k, v [n,G,D] such that query i of head h gives about half of its weight to key at[i, h]."""
    k, v = torch.randn(n, G, D, generator=gen), torch.randn(n, G, D, generator=gen)
    heads = torch.arange(H) // (H // G)
    q = k[at, heads.expand(n, H)]                        # its score with itself |k|^2 / sqrt(D), with others about |k| / sqrt(D)
    own = (q ** 2).sum(-1, keepdim=True) * D ** -0.5
    seen = torch.arange(1, n + 1, dtype=torch.float32)[:, None, None]
    return [(q * (torch.log(seen + 1) / own)).to(dtype), k.to(dtype), v.to(dtype)]
