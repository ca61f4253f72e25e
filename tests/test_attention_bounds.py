"""The bounds that the GPU tests hold attention to: kept by its definition with the roundings that the kernels are allowed, and
passed by mistakes that are planted in the definition (here, on the CPU): a key lost, a key twice, a weight rounded once more."""
import pytest
import torch

import attention_bounds as bounds
from serving_refs import f64

BF, F32 = torch.bfloat16, torch.float32


def _round(x, dtype):
    return x.to(dtype).double()


def _emulate(q, k, v, causal, terms, weights=None):
    """The definition with weights of ``terms`` terms of bfloat16 (0: unrounded), the output rounded to q's type.  ``weights``
    changes the unnormalised ones [n,t] of a head."""
    n, H, D = q.shape
    out = torch.zeros(n, H, D, dtype=torch.float64)
    for h in range(H):
        g = h // (H // k.shape[1])
        s = D ** -0.5 * (f64(q)[:, h] @ f64(k)[:, g].t())
        if causal:
            s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), -float("inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True) - 0.3)
        if weights is not None:
            p = weights(p)
        used = p if not terms else _round(p, BF)
        if terms == 2:
            used = used + _round(p - used, BF)
        out[:, h] = used @ f64(v)[:, g] / p.sum(-1, keepdim=True)
    return _round(out, q.dtype)


def _qkv(seed, n, t, H, G, D, dtype):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=gen).to(dtype) for s in ((n, H, D), (t, G, D), (t, G, D))]


def _over(got, q, k, v, causal, w):
    return bounds.over(got, *bounds.parts(f64(q), f64(k), f64(v), causal), k.shape[0], w, q.dtype)


def _without(t):
    return lambda p: p.index_fill(1, torch.tensor(t), 0.0)


STEPS = [(4097, 5, 5, 128), (2500, 6, 1, 192), (2000, 2, 1, 64), (257, 4, 2, 40)]


@pytest.mark.parametrize("t,H,G,D", STEPS)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_lost_key_of_a_long_cache(t, H, G, D, dtype):
    """Of thousands of keys, one of usual weight: too little for a bound on each value, enough for one on a head's."""
    q, k, v = _qkv(t, 1, t, H, G, D, dtype)
    terms = 2 if dtype == BF else 0
    assert max(_over(_emulate(q, k, v, False, terms), q, k, v, False, bounds.TWO_TERMS)) <= 1
    usual = (f64(q)[0, 0] @ f64(k)[:, 0].t()).argsort()[t // 2].item()                     # the median weight
    for gone in ([usual], list(range(t - 16, t))):
        assert _over(_emulate(q, k, v, False, terms, _without(gone)), q, k, v, False, bounds.TWO_TERMS)[1] > 1, gone


@pytest.mark.parametrize("t", [40, 300, 1000])
def test_a_weight_s_second_term(t):
    """Weights once rounded pass the bound of weights in two terms where the output is nearly 0."""
    q, k, v = _qkv(t, 1, t, 1, 1, 64, BF)
    v = bounds.balanced(q, k, v, BF)
    assert max(_over(_emulate(q, k, v, False, 2), q, k, v, False, bounds.TWO_TERMS)) <= 1
    assert max(_over(_emulate(q, k, v, False, 1), q, k, v, False, bounds.ONE_TERM)) <= 1
    assert _over(_emulate(q, k, v, False, 1), q, k, v, False, bounds.TWO_TERMS)[0] > 1.5


@pytest.mark.parametrize("dtype", [BF, F32])
def test_prompts(dtype):
    """A prompt's rows within the bounds of once rounded weights; not so where a tile's last key is lost, or every row's own."""
    n = 700
    q, k, v = _qkv(3, n, n, 2, 1, 64, dtype)
    terms = 1 if dtype == BF else 0
    assert max(_over(_emulate(q, k, v, True, terms), q, k, v, True, bounds.ONE_TERM)) <= 1
    for bad in (_without([31]), _without([640]), lambda p: p - torch.diag(p.diag())):
        p = lambda x, bad=bad: bad(x) + 1e-300  # noqa: E731  (a row may be left with none)
        assert _over(_emulate(q, k, v, True, terms, p), q, k, v, True, bounds.ONE_TERM)[1] > 1


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_pointed_weights(dtype, D):
    """A key of half of a query's weight, lost or twice, passes the bound on each value for that query alone."""
    n, gen = 150, torch.Generator().manual_seed(D)
    at = torch.stack([torch.arange(n), (torch.arange(n) // 32) * 32, (torch.rand(n, generator=gen) * torch.arange(1, n + 1)).long()], 1)
    q, k, v = bounds.pointed(gen, n, 3, 1, D, at, dtype)
    s = D ** -0.5 * (f64(q).transpose(0, 1) @ f64(k)[:, 0].t())
    p = torch.softmax(s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -float("inf")), -1)
    own = p.gather(-1, at.t()[..., None])[:, 1:]
    assert 0.2 < own.min() and own.max() < 0.9
    terms, want = (1 if dtype == BF else 0), bounds.parts(f64(q), f64(k), f64(v))
    good = _emulate(q, k, v, True, terms)
    assert bounds.over(good, *want, n, bounds.ONE_TERM, dtype)[0] <= 1
    tol = bounds.each(want[0], want[1], want[3], n, dtype, bounds.ONE_TERM)
    for factor in (0.0, 2.0):
        for h in range(3):
            pick = torch.nn.functional.one_hot(at[:, h], n).double() * (factor - 1)
            bad = _emulate(q[:, h:h + 1], k, v, True, terms, lambda p: p * (1 + pick) + (1e-300 if factor == 0 else 0))
            assert ((bad - want[0][:, h:h + 1]).abs() > tol[:, h:h + 1]).any(-1)[1:].all(), (factor, h)
