"""Infinities in the values of attention, on the GPU: where the definition gives an infinity or NaN the operators give the
same one, and every other output keeps its bits."""
import pytest
import torch

from conftest import announce
from pto_fuser_amd import attention_step, causal_attention
from test_gpu_attention import BF, DEV, F32, INF, NAN, _cu, _ints, _paged, _qkv, _rand

pytestmark = pytest.mark.gpu


def _same(got, want, what):
    """The same bits, a NaN of any bits for a NaN."""
    bad = ~((got == want) | (got.isnan() & want.isnan()))
    assert not bad.any(), f"{what}: {int(bad.sum())} values differ, the first at {bad.nonzero()[0].tolist()}"


# (column -> the values that its tokens hold) and what their weighted sum is, all weights being positive
MARKS = [((INF,), INF), ((-INF,), -INF), ((INF, INF), INF), ((INF, -INF), NAN), ((-INF, NAN), NAN)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,H,G,D,page", [
    ([300, 77, 20, 1, 33], 4, 2, 64, 16), ([1500, 300, 17, 64], 4, 2, 128, 16), ([90, 600, 2], 20, 1, 136, 64),
    ([1100, 3], 6, 3, 40, 32), ([700, 50], 8, 2, 256, 16)])
def test_step_infinities(dtype, lens, H, G, D, page):
    """In the first, a middle and the last token of a sequence: its column of the heads that share it takes the infinity, two
    of different signs a NaN."""
    announce(f"attention_step infinities {dtype} {lens} H{H} G{G} D{D} page{page}")
    (k, v), tables, _ = _paged(lens, G, D, page, dtype, sum(lens) + D)
    q, share = _rand(D)(len(lens), H, D).to(DEV, dtype), H // G
    clean = attention_step(q, k, v, tables, _ints(lens))
    for marks, want in MARKS:
        for b, n in enumerate(lens):
            for at in {(0, n // 2), (n - 1, n // 3), (n // 2, n - 1)}:
                g, col = (b + at[0]) % G, (7 * b + at[0]) % D
                new, good = v.clone(), clean.clone()
                for t, x in zip(at, marks):
                    new[tables[b, t // page], t % page, g, col] = x
                last = marks[-1] if n == 1 or at[0] == at[1] else want        # (one token, marked twice)
                good[b, g * share:(g + 1) * share, col] = last
                _same(attention_step(q, k, new, tables, _ints(lens)), good, (marks, b, at))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n", [200, 1000])
def test_step_infinities_beside_a_page_outside_the_pool(dtype, n):
    """Tokens of a page outside the pool weigh nothing, whatever stands in for them."""
    announce(f"attention_step infinities beside a page outside {dtype} n{n}")
    page = 16
    (k, v), tables, _ = _paged([n], 2, 64, page, dtype, n)
    for gone in (0, 1, 4, 7, 10):
        tables[0, gone] = -1
    q = _rand(n)(1, 4, 64).to(DEV, dtype)
    clean = attention_step(q, k, v, tables, _ints([n]))
    assert torch.isfinite(clean).all()
    for t in (2 * page, 3 * page + 5, 5 * page, 6 * page + 15, 8 * page, n - 1):
        new, good = v.clone(), clean.clone()
        new[tables[0, t // page], t % page, 1, 9] = INF
        good[0, 2:, 9] = INF
        _same(attention_step(q, k, new, tables, _ints([n])), good, t)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,G,D", [(4, 2, 64), (16, 2, 128), (256, 2, 64), (3, 1, 96), (4, 2, 256)])
def test_prompt_infinities(dtype, H, G, D):
    """From its own token on, in its column of the heads that share it; with one of the other sign, NaN from the later one on."""
    announce(f"causal_attention infinities {dtype} H{H} G{G} D{D}")
    lens, share = [230, 40], H // G
    q, k, v = _qkv(lens, H, G, D, dtype, 3 * D)
    clean = causal_attention(q, k, v, _cu(lens))
    for marks, _ in MARKS:
        for at in ((0, 100), (63, 64), (200, 229)):
            new, good, so_far = v.clone(), clean.clone(), 0.0
            for i, (t, x) in enumerate(zip(at, marks)):
                new[t, G - 1, 5] = x
                so_far += x
                good[t:lens[0], (G - 1) * share:, 5] = so_far
            _same(causal_attention(q, k, new, _cu(lens)), good, (marks, at))
