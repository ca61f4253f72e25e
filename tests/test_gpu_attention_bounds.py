"""Attention on the GPU within bounds that a lost key, a key counted twice or a weight rounded once too often would pass
(tests/test_attention_bounds.py plants those): long caches and prompts, half of the weight on one key at every position, sums that
cancel; and lengths that are cut at a table's end."""
import pytest
import torch

import attention_bounds as bounds
import attention_refs as att
import serving_refs as ref
from conftest import announce
from pto_fuser_amd import attention_step, causal_attention
from test_gpu_attention import BF, DEV, F32, NAN, _cu, _ints, _paged, _qkv, _rand

pytestmark = pytest.mark.gpu


def _store(kv, page, dtype, seed):
    """Caches in pages of no order, with NaN behind the tokens, for sequences' (k, v) [n,G,D]; their tables."""
    need = [att.pages_of(k.shape[0], page) for k, _ in kv]
    order = torch.randperm(sum(need) + 3, generator=torch.Generator().manual_seed(seed))
    G, D = kv[0][0].shape[1:]
    tables = torch.full((len(kv), max(need) + 1), -7, dtype=torch.int32)
    caches, at = [torch.full((len(order), page, G, D), NAN, dtype=dtype) for _ in range(2)], 0
    for b, pair in enumerate(kv):
        own, at = order[at:at + need[b]], at + need[b]
        tables[b, :need[b]] = own.int()
        for cache, x in zip(caches, pair):
            rows = torch.full((need[b] * page, G, D), NAN, dtype=dtype)
            rows[:x.shape[0]] = x
            cache[own] = rows.view(need[b], page, G, D)
    return [c.to(DEV) for c in caches], tables.to(DEV)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,H,G,D,page", [
    ([4097], 5, 5, 128, 16), ([2500], 6, 1, 192, 64), ([2000, 1999, 65], 2, 1, 64, 16), ([257, 300, 512], 4, 2, 40, 16),
    ([1100, 900], 40, 2, 128, 32), ([1500], 8, 4, 256, 16)])
def test_long_caches(dtype, lens, H, G, D, page):
    announce(f"attention_step bounds {dtype} {lens} H{H} G{G} D{D} page{page}")
    (k, v), tables, rows = _paged(lens, G, D, page, dtype, sum(lens) + H)
    q = _rand(D + 1)(len(lens), H, D).to(DEV, dtype)
    o = attention_step(q, k, v, tables, _ints(lens))
    for b, n in enumerate(lens):
        want = bounds.parts(ref.f64(q[b:b + 1]), *(ref.f64(t) for t in rows[b]), causal=False)
        bounds.within(o[b:b + 1], want, n, bounds.TWO_TERMS, f"sequence {b} of {n}")


@pytest.mark.parametrize("t,B", [(17, 1), (40, 3), (300, 2), (1000, 2)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_sums_that_cancel(t, B, D):
    """Single tokens whose outputs are nearly zero: weights hold 16 bits."""
    announce(f"attention_step sums that cancel t{t} B{B} D{D}")
    gen = torch.Generator().manual_seed(t + D)
    seqs = []
    for _ in range(B):
        q, k, v = (torch.randn(n, 1, D, generator=gen).to(BF) for n in (1, t, t))
        seqs.append((q, k, bounds.balanced(q, k, v, BF)))
    (k, v), tables = _store([s[1:] for s in seqs], 16, BF, t)
    o = attention_step(torch.cat([s[0] for s in seqs]).to(DEV), k, v, tables, _ints([t] * B))
    for b, s in enumerate(seqs):
        bounds.within(o[b:b + 1], bounds.parts(*(ref.f64(x) for x in s), causal=False), t, bounds.TWO_TERMS, f"sequence {b}")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,G,D,page", [(200, 4, 64, 16), (333, 3, 128, 32), (700, 7, 64, 16), (150, 2, 256, 16)])
def test_half_of_the_weight_at_every_position(dtype, n, G, D, page):
    """Sequence b's head g points at token b G + g: each token of a cache decides one output."""
    announce(f"attention_step pointed {dtype} n{n} G{G} D{D}")
    gen, B = torch.Generator().manual_seed(n), -(-n // G)
    qs, kv = [], []
    for b in range(B):
        k, v = (torch.randn(n, G, D, generator=gen).to(dtype) for _ in range(2))
        own = k[(b * G + torch.arange(G)) % n, torch.arange(G)].float()                    # [G, D]
        q = own * (torch.log(torch.tensor(n + 1.0)) / ((own ** 2).sum(-1, keepdim=True) * D ** -0.5))
        qs.append(q.to(dtype))
        kv.append((k, v))
    (k, v), tables = _store(kv, page, dtype, n)
    q = torch.stack(qs)
    o = attention_step(q.to(DEV), k, v, tables, _ints([n] * B))
    for b in range(B):
        want = bounds.parts(ref.f64(q[b:b + 1]), *(ref.f64(t) for t in kv[b]), causal=False)
        bounds.within(o[b:b + 1], want, n, bounds.TWO_TERMS, f"tokens {b * G} to {b * G + G - 1}")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,H,G,D", [
    ([700, 37], 4, 2, 64), ([513, 200], 3, 3, 128), ([1100], 16, 4, 80), ([300] * 3, 64, 8, 64), ([900], 2, 1, 256), ([640], 64, 32, 128)])
def test_prompts(dtype, lens, H, G, D):
    announce(f"causal_attention bounds {dtype} {lens} H{H} G{G} D{D}")
    q, k, v = _qkv(lens, H, G, D, dtype, sum(lens) + D + 1)
    o, at, share = causal_attention(q, k, v, _cu(lens)), 0, H // G
    for b, n in enumerate(lens):
        for g in {0, G - 1}:
            rows, heads = slice(at, at + n), slice(g * share, (g + 1) * share)
            want = bounds.parts(*(ref.f64(t) for t in (q[rows, heads], k[rows, g:g + 1], v[rows, g:g + 1])))
            bounds.within(o[rows, heads], want, n, bounds.ONE_TERM, f"prompt {b}, keys' head {g}")
        at += n


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,H,G,D,copies", [(300, 4, 1, 64, 1), (300, 4, 1, 64, 60), (450, 4, 2, 128, 1), (260, 4, 4, 128, 30), (200, 4, 1, 256, 1),
                                            (200, 8, 2, 96, 20)])
def test_prompts_that_point_at_a_key(dtype, n, H, G, D, copies):
    """Queries that point at their own token, the one before, their tile's first and any other, alone and in calls large enough
    that a wave walks all keys of its rows."""
    announce(f"causal_attention pointed {dtype} n{n} H{H} G{G} D{D} x{copies}")
    gen, i = torch.Generator().manual_seed(n + D), torch.arange(n)
    kinds = [i, (i - 1).clamp(min=0), i // 32 * 32, (torch.rand(n, generator=gen) * (i + 1)).long()]
    at = torch.stack([kinds[h % 4] for h in range(H)], 1)
    q, k, v = bounds.pointed(gen, n, H, G, D, at, dtype)
    many = [t.repeat(copies, 1, 1).to(DEV) for t in (q, k, v)]
    o = causal_attention(*many, _cu([n] * copies)).view(copies, n, H, D)
    want = bounds.parts(*(ref.f64(t) for t in (q, k, v)))
    for c in {0, copies // 2, copies - 1}:
        bounds.within(o[c], want, n, bounds.ONE_TERM, f"copy {c}")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M", [8, 32, 70])
def test_lengths_past_the_table(dtype, M):
    """Tables whose every page holds tokens: lengths of more are those of all of them; negative ones are none."""
    announce(f"attention_step lengths past the table {dtype} M{M}")
    page, n = 16, 16 * M
    (k, v), tables, rows = _paged([n, n, n, n], 2, 64, page, dtype, M)
    tables = tables[:, :M].contiguous()
    q = _rand(M)(4, 4, 64).to(DEV, dtype)
    o = attention_step(q, k, v, tables, _ints([2 ** 31 - 1, n + 1, -5, n]))
    assert not o[2].any()
    for b in (0, 1, 3):
        want = bounds.parts(ref.f64(q[b:b + 1]), *(ref.f64(t) for t in rows[b]), causal=False)
        bounds.within(o[b:b + 1], want, n, bounds.TWO_TERMS, f"sequence {b}")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_lengths_past_the_table_without_some_pages(dtype):
    """The same where pages are outside the pool, the table's last among them."""
    announce(f"attention_step lengths past a table with gaps {dtype}")
    page, n = 16, 1000
    (k, v), tables, rows = _paged([n], 2, 64, page, dtype, 19)
    keep, gone = torch.ones(n, dtype=torch.bool), [0, 1, 7, 20, 21, 33, 62]
    for i in gone:
        tables[0, i] = [-1, 10 ** 6, k.shape[0]][i % 3]
        keep[i * page:(i + 1) * page] = False
    tables[0, -1] = -1
    q = _rand(4)(1, 4, 64).to(DEV, dtype)
    o = attention_step(q, k, v, tables, _ints([2 ** 31 - 1]))
    want = bounds.parts(ref.f64(q), *(ref.f64(t[keep]) for t in rows[0]), causal=False)
    bounds.within(o, want, n, bounds.TWO_TERMS, "o")
