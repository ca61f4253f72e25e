"""Pages, cache rows and their storing on the GPU, against the definitions request by request."""
import random

import pytest
import torch

import attention_refs as att
from conftest import announce
from pto_fuser_amd import assign_pages, release_pages, store_kv

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _state(seed, B, T, page, spare, slots=False, M=None):
    """Requests with up to T tokens in a pool of pages in no order."""
    rng = random.Random(seed)
    lengths = [rng.choice([0, 1, page, rng.randint(0, T)]) if T else 0 for _ in range(B)]
    lengths = [min(n, T) for n in lengths]
    need = [att.pages_of(n, page) for n in lengths]
    free = list(range(sum(need) + spare))
    rng.shuffle(free)
    M = M or max(need + [0]) + 3
    S = B + 4 if slots else B
    where = rng.sample(range(S), B) if slots else None
    tables = [[-9] * M for _ in range(S)]
    at = 0
    for b, n in enumerate(need):
        s = where[b] if slots else b
        tables[s][:n] = free[at:at + n]
        at += n
    return rng, lengths, free, at, tables, where


def _assign(tables, lengths, tokens, free, taken, page, capacity, slots=None, one=False):
    t = torch.tensor(tables, dtype=torch.int32, device=DEV).view(len(tables), -1)
    plan = assign_pages(t, _ints(lengths), None if one else _ints(tokens), _ints(free), _ints([taken]), page_size=page,
                        capacity=None if one else capacity, slots=None if slots is None else _ints(slots))
    rows, cu, after, at, want = att.assign(tables, lengths, tokens, free, taken, page, capacity, slots)
    assert plan.rows.dtype == torch.int64 and plan.rows.tolist() == rows
    assert plan.cu_seqlens.tolist() == cu and plan.lengths.tolist() == after and plan.taken.tolist() == [at]
    assert t.tolist() == want
    return after, at, want


@pytest.mark.parametrize("B,T,new,page", [(1, 0, 1, 16), (3, 40, 50, 16), (70, 100, 33, 16), (5, 0, 3000, 32), (1500, 60, 3, 64),
                                          (2, 5000, 1, 128), (40, 200, 0, 16), (1, 1000, 20000, 16)])
@pytest.mark.parametrize("slots", [False, True])
def test_assign(B, T, new, page, slots):
    announce(f"assign_pages B{B} T{T} new{new} page{page} slots={slots}")
    rng, lengths, free, taken, tables, where = _state(B + T, B, T, page, 3 + B * att.pages_of(new, page) + B, slots,
                                                      M=att.pages_of(T + new, page) + 2)
    tokens = [rng.randint(0, new) for _ in range(B)]
    tokens[0] = new
    _assign(tables, lengths, tokens, free, taken, page, sum(tokens) + 9, where)


@pytest.mark.parametrize("B", [1, 64, 1024, 1025, 3000])
def test_assign_a_step(B):
    """One token each, several steps on: pages fill and the next begin."""
    announce(f"assign_pages step B{B}")
    page = 16
    _, lengths, free, taken, tables, _ = _state(B, B, 70, page, 2 * B)
    for _ in range(3):
        lengths, taken, tables = _assign(tables, lengths, [1] * B, free, taken, page, B, one=True)


def test_assign_refuses_whole_requests():
    """Too few pages, full tables, slots outside the pool, a capacity that ends inside a request."""
    announce("assign_pages refusals")
    page = 16
    for seed in range(6):
        rng, lengths, free, taken, tables, where = _state(seed, 20, 100, page, 11, True, M=9)
        where[3], where[9] = -1, 24 + seed
        tokens = [rng.randint(0, 60) for _ in range(20)]
        tokens[5] = 0
        _assign(tables, lengths, tokens, free, taken, page, sum(tokens), where)
        _assign(tables, lengths, tokens, free, taken, page, sum(tokens[:13]) + 5, where)
        _assign(tables, lengths, tokens, free, len(free), page, sum(tokens), where)
        _assign(tables, lengths, [160] + tokens[1:], free, taken, page, 400, where)


def test_assign_of_nothing():
    announce("assign_pages of nothing")
    tables = torch.zeros(0, 4, dtype=torch.int32, device=DEV)
    plan = assign_pages(tables, _ints([]), _ints([]), _ints([]), _ints([0]), page_size=16, capacity=5)
    assert plan.rows.tolist() == [-1] * 5 and plan.cu_seqlens.tolist() == [0] and plan.taken.tolist() == [0]
    plan = assign_pages(tables.new_zeros(2, 0), _ints([0, 0]), _ints([1, 0]), _ints([]), _ints([0]), page_size=16, capacity=0)
    assert plan.lengths.tolist() == [0, 0] and plan.rows.shape == (0,)


@pytest.mark.parametrize("B,T,slots", [(1, 50, False), (30, 300, True), (700, 90, False)])
def test_release(B, T, slots):
    announce(f"release_pages B{B} T{T}")
    page = 16
    rng, lengths, free, taken, tables, where = _state(B, B, T, page, 5, slots)
    some = sorted(rng.sample(range(B), (B + 1) // 2))
    own = [lengths[b] for b in some]
    at = [where[b] if slots else b for b in some]
    f = _ints(free)
    left = release_pages(_ints(tables), _ints(own), f, _ints([taken]), page_size=page, slots=_ints(at))
    want, count = att.release(tables, own, free, taken, page, at)
    assert left.tolist() == [count] and f.tolist() == want
    # no page is in two places
    held = [p for b in range(B) if b not in some for p in tables[where[b] if slots else b][:att.pages_of(lengths[b], page)]]
    assert sorted(held + f.tolist()[count:]) == list(range(len(free)))


def test_release_of_more_than_was_taken():
    """Slots outside the pool have no pages; what would come back past the pool's start stays out."""
    announce("release_pages past the start")
    page, tables = 16, [[i * 3, i * 3 + 1, i * 3 + 2] for i in range(4)]
    for lengths, slots, taken in (([40, 16, 48, 3], [0, 1, 2, 3], 5), ([40, 40], [-1, 9], 4), ([48, 48, 0, 16], [2, 1, 0, 3], 4)):
        free = list(range(100, 112))
        f = _ints(free)
        left = release_pages(_ints(tables), _ints(lengths), f, _ints([taken]), page_size=page, slots=_ints(slots))
        want, count = att.release(tables, lengths, free, taken, page, slots)
        assert left.tolist() == [count] and f.tolist() == want


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,G,D,page", [(1, 1, 8, 16), (77, 3, 40, 16), (300, 2, 128, 64), (5, 8, 256, 32)])
@pytest.mark.parametrize("layout", ["plain", "one", "heads first"])
def test_store(dtype, N, G, D, page, layout):
    """Rows in no order, some skipped or outside the cache; the rest of the cache keeps its bits."""
    announce(f"store_kv {dtype} N{N} G{G} D{D} page{page} {layout}")
    gen = torch.Generator().manual_seed(N)
    pages = att.pages_of(N, page) + 2
    row = torch.randn(N, 2 * G * D + 3, generator=gen).to(DEV, dtype)
    k, v = (t.unflatten(-1, (G, D)) for t in (row[:, 1:1 + G * D], row[:, 1 + G * D:1 + 2 * G * D]))
    rows = torch.randperm(pages * page, generator=gen)[:N]
    rows[::7] = torch.tensor([-1, pages * page, -(1 << 40), 1 << 40])[torch.arange(len(rows[::7])) % 4]
    old = torch.randn(2, pages, page, G, D, generator=gen).to(DEV, dtype)
    if layout == "one":
        both = old.transpose(0, 1).contiguous()
        kc, vc = both[:, 0], both[:, 1]
    elif layout == "heads first":
        kc, vc = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in old)
    else:
        kc, vc = old[0].clone(), old[1].clone()
    want = old.clone().view(2, pages * page, G, D)
    for t, r in enumerate(rows.tolist()):
        if 0 <= r < pages * page:
            want[0, r], want[1, r] = k[t], v[t]
    assert store_kv(k, v, kc, vc, rows.to(DEV)) is None
    assert torch.equal(kc, want[0].view_as(kc)) and torch.equal(vc, want[1].view_as(vc))


def test_store_past_32_bits():
    announce("store_kv past 4 GiB")
    pages = (5 << 30) // (16 * 8 * 128 * 2)
    kc, vc = (torch.zeros(pages, 16, 8, 128, device=DEV, dtype=BF) for _ in range(2))
    k, v = (torch.randn(3, 8, 128, device=DEV).to(BF) for _ in range(2))
    rows = torch.tensor([pages * 16 - 1, 0, pages * 16 - 33], device=DEV)
    store_kv(k, v, kc, vc, rows)
    for cache, x in ((kc, k), (vc, v)):
        assert torch.equal(cache.view(-1, 8, 128)[rows], x)
        assert int(cache.view(torch.int32).count_nonzero()) <= 3 * 8 * 64


def test_assign_of_numbers_at_their_limits():
    """Sums of tokens past 32 bits, lengths at a table's end: refused requests stay refused, and the rest is served."""
    announce("assign_pages at the limits")
    page, big = 65536, 2 ** 31 - 1
    M = (1 << 30) // page
    for lengths, tokens, capacity in (([0, 0, 0, 5], [big, big, big, 1], 40), ([(1 << 30) - 1, (1 << 30) - 1, 3], [1, 2, 4], 90),
                                      ([7, 0, 0], [3, big, 2], 10)):
        B = len(lengths)
        tables = [[b * 3 + i for i in range(3)] + [5] * (M - 3) for b in range(B)]
        _assign(tables, lengths, tokens, list(range(50, 90)), 2, page, capacity)
    lengths = _ints([-3, 4])
    tables = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    plan = assign_pages(tables, lengths, _ints([-7, 2]), _ints([9]), _ints([-1]), page_size=16, capacity=5)
    assert plan.cu_seqlens.tolist() == [0, 0, 2] and plan.rows.tolist() == [4, 5, -1, -1, -1] and plan.lengths.tolist() == [0, 6]
    assert plan.taken.tolist() == [0]
