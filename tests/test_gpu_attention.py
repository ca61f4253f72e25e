"""Attention over prompts and over a paged cache on the GPU, against its definition in float64: odd sizes, views, lengths of
zero and one, groups of heads, values that are not finite, pages in any order and rows behind the last token."""
import pytest
import torch

import attention_refs as att
import serving_refs as ref
from conftest import announce
from pto_fuser_amd import attention_step, causal_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


def _rand(seed):
    gen = torch.Generator().manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=gen)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _cu(lens):
    return _ints([sum(lens[:i]) for i in range(len(lens) + 1)])


def _wide(t, extra, at=1):
    """The same values as a view of rows that are ``extra`` wider, starting ``at`` elements in; NaN around them."""
    buf = torch.full((*t.shape[:-1], t.shape[-1] + extra), NAN, dtype=t.dtype, device=t.device)
    view = buf[..., at:at + t.shape[-1]]
    view.copy_(t)
    return view


def _qkv(lens, H, G, D, dtype, seed, size=1.0):
    r, N = _rand(seed), sum(lens)
    return [(size * r(N, h, D)).to(DEV, dtype) for h in (H, G)] + [r(N, G, D).to(DEV, dtype)]


def _check_prompts(o, q, k, v, lens, what, scale=None):
    at = 0
    for i, n in enumerate(lens):
        rows = slice(at, at + n)
        want = att.attention(*(ref.f64(t[rows]) for t in (q, k, v)), scale=scale)
        att.check(o[rows], *want, n, f"{what}, prompt {i}")
        at += n


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,H,G,D", [
    ([1], 1, 1, 8), ([2, 0, 1], 2, 1, 64), ([31, 33, 64, 65], 4, 2, 64), ([127, 128, 129], 2, 2, 128), ([300], 6, 1, 40),
    ([5, 0, 0, 257, 3], 5, 5, 80), ([200, 56], 8, 2, 120), ([513], 3, 3, 128), ([1] * 70 + [90], 2, 1, 32), ([0, 0], 2, 1, 64),
    ([1, 65, 0, 130], 4, 2, 256), ([33, 300], 3, 1, 200), ([64], 2, 2, 136)])
def test_prompts(dtype, lens, H, G, D):
    announce(f"causal_attention {dtype} {lens[:5]} H{H} G{G} D{D}")
    q, k, v = _qkv(lens, H, G, D, dtype, sum(lens) + D)
    o = causal_attention(q, k, v, _cu(lens))
    _check_prompts(o, q, k, v, lens, "o")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,H,G,D", [
    ([1100, 37], 64, 8, 64), ([900], 80, 16, 128), ([1] * 100 + [700, 0, 65], 64, 4, 128), ([700, 500], 24, 3, 64), ([1025], 32, 2, 128),
    ([130] * 9, 16, 4, 72), ([1100, 37], 64, 8, 256), ([500, 129], 64, 16, 168)])
def test_many_workgroups(dtype, lens, H, G, D):
    """Sizes at which a row is one wave's, two waves' and four waves', up to 64 prompts and more of them; some heads of each."""
    announce(f"causal_attention {dtype} {lens[-2:]} of {len(lens)} H{H} G{G} D{D}")
    q, k, v = _qkv(lens, H, G, D, dtype, sum(lens) + H)
    o = causal_attention(q, k, v, _cu(lens))
    r = H // G
    for h in (0, r - 1, H - 1):
        g = h // r
        _check_prompts(o[:, h:h + 1], q[:, h:h + 1], k[:, g:g + 1], v[:, g:g + 1], lens, f"head {h}")


@pytest.mark.parametrize("H", [2, 64])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_prompts_that_share_a_buffer_with_others(dtype, H):
    """70 prompts, some of no rows, behind rows of none and before others: each is itself, and the rest is zero."""
    announce(f"causal_attention 70 prompts {dtype} H{H}")
    lens = [(i * 37) % 150 for i in range(70)]
    starts = [11 + sum(lens[:i]) for i in range(71)]
    N = starts[-1] + 500
    q, k, v = _qkv([N], H, 2, 64, dtype, 41)
    o = causal_attention(q, k, v, _ints(starts))
    assert not o[:11].any() and not o[starts[-1]:].any()
    inside = slice(11, starts[-1])
    _check_prompts(o[inside, H - 1:], q[inside, H - 1:], k[inside, 1:], v[inside, 1:], lens, "o")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D,extra,at", [(64, 8, 8), (128, 5, 1), (80, 16, 8), (96, 3, 2)])
def test_prompts_of_views(dtype, D, extra, at):
    """Rows inside wider rows, on 16-byte vectors and off them; heads stored before tokens; an output that is a view."""
    announce(f"causal_attention views {dtype} D{D} extra={extra}")
    lens = [67, 130]
    q, k, v = _qkv(lens, 4, 2, D, dtype, D)
    out = _wide(torch.zeros(sum(lens), 4, D, device=DEV, dtype=dtype), 3)
    o = causal_attention(_wide(q, extra, at), k.transpose(0, 1).contiguous().transpose(0, 1), _wide(v, extra, at), _cu(lens),
                         out=out, scale=0.2)
    assert o is out
    _check_prompts(o, q, k, v, lens, "o", scale=0.2)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_padded_prompts(dtype):
    """A padded batch: what lies past a prompt's length is NaN and is not read, and the output is zero there; in a given
    output it is left as it was."""
    announce(f"causal_attention padded {dtype}")
    T, lens = 150, [150, 0, 1, 129, 64]
    q, k, v = _qkv([T] * len(lens), 4, 2, 64, dtype, 7)
    live = torch.cat([torch.arange(T) < n for n in lens])
    for t in (q, k, v):
        t[~live.to(DEV)] = NAN
    cu, lengths = _ints([T * i for i in range(len(lens) + 1)]), _ints(lens)
    o = causal_attention(q, k, v, cu, lengths=lengths)
    assert not o[~live.to(DEV)].any()
    _check_prompts(o[live.to(DEV)], *(t[live.to(DEV)] for t in (q, k, v)), lens, "o")
    given = torch.full_like(o, 7.0)
    causal_attention(q, k, v, cu, lengths=lengths, out=given)
    assert torch.equal(given[live.to(DEV)], o[live.to(DEV)]) and bool((given[~live.to(DEV)] == 7.0).all())


def test_rows_of_no_prompt():
    """Rows before the first prompt and behind the last one: zero in an output of the call's, untouched in a given one."""
    announce("causal_attention rows of no prompt")
    N, first, lens = 1000, 37, [40, 0, 100]
    q, k, v = _qkv([N], 3, 1, 64, BF, 3)
    cu = _ints([first, first + 40, first + 40, first + 140])
    rows = slice(first, first + 140)
    outside = torch.ones(N, dtype=torch.bool)
    outside[rows] = False
    o = causal_attention(q, k, v, cu)
    _check_prompts(o[rows], q[rows], k[rows], v[rows], lens, "o")
    assert not o[outside.to(DEV)].any()
    given = torch.full_like(o, -3.0)
    causal_attention(q, k, v, cu, out=given)
    assert torch.equal(given[rows], o[rows]) and bool((given[outside.to(DEV)] == -3.0).all())
    for empty in (_ints([0]), _ints([5, 5])):
        assert not causal_attention(q, k, v, empty).any()
    assert causal_attention(q[:0], k[:0], v[:0], _ints([0])).shape == (0, 3, 64)


def test_offsets_outside_the_rows_are_cut():
    """Offsets past the rows or falling: every access stays inside, and prompts inside the rows are right."""
    announce("causal_attention offsets outside")
    q, k, v = _qkv([100], 2, 1, 64, F32, 5)
    o = causal_attention(q, k, v, _ints([-4, 50, 4000]))
    _check_prompts(o, q, k, v, [50, 50], "o")
    causal_attention(q, k, v, _ints([60, 20, 100, 7]), lengths=_ints([-5, 1 << 30, 9]))
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("size", [0.0, 30.0, 1e4])
def test_flat_and_sharp_weights(dtype, size):
    """All weights equal; scores of hundreds and of 1e8, whose weights are one and zeros."""
    announce(f"causal_attention {dtype} scores of size {size}")
    lens = [200, 70]
    q, k, v = _qkv(lens, 2, 2, 64, dtype, 11, size)
    o = causal_attention(q, k, v, _cu(lens))
    if size < 1e4:
        _check_prompts(o, q, k, v, lens, "o")
    else:
        assert torch.isfinite(o).all() and bool((o.abs() <= v.abs().amax() * (1 + 2.0 ** -7)).all())


def test_scores_that_rise_along_the_keys():
    """Each key's score is higher than all before: the carried bound moves at every tile."""
    announce("causal_attention rising scores")
    n, D = 700, 64
    q = torch.ones(n, 1, D, device=DEV)
    k = (torch.arange(n, device=DEV, dtype=F32) * 0.05)[:, None, None].expand(n, 1, D).contiguous()
    v = _rand(1)(n, 1, D).to(DEV)
    for dtype in (BF, F32):
        a = [t.to(dtype) for t in (q, k, v)]
        _check_prompts(causal_attention(*a, _cu([n])), *a, [n], "o")
        b = [a[0], a[1].flip(0).contiguous(), a[2]]
        _check_prompts(causal_attention(*b, _cu([n])), *b, [n], "o, falling")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("what,H,G,D", [(NAN, 4, 2, 64), (INF, 4, 2, 128), (NAN, 256, 2, 64), (INF, 80, 2, 128), (NAN, 6, 2, 40),
                                        (INF, 256, 2, 96), (NAN, 80, 2, 120), (INF, 96, 2, 32), (NAN, 4, 2, 256), (INF, 160, 2, 144)])
def test_values_that_are_not_finite(dtype, D, what, H, G):
    """In v they reach their own column from their own token on, in a key the tokens from it on, in a query its own row;
    the next prompt and the other heads stay as they are."""
    announce(f"causal_attention not finite {dtype} D{D} {what} H{H}")
    n = 330
    lens = [n, 100]
    clean = _qkv(lens, H, G, D, dtype, 13)
    good = ref.f64(causal_attention(*clean, _cu(lens)))
    for t in (0, 5, 63, 64, 200, 329):
        q, k, v = (x.clone() for x in clean)
        v[t, 1, 3] = what
        bad = torch.zeros(sum(lens), H, D, dtype=torch.bool)
        bad[t:n, H // 2:, 3] = True
        o = ref.f64(causal_attention(q, k, v, _cu(lens)))
        assert torch.equal(~torch.isfinite(o), bad), t
        assert torch.equal(o[~bad], good[~bad]), t
    q, k, v = (x.clone() for x in clean)                 # a later token's, and another's of the same tile
    v[300, 0, D - 1], v[302, 0, 0] = what, -INF
    bad = torch.zeros(sum(lens), H, D, dtype=torch.bool)
    bad[300:n, :H // 2, D - 1] = bad[302:n, :H // 2, 0] = True
    o = ref.f64(causal_attention(q, k, v, _cu(lens)))
    assert torch.equal(~torch.isfinite(o), bad) and torch.equal(o[~bad], good[~bad])
    for t in (0, 70, 329):
        q, k, v = (x.clone() for x in clean)
        k[t, 0, 5] = NAN
        bad = torch.zeros(sum(lens), H, D, dtype=torch.bool)
        bad[t:n, :H // 2] = True
        o = ref.f64(causal_attention(q, k, v, _cu(lens)))
        assert torch.equal(~torch.isfinite(o), bad) and torch.equal(o[~bad], good[~bad]), t
        q, k, v = (x.clone() for x in clean)
        q[t, 1, 5] = NAN
        bad = torch.zeros(sum(lens), H, D, dtype=torch.bool)
        bad[t, 1] = True
        o = ref.f64(causal_attention(q, k, v, _cu(lens)))
        assert torch.equal(~torch.isfinite(o), bad) and torch.equal(o[~bad], good[~bad]), t


def test_keys_of_minus_infinity():
    """A key whose scores are minus infinity weighs nothing; a query that sees no other gives zeros."""
    announce("causal_attention scores of minus infinity")
    n, D = 90, 64
    q, k, v = _qkv([n], 1, 1, D, F32, 4)
    q[:, :, 0] = 1.0
    k[:3, :, 0] = -INF
    o = causal_attention(q, k, v, _cu([n]))
    assert not o[:3].any()
    want, mag, size = att.attention(ref.f64(q)[3:], ref.f64(k)[3:], ref.f64(v)[3:])
    att.check(o[3:], want, mag, size, n, "o")


def test_rows_far_apart():
    """Token strides that take a prompt's rows past 4 GiB of its first."""
    announce("causal_attention rows far apart")
    n, stride = 700, 1 << 22
    q, k, v = _qkv([n], 1, 1, 64, BF, 6)
    far = [torch.empty((n - 1) * stride + 64, device=DEV, dtype=BF).as_strided((n, 1, 64), (stride, 64, 1)) for _ in range(2)]
    far[0].copy_(k)
    far[1].copy_(v)
    assert torch.equal(causal_attention(q, *far, _cu([n])), causal_attention(q, k, v, _cu([n])))


# ------------------------------------------------------------------------------------------
#  Single tokens
# ------------------------------------------------------------------------------------------
def _paged(lens, G, D, page, dtype, seed, extra=2, slots=None, S=None):
    """Caches whose pages are in no order, tables of them, and the keys and values that they hold; NaN everywhere else."""
    r, gen = _rand(seed), torch.Generator().manual_seed(seed)
    need = [att.pages_of(n, page) for n in lens]
    pages = sum(need) + extra
    order, M = torch.randperm(pages, generator=gen), max(need + [1]) + 1
    tables = torch.full((S or len(lens), M), -7, dtype=torch.int32)
    caches = [torch.full((pages, page, G, D), NAN) for _ in range(2)]
    rows, at = [], 0
    for b, n in enumerate(lens):
        own = order[at:at + need[b]]
        at += need[b]
        tables[b if slots is None else slots[b], :need[b]] = own.int()
        kv = [r(n, G, D).to(dtype) for _ in range(2)]
        for cache, x in zip(caches, kv):
            flat = cache[own].flatten(0, 1)
            flat[:n] = x.float()
            cache[own] = flat.view(need[b], page, G, D)
        rows.append(kv)
    return [c.to(DEV, dtype) for c in caches], tables.to(DEV), rows


def _check_step(o, q, rows, lens, what, scale=None):
    for b, n in enumerate(lens):
        if not n:
            assert not o[b].any(), (what, b)
            continue
        want = att.attention(ref.f64(q[b:b + 1]), ref.f64(rows[b][0]), ref.f64(rows[b][1]), causal=False, scale=scale)
        att.check(o[b:b + 1], *want, n, f"{what}, sequence {b} of {n}")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,H,G,D,page", [
    ([1], 1, 1, 8, 16), ([0, 1, 2, 15, 16, 17], 4, 2, 64, 16), ([127, 128, 129, 31, 33], 8, 1, 128, 16), ([600], 16, 1, 64, 32),
    ([700, 3], 20, 1, 80, 16), ([5, 900], 40, 2, 128, 64), ([1023, 0, 1], 6, 2, 64, 128), ([4097], 5, 5, 128, 16),
    ([64] * 70 + [2000], 2, 1, 64, 16), ([300, 40], 2, 2, 120, 256),
    ([1, 0, 700, 33], 8, 2, 256, 16), ([2500], 6, 1, 192, 64), ([90, 600], 20, 1, 136, 16)])
def test_step(dtype, lens, H, G, D, page):
    announce(f"attention_step {dtype} {lens[:5]} H{H} G{G} D{D} page{page}")
    (k, v), tables, rows = _paged(lens, G, D, page, dtype, sum(lens) + D)
    q = _rand(D)(len(lens), H, D).to(DEV, dtype)
    o = attention_step(q, k, v, tables, _ints(lens))
    _check_step(o, q, rows, lens, "o")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["one", "heads first"])
def test_step_of_views_and_slots(dtype, layout):
    """Keys and values in one buffer, heads before rows; tables by slot, slots outside the pool; queries inside wider rows."""
    announce(f"attention_step views {dtype} {layout}")
    lens, slots, S = [700, 40, 900, 77], [5, -1, 2, 9], 9
    (k, v), tables, rows = _paged(lens, 2, 64, 16, dtype, 17, slots=[5, 0, 2, 1], S=S)
    tables[1] = -7
    if layout == "one":
        both = torch.stack([k, v], 1)
        k, v = both[:, 0], both[:, 1]
    else:
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    q = _rand(3)(4, 6, 64).to(DEV, dtype)
    out = _wide(torch.full((4, 6, 64), 5.0, device=DEV, dtype=dtype), 3)
    o = attention_step(_wide(q, 5), k, v, tables, _ints(lens), slots=_ints(slots), out=out, scale=0.3)
    assert o is out and not o[1].any() and not o[3].any()
    for b in (0, 2):
        _check_step(o[b:b + 1], q[b:b + 1], rows[b:b + 1], lens[b:b + 1], "o", scale=0.3)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_step_pages_outside_the_pool(dtype):
    """They hold no tokens: the sequence is attended to without them; lengths past the table are cut."""
    announce(f"attention_step pages outside {dtype}")
    page, n = 16, 1000
    (k, v), tables, rows = _paged([n, 50], 2, 64, page, dtype, 19)
    q = _rand(4)(2, 4, 64).to(DEV, dtype)
    gone, keep = [0, 1, 7, 20, 21, 33, 62], torch.ones(n, dtype=torch.bool)
    for i in gone:
        tables[0, i] = [-1, 10 ** 6, k.shape[0]][i % 3]
        keep[i * page:(i + 1) * page] = False
    kept = [[t[keep] for t in rows[0]], rows[1]]
    o = attention_step(q, k, v, tables, _ints([n, 50]))
    _check_step(o, q, kept, [int(keep.sum()), 50], "o")
    tables[1] = -1
    assert not attention_step(q, k, v, tables, _ints([n, 50]))[1].any()
    M = tables.shape[1]
    full = (M - 1) * page if n > (M - 1) * page else n
    tables[0, M - 1] = -1
    o = attention_step(q, k, v, tables, _ints([2 ** 31 - 1, -5]))
    assert not o[1].any() and (torch.isfinite(o[0]).all() or full < (M - 1) * page)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_step_values_that_are_not_finite(dtype):
    """A NaN in v reaches its column of the heads that share it, in a key those heads, in a query its own head."""
    announce(f"attention_step not finite {dtype}")
    lens = [1500, 300, 20]
    (k, v), tables, _ = _paged(lens, 2, 64, 16, dtype, 23)
    q = _rand(5)(3, 4, 64).to(DEV, dtype)
    good = ref.f64(attention_step(q, k, v, tables, _ints(lens)))
    at = int(tables[0, 50])
    bad = torch.zeros(3, 4, 64, dtype=torch.bool)
    for cache, mark in ((v, (0, slice(2, 4), 9)), (k, (0, slice(2, 4)))):
        new = cache.clone()
        new[at, 3, 1, 9] = NAN
        o = ref.f64(attention_step(q, new if cache is k else k, new if cache is v else v, tables, _ints(lens)))
        bad.zero_()
        bad[mark] = True
        assert torch.equal(~torch.isfinite(o), bad) and torch.equal(o[~bad], good[~bad])
    q[1, 3, 0] = NAN
    o = ref.f64(attention_step(q, k, v, tables, _ints(lens)))
    bad.zero_()
    bad[1, 3] = True
    assert torch.equal(~torch.isfinite(o), bad) and torch.equal(o[~bad], good[~bad])


def test_step_offsets_past_32_bits():
    """A cache of 6 GiB: pages whose bytes lie past 2^32."""
    announce("attention_step pages past 4 GiB")
    page, G, D, n = 64, 8, 128, 2000
    pages = (6 << 30) // (page * G * D * 2)
    k, v = (torch.empty(pages, page, G, D, device=DEV, dtype=BF) for _ in range(2))
    r = _rand(8)
    rows = [[r(n, G, D).to(BF) for _ in range(2)]]
    need = att.pages_of(n, page)
    own = torch.linspace(0, pages - 1, need).long().flip(0)
    for cache, x in zip((k, v), rows[0]):
        padded = torch.zeros(need * page, G, D, dtype=BF)
        padded[:n] = x
        cache[own.to(DEV)] = padded.view(need, page, G, D).to(DEV)
    q = r(1, 16, D).to(DEV, BF)
    o = attention_step(q, k, v, own[None].int().to(DEV), _ints([n]))
    _check_step(o, q, rows, [n], "o")


def test_step_of_nothing():
    announce("attention_step of nothing")
    k = torch.empty(0, 16, 2, 64, device=DEV)
    q = torch.ones(3, 4, 64, device=DEV)
    o = attention_step(q, k, k, torch.zeros(3, 5, dtype=torch.int32, device=DEV), _ints([9, 0, 2]))
    assert not o.any()
    assert attention_step(q[:0], k, k, torch.zeros(0, 5, dtype=torch.int32, device=DEV), _ints([])).shape == (0, 4, 64)
    k = torch.ones(4, 16, 2, 64, device=DEV)
    assert not attention_step(q, k, k, torch.zeros(3, 0, dtype=torch.int32, device=DEV), _ints([9, 0, 2])).any()


def test_results_do_not_vary():
    """The same call gives the same bits: no order of atomics enters."""
    announce("attention twice")
    lens = [900, 33, 512]
    q, k, v = _qkv(lens, 4, 2, 128, BF, 29)
    first = causal_attention(q, k, v, _cu(lens))
    (kc, vc), tables, _ = _paged(lens, 2, 128, 16, BF, 31)
    q1 = q[:3].contiguous()
    step = attention_step(q1, kc, vc, tables, _ints(lens))
    for _ in range(5):
        assert torch.equal(causal_attention(q, k, v, _cu(lens)), first)
        assert torch.equal(attention_step(q1, kc, vc, tables, _ints(lens)), step)
