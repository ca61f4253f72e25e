"""An attention layer among recurrent ones as it is served: prompts into pages, single tokens over them, requests that leave
and others that take their pages; against the definition in float64, and captured."""
import pytest
import torch

import attention_refs as att
import serving_refs as ref
from conftest import announce
from pto_fuser_amd import assign_pages, attention_step, causal_attention, release_pages, store_kv
from pto_fuser_amd.forwards import make_attention_layer, make_gdn_layer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
D, PAGE = 128, 16
# Two ways to the same bfloat16 layer differ by the roundings of the rows between (2^-9 a value) and of the 8-bit codes (2^-4,
# of which a fraction moves): in the 2-norm less than the rounding of every code at once.
CLOSE = 2.0 ** -4


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _hidden(N, seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(N, D, generator=gen).to(DEV, torch.bfloat16) for _ in range(2)]


def _far(a, b):
    a, b = ref.f64(a), ref.f64(b)
    return ((a - b).norm() / b.norm()).item()


def _definition(layer, hidden, residual):
    """One prompt through the layer's formulas in float64 (weights as they are stored)."""
    y, h = ref.norm(ref.f64(hidden), ref.f64(layer.norm_w), ref.f64(residual))
    row = y @ ref.f64(layer.in_w)
    q, k, v = (t.unflatten(-1, (-1, layer.head)) for t in row.split([layer.H * layer.head] + [layer.G * layer.head] * 2, dim=-1))
    o, _, _ = att.attention(q, k, v)
    y, _ = ref.norm(o.flatten(-2), ref.f64(layer.out_norm_w))
    return y @ ref.f64(layer.out.plain()).t(), h


class Pool:
    """What the layers of a model share: tables, the free list and how much of it is taken."""

    def __init__(self, slots, pages, width):
        gen = torch.Generator().manual_seed(pages)
        self.tables = torch.full((slots, width), -1, dtype=torch.int32, device=DEV)
        self.free, self.taken = torch.randperm(pages, generator=gen).int().to(DEV), _ints([0])

    def assign(self, lengths, tokens, slots, capacity=None):
        plan = assign_pages(self.tables, lengths, tokens, self.free, self.taken, page_size=PAGE, capacity=capacity, slots=slots)
        self.taken = plan.taken
        return plan


def test_prompts_then_tokens_against_the_definition():
    """Prompts of uneven length into slots of a pool, tokens one by one, one request leaves and a new one takes its pages:
    every output is that of the longer prompt alone."""
    announce("attention layer: prompts, tokens, requests that leave and come")
    layer, pool = make_attention_layer(D, 6, 2, 64, seed=3), Pool(5, 14, 6)
    cache = layer.cache(14, PAGE)
    lens, more, slots = [50, 17, 1], 20, _ints([3, 0, 4])
    seqs = [_hidden(n + more, 10 + n) for n in lens]
    pack = [torch.cat([s[i][:n] for s, n in zip(seqs, lens)] + [s[i][:2] for s in seqs[:1]]) for i in range(2)]   # two rows of none
    want = [_definition(layer, *s) for s in seqs]
    plan = pool.assign(_ints([0] * 3), _ints(lens), slots, capacity=sum(lens) + 2)
    assert plan.rows[sum(lens):].tolist() == [-1, -1]
    out, stream = layer.prefill(*pack, cache, plan)
    at = 0
    for (o, h), n in zip(want, lens):
        assert _far(out[at:at + n], o[:n]) < CLOSE and _far(stream[at:at + n], h[:n]) < 2.0 ** -8
        at += n
    lengths, got = plan.lengths, []
    for t in range(more):
        plan = pool.assign(lengths, None, slots)
        rows = [torch.stack([s[i][n + t] for s, n in zip(seqs, lens)]) for i in range(2)]
        got.append(layer.step(*rows, cache, plan, pool.tables, slots)[0])
        lengths = plan.lengths
    assert lengths.tolist() == [n + more for n in lens]
    for b, ((o, _), n) in enumerate(zip(want, lens)):
        assert _far(torch.stack([g[b] for g in got]), o[n:]) < CLOSE, b
    # the first leaves; a prompt that needs its pages comes into another slot, and the others go on undisturbed
    left = pool.taken.item()
    pool.taken = release_pages(pool.tables, lengths[:1].contiguous(), pool.free, pool.taken, page_size=PAGE, slots=slots[:1].contiguous())
    assert pool.taken.item() == left - att.pages_of(lens[0] + more, PAGE)
    new = _hidden(90, 5)
    plan = pool.assign(_ints([0]), _ints([90]), _ints([1]), capacity=90)
    assert plan.lengths.tolist() == [90] and pool.taken.item() == left - 5 + 6
    out, _ = layer.prefill(*new, cache, plan)
    assert _far(out, _definition(layer, *new)[0]) < CLOSE
    both = torch.cat([lengths[1:], plan.lengths])
    plan = pool.assign(both, None, _ints([0, 4, 1]))
    last = [_hidden(1, 70 + b) for b in range(3)]
    out, _ = layer.step(*(torch.cat([x[i] for x in last]) for i in range(2)), cache, plan, pool.tables, _ints([0, 4, 1]))
    for b, s in enumerate((seqs[1], seqs[2], new)):
        o, _ = _definition(layer, *(torch.cat([x, y]) for x, y in zip(s, last[b])))
        assert _far(out[b:b + 1], o[-1:]) < CLOSE, b


def test_a_request_that_gets_no_page():
    """The pool is empty: the prompt and the token are computed, nothing is stored, and the others are as if it were not
    there."""
    announce("attention layer: no page left")
    layer, pool = make_attention_layer(D, 4, 4, 32, seed=4), Pool(3, 4, 4)
    cache = layer.cache(4, PAGE)
    lens, slots = [40, 30, 10], _ints([0, 1, 2])
    hidden, residual = _hidden(80, 1)
    plan = pool.assign(_ints([0] * 3), _ints(lens), slots, capacity=80)
    assert plan.lengths.tolist() == [40, 0, 0] and pool.taken.tolist() == [3]
    before = [t.clone() for t in (cache.k, cache.v)]
    out, _ = layer.prefill(hidden, residual, cache, plan)
    for a, b in ((0, 40), (40, 70), (70, 80)):
        assert _far(out[a:b], _definition(layer, hidden[a:b], residual[a:b])[0]) < CLOSE
    idle = int(pool.free[3])
    assert torch.equal(cache.k[idle], before[0][idle]) and torch.equal(cache.v[idle], before[1][idle])
    plan = pool.assign(_ints([48, 0, 0]), None, slots)                     # its third page is full, the fourth the last
    assert plan.lengths.tolist() == [49, 0, 0] and pool.taken.tolist() == [4]
    q = torch.ones(3, 4, 32, device=DEV, dtype=torch.bfloat16)
    o = attention_step(q, cache.k, cache.v, pool.tables, plan.lengths, slots=slots)
    assert o[0].any() and not o[1:].any()


def test_decode_loop_in_a_graph():
    """A recurrent and an attention layer's step, the plan and the lengths' carrying captured as one graph: replays over
    changing tokens, with eager work between, are what the eager loop gives."""
    announce("captured decode step of a hybrid model")
    gdn, layer, B = make_gdn_layer(D, 2, seed=4), make_attention_layer(D, 4, 2, 64, seed=5), 3
    hidden, residual = _hidden(B, 6)
    slots, lens = _ints([2, 0, 3]), [30, 15, 700]

    def state():
        pool = Pool(4, 64, 60)
        plan = pool.assign(_ints([0] * B), _ints(lens), slots, capacity=sum(lens))
        kv, states = layer.cache(64, PAGE), gdn.cache(B)
        layer.prefill(*_hidden(sum(lens), 7), kv, plan)
        return pool, kv, states, plan.lengths.clone()

    def step(pool, kv, states, lengths):
        x, r = gdn.step(hidden, residual, states)
        plan = assign_pages(pool.tables, lengths, None, pool.free, pool.taken, page_size=PAGE, slots=slots)
        x, r = layer.step(x, r, kv, plan, pool.tables, slots)
        lengths.copy_(plan.lengths)
        pool.taken.copy_(plan.taken)
        return x, r

    eager, captured = state(), state()
    captured[0].taken, eager[0].taken = captured[0].taken.clone(), eager[0].taken.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step(*state())
        with torch.cuda.graph(graph, stream=stream):
            x, r = step(*captured)
    torch.cuda.synchronize()
    for i in range(6):
        for t, new in zip((hidden, residual), _hidden(B, 20 + i)):
            t.copy_(new)
        want = step(*eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, want[0]) and torch.equal(r, want[1])
        for a, b in zip((captured[0].tables, captured[0].taken, captured[1].k, captured[1].v, captured[2].state, captured[3]),
                        (eager[0].tables, eager[0].taken, eager[1].k, eager[1].v, eager[2].state, eager[3])):
            assert torch.equal(a, b)
    assert captured[3].tolist() == [n + 6 for n in lens]


def test_two_graphs_and_another_stream():
    """Two captured calls of different shapes, replayed in turn and on two streams at once: no workspace is shared."""
    announce("two captured attention steps, two streams")
    gen = torch.Generator().manual_seed(8)
    calls = []
    for B, n, G in ((2, 3000, 2), (9, 900, 1)):
        need = att.pages_of(n, PAGE)
        k, v = (torch.randn(B * need, PAGE, G, 64, generator=gen).to(DEV, torch.bfloat16) for _ in range(2))
        tables = torch.randperm(B * need, generator=gen).int().view(B, need).to(DEV)
        q = torch.randn(B, 4, 64, generator=gen).to(DEV, torch.bfloat16)
        p = torch.randn(400, 4, 64, generator=gen).to(DEV, torch.bfloat16)
        calls.append((q, k, v, tables, _ints([n] * B), p, _ints([0, 150, 400])))

    def run(c):
        return attention_step(*c[:5]), causal_attention(c[5], c[5][:, :2], c[5][:, 2:], c[6])

    want = [run(c) for c in calls]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for c, stream in zip(calls, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            run(c)
            with torch.cuda.graph(graph, stream=stream):
                outs.append(run(c))
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(4):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        eager = [run(c) for c in calls]
        torch.cuda.synchronize()
        for a, b, c in zip(outs, want, eager):
            assert all(torch.equal(x, y) for x, y in zip(a, b)) and all(torch.equal(x, y) for x, y in zip(c, b))


def test_prefill_rows_are_what_steps_read():
    """The last row of a prompt through causal_attention, and the same token through the cache."""
    announce("prompt's last row and the step")
    for dtype in (torch.bfloat16, torch.float32):
        gen = torch.Generator().manual_seed(9)
        n, pages = 333, 21
        q, k, v = (torch.randn(n, h, 128, generator=gen).to(DEV, dtype) for h in (8, 2, 2))
        kc, vc = (torch.full((pages, PAGE, 2, 128), float("nan"), device=DEV, dtype=dtype) for _ in range(2))
        tables = torch.full((1, pages), -1, dtype=torch.int32, device=DEV)
        free = torch.randperm(pages, generator=gen).int().to(DEV)
        plan = assign_pages(tables, _ints([0]), _ints([n]), free, _ints([0]), page_size=PAGE, capacity=n)
        store_kv(k, v, kc, vc, plan.rows)
        o, s = causal_attention(q, k, v, plan.cu_seqlens)[-1:], attention_step(q[-1:].contiguous(), kc, vc, tables, plan.lengths)
        want = att.attention(ref.f64(q[-1:]), ref.f64(k), ref.f64(v), causal=False)
        att.check(o, *want, n, "prompt")
        att.check(s, *want, n, "step")
