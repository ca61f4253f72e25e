"""What an attention layer's prefill does not compute: the new tokens of a request whose earlier ones the cache holds.  Only the
device knows which those are; their rows come out as NaN, and the others as they would alone."""
import pytest
import torch

from conftest import announce
from pto_fuser_amd.forwards import make_attention_layer
from test_gpu_attention_layer import CLOSE, PAGE, Pool, _definition, _far, _hidden, _ints

pytestmark = pytest.mark.gpu


def _check(out, pack, layer, cu, held):
    """Rows of requests that are ``held`` are NaN, the others the definition's."""
    for b, (lo, hi) in enumerate(zip(cu, cu[1:])):
        if held[b]:
            assert out[lo:hi].isnan().all(), b
        elif hi > lo:
            assert _far(out[lo:hi], _definition(layer, *(t[lo:hi] for t in pack))[0]) < CLOSE, b


@pytest.mark.parametrize("H,G,head", [(6, 2, 64), (4, 4, 32), (8, 2, 128)])
def test_requests_that_hold_tokens(H, G, head):
    """Held tokens that end a page and that do not, more and fewer of them than new ones; requests of no new token among
    and behind them; two that get no page, one of which holds tokens."""
    announce(f"attention layer: prefill of requests that hold tokens H{H} G{G} D{head}")
    layer, pool = make_attention_layer(128, H, G, head, seed=5), Pool(9, 20, 6)
    cache = layer.cache(20, PAGE)
    before = [PAGE, 0, 40, 3, 0, 1, 7, 0, 0]
    first = pool.assign(_ints([0] * 9), _ints(before), None, capacity=sum(before))
    layer.prefill(*_hidden(sum(before), 1), cache, first)
    new = [5, 33, 2, 0, 1, 60, 0, 90, 12]
    plan = pool.assign(first.lengths, _ints(new), None, capacity=sum(new))
    assert plan.lengths.tolist() == [21, 33, 42, 3, 1, 61, 7, 0, 0]
    cu = [sum(new[:i]) for i in range(10)]
    pack = _hidden(sum(new), 2)
    out, _ = layer.prefill(*pack, cache, plan)
    held = [b > 0 for b in before]
    _check(out, pack, layer, cu, held)
    assert torch.isfinite(cache.k).all() and torch.isfinite(cache.v).all()        # (what is stored is right)
    # too few pages: most requests are not served, with fewer tokens held than new ones and with more
    short = [50, 50, 50, 20, 1, 1, 1, 1, 3]
    plan = pool.assign(plan.lengths, _ints(short), None, capacity=sum(short))
    assert plan.lengths.tolist() == [71, 33, 42, 3, 2, 62, 8, 0, 0] and plan.rows[50] == -1
    pack = _hidden(sum(short), 3)
    out, _ = layer.prefill(*pack, cache, plan)
    _check(out, pack, layer, [sum(short[:i]) for i in range(10)], [True] * 7 + [False] * 2)


def test_capacity_that_ends_before_a_request():
    """A request that holds tokens and whose new ones all lie past the capacity refuses nobody else's rows."""
    announce("attention layer: prefill, held requests past the capacity")
    layer, pool = make_attention_layer(128, 4, 2, 64, seed=6), Pool(3, 20, 6)
    cache = layer.cache(20, PAGE)
    first = pool.assign(_ints([0] * 3), _ints([0, 5, 20]), None, capacity=25)
    plan = pool.assign(first.lengths, _ints([30, 4, 9]), None, capacity=30)
    assert plan.cu_seqlens.tolist() == [0, 30, 30, 30] and plan.lengths.tolist() == [30, 5, 20]
    pack = _hidden(30, 7)
    out, _ = layer.prefill(*pack, cache, plan)
    _check(out, pack, layer, [0, 30, 30, 30], [False, True, True])


def test_more_requests_than_a_workgroup_has_threads():
    announce("attention layer: prefill of 600 requests, a third of which hold tokens")
    layer, B = make_attention_layer(128, 2, 1, 64, seed=8), 600
    pool, cache = Pool(B, 2 * B, 4), layer.cache(2 * B, PAGE)
    before, new = [int(b % 3 == 1) for b in range(B)], [b % 4 for b in range(B)]
    first = pool.assign(_ints([0] * B), _ints(before), None, capacity=sum(before))
    plan = pool.assign(first.lengths, _ints(new), None, capacity=sum(new))
    cu, pack = [sum(new[:b]) for b in range(B + 1)], _hidden(sum(new), 9)
    out, _ = layer.prefill(*pack, cache, plan)
    bad = torch.tensor([before[b] > 0 for b in range(B) for _ in range(new[b])])
    assert torch.equal(out.isnan().all(-1).cpu(), bad) and torch.equal(out.isnan().any(-1).cpu(), bad)
    for b in (0, 3, 597):
        if cu[b] < cu[b + 1]:
            assert _far(out[cu[b]:cu[b + 1]], _definition(layer, *(t[cu[b]:cu[b + 1]] for t in pack))[0]) < CLOSE


def test_captured_prefill():
    """Replayed with lengths that change: a request is refused in the replays in which it holds tokens."""
    announce("attention layer: captured prefill")
    layer, pool = make_attention_layer(128, 4, 2, 64, seed=10), Pool(2, 20, 6)
    cache, tokens, lengths = layer.cache(20, PAGE), _ints([20, 7]), _ints([0, 0])
    pack, free = _hidden(27, 11), pool.taken

    def call():
        pool.taken = free
        return layer.prefill(*pack, cache, pool.assign(lengths, tokens, None, capacity=27))[0]

    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
        with torch.cuda.graph(graph, stream=stream):
            out = call()
    for held in ([0, 0], [5, 0], [0, 16], [0, 0]):
        lengths.copy_(_ints(held))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _check(out, pack, layer, [0, 20, 27], [h > 0 for h in held])
        want = call()
        assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(), want.nan_to_num())
