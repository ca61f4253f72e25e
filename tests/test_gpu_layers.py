"""Recurrent layers as they are served: a ragged batch of prompts against its prompts alone and against the definitions
in float64, then single tokens from pools of states against longer prompts."""
import pytest
import torch

import serving_refs as ref
from conftest import announce
from pto_fuser_amd.forwards import make_gdn_layer, make_ssm_layer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
D = 128


def _layer(kind):
    return make_ssm_layer(D, 4, P=64, G=2, N=32, seed=3) if kind == "ssm" else make_gdn_layer(D, 2, seed=4)


def _hidden(B, T, seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(B, T, D, generator=gen).to(DEV, torch.bfloat16) for _ in range(2)]


def _far(a, b):
    """Distance over size, in the 2-norm."""
    a, b = ref.f64(a), ref.f64(b)
    return ((a - b).norm() / b.norm()).item()


# What two ways to the same bfloat16 layer differ by: the intermediate rows are rounded to bfloat16 (2^-9 a value) in six
# places and to 8 bits with 4 significant (2^-4) in one, each of which moves a value by at most its rounding where the
# inputs differ by theirs; in the 2-norm over thousands of values roundings add as their squares and a code moves for a
# fraction of the values only.  A sixteenth is the rounding of every code at once.
CLOSE = 2.0 ** -4


@pytest.mark.parametrize("kind", ["ssm", "gdn"])
def test_ragged_prefill_is_each_prompt_alone(kind):
    announce(f"{kind} layer, ragged prefill")
    layer, (hidden, residual) = _layer(kind), _hidden(3, 150, 1)
    lengths = [150, 37, 1]
    out, stream, cache = layer.prefill(hidden, residual, torch.tensor(lengths, dtype=torch.int32, device=DEV))
    for b, n in enumerate(lengths):
        o, s, c = layer.prefill(hidden[b:b + 1, :n].contiguous(), residual[b:b + 1, :n].contiguous())
        assert torch.equal(s[0], stream[b, :n])
        # (the library's product may round otherwise for another number of rows)
        assert _far(cache.conv[b], c.conv[0]) < 1e-2 and _far(cache.state[b], c.state[0]) < 1e-2 and _far(out[b, :n], o[0]) < CLOSE


@pytest.mark.parametrize("kind", ["ssm", "gdn"])
def test_steps_continue_the_prefill(kind):
    """Prompts of two sequences into slots of a pool, then tokens one by one: the outputs and states of the longer
    prompts; the pool's other slots keep their bits."""
    announce(f"{kind} layer, steps after prefill")
    T, n, B = 72, 64, 2
    layer, (hidden, residual) = _layer(kind), _hidden(B, T, 2)
    want, _, last = layer.prefill(hidden, residual)
    _, _, first = layer.prefill(hidden[:, :n].contiguous(), residual[:, :n].contiguous())
    pool, slots = layer.cache(5), torch.tensor([3, 1], dtype=torch.int32, device=DEV)
    pool.conv[slots.long()], pool.state[slots.long()] = first.conv, first.state
    got = [layer.step(hidden[:, t].contiguous(), residual[:, t].contiguous(), pool, slots)[0] for t in range(n, T)]
    assert _far(torch.stack(got, 1), want[:, n:]) < CLOSE
    assert _far(pool.state[slots.long()], last.state) < 1e-2
    assert not pool.state[[0, 2, 4]].any() and not pool.conv[[0, 2, 4]].any()


def test_ssm_layer_against_its_definition():
    """One prompt through the layer's formulas in float64 (weights as they are stored)."""
    announce("ssm layer in float64")
    layer, (hidden, residual) = _layer("ssm"), _hidden(1, 70, 5)
    out, stream, cache = layer.prefill(hidden, residual)
    y, h = ref.norm(ref.f64(hidden), ref.f64(layer.norm_w), ref.f64(residual))
    row = y @ ref.f64(layer.in_w)
    z, xbc, dt = layer._split(row)
    xbc, _, _ = ref.conv(xbc, ref.f64(layer.conv_w), ref.f64(layer.conv_b))
    x, b, c = (t.transpose(1, 2) for t in layer._operands(xbc))
    s, _, S, _ = ref.ssm(x, dt.transpose(1, 2), ref.f64(layer.A), b, c, ref.f64(layer.D),
                         z.unflatten(-1, (layer.H, layer.P)).transpose(1, 2), ref.f64(layer.dt_bias), True)
    y, _ = ref.norm(s.transpose(1, 2).flatten(-2), ref.f64(layer.gate_w))
    want = y @ ref.f64(layer.out.plain()).t()
    assert _far(out, want) < CLOSE and _far(stream, h) < 2.0 ** -8 and _far(cache.state, S) < 2e-2


def test_decode_step_in_a_graph():
    """A step of both layers, one after the other, captured and replayed over changing tokens."""
    announce("captured decode step of two layers")
    layers = [_layer("ssm"), _layer("gdn")]
    caches, eager = [l.cache(2) for l in layers], [l.cache(2) for l in layers]
    hidden, residual = (t[:, 0].contiguous() for t in _hidden(2, 1, 6))

    def step(caches):
        x, r = hidden, residual
        for layer, cache in zip(layers, caches):
            x, r = layer.step(x, r, cache)
        return x, r

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step([l.cache(2) for l in layers])
        with torch.cuda.graph(graph, stream=stream):
            x, r = step(caches)
    torch.cuda.synchronize()
    for i in range(4):
        for t, new in zip((hidden, residual), _hidden(2, 1, 10 + i)):
            t.copy_(new[:, 0])
        want_x, want_r = step(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, want_x) and torch.equal(r, want_r)
        for a, b in zip(caches, eager):
            assert torch.equal(a.state, b.state) and torch.equal(a.conv, b.conv)
