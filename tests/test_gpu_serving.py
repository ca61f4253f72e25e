"""The short convolution, single tokens of the recurrences and the norm on the GPU, against their definitions in
float64: odd sizes, views, lengths of zero and one, pools of states, rows of zeros and of infinities."""
import pytest
import torch

import serving_refs as ref
from conftest import announce
from pto_fuser_amd import (add_rms_norm, add_rms_norm_fp8, causal_conv, causal_conv_step, gdn_chunk_forward, gdn_step,
                           ssm_step)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


def _rand(seed):
    gen = torch.Generator().manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=gen)


def _dev(t, dtype=None):
    return None if t is None else t.to(DEV, dtype)


def _wide(t, extra):
    """The same values as a view of rows that are ``extra`` wider, starting one element in; NaN around them."""
    buf = torch.full((*t.shape[:-1], t.shape[-1] + extra), NAN, dtype=t.dtype, device=t.device)
    view = buf[..., 1:1 + t.shape[-1]]
    view.copy_(t)
    return view


# ------------------------------------------------------------------------------------------
#  Convolution.  32-bit operations on a term: its product, at most K + 1 additions, and the activation's six.
# ------------------------------------------------------------------------------------------
CONV_OPS = 16


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,W,K", [(1, 1, 8, 4), (2, 2, 64, 4), (3, 3, 24, 3), (1, 8, 7, 2), (2, 9, 1, 4), (2, 37, 520, 4),
                                     (1, 131, 40, 3), (5, 16, 13, 2)])
@pytest.mark.parametrize("plain", [True, False])
def test_conv(dtype, B, T, W, K, plain):
    announce(f"causal_conv {dtype} B{B} T{T} W{W} K{K} plain={plain}")
    r = _rand(B * T + W)
    x, w = _dev(r(B, T, W), dtype), _dev(0.5 * r(W, K), dtype if plain else F32)
    bias = None if plain else _dev(0.2 * r(W), F32)
    state = None if plain else _dev(r(B, K - 1, W), dtype)
    xin = x if plain else _wide(x, 5)
    y, final = causal_conv(xin, w, bias, activation=None if plain else "silu", initial_state=state)
    want, mag, last = ref.conv(ref.f64(x), ref.f64(w), ref.f64(bias), not plain, ref.f64(state))
    ref.check(y, want, mag, CONV_OPS, "y")
    assert torch.equal(ref.f64(final), last)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("K", [2, 3, 4])
def test_conv_lengths(dtype, K):
    """Sequences of 0, 1, 2, .. tokens in one batch: what follows them is NaN and is not read; the state is of the last
    live token, written over the one that came in."""
    announce(f"causal_conv lengths {dtype} K{K}")
    T, W = 19, 48
    lengths = [0, 1, 2, 3, T - 1, T]
    B, r = len(lengths), _rand(K)
    x, w, bias = _dev(r(B, T, W), dtype), _dev(0.5 * r(W, K), dtype), _dev(0.2 * r(W), dtype)
    state = _dev(r(B, K - 1, W), dtype)
    want, mag, last = ref.conv(ref.f64(x), ref.f64(w), ref.f64(bias), True, ref.f64(state), lengths)
    for b, n in enumerate(lengths):
        x[b, n:] = NAN
    y, final = causal_conv(x, w, bias, initial_state=state, lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV),
                           final_out=state)
    assert final is state
    ref.check(y, want, mag, CONV_OPS, "y")
    assert torch.equal(ref.f64(final), last)


def test_conv_of_no_tokens():
    announce("causal_conv T=0, B=0")
    state = torch.randn(2, 3, 16, device=DEV)
    w = torch.randn(16, 4, device=DEV)
    y, final = causal_conv(torch.empty(2, 0, 16, device=DEV), w, initial_state=state)
    assert y.shape == (2, 0, 16) and torch.equal(final, state)
    y, final = causal_conv(torch.empty(2, 0, 16, device=DEV), w)
    assert not final.any()
    y, final = causal_conv(torch.empty(0, 5, 16, device=DEV), w)
    assert y.shape == (0, 5, 16) and final.shape == (0, 3, 16)


def test_conv_keeps_nan_where_it_is():
    """A NaN or infinity reaches the K tokens that read it and no other, and no other channel."""
    announce("causal_conv NaN")
    x = torch.ones(1, 40, 64, device=DEV, dtype=BF)
    x[0, 11, 3], x[0, 20, 5] = NAN, INF
    y, _ = causal_conv(x, torch.ones(64, 4, device=DEV, dtype=BF), activation=None)
    bad = ~torch.isfinite(y[0].cpu())
    want = torch.zeros(40, 64, dtype=torch.bool)
    want[11:15, 3] = want[20:24, 5] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("W,K", [(64, 4), (520, 3), (7, 2), (24, 4)])
def test_conv_step_continues_the_prompt(dtype, W, K):
    """A prompt, then single tokens from its state: the bits of the whole prompt at once."""
    announce(f"causal_conv_step {dtype} W{W} K{K}")
    B, T, n, r = 3, 12, 5, _rand(W)
    x, w, bias = _dev(r(B, T, W), dtype), _dev(0.5 * r(W, K), dtype), _dev(0.2 * r(W), F32).to(dtype)
    whole, last = causal_conv(x, w, bias)
    first, state = causal_conv(x[:, :n], w, bias)
    rest = [causal_conv_step(x[:, t], state, w, bias) for t in range(n, T)]
    assert torch.equal(torch.cat([first, torch.stack(rest, 1)], 1), whole)
    assert torch.equal(state, last)


def test_conv_step_slots():
    """States in a pool: the named ones move, all others keep their bits, and a slot outside the pool is skipped."""
    announce("causal_conv_step slots")
    r = _rand(2)
    pool, x, w = _dev(r(9, 3, 40)), _dev(r(4, 40)), _dev(r(40, 4))
    before = pool.clone()
    slots = torch.tensor([7, -1, 0, 9], dtype=torch.int32, device=DEV)
    y = causal_conv_step(x, pool, w, slots=slots)
    picked = before[[7, 0]].clone()
    want = causal_conv_step(x[[0, 2]], picked, w)
    assert torch.equal(y[[0, 2]], want) and not y[[1, 3]].any()
    before[[7, 0]] = picked
    assert torch.equal(pool, before)


# ------------------------------------------------------------------------------------------
#  Single tokens.  Operations on a term: decay (with the exponential's and its argument's), products, and sums over up
#  to 256 rows: at most 32 additions on a term's way (eight rows of a thread, a tree, four waves), with 12 more.
# ------------------------------------------------------------------------------------------
STEP_OPS = 48


def _step_case(seed, dtype, B, H, P, G, N, z=True):
    r = _rand(seed)
    s = {"x": _dev(r(B, H, P), dtype), "dt": _dev(r(B, H), dtype), "A": _dev(-1 - r(H).abs()), "B": _dev(r(B, G, N), dtype),
         "C": _dev(r(B, G, N), dtype), "D": _dev(r(H)), "z": _dev(r(B, H, P), dtype) if z else None, "dt_bias": _dev(r(H) - 3)}
    return s, _dev(r(B, H, N, P))


def _one_token(s, state):
    add = lambda t: None if t is None else ref.f64(t).unsqueeze(2)  # noqa: E731
    y, mag, S, M = ref.ssm(add(s["x"]), add(s["dt"]), ref.f64(s["A"]), add(s["B"]), add(s["C"]), ref.f64(s["D"]), add(s["z"]),
                           ref.f64(s["dt_bias"]), True, ref.f64(state))
    return y[:, :, 0], mag[:, :, 0], S, M


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,H,P,G,N", [(1, 1, 4, 1, 1), (2, 6, 64, 2, 128), (3, 5, 36, 5, 17), (1, 8, 96, 1, 64), (2, 3, 128, 1, 200),
                                       (1, 2, 260, 2, 256)])
def test_ssm_step(dtype, B, H, P, G, N):
    announce(f"ssm_step {dtype} B{B} H{H} P{P} G{G} N{N}")
    s, state = _step_case(B + N, dtype, B, H, P, G, N)
    want, mag, S, M = _one_token(s, state)
    y = ssm_step(state, dt_softplus=True, **s)
    ref.check(y, want, mag, STEP_OPS, "y")
    ref.check(state, S, M, STEP_OPS, "state")


def test_ssm_step_views_and_plain_dt():
    """Operands as slices of one projected row, dt in float32 and used as it is, no D, no z."""
    announce("ssm_step views")
    r = _rand(3)
    row = _dev(r(4, 3 * 64 + 2 * 2 * 16 + 3), BF)
    s = {"x": row[:, :192].unflatten(-1, (3, 64)), "B": row[:, 192:208].unflatten(-1, (1, 16)),
         "C": row[:, 208:224].unflatten(-1, (1, 16)), "dt": _dev(r(4, 6).abs() * 0.1)[:, ::2], "A": _dev(-r(3).abs())}
    state = _dev(r(4, 3, 16, 64))
    add = lambda t: ref.f64(t).unsqueeze(2)  # noqa: E731
    want, mag, S, M = ref.ssm(add(s["x"]), add(s["dt"]), ref.f64(s["A"]), add(s["B"]), add(s["C"]), h0=ref.f64(state))
    out = torch.empty(4, 3, 80, device=DEV, dtype=BF)[..., 8:72]
    y = ssm_step(state, out=out, **s)
    assert y.data_ptr() == out.data_ptr()
    ref.check(y, want[:, :, 0], mag[:, :, 0], STEP_OPS, "y")
    ref.check(state, S, M, STEP_OPS, "state")


def test_ssm_step_slots():
    announce("ssm_step slots")
    s, _ = _step_case(11, F32, 4, 2, 64, 1, 32)
    pool = _dev(_rand(12)(6, 2, 32, 64))
    before = pool.clone()
    y = ssm_step(pool, dt_softplus=True, slots=torch.tensor([5, 6, 2, -3], dtype=torch.int32, device=DEV), **s)
    picked = before[[5, 2]].clone()
    want = ssm_step(picked, dt_softplus=True, **{k: v if k in ("A", "D", "dt_bias") else v[[0, 2]] for k, v in s.items()})
    assert torch.equal(y[[0, 2]], want) and not y[[1, 3]].any()
    before[[5, 2]] = picked
    assert torch.equal(pool, before)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("gate", ["none", "head", "channel"])
@pytest.mark.parametrize("B,H,DK,DV", [(1, 1, 128, 128), (2, 3, 128, 128), (2, 2, 64, 128), (1, 3, 256, 36), (3, 1, 5, 4)])
def test_gdn_step(dtype, gate, B, H, DK, DV):
    announce(f"gdn_step {dtype} {gate} B{B} H{H} DK{DK} DV{DV}")
    r = _rand(DK + DV)
    unit = torch.nn.functional.normalize
    q, k = _dev(unit(r(B, H, DK), dim=-1), dtype), _dev(unit(r(B, H, DK), dim=-1), dtype)
    v, beta = _dev(r(B, H, DV), dtype), _dev(torch.sigmoid(r(B, H)))
    g = {"none": None, "head": -r(B, H).abs(), "channel": -r(B, H, DK).abs()}[gate]
    g, state = _dev(g), _dev(r(B, H, DK, DV))
    want, mag, S, M = ref.delta_step(*(ref.f64(t) for t in (state, q, k, v, beta, g)))
    o = gdn_step(state, q, k, v, beta, g)
    assert o.dtype is F32
    ref.check(o, want, mag, 2 * STEP_OPS, "o")            # the two sums follow one another
    ref.check(state, S, M, 2 * STEP_OPS, "state")


def test_gdn_step_continues_the_chunked_forward():
    """64 tokens through the chunked forward, four more one by one: the float64 recurrence over all 68."""
    announce("gdn_step after gdn_chunk_forward")
    B, H, T, n, D = 1, 2, 68, 64, 128
    r = _rand(5)
    unit = torch.nn.functional.normalize
    q, k, v = unit(r(B, H, T, D), dim=-1), unit(r(B, H, T, D), dim=-1), r(B, H, T, D)
    beta, g = torch.sigmoid(r(B, H, T)), -0.1 * r(B, H, T).abs()
    S, M = (torch.zeros(B, H, D, D, dtype=torch.float64) for _ in range(2))
    want = []
    for t in range(T):
        o, _, S, _ = ref.delta_step(S, *(a[:, :, t].double() for a in (q, k, v, beta, g)))
        want.append(o)
    d = [_dev(a) for a in (q, k, v, beta, g)]
    _, state = gdn_chunk_forward(*(a[:, :, :n].contiguous() for a in d))
    got = [gdn_step(state, *(a[:, :, t].contiguous() for a in d)) for t in range(n, T)]
    # the chunked forward in fp32 is within 1e-4 of the largest value (its documented parity); the steps keep that
    want = torch.stack(want[n:], 2)
    assert (ref.f64(torch.stack(got, 2)) - want).abs().max() <= 1e-4 * want.abs().max()
    assert (ref.f64(state) - S).abs().max() <= 1e-4 * S.abs().max()


# ------------------------------------------------------------------------------------------
#  Norm.  A value carries the residual's addition, half the relative error of the mean of squares (a tree over at most
#  64 values of a thread: under 80 additions, halved by the root), the root, the quotient and two products.
# ------------------------------------------------------------------------------------------
NORM_OPS = 56
WIDTHS = [1, 7, 8, 100, 513, 1024, 2048, 2056, 4096, 6144, 9000, 16384, 32768]


def _norm_case(seed, dtype, rows, D, residual, w_dtype):
    r = _rand(seed)
    return (_dev(r(rows, D), dtype), _dev(1 + 0.1 * r(D), w_dtype), None if residual is None else _dev(3 * r(rows, D), residual))


def _check_norm(y, h, x, w, res, what):
    want, sums = ref.norm(ref.f64(x), ref.f64(w), ref.f64(res))
    mag = want.abs()
    if res is not None:      # the sum's own rounding, carried by the row's factor
        mag = mag + ref.norm(ref.f64(x).abs() + ref.f64(res).abs(), ref.f64(w).abs())[0]
        ref.check(h, sums, ref.f64(x).abs() + ref.f64(res).abs(), 1, what + " h")
    ref.check(y, want, mag, NORM_OPS, what + " y")


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype,residual,w_dtype", [(BF, None, BF), (BF, BF, F32), (BF, F32, BF), (F32, F32, F32), (F32, None, F32)])
def test_norm(D, dtype, residual, w_dtype):
    announce(f"add_rms_norm {dtype} residual {residual} D{D}")
    x, w, res = _norm_case(D, dtype, 5, D, residual, w_dtype)
    y, h = add_rms_norm(x, w, res)
    assert y.dtype is dtype and (h is None) == (res is None) and (h is None or h.dtype is residual)
    _check_norm(y, h, x, w, res, f"D{D}")


def test_norm_layouts():
    """Rows that are slices of wider ones, several leading dimensions, float32 rows to bfloat16, the stream in place."""
    announce("add_rms_norm layouts")
    x, w, res = _norm_case(1, F32, 12, 200, F32, F32)
    want, sums = add_rms_norm(x, w, res)
    y, h = add_rms_norm(_wide(x, 9), w, _wide(res, 3))
    assert torch.equal(y, want) and torch.equal(h, sums)
    y, _ = add_rms_norm(x.view(3, 4, 200), w, res.view(3, 4, 200))
    assert y.shape == (3, 4, 200) and torch.equal(y.view(12, 200), want)
    y, _ = add_rms_norm(x, w, res, out_dtype=BF)
    assert torch.equal(y, want.to(BF))
    stream = res.clone()
    y, h = add_rms_norm(x, w, stream, residual_out=stream)
    assert h is stream and torch.equal(stream, sums) and torch.equal(y, want)
    y, h = add_rms_norm(x[:0], w, res[:0])
    assert y.shape == (0, 200) and h.shape == (0, 200)


def test_norm_rows_of_their_own():
    """Rows of zeros, an infinity, a NaN, values whose squares overflow: each keeps to itself."""
    announce("add_rms_norm special rows")
    x = torch.ones(6, 96, device=DEV)
    x[1] = 0
    x[2, 5] = INF
    x[3, 7] = NAN
    x[4] = 1e30
    w = torch.full((96,), 2.0, device=DEV)
    y = add_rms_norm(x, w)[0].cpu()
    assert torch.allclose(y[[0, 5]], torch.full((2, 96), 2.0), rtol=1e-6) and not y[1].any()
    assert torch.isnan(y[2, 5]) and not y[2, :5].any() and torch.isnan(y[3]).all() and not y[4].any()
    codes, scales, _ = add_rms_norm_fp8(x, w)
    codes, scales = codes.float().cpu(), scales.cpu()
    assert (codes[[0, 5]] == 448).all() and not codes[1].any() and scales[1] == 0
    assert torch.isnan(codes[3]).all() and torch.isnan(scales[3])
    assert torch.allclose(scales[[0, 5]], torch.full((2, 1), 2 / 448), rtol=1e-6)


def _check_fp8(codes, scales, want, block, what):
    """Each code is the value's nearest, up to the value's own 32-bit error: off by half a step (a sixteenth of the
    power of two below, at least 2^-10 for the smallest) and NORM_OPS roundings."""
    rows, D = want.shape
    top = want.view(rows, -1, block).abs().amax(-1)
    ref.check(scales, top / 448, top / 448, NORM_OPS + 2, what + " scales")
    scaled = want.view(rows, -1, block) * torch.where(top > 0, 448 / top, 0.0)[..., None]
    got = codes.float().cpu().double().view_as(scaled)
    step = torch.maximum(2.0 ** torch.floor(torch.log2(scaled.abs().clamp(min=1e-30))) / 16, torch.tensor(2.0 ** -10, dtype=torch.float64))
    over = (got - scaled).abs() - step - 2 * (NORM_OPS + 4) * ref.EPS32 * 448
    assert over.max() <= 0, f"{what}: a code is {over.max():.3e} further off than half a step"


@pytest.mark.parametrize("D,block", [(7, None), (128, None), (513, None), (2048, None), (6144, None), (16384, None), (128, 128),
                                     (640, 128), (2048, 128), (6144, 128), (16384, 128), (32768, 128)])
@pytest.mark.parametrize("dtype,residual", [(BF, None), (BF, BF), (BF, F32), (F32, F32)])
def test_norm_fp8(D, block, dtype, residual):
    announce(f"add_rms_norm_fp8 {dtype} residual {residual} D{D} block {block}")
    x, w, res = _norm_case(D, dtype, 5, D, residual, dtype)
    x[2] = 0
    if res is not None:
        res[2] = 0
    codes, scales, h = add_rms_norm_fp8(x, w, res, scale_block=block)
    assert codes.dtype is torch.float8_e4m3fn and scales.shape == (5, D // block if block else 1)
    want, sums = ref.norm(ref.f64(x), ref.f64(w), ref.f64(res))
    _check_fp8(codes, scales, want, block or D, f"D{D}")
    if res is not None:
        ref.check(h, sums, ref.f64(x).abs() + ref.f64(res).abs(), 1, "h")


# ------------------------------------------------------------------------------------------
#  Streams and graphs
# ------------------------------------------------------------------------------------------
def test_steps_in_a_graph():
    """One decode step (norm, convolution, state space, delta rule) captured on a stream of its own and replayed, with
    eager work between: every replay is the eager step's bits."""
    announce("captured decode step")
    s, state = _step_case(21, BF, 2, 4, 64, 1, 32)
    r = _rand(22)
    conv_x, conv_w, conv_s = _dev(r(2, 64), BF), _dev(r(64, 4), BF), _dev(r(2, 3, 64), BF)
    rows, w = _dev(r(2, 96), BF), _dev(r(96), BF)
    q = _dev(torch.nn.functional.normalize(r(2, 4, 32), dim=-1), BF)
    beta, S2 = _dev(torch.sigmoid(r(2, 4))), _dev(r(2, 4, 32, 64))

    def step(states):
        return (add_rms_norm_fp8(rows, w, rows), causal_conv_step(conv_x, states[0], conv_w),
                ssm_step(states[1], dt_softplus=True, **s), gdn_step(states[2], q, q, s["x"], beta))

    def flat(outs):
        return [t.float() for o in outs for t in (o if isinstance(o, tuple) else (o,))]

    eager, captured = ([t.clone() for t in (conv_s, state, S2)] for _ in range(2))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step([t.clone() for t in captured])
        with torch.cuda.graph(graph, stream=stream):
            outs = step(captured)
    torch.cuda.synchronize()
    for _ in range(4):
        want = flat(step(eager))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(flat(outs), want))
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))


# ------------------------------------------------------------------------------------------
#  State space scan over prompts.  32-bit operations on a term of the state or of y: the step and its softplus, the chunk's
#  decay (an exponential of a sum of up to 64 gates, whose own error is relative to its size: the tests keep a chunk's
#  under 2^4, so 64 gates' roundings cost 2^4 of the 2^-24), a product a chunk from there on, and additions in a tree over
#  64 tokens and 128 rows.  bfloat16 operands besides: the score's and the entering state's rounding to 8 bits, of each
#  term, by at most 2^-9 (the state's update has its weighted x in 16 bits or more, 2^-17 of each term).
# ------------------------------------------------------------------------------------------
def _ssm_ops(T):
    return 160 + (T + 63) // 64


def _ssm_case(seed, dtype, B, H, T, P, G, N, z=True, h0=True, D=True):
    r = _rand(seed)
    s = {"x": _dev(r(B, H, T, P), dtype), "dt": _dev(0.5 * r(B, H, T), dtype), "A": _dev(-1 - r(H).abs()),
         "B": _dev(r(B, G, T, N), dtype), "C": _dev(r(B, G, T, N), dtype), "D": _dev(r(H)) if D else None,
         "z": _dev(r(B, H, T, P), dtype) if z else None, "dt_bias": _dev(0.3 * r(H) - 3.5)}
    s["h0"] = _dev(r(B, H, N, P)) if h0 else None
    return s


def _check_ssm(s, y, final, lengths=None, what="", softplus=True):
    args = {k: ref.f64(v) for k, v in s.items()}
    want, mag, S, M = ref.ssm(args["x"], args["dt"], args["A"], args["B"], args["C"], args["D"], args["z"], args["dt_bias"],
                              softplus, args["h0"], lengths)
    ops = _ssm_ops(s["x"].shape[2])
    if y.dtype is BF:
        # the roundings to 8 bits are independent from term to term: over n terms their sum is some sqrt(n) of one, and
        # far below the sum of their bounds, which is what is allowed here
        ops += 2 * 2 ** 24 / 2 ** 9
    ref.check(y, want, mag, ops, what + " y")
    if final is not None:
        # of the state's terms nothing is rounded below 24 bits
        ref.check(final, S, M, _ssm_ops(s["x"].shape[2]), what + " state")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,H,T,P,G,N", [(1, 1, 1, 32, 1, 16), (1, 2, 5, 64, 1, 128), (2, 3, 64, 64, 1, 64), (1, 4, 65, 32, 2, 128),
                                         (1, 4, 131, 64, 1, 128), (2, 2, 200, 128, 2, 32), (1, 5, 333, 96, 1, 48), (1, 1, 300, 256, 1, 112),
                                         (3, 6, 90, 64, 3, 80), (1, 9, 520, 64, 1, 128)])
def test_ssm(dtype, B, H, T, P, G, N):
    announce(f"ssm_chunk_forward {dtype} B{B} H{H} T{T} P{P} G{G} N{N}")
    s = _ssm_case(T + N, dtype, B, H, T, P, G, N)
    y, final = pf_ssm(s)
    _check_ssm(s, y, final)


@pytest.mark.parametrize("dtype,B,H,T,P,G,N,segments", [
    (BF, 9, 64, 130, 64, 1, 16, False),        # whole sequences, blocks of 256 columns
    (BF, 1, 32, 4096, 64, 1, 80, True),        # segments of 256 columns, batches of tables begun again
    (BF, 4, 13, 700, 96, 1, 32, True),         # heads cut by the blocks' ends
    (BF, 2, 48, 180, 32, 2, 16, True), (F32, 3, 24, 300, 32, 2, 32, True), (F32, 40, 12, 129, 64, 1, 16, False)])
def test_ssm_of_many_columns(dtype, B, H, T, P, G, N, segments):
    """Shapes that take the wide blocks of columns, with and without segments."""
    from pto_fuser_amd import _hip
    announce(f"ssm_chunk_forward {dtype} B{B} H{H} T{T} P{P} G{G} N{N}")
    assert (_hip.load().pf_ssm_workspace_bytes(B, H, G, T, N, P, int(dtype is BF)) > 0) == segments
    s = _ssm_case(T + P, dtype, B, H, T, P, G, N, z=False)
    _check_ssm(s, *pf_ssm(s))


def pf_ssm(s, **kw):
    from pto_fuser_amd import ssm_chunk_forward
    return ssm_chunk_forward(s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], z=s["z"], dt_bias=s["dt_bias"],
                             dt_softplus=True, h0=s["h0"], **kw)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_ssm_views(dtype):
    """x, B and C in place in one convolved row per token, dt and z of projections; no state in, no D; y comes token-major."""
    announce(f"ssm_chunk_forward views {dtype}")
    B, T, H, P, G, N = 2, 150, 4, 64, 2, 32
    r = _rand(1)
    row = _wide(_dev(r(B, T, H * P + 2 * G * N), dtype), 9)
    x, b, c = row.split([H * P, G * N, G * N], dim=-1)
    s = {"x": x.unflatten(-1, (H, P)).transpose(1, 2), "B": b.unflatten(-1, (G, N)).transpose(1, 2),
         "C": c.unflatten(-1, (G, N)).transpose(1, 2), "dt": _dev(0.5 * r(B, T, H)).transpose(1, 2), "A": _dev(-1 - r(H).abs()),
         "D": None, "z": _wide(_dev(r(B, T, H, P), dtype), 3).transpose(1, 2), "dt_bias": _dev(r(H) - 4), "h0": None}
    y, final = pf_ssm(s)
    assert y.transpose(1, 2).is_contiguous()
    _check_ssm(s, y, final)
    again, none = pf_ssm(s, output_final_state=False, out=torch.empty(B, H, T, P + 4, device=DEV, dtype=dtype)[..., :P])
    assert none is None and torch.equal(again, y)
    packed = {k: None if v is None else v.contiguous() for k, v in s.items()}
    assert all(torch.equal(a, b) for a, b in zip(pf_ssm(packed), (y, final)))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_ssm_lengths(dtype):
    """Sequences of 0, 1, 63, 64, 65 .. tokens in one batch of segments: what follows them is NaN and is not read."""
    announce(f"ssm_chunk_forward lengths {dtype}")
    lengths = [0, 1, 63, 64, 65, 128, 200, 299, 300]
    B, H, T, P, G, N = len(lengths), 2, 300, 32, 1, 32
    s = _ssm_case(7, dtype, B, H, T, P, G, N)
    clean = {k: None if v is None else v.clone() for k, v in s.items()}
    for i, n in enumerate(lengths):
        for k in ("x", "dt", "B", "C", "z"):
            s[k][i, :, n:] = NAN
    final = s["h0"]
    y, got = pf_ssm(s, lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV), final_out=final)
    assert got is final
    _check_ssm(clean, y, got, lengths)
    for i, n in enumerate(lengths):
        assert not y[i, :, n:].any()
    assert torch.equal(final[0], clean["h0"][0])


def test_ssm_of_no_tokens():
    announce("ssm_chunk_forward T=0, B=0")
    s = _ssm_case(1, F32, 2, 2, 0, 32, 1, 16)
    y, final = pf_ssm(s)
    assert y.shape == (2, 2, 0, 32) and torch.equal(final, s["h0"])
    y, final = pf_ssm(_ssm_case(1, F32, 0, 2, 5, 32, 1, 16))
    assert y.shape == (0, 2, 5, 32) and final.shape == (0, 2, 16, 32)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_ssm_strong_and_no_decay(dtype):
    """Heads whose state is gone within a token, heads that never decay, and one that grows: no overflow where the result
    has none."""
    announce(f"ssm_chunk_forward decays {dtype}")
    s = _ssm_case(3, dtype, 1, 4, 200, 32, 1, 32)
    s["dt_bias"] = torch.tensor([3.0, -4.0, -4.0, 1.0], device=DEV)
    s["A"] = torch.tensor([-60.0, 0.0, 0.01, -3.0], device=DEV)
    y, final = pf_ssm(s)
    args = {k: ref.f64(v) for k, v in s.items()}
    want, mag, S, M = ref.ssm(args["x"], args["dt"], args["A"], args["B"], args["C"], args["D"], args["z"], args["dt_bias"], True,
                              args["h0"])
    # a chunk's gates sum to 64 * 4 * 60 at most here, 2^14: 10 bits more than the tests above allow for
    ops = _ssm_ops(200) + 64 * 2 ** 10 + (2 ** 16 if dtype is BF else 0)
    ref.check(y, want, mag, ops, "y")
    ref.check(final, S, M, ops, "state")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("step", [300.0, 1e4, 1e30])
def test_ssm_after_a_token_that_ends_the_state(dtype, step):
    """A token whose step decays all that was (and adds nothing): those after it keep their own decays."""
    announce(f"ssm_chunk_forward reset by a step of {step} {dtype}")
    s = _ssm_case(8, dtype, 1, 3, 190, 32, 1, 32)
    for t in (5, 70, 100):
        s["x"][:, :, t], s["dt"][:, :, t] = 0.0, step
    y, final = pf_ssm(s)
    args = {k: ref.f64(v) for k, v in s.items()}
    want, mag, S, M = ref.ssm(args["x"], args["dt"], args["A"], args["B"], args["C"], args["D"], args["z"], args["dt_bias"], True,
                              args["h0"])
    # two such tokens of a chunk sum to 2 * 2^8 in log2: 2^9, or 5 bits more than the tests above allow for
    ops = _ssm_ops(190) + 64 * 2 ** 5 + (2 ** 16 if dtype is BF else 0)
    ref.check(y, want, mag, ops, "y")
    ref.check(final, S, M, ops, "state")


def test_ssm_workspace_is_optional():
    """Through the C entry without a workspace: whole sequences, within rounding of the segments."""
    from pto_fuser_amd import _hip, serving
    announce("pf_ssm_exec without a workspace")
    s = _ssm_case(5, F32, 1, 2, 1000, 64, 1, 64)
    assert _hip.load().pf_ssm_workspace_bytes(1, 2, 1, 1000, 64, 64, 0) > 0
    y, final = pf_ssm(s)
    y2, final2 = torch.empty_like(y), torch.empty_like(final)
    st = lambda t: t.stride()[:3]  # noqa: E731
    serving._exec("pf_ssm_exec", s["x"].device, serving._SSM, serving._SSM_SIZE, s["x"].data_ptr(), s["dt"].data_ptr(),
                  s["B"].data_ptr(), s["C"].data_ptr(), s["z"].data_ptr(), s["A"].data_ptr(), s["D"].data_ptr(),
                  s["dt_bias"].data_ptr(), s["h0"].data_ptr(), 0, y2.data_ptr(), final2.data_ptr(), 0, 0, *st(s["x"]),
                  *s["dt"].stride(), *st(s["B"]), *st(s["C"]), *st(s["z"]), *st(y2), 1, 2, 1, 1000, 64, 64, 0, 0, 1)
    _check_ssm(s, y, final, what="segments")
    _check_ssm(s, y2, final2, what="whole")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_ssm_step_continues_the_prompt(dtype):
    announce(f"ssm_step after ssm_chunk_forward {dtype}")
    s = _ssm_case(9, dtype, 2, 4, 71, 64, 2, 64, h0=False)
    cut = {k: v[:, :, :67] if k in ("x", "dt", "B", "C", "z") else v for k, v in s.items()}
    first, state = pf_ssm(cut)
    rest = [ssm_step(state, *(s[k][:, :, t] for k in ("x", "dt")), s["A"], s["B"][:, :, t], s["C"][:, :, t], s["D"],
                     z=s["z"][:, :, t], dt_bias=s["dt_bias"], dt_softplus=True) for t in range(67, 71)]
    _check_ssm(s, torch.cat([first, torch.stack(rest, 2)], 2), state)


def test_ssm_in_a_graph():
    """Captured, segments and all, and replayed on changing inputs with eager calls between."""
    announce("captured ssm_chunk_forward")
    s = _ssm_case(13, BF, 1, 4, 700, 64, 1, 128)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        pf_ssm(s)
        with torch.cuda.graph(graph, stream=stream):
            y, final = pf_ssm(s)
    torch.cuda.synchronize()
    for i in range(4):
        s["x"].copy_(_dev(_rand(100 + i)(*s["x"].shape), BF))
        want = pf_ssm(s)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(final, want[1])


# ------------------------------------------------------------------------------------------
#  The scan where its weights are differences of long sums: a weight is as exact as the gates between its two tokens,
#  whatever came before them in the chunk.  The same operations as above, so the same count of roundings; a weight of
#  2^-d has a relative error of some d roundings, and d 2^-d < 1.
# ------------------------------------------------------------------------------------------
def _steps_case(seed, dtype, T, strong, step, A, N=32):
    """Steps as they are (no softplus): ``step`` at the ``strong`` tokens, 2^-7 to 2^-5 elsewhere; x everywhere."""
    s = _ssm_case(seed, dtype, 2, 3, T, 32, 1, N)
    s["A"] = torch.full((3,), A, device=DEV)
    s["dt"] = _dev(2.0 ** -7 * (1 + 3 * torch.rand(2, 3, T, generator=torch.Generator().manual_seed(seed))), F32)
    s["dt"][:, :, strong] = step
    s["dt_bias"] = None
    return s


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,h0", [(64, True), (64, False), (391, True)])
@pytest.mark.parametrize("strong,step,A", [
    (range(48), 1.0, -16.0), (range(8), 11.0, -16.0), (range(32), 11.0, -16.0), (range(48), 11.0, -16.0),
    (range(0, 60, 3), 7.0, -20.0), ([5, 6, 21, 63], 1e4, -2.0), ([0], 3e30, -1.0)])
def test_ssm_weak_tokens_between_strong_ones(dtype, T, h0, strong, step, A):
    from pto_fuser_amd import ssm_chunk_forward
    strong = [t + c for c in range(0, T, 64) for t in strong if t + c < T]
    announce(f"ssm_chunk_forward {len(strong)} steps of {step} and weak ones {dtype} T{T} h0={h0}")
    s = _steps_case(17, dtype, T, strong, step, A)
    if step > 1e6:                       # the square of what such a step adds is past fp32
        s["x"][:, :, strong] *= 1e-20
        s["B"][:, :, strong] *= 1e-10
    if not h0:
        s["h0"] = None
    y, final = ssm_chunk_forward(s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], z=s["z"], h0=s["h0"])
    _check_ssm(s, y, final, softplus=False)


# ------------------------------------------------------------------------------------------
#  Values that are not finite: the recurrence takes one to its own token and to those after it.
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,H,T,P,N,t", [(1, 3, 64, 32, 32, 37), (2, 4, 150, 64, 128, 100), (1, 4, 700, 64, 64, 331),
                                         (17, 16, 70, 64, 128, 66), (9, 64, 70, 32, 16, 13)])
@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("name", ["x", "z", "dt", "B", "C", "h0"])
def test_ssm_keeps_nan_where_it_is(dtype, B, H, T, P, N, t, bad, name):
    announce(f"ssm_chunk_forward {bad} in {name} {dtype} B{B} H{H} T{T} P{P} N{N}")
    s = _ssm_case(23, dtype, B, H, T, P, 1, N)
    s["D"] = torch.ones(H, device=DEV)
    clean, clean_state = pf_ssm(s)
    b, h, p, n = B - 1, H - 2, P - 3, N // 2 + 1
    at = {"x": (b, h, t, p), "z": (b, h, t, p), "dt": (b, h, t), "B": (b, 0, t, n), "C": (b, 0, t, n), "h0": (b, h, n, p)}[name]
    s[name][at] = bad
    y, state = pf_ssm(s)
    # where the definition has it
    want, want_state = torch.zeros(B, H, T, P, dtype=torch.bool), torch.zeros(B, H, N, P, dtype=torch.bool)
    if name == "x":
        want[b, h, t:, p] = want_state[b, h, :, p] = True
    elif name == "dt":
        want[b, h, t:] = want_state[b, h] = True
    elif name == "B":
        want[b, :, t:] = want_state[b, :, n] = True
    elif name == "C":
        want[b, :, t] = True
    elif name == "h0":
        want[b, h, :, p] = want_state[b, h, n, p] = True
    else:
        want[b, h, t, p] = True
    assert torch.equal(~torch.isfinite(y.cpu()), want) and torch.equal(~torch.isfinite(state.cpu()), want_state)
    # and the bits of everything else stay
    assert torch.equal(torch.where(want, 0, y.float().cpu()), torch.where(want, 0, clean.float().cpu()))
    assert torch.equal(torch.where(want_state, 0, state.cpu()), torch.where(want_state, 0, clean_state.cpu()))


def test_outputs_over_their_own_operands():
    """What the descriptions let be one view: the bits of separate ones."""
    announce("outputs over operands")
    s, state = _step_case(31, BF, 5, 4, 64, 2, 32)
    r = _rand(32)

    def both(call, *over):
        """call(out) with fresh memory, and with each of ``over`` (restored) as the output."""
        want = call(None).clone()
        for t in over:
            kept = t.clone()
            got = call(t)
            assert got is t and torch.equal(got, want)
            t.copy_(kept)

    both(lambda o: ssm_step(state.clone(), dt_softplus=True, out=o, **s), s["x"], s["z"])
    q, v, beta, S = _dev(0.1 * r(5, 4, 32)), _dev(r(5, 4, 64)), _dev(torch.sigmoid(r(5, 4))), _dev(r(5, 4, 32, 64))
    both(lambda o: gdn_step(S.clone(), q, q, v, beta, out=o), v)
    x, w, conv = _dev(r(5, 520), BF), _dev(r(520, 4), BF), _dev(r(5, 3, 520), BF)
    both(lambda o: causal_conv_step(x, conv.clone(), w, out=o), x)
    for D in (520, 4096):                    # a wave and a workgroup a row
        rows, res, w = _dev(r(37, D), BF), _dev(r(37, D), BF), _dev(r(D), BF)
        both(lambda o: add_rms_norm(rows, w, res, out=o)[0], rows, res)
        both(lambda o: add_rms_norm(rows, w, res, residual_out=o)[1], rows, res)
    wide = _dev(r(2, 33, 3 * 64), BF)
    both(lambda o: causal_conv(wide[..., :64], _dev(torch.ones(64, 4), BF), out=o)[0], wide[..., 64:128])


def test_steps_of_empty_batches_and_pools():
    announce("steps of no sequences, and of a pool of none")
    s, state = _step_case(33, BF, 3, 4, 64, 1, 32)
    none = {k: t[:0] if t is not None and t.shape[0] == 3 else t for k, t in s.items()}
    before = state.clone()
    slots = torch.zeros(0, dtype=torch.int32, device=DEV)
    q, v, beta = torch.zeros(0, 4, 32, device=DEV, dtype=BF), none["x"], torch.zeros(0, 4, device=DEV)
    x, conv, w = torch.zeros(0, 64, device=DEV, dtype=BF), torch.zeros(2, 3, 64, device=DEV, dtype=BF), torch.ones(64, 4, device=DEV, dtype=BF)
    assert ssm_step(state, slots=slots, **none).shape == ssm_step(state[:0], **none).shape == (0, 4, 64)
    assert gdn_step(state, q, q, v, beta, slots=slots).shape == gdn_step(state[:0], q, q, v, beta).shape == (0, 4, 64)
    assert causal_conv_step(x, conv, w, slots=slots).shape == causal_conv_step(x, conv[:0], w).shape == (0, 64)
    assert torch.equal(state, before)
    # a pool of no states: every slot is outside it
    slots = torch.tensor([0, 1, -1], dtype=torch.int32, device=DEV)
    assert not ssm_step(state[:0], slots=slots, **s).any()
    q, beta = torch.ones(3, 4, 32, device=DEV, dtype=BF), torch.ones(3, 4, device=DEV)
    assert not gdn_step(state[:0], q, q, s["x"], beta, slots=slots).any()
    assert not causal_conv_step(torch.ones(3, 64, device=DEV, dtype=BF), conv[:0], w, slots=slots).any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_ssm_of_tokens_far_apart(dtype):
    """Token strides at the kernel's bound, read in place, and past it: the bits of packed operands."""
    announce(f"ssm_chunk_forward token strides of 2^22 {dtype}")
    s = _ssm_case(41, dtype, 1, 2, 3, 32, 1, 16)
    want = pf_ssm(s)
    for stride in (1 << 22, (1 << 22) + 8):
        far = dict(s)
        for k in ("x", "B", "C", "z"):
            t = s[k]
            buf = torch.full((3 * stride,), NAN, device=DEV, dtype=dtype)
            far[k] = buf.as_strided(t.shape, (0, t.shape[3], stride, 1))
            far[k].copy_(t)
        assert all(torch.equal(a, b) for a, b in zip(pf_ssm(far), want))
