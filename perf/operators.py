"""The serving operators around the chunked forwards, over the sizes they are used at: the short causal
convolution, the selective state space scan and the gated delta rule's single tokens, and the norm with the
residual's addition.

With ``own`` false, ``run`` computes them in plain 32-bit torch (products, sums, exponentials, indexing) and rounds
once at the end; with ``own`` true it makes the calls of ``pto_fuser_amd`` that a program makes.  ``exact`` evaluates
the definitions in 64 bits, the recurrences token by token.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp32": 4}
EPS = 1e-6
FP8_MAX = 448.0


# ------------------------------------------------------------------------------------------
#  The cases
# ------------------------------------------------------------------------------------------
def _conv(dtype, B, T, W, K=4, extra=0, bias=True, state=False, ragged=False):
    return {"op": "conv", "dtype": dtype, "B": B, "T": T, "W": W, "K": K, "extra": extra, "bias": bias, "state": state,
            "ragged": ragged}


def _conv_step(dtype, B, W, K=4, pool=0):
    return {"op": "conv_step", "dtype": dtype, "B": B, "W": W, "K": K, "pool": pool}


def _ssm(dtype, B, H, T, P=64, N=128, G=1, z=False, h0=False, ragged=False):
    return {"op": "ssm", "dtype": dtype, "B": B, "H": H, "T": T, "P": P, "N": N, "G": G, "z": z, "h0": h0, "ragged": ragged}


def _ssm_step(dtype, B, H, P=64, N=128, G=1, z=False, pool=0):
    return {"op": "ssm_step", "dtype": dtype, "B": B, "H": H, "P": P, "N": N, "G": G, "z": z, "pool": pool}


def _gdn_step(dtype, B, H, gate="head", pool=0):
    return {"op": "gdn_step", "dtype": dtype, "B": B, "H": H, "gate": gate, "pool": pool}


def _norm(dtype, rows, D, residual=True):
    return {"op": "norm", "dtype": dtype, "rows": rows, "D": D, "residual": residual}


def _norm_fp8(dtype, rows, D, residual=True, block=0):
    return {"op": "norm_fp8", "dtype": dtype, "rows": rows, "D": D, "residual": residual, "block": block}


def listed():
    return [
        # the convolution of a layer's q, k and v (16 heads of 128) over the benchmark's prompts, read in place from
        # a projection that also holds gates
        dict(_conv("bf16", 4, 4096, 6144, extra=2080, bias=False), name="conv_prefill"),
        # three prompts of uneven length in full precision, continued from a state, 5 heads, three taps
        dict(_conv("fp32", 3, 1471, 1920, K=3, state=True, ragged=True), name="conv_ragged_fp32"),
        # one token each of 64 running sequences, states in a pool
        dict(_conv_step("bf16", 64, 6144, pool=96), name="conv_step"),
        # a state space layer over two prompts: 32 heads that share B and C
        dict(_ssm("bf16", 2, 32, 8192), name="ssm_prefill"),
        # one long context, gated, continued from a state
        dict(_ssm("bf16", 1, 32, 32768, z=True, h0=True), name="ssm_long_context"),
        # three prompts of uneven length in full precision, two groups of three heads
        dict(_ssm("fp32", 3, 6, 1471, N=64, G=2, z=True, h0=True, ragged=True), name="ssm_ragged_fp32"),
        # one token each of 64 running sequences
        dict(_ssm_step("bf16", 64, 32, pool=80), name="ssm_step"),
        # the same of the delta rule: a GDN layer's 64 sequences, and a KDA layer's single one
        dict(_gdn_step("bf16", 64, 16), name="gdn_step"),
        dict(_gdn_step("bf16", 1, 32, gate="channel"), name="kda_step_single"),
        # the norm before a layer over the benchmark's 16384 tokens, 16 heads of 128 wide
        dict(_norm("bf16", 16384, 2048), name="norm_prefill"),
        # with 8-bit output in blocks of 128 for a wide projection, an odd number of tokens
        dict(_norm_fp8("bf16", 8191, 6144, block=128), name="norm_fp8_prefill"),
        # the same for four running sequences, one scale a token
        dict(_norm_fp8("bf16", 4, 2048), name="norm_fp8_decode"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    op = rng.choice(["conv", "conv", "conv_step", "ssm", "ssm", "ssm", "ssm_step", "ssm_step", "gdn_step", "norm",
                     "norm_fp8", "norm_fp8"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    flip = lambda p=0.5: rng.random() < p  # noqa: E731
    if op == "conv":
        W = rng.choice([_log_int(rng, 64, 8192), 8 * _log_int(rng, 8, 1024), 8 * _log_int(rng, 8, 1024)])
        most = 200_000_000 // ESIZE[dtype] // W
        T = _log_int(rng, 1, min(32768, most))
        B = _log_int(rng, 1, max(1, min(64, most // T)))
        return _conv(dtype, B, T, W, K=rng.choice([2, 3, 4, 4]), extra=rng.choice([0, 32, 2080]), bias=flip(), state=flip(),
                     ragged=flip())
    if op == "conv_step":
        B = _log_int(rng, 1, 512)
        return _conv_step(dtype, B, 8 * _log_int(rng, 8, 1024), K=rng.choice([2, 3, 4, 4]), pool=B + 7 if flip() else 0)
    if op in ("ssm", "ssm_step"):
        P, N = rng.choice([32, 64, 64, 96, 128]), rng.choice([16, 32, 64, 128, 128])
        if op == "ssm_step":
            G = rng.choice([1, 1, 1, 2, 4, 8])
            H = G * _log_int(rng, 1, 64 // G)
            B = _log_int(rng, 1, max(1, min(256, 33_000_000 // (H * P * N))))
            return _ssm_step(dtype, B, H, P, N, G, z=flip(), pool=B + 5 if flip() else 0)
        T = _log_int(rng, 1, 32768)
        most = (180_000_000 if dtype == "bf16" else 60_000_000) // T     # values of x, y, z, B and C a token
        G = rng.choice([g for g in (1, 1, 1, 2, 4, 8) if g * (3 * P + 2 * N) <= most])
        H = G * _log_int(rng, 1, max(1, min(64 // G, (most // G - 2 * N) // (3 * P))))
        B = _log_int(rng, 1, max(1, min(16, most // (3 * H * P + 2 * G * N))))
        return _ssm(dtype, B, H, T, P, N, G, z=flip(), h0=flip(), ragged=flip(0.3))
    if op == "gdn_step":
        H = _log_int(rng, 1, 64)
        B = _log_int(rng, 1, max(1, min(256, 2048 // H)))
        return _gdn_step(dtype, B, H, gate=rng.choice(["none", "head", "head", "channel"]), pool=B + 3 if flip() else 0)
    rows = _log_int(rng, 1, 16384)
    D = rng.choice([_log_int(rng, 64, 16384), 128 * _log_int(rng, 1, 128), 128 * _log_int(rng, 1, 128)])
    rows = max(1, min(rows, 100_000_000 // ESIZE[dtype] // D))
    if op == "norm":
        return _norm(dtype, rows, D, residual=flip(0.7))
    return _norm_fp8(dtype, rows, D, residual=flip(0.7), block=rng.choice([0, 128]) if D % 128 == 0 else 0)


# ------------------------------------------------------------------------------------------
#  What a program has in hand before the call
# ------------------------------------------------------------------------------------------
def _gen(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)
    return gen


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _rand(gen, *shape):
    return torch.rand(*shape, generator=gen, device="cuda")


def _slots(gen, B, pool):
    """B different slots of a pool, in no order."""
    return torch.randperm(pool, generator=gen, device="cuda")[:B].to(torch.int32)


def _lengths(gen, B, T):
    """Uneven prompt lengths: the first is whole, and with three or more the last is empty."""
    n = (_rand(gen, B) * (T + 1)).to(torch.int32).clamp_(0, T)
    n[0] = T
    if B > 2:
        n[-1] = 0
    return n


def _ssm_inputs(gen, case, T):
    """x, B, C as views of one convolved row per token and dt of another, as a layer has them."""
    B, H, P, N, G = (case[k] for k in "BHPNG")
    dt = DTYPES[case["dtype"]]
    xbc = torch.nn.functional.silu(_randn(gen, B, T, H * P + 2 * G * N)).to(dt)
    x, b, c = xbc.split([H * P, G * N, G * N], dim=-1)
    s = {"x": x.unflatten(-1, (H, P)).transpose(1, 2), "b": b.unflatten(-1, (G, N)).transpose(1, 2),
         "c": c.unflatten(-1, (G, N)).transpose(1, 2), "dt": (0.5 * _randn(gen, B, T, H)).to(dt).transpose(1, 2),
         "a": -1 - 15 * _rand(gen, H), "d": 1 + 0.1 * _randn(gen, H), "z": None}
    step = torch.exp(math.log(1e-3) + _rand(gen, H) * math.log(100.0))   # dt between 1e-3 and 1e-1
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    if case["z"]:
        s["z"] = _randn(gen, B, T, H, P).to(dt).transpose(1, 2)
    return s


def prepare(case, seed):
    gen, dt, op = _gen(seed), DTYPES[case["dtype"]], case["op"]
    if op == "conv":
        B, T, W, K = (case[k] for k in "BTWK")
        s = {"x": _randn(gen, B, T, W + case["extra"]).to(dt)[..., :W], "w": ((2 * _rand(gen, W, K) - 1) * K ** -0.5).to(dt)}
        s["bias"] = (0.1 * _randn(gen, W)).to(dt) if case["bias"] else None
        s["state"] = _randn(gen, B, K - 1, W).to(dt) if case["state"] else None
        s["lengths"] = _lengths(gen, B, T) if case["ragged"] else None
    elif op == "conv_step":
        B, W, K, pool = case["B"], case["W"], case["K"], case["pool"]
        s = {"x": _randn(gen, B, W).to(dt), "w": ((2 * _rand(gen, W, K) - 1) * K ** -0.5).to(dt),
             "bias": (0.1 * _randn(gen, W)).to(dt), "state": _randn(gen, pool or B, K - 1, W).to(dt),
             "slots": _slots(gen, B, pool) if pool else None}
    elif op == "ssm":
        s = _ssm_inputs(gen, case, case["T"])
        s["h0"] = 0.1 * _randn(gen, case["B"], case["H"], case["N"], case["P"]) if case["h0"] else None
        s["lengths"] = _lengths(gen, case["B"], case["T"]) if case["ragged"] else None
    elif op == "ssm_step":
        s = {k: v.squeeze(2) if torch.is_tensor(v) and v.dim() > 2 else v for k, v in _ssm_inputs(gen, case, 1).items()}
        s["state"] = 0.1 * _randn(gen, case["pool"] or case["B"], case["H"], case["N"], case["P"])
        s["slots"] = _slots(gen, case["B"], case["pool"]) if case["pool"] else None
    elif op == "gdn_step":
        B, H, D, pool = case["B"], case["H"], 128, case["pool"]
        unit = lambda t: torch.nn.functional.normalize(t, dim=-1)  # noqa: E731
        s = {"q": unit(_randn(gen, B, H, D)).to(dt), "k": unit(_randn(gen, B, H, D)).to(dt), "v": _randn(gen, B, H, D).to(dt),
             "beta": torch.sigmoid(_randn(gen, B, H)), "g": None, "state": 0.1 * _randn(gen, pool or B, H, D, D),
             "slots": _slots(gen, B, pool) if pool else None}
        if case["gate"] != "none":
            shape = (B, H) if case["gate"] == "head" else (B, H, D)
            s["g"] = -0.1 * torch.nn.functional.softplus(_randn(gen, *shape))
    else:
        rows, D = case["rows"], case["D"]
        s = {"x": _randn(gen, rows, D).to(dt), "w": (1 + 0.1 * _randn(gen, D)).to(dt),
             "residual": (3 * _randn(gen, rows, D)).to(dt) if case["residual"] else None}
    s["case"] = case
    return s


# ------------------------------------------------------------------------------------------
#  One pass
# ------------------------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    pf = _package()
    op = s["case"]["op"]
    if op == "conv":
        return pf.causal_conv(s["x"], s["w"], s["bias"], initial_state=s["state"], lengths=s["lengths"])
    if op == "conv_step":
        return pf.causal_conv_step(s["x"], s["state"], s["w"], s["bias"], slots=s["slots"]), s["state"]
    if op == "ssm":
        return pf.ssm_chunk_forward(s["x"], s["dt"], s["a"], s["b"], s["c"], s["d"], z=s["z"], dt_bias=s["dt_bias"],
                                    dt_softplus=True, h0=s["h0"], lengths=s["lengths"])
    if op == "ssm_step":
        y = pf.ssm_step(s["state"], s["x"], s["dt"], s["a"], s["b"], s["c"], s["d"], z=s["z"], dt_bias=s["dt_bias"],
                        dt_softplus=True, slots=s["slots"])
        return y, s["state"]
    if op == "gdn_step":
        return pf.gdn_step(s["state"], s["q"], s["k"], s["v"], s["beta"], s["g"], slots=s["slots"]), s["state"]
    if op == "norm":
        return pf.add_rms_norm(s["x"], s["w"], s["residual"], eps=EPS)
    return pf.add_rms_norm_fp8(s["x"], s["w"], s["residual"], eps=EPS, scale_block=s["case"]["block"] or None)


_PACKAGE = []


def _package():
    if not _PACKAGE:
        sys.path.insert(0, os.path.join(os.getcwd(), "pto-fuser_amd"))
        import pto_fuser_amd
        _PACKAGE.append(pto_fuser_amd)
    return _PACKAGE[0]


def _silu(v):
    return v / (1 + torch.exp(-v))


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(torch.clamp(v, max=20.0))))


def _run_plain(s):
    return {"conv": _plain_conv, "conv_step": _plain_conv_step, "ssm": _plain_ssm, "ssm_step": _plain_ssm_step,
            "gdn_step": _plain_gdn_step, "norm": _plain_norm, "norm_fp8": _plain_norm}[s["case"]["op"]](s)


def _plain_conv(s):
    x, w = s["x"], s["w"]
    (B, T, W), K = x.shape, w.shape[1]
    before = torch.zeros(B, K - 1, W, device=x.device) if s["state"] is None else s["state"].float()
    ext = torch.cat([before, x.float()], 1)                                  # [B, K-1+T, W]
    y = (ext.unfold(1, K, 1) * w.float()).sum(-1)
    y = _silu(y if s["bias"] is None else y + s["bias"].float())
    if s["lengths"] is None:
        return y.to(x.dtype), ext[:, T:].to(x.dtype)
    n = s["lengths"].long()
    y = torch.where(torch.arange(T, device=x.device)[None, :, None] < n[:, None, None], y, 0.0)
    last = n[:, None] + torch.arange(K - 1, device=x.device)
    return y.to(x.dtype), ext.gather(1, last[..., None].expand(B, K - 1, W)).to(x.dtype)


def _plain_conv_step(s):
    at = slice(None) if s["slots"] is None else s["slots"].long()
    ext = torch.cat([s["state"][at], s["x"][:, None]], 1)                    # [B, K, W]
    y = _silu((ext.float() * s["w"].float().t()).sum(1) + s["bias"].float())
    s["state"][at] = ext[:, 1:]
    return y.to(s["x"].dtype), s["state"]


def _segment_sums(g):
    """[..., i, j] = g_{j+1} + .. + g_i for j <= i, -inf above: each sum starts at its own j, so none is the
    difference of two long ones."""
    n = g.shape[-1]
    i = torch.arange(n, device=g.device)
    v = torch.where(i[:, None] > i, g[..., :, None], 0.0).cumsum(-2)
    return torch.where(i[:, None] >= i, v, -math.inf)


def _plain_ssm(s, L=64):
    x, dt = s["x"].float(), _softplus(s["dt"].float() + s["dt_bias"][:, None])
    B, H, T, P = x.shape
    G, N = s["b"].shape[1], s["b"].shape[-1]
    if s["lengths"] is not None:
        live = torch.arange(T, device=x.device) < s["lengths"][:, None]      # [B, T]
        dt = torch.where(live[:, None], dt, 0.0)
    nc = (T + L - 1) // L
    pad = lambda t: torch.nn.functional.pad(t, (0, 0, 0, nc * L - T))        # noqa: E731
    heads = lambda t: t[:, :, None].expand(B, G, H // G, *t.shape[2:]).reshape(B, H, *t.shape[2:])  # noqa: E731
    xc = pad(x).reshape(B, H, nc, L, P)
    b = pad(s["b"].float()).reshape(B, G, nc, L, N)
    c = pad(s["c"].float()).reshape(B, G, nc, L, N)
    dtc = pad(dt[..., None]).reshape(B, H, nc, L)
    g = dtc * s["a"][:, None, None]
    seg = _segment_sums(g)                                                   # [B, H, nc, L, L]
    score = heads(torch.matmul(c, b.transpose(-1, -2).contiguous())) * torch.exp(seg) * dtc[..., None, :]
    y = torch.matmul(score, xc)
    wx = xc * (torch.exp(seg[..., -1, :]) * dtc)[..., None]
    states = torch.matmul(heads(b.transpose(-1, -2).contiguous()), wx)       # [B, H, nc, N, P]
    h0 = torch.zeros(B, H, N, P, device=x.device) if s["h0"] is None else s["h0"]
    states = torch.cat([h0[:, :, None], states], 2).reshape(B, H, nc + 1, N * P)
    total = torch.nn.functional.pad(g.sum(-1), (1, 0))                       # log decay of a chunk; of h0 none
    entry = torch.matmul(torch.exp(_segment_sums(total)), states).reshape(B, H, nc + 1, N, P)
    y = y + torch.exp(g.cumsum(-1))[..., None] * torch.matmul(heads(c), entry[:, :, :-1])
    y = y.reshape(B, H, nc * L, P)[:, :, :T] + s["d"][:, None, None] * x
    if s["z"] is not None:
        y = y * _silu(s["z"].float())
    if s["lengths"] is not None:
        y = torch.where(live[:, None, :, None], y, 0.0)
    return y.to(s["x"].dtype), entry[:, :, -1].contiguous()


def _plain_ssm_step(s):
    at = slice(None) if s["slots"] is None else s["slots"].long()
    x, dt = s["x"].float(), _softplus(s["dt"].float() + s["dt_bias"])
    B, H, P = x.shape
    G, N = s["b"].shape[1:]
    heads = lambda t: t.float()[:, :, None].expand(B, G, H // G, N).reshape(B, H, N)  # noqa: E731
    new = s["state"][at] * torch.exp(dt * s["a"])[..., None, None] + heads(s["b"])[..., None] * (dt[..., None] * x)[:, :, None]
    s["state"][at] = new
    y = (heads(s["c"])[..., None] * new).sum(2) + s["d"][:, None] * x
    if s["z"] is not None:
        y = y * _silu(s["z"].float())
    return y.to(s["x"].dtype), s["state"]


def _plain_gdn_step(s):
    at = slice(None) if s["slots"] is None else s["slots"].long()
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    S = s["state"][at]
    if s["g"] is not None:
        S = S * torch.exp(s["g"] if s["g"].dim() == 3 else s["g"][..., None])[..., None]
    r = s["beta"][..., None] * (v - (k[..., None] * S).sum(2))
    S = S + k[..., None] * r[:, :, None]
    s["state"][at] = S
    return (q[..., None] * S).sum(2) * q.shape[-1] ** -0.5, s["state"]


def _plain_norm(s):
    case, h = s["case"], s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["w"].float()
    h = None if s["residual"] is None else h.to(s["x"].dtype)
    if case["op"] == "norm":
        return y.to(s["x"].dtype), h
    block = case["block"] or case["D"]
    y = y.reshape(case["rows"], -1, block)
    top = y.abs().amax(-1, keepdim=True)
    # e4m3 is a floating type: the codes come back as the values they are, beside the scales
    codes = (y * torch.where(top > 0, FP8_MAX / top, 0.0)).to(torch.float8_e4m3fn).reshape(case["rows"], case["D"])
    return codes, (top / FP8_MAX).squeeze(-1), h


# ------------------------------------------------------------------------------------------
#  What one pass cannot do without
# ------------------------------------------------------------------------------------------
def work(case):
    op, e = case["op"], ESIZE[case["dtype"]]
    if op == "conv":
        B, T, W, K = (case[k] for k in "BTWK")
        state = B * (K - 1) * W * e
        return {"bytes": 2 * B * T * W * e + state * (2 if case["state"] else 1) + W * K * e, "flops": B * T * W * (2 * K + 4)}
    if op == "conv_step":
        B, W, K = case["B"], case["W"], case["K"]
        return {"bytes": 2 * B * W * e + 2 * B * (K - 1) * W * e + W * (K + 1) * e, "flops": B * W * (2 * K + 4)}
    if op == "ssm":
        B, H, T, P, N, G = (case[k] for k in "BHTPNG")
        state = 4 * B * H * N * P
        rows = e * B * T * (H * P * (3 if case["z"] else 2) + 2 * G * N + H)
        L = min(T, 64)                       # chunks of 64: the causal half of the score, its product, C S and the update
        return {"bytes": rows + state * (2 if case["h0"] else 1), "flops": B * T * (G * L * N + H * (L * P + 4 * N * P))}
    if op == "ssm_step":
        B, H, P, N, G = (case[k] for k in "BHPNG")
        rows = e * B * (H * P * (3 if case["z"] else 2) + 2 * G * N + H)
        return {"bytes": rows + 8 * B * H * N * P, "flops": 5 * B * H * N * P}
    if op == "gdn_step":
        B, H, D = case["B"], case["H"], 128
        gate = {"none": 0, "head": 1, "channel": D}[case["gate"]]
        return {"bytes": B * H * (8 * D * D + 3 * D * e + 4 * D + 4 + 4 * gate), "flops": 7 * B * H * D * D}
    rows, D = case["rows"], case["D"]
    n = rows * D
    moved = n * e * (3 if case["residual"] else 1) + D * e
    if op == "norm":
        return {"bytes": moved + n * e, "flops": 5 * n}
    return {"bytes": moved + n + 4 * rows * (D // case["block"] if case["block"] else 1), "flops": 7 * n}


# ------------------------------------------------------------------------------------------
#  The definitions in 64 bits
# ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    f = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    silu = lambda v: v * torch.sigmoid(v)  # noqa: E731
    softplus = lambda v: torch.logaddexp(v, torch.zeros_like(v))  # noqa: E731
    op = case["op"]
    if op == "conv":
        x, w, K = f["x"], f["w"], case["K"]
        B, T, W = x.shape
        y = torch.zeros_like(x) if f["bias"] is None else f["bias"].expand(B, T, W).clone()
        for k in range(K):
            back = K - 1 - k
            y[:, back:] += w[:, k] * x[:, :max(T - back, 0)]
            if f["state"] is not None:                      # tap k of token t < back is state row t + k
                n = min(back, T)
                y[:, :n] += w[:, k] * f["state"][:, k:k + n]
        y = silu(y)
        state = torch.zeros(B, K - 1, W, dtype=torch.float64, device=x.device)
        lengths = [T] * B if s["lengths"] is None else s["lengths"].tolist()
        for i, n in enumerate(lengths):
            y[i, n:] = 0
            for r in range(K - 1):
                t = n - (K - 1) + r
                if t >= 0:
                    state[i, r] = x[i, t]
                elif f["state"] is not None:
                    state[i, r] = f["state"][i, t + K - 1]
        return y, state
    if op == "conv_step":
        at = list(range(case["B"])) if s["slots"] is None else s["slots"].long()
        old, w = f["state"][at].clone(), f["w"]
        y = f["bias"] + f["x"] * w[:, -1]
        for k in range(case["K"] - 1):
            y = y + old[:, k] * w[:, k]
        f["state"][at] = torch.cat([old[:, 1:], f["x"][:, None]], 1)
        return silu(y), f["state"]
    if op in ("ssm", "ssm_step"):
        one = op == "ssm_step"
        rep = case["H"] // case["G"]
        add = lambda t: t.unsqueeze(2) if one else t  # noqa: E731
        x, b, c = add(f["x"]), add(f["b"]).repeat_interleave(rep, 1), add(f["c"]).repeat_interleave(rep, 1)
        dt = softplus(add(f["dt"]) + f["dt_bias"][:, None])
        if one:
            at = list(range(case["B"])) if s["slots"] is None else s["slots"].long()
            h = f["state"][at].clone()
        else:
            shape = (case["B"], case["H"], case["N"], case["P"])
            h = torch.zeros(shape, dtype=torch.float64, device=x.device) if f["h0"] is None else f["h0"].clone()
        T = x.shape[2]
        live = None
        if s.get("lengths") is not None:
            live = torch.arange(T, device=x.device) < s["lengths"][:, None]
            dt = dt * live[:, None]                         # a token past the end neither decays nor adds
        decay, step = torch.exp(dt * f["a"][:, None]), dt[..., None] * x
        y = torch.empty_like(x)
        for t in range(T):
            h = h.mul_(decay[:, :, t, None, None]).addcmul_(b[:, :, t, :, None], step[:, :, t, None, :])
            y[:, :, t] = torch.matmul(c[:, :, t, None, :], h)[:, :, 0]
        y = y + f["d"][:, None, None] * x
        if f["z"] is not None:
            y = y * silu(add(f["z"]))
        if live is not None:
            y = y * live[:, None, :, None]
        if one:
            f["state"][at] = h
            return y[:, :, 0], f["state"]
        return y, h
    if op == "gdn_step":
        at = list(range(case["B"])) if s["slots"] is None else s["slots"].long()
        S = f["state"][at]
        if f["g"] is not None:
            S = S * torch.exp(f["g"].reshape(*f["g"].shape[:2], -1, 1))
        r = f["beta"][..., None] * (f["v"] - torch.matmul(f["k"][:, :, None], S)[:, :, 0])
        S = S + f["k"][..., None] * r[:, :, None]
        f["state"][at] = S
        return torch.matmul(f["q"][:, :, None], S)[:, :, 0] / math.sqrt(S.shape[-2]), f["state"]
    h = f["x"] if f["residual"] is None else f["x"] + f["residual"]
    y = h / torch.sqrt((h ** 2).mean(-1, keepdim=True) + EPS) * f["w"]
    h = None if f["residual"] is None else h
    if op == "norm":
        return y, h
    y = y.unflatten(-1, (-1, case["block"] or case["D"]))
    top = y.abs().amax(-1, keepdim=True)
    return (y / top * FP8_MAX).flatten(-2), top.squeeze(-1) / FP8_MAX, h
