"""The serving operators from their definitions, in float64 on the CPU, each with the sum of the magnitudes of the
terms it adds: 32-bit arithmetic is off by a small multiple of 2^-24 of that sum, whatever cancels in the result."""
import torch

EPS32 = 2.0 ** -24


def f64(t):
    return None if t is None else t.detach().cpu().double()


def silu(v):
    return v * torch.sigmoid(v)


def softplus(v):
    return torch.logaddexp(v, torch.zeros_like(v))


def tolerance(ref, mag, dtype, ops):
    """``ops`` roundings of 2^-24 on the terms, the output's own rounding (2^-9 of it for bfloat16: half a unit in the
    last of 8 bits), and as much again for a value that 32-bit error moves across a rounding boundary."""
    tol = ops * EPS32 * (mag + ref.abs()) + 1e-30
    return tol + 2.0 ** -8 * ref.abs() if dtype == torch.bfloat16 else tol


def check(got, ref, mag, ops, what):
    got64 = f64(got)
    assert got64.shape == ref.shape, (what, got64.shape, ref.shape)
    tol = tolerance(ref, mag, got.dtype, ops)
    over = (got64 - ref).abs() - tol
    worst = over.max().item() if over.numel() else -1.0
    assert not over.numel() or worst <= 0, f"{what}: {int((over > 0).sum())} of {over.numel()} values off, worst by {worst:.3e} past its tolerance"
    assert torch.isfinite(got64).all(), what


def conv(x, w, bias=None, act=True, state=None, lengths=None):
    """(y, mag, final state) with x [B,T,W] in float64."""
    B, T, W = x.shape
    K = w.shape[1]
    y, mag = torch.zeros(B, T, W, dtype=torch.float64), torch.zeros(B, T, W, dtype=torch.float64)
    final = torch.zeros(B, K - 1, W, dtype=torch.float64)
    for b in range(B):
        n = T if lengths is None else int(lengths[b])
        ext = torch.cat([torch.zeros(K - 1, W, dtype=torch.float64) if state is None else state[b], x[b, :n]])
        for t in range(n):
            terms = ext[t:t + K] * w.t()
            s, m = terms.sum(0), terms.abs().sum(0)
            if bias is not None:
                s, m = s + bias, m + bias.abs()
            y[b, t], mag[b, t] = (silu(s), 1.1 * m + s.abs()) if act else (s, m)   # |silu'| < 1.1
        final[b] = ext[n:n + K - 1]
    return y, mag, final


def ssm(x, dt, A, Bm, Cm, D=None, z=None, dt_bias=None, dt_softplus=False, h0=None, lengths=None):
    """(y, mag of y, final state, mag of the state): token by token, x [B,H,T,P], dt [B,H,T], B, C [B,G,T,N]."""
    B, H, T, P = x.shape
    G, N = Bm.shape[1], Bm.shape[3]
    Bm, Cm = Bm.repeat_interleave(H // G, 1), Cm.repeat_interleave(H // G, 1)
    dt = dt if dt_bias is None else dt + dt_bias[:, None]
    dt = softplus(dt) if dt_softplus else dt
    S = torch.zeros(B, H, N, P, dtype=torch.float64) if h0 is None else h0.clone()
    M = S.abs()
    y, mag = torch.zeros_like(x), torch.zeros_like(x)
    live = torch.ones(B, T, dtype=torch.bool)
    if lengths is not None:
        live = torch.arange(T)[None] < torch.as_tensor(lengths)[:, None]
    for t in range(T):
        on = live[:, t][:, None, None, None]
        xt = torch.where(on[..., 0], x[:, :, t], 0.0)
        dx = dt[:, :, t, None] * xt
        decay = torch.exp(dt[:, :, t] * A)[..., None, None]
        kt, qt = torch.where(on[..., 0], Bm[:, :, t], 0.0), torch.where(on[..., 0], Cm[:, :, t], 0.0)
        S = torch.where(on, decay * S + kt[..., None] * dx[:, :, None], S)
        M = torch.where(on, decay * M + (kt[..., None] * dx[:, :, None]).abs(), M)
        o, m = (qt[..., None] * S).sum(2), (qt[..., None].abs() * M).sum(2)
        if D is not None:
            o, m = o + D[:, None] * xt, m + (D[:, None] * xt).abs()
        if z is not None:
            zt = torch.where(on[..., 0], z[:, :, t], 0.0)
            o, m = o * silu(zt), m * silu(zt).abs()
        y[:, :, t], mag[:, :, t] = torch.where(on[..., 0], o, 0.0), m
    return y, mag, S, M


def delta_step(S, q, k, v, beta, g=None, scale=None):
    """(o, mag of o, new state, mag of the state) of one token of the gated delta rule."""
    M = S.abs()
    if g is not None:
        e = torch.exp(g if g.dim() == 3 else g[..., None])[..., None]
        S, M = S * e, M * e
    r = beta[..., None] * (v - (k[..., None] * S).sum(2))
    mr = beta[..., None].abs() * (v.abs() + (k[..., None].abs() * M).sum(2))
    S, M = S + k[..., None] * r[:, :, None], M + k[..., None].abs() * mr[:, :, None]
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    return (q[..., None] * S).sum(2) * sc, (q[..., None].abs() * M).sum(2) * abs(sc), S, M


def norm(x, w, residual=None, eps=1e-6):
    """(y, h): the norm of rows in float64."""
    h = x if residual is None else x + residual
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w, h
