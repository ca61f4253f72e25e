"""Serving operators around the chunked forwards: what stands before and after the recurrence in a layer, and single
tokens.

* :func:`causal_conv`, :func:`causal_conv_step` — the short depthwise convolution along the tokens, for prompts and for
  single tokens, with its state.
* :func:`ssm_chunk_forward`, :func:`ssm_step` — the selective state space scan, over prompts and for single tokens.
* :func:`gdn_step` — one token of the gated delta rule (GDN; DeltaNet with ``g is None``; KDA with a gate per channel):
  continues the final state of ``gdn_chunk_forward`` and ``kda_chunk_forward``.
* :func:`add_rms_norm`, :func:`add_rms_norm_fp8` — the norm with the residual's addition, in the rows' type or in 8 bits
  with scales.

No counterpart in the reference, whose path ends at the chunked forward.  Forward only, like the chunked forwards.

Unlike those, the operands may be views: batch, head and token strides are free (a slice of a projection's output, a
transposed head layout); only the innermost dimension is contiguous.  Every operator raises ``ValueError`` before
launching for what it does not support, works on the current stream of the operands' device, and neither synchronises nor
allocates anything but its outputs and (the scan) a workspace and operands that it has to copy, from torch's allocator: each can
be captured in a HIP graph.  What a call is given to write (``out`` and the like) shares memory with no other operand, unless its description
names one that it may be; slices of one buffer that lie side by side are apart.
"""
from __future__ import annotations

import math
import struct
from typing import Optional, Tuple

import torch

from . import _hip
from .ops import _dtype_code, _require

# The argument structs of include/pto_fuser_hip.h: pointers, strides, then sizes and flags, in C's own layout.
_CONV = struct.Struct("@N7P6q7i")
_CONV_STEP = struct.Struct("@N6P3q7i")
_STEP = struct.Struct("@N13P13q10if")
_SSM = struct.Struct("@N13PN18q9i")
_NORM = struct.Struct("@N6P4q7if")


def _size(layout: struct.Struct) -> int:
    """sizeof the C struct: its fields and the tail padding to 8 bytes."""
    return (layout.size + 7) & ~7


_CONV_SIZE, _CONV_STEP_SIZE, _STEP_SIZE, _SSM_SIZE, _NORM_SIZE = (
    _size(s) for s in (_CONV, _CONV_STEP, _STEP, _SSM, _NORM))

CONV_TAPS = (2, 3, 4)
STEP_MAX_ROWS = 256
SSM_MAX_ROWS, SSM_MAX_COLS, SSM_MAX_STRIDE = 128, 256, 1 << 22
NORM_MAX_WIDTH = 32768
_ACTIVATIONS = {None: 0, "silu": 1}


_FUNCTIONS = {}


def _exec(name: str, dev: torch.device, layout: struct.Struct, *fields) -> None:
    """One call on the current stream of ``dev``, with it as the current device."""
    fn = _FUNCTIONS.get(name)
    if fn is None:
        fn = _FUNCTIONS[name] = getattr(_hip.load(), name)
    try:
        args = layout.pack(*fields)
    except struct.error as e:
        raise ValueError(f"a size of this call is past what {name} takes: {e}") from None
    index = dev.index
    if torch._C._cuda_getDevice() == index:
        st = fn(args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            st = fn(args, torch._C._cuda_getCurrentRawStream(index))
    if st == _hip.PF_ERR_ARG:
        raise ValueError(f"{name} does not take a call of this size: a stride or its grid is past what one launch covers")
    if st:
        _hip.check(name, st)


def _device_of(t, name: str) -> torch.device:
    if isinstance(t, torch.Tensor) and t.is_cuda:
        return t.device
    raise ValueError(f"{name} must be a tensor on a HIP device")


def _require_view(t, name: str, shape, dtype, dev) -> None:
    """``t`` is a tensor of this shape, dtype and device whose innermost dimension is contiguous."""
    if (isinstance(t, torch.Tensor) and t.shape == shape and t.dtype is dtype and t.get_device() == dev.index
            and (t.stride(-1) == 1 or shape[-1] == 1)):
        return
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.dim() != len(shape) or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, expected {dev}")
    raise ValueError(f"{name} must be contiguous along its last dimension")


def _param_f32(t: torch.Tensor, name: str, dtype: torch.dtype) -> int:
    """1 for a float32 parameter, 0 for one of the operands' type."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.dtype is torch.float32:
        return 1
    if t.dtype is not dtype:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype} or float32")
    return 0


def _dim(t, name: str, dims: int, layout: str) -> None:
    if not isinstance(t, torch.Tensor) or t.dim() != dims:
        got = tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__
        raise ValueError(f"{name} must be {layout}, got {got}")


def _act(activation) -> int:
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be 'silu' or None, got {activation!r}")
    return _ACTIVATIONS[activation]


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _span(t: torch.Tensor) -> int:
    """Bytes from a tensor's first element to the end of its last."""
    return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _once(t: torch.Tensor, name: str) -> None:
    """No two elements of ``t``, which a call writes, are one place (an expanded dimension, rows closer than they are long)."""
    if t.is_contiguous():
        return
    end = 1
    for stride, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if stride < end:
            raise ValueError(f"{name} has overlapping rows")
        end = stride * (n - 1) + end


def _share(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors may have memory in common.  Blocks that lie side by side in one buffer (slices of a projection's
    output) do not: all offsets of both are multiples of one pitch, apart from their start and their place in a block."""
    at, bt = a.data_ptr(), b.data_ptr()
    if not a.numel() or not b.numel() or at + _span(a) <= bt or bt + _span(b) <= at:
        return False
    pitch, widths = 0, []
    for t in (a, b):
        width, size = 1, t.element_size()
        for stride, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
            if stride == width:
                width *= n                        # the block goes on
            else:
                pitch = math.gcd(pitch, stride * size)
        widths.append(width * size)
    if not pitch:
        return True
    ahead = (bt - at) % pitch
    return ahead < widths[0] or ahead + widths[1] > pitch


def _apart(name: str, t: Optional[torch.Tensor], same=(), **others) -> None:
    """``t``, which a call writes, is written once an element and has no memory in common with what other threads of it read
    or write.  It may be the very view ``others`` name in ``same``: those elements are read by the thread that writes them."""
    if t is None:
        return
    _once(t, name)
    for other, u in others.items():
        if u is None or not _share(t, u):
            continue
        if other in same and t.data_ptr() == u.data_ptr() and t.dtype == u.dtype and t.stride() == u.stride():
            continue
        raise ValueError(f"{name} may not be {other} nor share memory with it")


def _pool(state: torch.Tensor, slots, B: int, dev) -> None:
    if slots is not None:
        _require(slots, "slots", (B,), torch.int32, dev)
    elif state.shape[0] != B:
        raise ValueError(f"state holds {state.shape[0]} sequences, expected {B} (or name their slots)")


# ------------------------------------------------------------------------------------------
#  Short causal convolution
# ------------------------------------------------------------------------------------------
def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                activation: Optional[str] = "silu", initial_state: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None, output_final_state: bool = True,
                out: Optional[torch.Tensor] = None, final_out: Optional[torch.Tensor] = None,
                ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Depthwise causal convolution along the tokens: y[b,t,c] = act(bias[c] + Σ_k w[c,k] x[b,t-(K-1)+k,c]).

    x [B,T,W] float32 or bfloat16, T up to 2^30, token and batch strides free; weight [W,K], K in 2..4, and bias [W] in x's type or
    float32 (both in one).  ``initial_state`` [B,K-1,W] holds the last K-1 inputs of what came before (None: zeros).
    ``lengths`` [B] int32 (None: all T): tokens of each sequence; what follows them is not read, and y is zero there.
    Returns (y [B,T,W] in x's type, the state after the last token [B,K-1,W] or None).  ``final_out`` may be
    ``initial_state``."""
    dev = _device_of(x, "x")
    _dim(x, "x", 3, "[B,T,W]")
    _dim(weight, "weight", 2, "[W,K]")
    B, T, W = x.shape
    K = weight.shape[1]
    code, dtype = _dtype_code(x.dtype), x.dtype
    if K not in CONV_TAPS or W == 0:
        raise ValueError(f"unsupported convolution of {W} channels and {K} taps (taps in {CONV_TAPS})")
    _require_view(x, "x", (B, T, W), dtype, dev)
    w_f32 = _param_f32(weight, "weight", dtype)
    _require(weight, "weight", (W, K), weight.dtype, dev)
    if bias is not None:
        _require(bias, "bias", (W,), weight.dtype, dev)
    if initial_state is not None:
        _require(initial_state, "initial_state", (B, K - 1, W), dtype, dev)
    if lengths is not None:
        _require(lengths, "lengths", (B,), torch.int32, dev)
    if out is None:
        y = torch.empty(B, T, W, device=dev, dtype=dtype)
    else:
        _require_view(out, "out", (B, T, W), dtype, dev)
        _apart("out", out, x=x, weight=weight, bias=bias, initial_state=initial_state, lengths=lengths)
        y = out
    final = None
    if output_final_state:
        final = final_out
        if final is None:
            final = torch.empty((B, K - 1, W), device=dev, dtype=dtype)
        else:
            _require(final, "final_out", (B, K - 1, W), dtype, dev)
            _apart("final_out", final, ("initial_state",), x=x, weight=weight, bias=bias, initial_state=initial_state,
                   lengths=lengths, out=y)
    sx, sy, state = x.stride(), y.stride(), (K - 1) * W
    _exec("pf_conv_exec", dev, _CONV, _CONV_SIZE, x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(initial_state),
          _ptr(lengths), y.data_ptr(), _ptr(final), sx[0], sx[1], sy[0], sy[1], state, state, B, T, W, K,
          code, w_f32, _act(activation))
    return y, final


def causal_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor,
                     bias: Optional[torch.Tensor] = None, *, activation: Optional[str] = "silu",
                     slots: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of :func:`causal_conv` for each of B sequences: x [B,W]; returns y [B,W].

    ``state`` [S,K-1,W] in x's type is updated in place.  Sequence b's is ``state[slots[b]]`` (``slots`` [B] int32, no two
    the same; one outside the pool is skipped and its y zero), or ``state[b]`` with S = B.  ``out`` may be x."""
    dev = _device_of(x, "x")
    _dim(x, "x", 2, "[B,W]")
    _dim(weight, "weight", 2, "[W,K]")
    _dim(state, "state", 3, "[S,K-1,W]")
    B, W = x.shape
    K = weight.shape[1]
    code, dtype = _dtype_code(x.dtype), x.dtype
    if K not in CONV_TAPS or W == 0:
        raise ValueError(f"unsupported convolution of {W} channels and {K} taps (taps in {CONV_TAPS})")
    _require_view(x, "x", (B, W), dtype, dev)
    w_f32 = _param_f32(weight, "weight", dtype)
    _require(weight, "weight", (W, K), weight.dtype, dev)
    if bias is not None:
        _require(bias, "bias", (W,), weight.dtype, dev)
    _require(state, "state", (state.shape[0], K - 1, W), dtype, dev)
    _pool(state, slots, B, dev)
    if out is None:
        y = torch.empty(B, W, device=dev, dtype=dtype)
    else:
        _require_view(out, "out", (B, W), dtype, dev)
        _apart("out", out, ("x",), x=x, state=state, weight=weight, bias=bias, slots=slots)
        y = out
    _exec("pf_conv_step_exec", dev, _CONV_STEP, _CONV_STEP_SIZE, x.data_ptr(), weight.data_ptr(), _ptr(bias),
          state.data_ptr(), _ptr(slots), y.data_ptr(), x.stride(0), y.stride(0), (K - 1) * W, B,
          state.shape[0], W, K, code, w_f32, _act(activation))
    return y


# ------------------------------------------------------------------------------------------
#  Selective state space scan
# ------------------------------------------------------------------------------------------
def ssm_chunk_forward(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                      D: Optional[torch.Tensor] = None, *, z: Optional[torch.Tensor] = None,
                      dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False,
                      h0: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                      output_final_state: bool = True, out: Optional[torch.Tensor] = None,
                      final_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Selective state space scan over prompts, in chunks of 64 tokens:

        dt = softplus(dt + dt_bias),  S_t = e^{dt·A} S_{t-1} + B_t (dt·x_t)ᵀ,  y_t = C_tᵀ S_t + D·x_t  (times silu(z_t))

    x, z [B,H,T,P] float32 or bfloat16, P a multiple of 32 up to 256; dt [B,H,T] in x's type or float32; B, C [B,G,T,N], N a
    multiple of 16 up to 128, head h reading group h // (H // G); A, D, dt_bias [H] float32 (A < 0: it decays); h0
    [B,H,N,P] float32.  T up to 2^30.  Batch, head and token strides are free: ``xbc[..., :H*P].unflatten(-1, (H,
    P)).transpose(1, 2)`` of a convolved row [B,T,..] is read in place; tokens that overlap or lie more than 2^22 elements
    apart are copied first, and not written (``out``).  ``lengths`` [B] int32 (None: all T): tokens of each sequence; what
    follows them is not read, y is zero there, and the state is that after the last one.  A NaN or infinity reaches
    its own token and those after it, as in the recurrence, and none before.

    Returns (y [B,H,T,P] in x's type, token-major in memory where x is; the final state [B,H,N,P] float32 or None).
    ``final_out`` may be h0.  Few sequences run as segments side by side, whose number follows from the call's shape: the
    same bfloat16 sequence alone and in a batch differs by its rounding."""
    dev = _device_of(x, "x")
    _dim(x, "x", 4, "[B,H,T,P]")
    _dim(B, "B", 4, "[B,G,T,N]")
    nb, H, T, P = x.shape
    G, N = B.shape[1], B.shape[3]
    code, dtype = _dtype_code(x.dtype), x.dtype
    if H == 0 or G == 0 or H % G or not 0 < P <= SSM_MAX_COLS or P % 32 or not 0 < N <= SSM_MAX_ROWS or N % 16:
        raise ValueError(f"unsupported shape H={H} G={G} N={N} P={P} (H a multiple of G, N of 16 up to {SSM_MAX_ROWS}, "
                         f"P of 32 up to {SSM_MAX_COLS})")
    _require_view(x, "x", (nb, H, T, P), dtype, dev)
    _require_view(B, "B", (nb, G, T, N), dtype, dev)
    _require_view(C, "C", (nb, G, T, N), dtype, dev)
    _dim(dt, "dt", 3, "[B,H,T]")
    dt_f32 = _param_f32(dt, "dt", dtype)
    if dt.shape != (nb, H, T) or dt.get_device() != dev.index:
        raise ValueError(f"dt is {tuple(dt.shape)} on {dt.device}, expected {(nb, H, T)} on {dev}")
    if A is None:
        raise ValueError("A must be a tensor")
    _require(A, "A", (H,), torch.float32, dev)
    if D is not None:
        _require(D, "D", (H,), torch.float32, dev)
    if dt_bias is not None:
        _require(dt_bias, "dt_bias", (H,), torch.float32, dev)
    if z is not None:
        _require_view(z, "z", (nb, H, T, P), dtype, dev)
    if h0 is not None:
        _require(h0, "h0", (nb, H, N, P), torch.float32, dev)
    if lengths is not None:
        _require(lengths, "lengths", (nb,), torch.int32, dev)
    token_major = x.stride(1) < x.stride(2)
    if T > 1:      # rows that overlap (a token expanded along the sequence) or lie far apart are laid out first
        x, B, C, z = (t if t is None or t.shape[3] <= t.stride(2) <= SSM_MAX_STRIDE else t.contiguous() for t in (x, B, C, z))
    sx = x.stride()
    if out is not None:
        _require_view(out, "out", (nb, H, T, P), dtype, dev)
        if T > 1 and out.stride(2) > SSM_MAX_STRIDE:
            raise ValueError(f"out's tokens are {out.stride(2)} elements apart (up to {SSM_MAX_STRIDE})")
        _apart("out", out, x=x, dt=dt, A=A, B=B, C=C, D=D, z=z, dt_bias=dt_bias, h0=h0, lengths=lengths)
        y = out
    elif token_major:
        y = torch.empty(nb, T, H, P, device=dev, dtype=dtype).transpose(1, 2)
    else:
        y = torch.empty(nb, H, T, P, device=dev, dtype=dtype)
    final = None
    if output_final_state:
        final = final_out
        if final is None:
            final = torch.empty((nb, H, N, P), device=dev, dtype=torch.float32)
        else:
            _require(final, "final_out", (nb, H, N, P), torch.float32, dev)
            _apart("final_out", final, ("h0",), x=x, dt=dt, A=A, B=B, C=C, D=D, z=z, dt_bias=dt_bias, h0=h0,
                   lengths=lengths, out=y)
    need = _hip.load().pf_ssm_workspace_bytes(nb, H, G, T, N, P, code)
    ws = torch.empty(need, device=dev, dtype=torch.uint8) if need else None
    sb, sc, sy, st = B.stride(), C.stride(), y.stride(), dt.stride()
    sz = (0, 0, 0) if z is None else z.stride()
    _exec("pf_ssm_exec", dev, _SSM, _SSM_SIZE, x.data_ptr(), dt.data_ptr(), B.data_ptr(), C.data_ptr(), _ptr(z),
          A.data_ptr(), _ptr(D), _ptr(dt_bias), _ptr(h0), _ptr(lengths), y.data_ptr(), _ptr(final), _ptr(ws), need,
          sx[0], sx[1], sx[2], st[0], st[1], st[2], sb[0], sb[1], sb[2], sc[0], sc[1], sc[2], sz[0], sz[1], sz[2],
          sy[0], sy[1], sy[2], nb, H, G, T, N, P, code, dt_f32, int(bool(dt_softplus)))
    return y, final


# ------------------------------------------------------------------------------------------
#  Single tokens of the recurrences
# ------------------------------------------------------------------------------------------
def ssm_step(state: torch.Tensor, x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
             C: torch.Tensor, D: Optional[torch.Tensor] = None, *, z: Optional[torch.Tensor] = None,
             dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False,
             slots: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of the selective state space recurrence for each of B sequences:

        dt = softplus(dt + dt_bias),  S ← e^{dt·A} S + B (dt·x)ᵀ,  y = Cᵀ S + D·x  (times silu(z))

    x, z [B,H,P] float32 or bfloat16 (P a multiple of 4); dt [B,H] in x's type or float32; B, C [B,G,N], N up to 256, head
    h reading group h // (H // G); A, D, dt_bias [H] float32 (A < 0: it decays).  ``state`` [S,H,N,P] float32 is updated
    in place, with ``slots`` as in :func:`causal_conv_step`.  Returns y [B,H,P] in x's type; ``out`` may be x or z."""
    dev = _device_of(x, "x")
    _dim(x, "x", 3, "[B,H,P]")
    _dim(B, "B", 3, "[B,G,N]")
    _dim(state, "state", 4, "[S,H,N,P]")
    nb, H, P = x.shape
    G, N = B.shape[1:]
    code, dtype = _dtype_code(x.dtype), x.dtype
    if H == 0 or G == 0 or H % G or P == 0 or P % 4 or not 0 < N <= STEP_MAX_ROWS:
        raise ValueError(f"unsupported shape H={H} G={G} N={N} P={P} (H a multiple of G, N up to {STEP_MAX_ROWS}, "
                         f"P a multiple of 4)")
    _require_view(x, "x", (nb, H, P), dtype, dev)
    _require_view(B, "B", (nb, G, N), dtype, dev)
    _require_view(C, "C", (nb, G, N), dtype, dev)
    _dim(dt, "dt", 2, "[B,H]")
    dt_f32 = _param_f32(dt, "dt", dtype)
    if dt.shape != (nb, H) or dt.get_device() != dev.index:
        raise ValueError(f"dt is {tuple(dt.shape)} on {dt.device}, expected {(nb, H)} on {dev}")
    if A is None:
        raise ValueError("A must be a tensor")
    _require(A, "A", (H,), torch.float32, dev)
    if D is not None:
        _require(D, "D", (H,), torch.float32, dev)
    if dt_bias is not None:
        _require(dt_bias, "dt_bias", (H,), torch.float32, dev)
    if z is not None:
        _require_view(z, "z", (nb, H, P), dtype, dev)
    _require(state, "state", (state.shape[0], H, N, P), torch.float32, dev)
    _pool(state, slots, nb, dev)
    if out is None:
        y = torch.empty(nb, H, P, device=dev, dtype=dtype)
    else:
        _require_view(out, "out", (nb, H, P), dtype, dev)
        _apart("out", out, ("x", "z"), x=x, dt=dt, A=A, B=B, C=C, D=D, z=z, dt_bias=dt_bias, state=state, slots=slots)
        y = out
    sx, sb, sc, sy, st = x.stride(), B.stride(), C.stride(), y.stride(), dt.stride()
    sz = (0, 0) if z is None else z.stride()
    _exec("pf_ssm_step_exec", dev, _STEP, _STEP_SIZE, state.data_ptr(), _ptr(slots), x.data_ptr(), B.data_ptr(),
          C.data_ptr(), y.data_ptr(), dt.data_ptr(), _ptr(z), A.data_ptr(), _ptr(D), _ptr(dt_bias), 0, 0,
          sx[0], sx[1], sb[0], sb[1], sc[0], sc[1], sy[0], sy[1], st[0], st[1], sz[0], sz[1], H * N * P, nb,
          state.shape[0], H, G, N, P, code, dt_f32, int(bool(dt_softplus)), 0, 0.0)
    return y


def gdn_step(state: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, beta: torch.Tensor,
             g: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
             slots: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of the gated delta rule for each of B sequences:

        S ← e^g S,  r = β (v − kᵀ S),  S ← S + k rᵀ,  o = scale · qᵀ S

    q, k [B,H,DK] (DK up to 256) and v [B,H,DV] (DV a multiple of 4) float32 or bfloat16; beta [B,H] float32; g float32:
    [B,H] (GDN), [B,H,DK] (KDA: row d of S decays by g[..., d]) or None (DeltaNet).  ``state`` [S,H,DK,DV] float32 — the
    chunked forwards' ``h_final`` — is updated in place, with ``slots`` as in :func:`causal_conv_step`.  Returns
    o [B,H,DV] float32 scaled by ``scale`` (default DK^-1/2), as the chunked forwards do; ``out`` may be v."""
    dev = _device_of(q, "q")
    _dim(q, "q", 3, "[B,H,DK]")
    _dim(v, "v", 3, "[B,H,DV]")
    _dim(state, "state", 4, "[S,H,DK,DV]")
    nb, H, N = q.shape
    P = v.shape[2]
    code, dtype = _dtype_code(q.dtype), q.dtype
    if H == 0 or P == 0 or P % 4 or not 0 < N <= STEP_MAX_ROWS:
        raise ValueError(f"unsupported shape H={H} DK={N} DV={P} (DK up to {STEP_MAX_ROWS}, DV a multiple of 4)")
    _require_view(q, "q", (nb, H, N), dtype, dev)
    _require_view(k, "k", (nb, H, N), dtype, dev)
    _require_view(v, "v", (nb, H, P), dtype, dev)
    if beta is None:
        raise ValueError("beta must be a tensor")
    _require(beta, "beta", (nb, H), torch.float32, dev)
    rows = False
    if g is not None:
        rows = isinstance(g, torch.Tensor) and g.dim() == 3
        _require(g, "g", (nb, H, N) if rows else (nb, H), torch.float32, dev)
    _require(state, "state", (state.shape[0], H, N, P), torch.float32, dev)
    _pool(state, slots, nb, dev)
    if out is None:
        o = torch.empty(nb, H, P, device=dev, dtype=torch.float32)
    else:
        _require_view(out, "out", (nb, H, P), torch.float32, dev)
        _apart("out", out, ("v",), q=q, k=k, v=v, beta=beta, g=g, state=state, slots=slots)
        o = out
    sq, sk, sv, so = q.stride(), k.stride(), v.stride(), o.stride()
    _exec("pf_gdn_step_exec", dev, _STEP, _STEP_SIZE, state.data_ptr(), _ptr(slots), v.data_ptr(), k.data_ptr(),
          q.data_ptr(), o.data_ptr(), 0, 0, 0, 0, 0, beta.data_ptr(), _ptr(g), sv[0], sv[1], sk[0], sk[1],
          sq[0], sq[1], so[0], so[1], 0, 0, 0, 0, H * N * P, nb, state.shape[0], H, H, N, P, code, 0, 0,
          int(rows), float(N ** -0.5 if scale is None else scale))
    return o


# ------------------------------------------------------------------------------------------
#  Norm
# ------------------------------------------------------------------------------------------
def _rows_of(t: torch.Tensor, name: str, D: int) -> int:
    """The row stride of a tensor [..., D] whose leading dimensions are evenly spaced rows."""
    if t.is_contiguous():
        return D
    try:
        flat = t.view(-1, D)
    except RuntimeError:
        flat = None
    if flat is None or (flat.stride(1) != 1 and D != 1):
        raise ValueError(f"{name} must be rows of {D} contiguous values, evenly spaced")
    return flat.stride(0)


def _norm(x, weight, residual, eps, y, y_code, block, scales, residual_out, given):
    dev, D, dtype = x.device, x.shape[-1], x.dtype
    if weight is None:
        raise ValueError("weight must be a tensor")
    w_f32 = _param_f32(weight, "weight", dtype)
    _require(weight, "weight", (D,), weight.dtype, dev)
    h, r_f32, r_row, h_row = None, 0, 0, 0
    if residual is not None:
        r_f32 = _param_f32(residual, "residual", dtype)
        if residual.shape != x.shape or residual.get_device() != dev.index:
            raise ValueError(f"residual is {tuple(residual.shape)} on {residual.device}, expected {tuple(x.shape)} on {dev}")
        r_row = _rows_of(residual, "residual", D)
        if residual_out is None:
            h = torch.empty(x.shape, device=dev, dtype=residual.dtype)
            h_row = D
        else:
            h = residual_out
            if h.shape != x.shape or h.dtype != residual.dtype or h.device != dev:
                raise ValueError(f"residual_out is {tuple(h.shape)} {h.dtype} on {h.device}, expected {tuple(x.shape)} "
                                 f"{residual.dtype} on {dev}")
            h_row = _rows_of(h, "residual_out", D)
            _apart("residual_out", h, ("x", "residual"), x=x, residual=residual, weight=weight, out=y, scales_out=scales)
    elif residual_out is not None:
        raise ValueError("residual_out without a residual")
    if given:
        _apart("out", y, ("x", "residual"), x=x, residual=residual, weight=weight, scales_out=scales)
        _apart("scales_out", scales, x=x, residual=residual, weight=weight)
    _exec("pf_norm_exec", dev, _NORM, _NORM_SIZE, x.data_ptr(), _ptr(residual), weight.data_ptr(), y.data_ptr(),
          _ptr(scales), _ptr(h), _rows_of(x, "x", D), r_row, _rows_of(y, "out", D), h_row, x.numel() // D,
          D, _dtype_code(dtype), y_code, r_f32, w_f32, block, float(eps))
    return h


def _norm_operand(x) -> None:
    _device_of(x, "x")
    if x.dim() == 0 or not 0 < x.shape[-1] <= NORM_MAX_WIDTH:
        raise ValueError(f"x must be [..., D] with D in 1..{NORM_MAX_WIDTH}, got {tuple(x.shape)}")


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                 out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
                 residual_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """h = x + residual;  y = h · rsqrt(mean(h²) + eps) · weight, over the last dimension.

    x [..., D] float32 or bfloat16, D up to 32768; residual of x's shape and weight [D] in x's type or float32.  Returns
    (y, h): y in x's type (bfloat16 also of float32 rows: ``out_dtype``), h in the residual's, or None without one.  The
    norm is of h before it is rounded.  ``residual_out`` may be ``residual`` (the stream updated in place) or x, and ``out``
    too, where it has their type; not both the same."""
    _norm_operand(x)
    dtype = x.dtype if out_dtype is None else out_dtype
    if dtype is not x.dtype and dtype is not torch.bfloat16:
        raise ValueError(f"out_dtype {dtype} of {x.dtype} rows ({x.dtype} or bfloat16)")
    given = out is not None
    if out is None:
        out = torch.empty(x.shape, device=x.device, dtype=dtype)
    elif out.shape != x.shape or out.dtype != dtype or out.device != x.device:
        raise ValueError(f"out is {tuple(out.shape)} {out.dtype} on {out.device}, expected {tuple(x.shape)} {dtype} on {x.device}")
    h = _norm(x, weight, residual, eps, out, _dtype_code(dtype), 0, None, residual_out, given)
    return out, h


def add_rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *,
                     eps: float = 1e-6, scale_block: Optional[int] = None, out: Optional[torch.Tensor] = None,
                     scales_out: Optional[torch.Tensor] = None, residual_out: Optional[torch.Tensor] = None,
                     ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """:func:`add_rms_norm` with the output in 8 bits: (codes, scales, h), y ≈ codes · scales.

    codes [..., D] are ``torch.float8_e4m3fn``, scales float32: the largest |y| of a row over 448, [..., 1], or with
    ``scale_block=128`` that of each 128 columns, [..., D // 128] (D a multiple of 128).  codes = y · (448 / largest) rounded
    to nearest even; a row or block of zeros has scale 0.  Operands as in :func:`add_rms_norm`."""
    _norm_operand(x)
    D = x.shape[-1]
    if scale_block is not None and (scale_block != 128 or D % 128):
        raise ValueError(f"scale_block must be None or 128, of rows of a multiple of 128: got {scale_block} of {D}")
    shape = (*x.shape[:-1], 1 if scale_block is None else D // 128)
    given = out is not None or scales_out is not None
    if out is None:
        out = torch.empty(x.shape, device=x.device, dtype=torch.float8_e4m3fn)
    elif out.shape != x.shape or out.dtype != torch.float8_e4m3fn or out.device != x.device:
        raise ValueError(f"out is {tuple(out.shape)} {out.dtype} on {out.device}, expected {tuple(x.shape)} float8_e4m3fn on {x.device}")
    if scales_out is None:
        scales_out = torch.empty(shape, device=x.device, dtype=torch.float32)
    else:
        _require(scales_out, "scales_out", shape, torch.float32, x.device)
    h = _norm(x, weight, residual, eps, out, _hip.PF_NORM_FP8, 128 if scale_block else 0, scales_out, residual_out,
              given)
    return out, scales_out, h
