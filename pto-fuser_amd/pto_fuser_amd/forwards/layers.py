"""Recurrent layers as they are served: a prompt (or a ragged batch of them), then single tokens from its state.

Two layers over the package's operators, with torch's library products for the projections:

* a state space layer — norm with the residual's addition, one projection to z, x, B, C and dt, the short convolution
  over x, B and C in place, the scan, the norm of its output in 8 bits with a scale a token, and the projection of those;
* a gated delta rule layer — the same around the chunked forward (``gdn_chunk_forward``) and ``gdn_step``.

``prefill`` returns the states after each prompt; ``step`` moves states in a pool on, which its ``slots`` name.  No
counterpart in the reference, whose path ends at the chunked forward.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from ..ops import gdn_chunk_forward
from ..serving import (add_rms_norm, add_rms_norm_fp8, causal_conv, causal_conv_step, gdn_step, ssm_chunk_forward,
                       ssm_step)

__all__ = ["LayerCache", "SsmLayer", "GdnLayer", "make_ssm_layer", "make_gdn_layer"]

_FP8_MAX = 448.0


@dataclass
class LayerCache:
    """The states of one layer's sequences: the last inputs of the convolution, and the recurrence's matrices."""
    conv: torch.Tensor    # [S, K-1, W]
    state: torch.Tensor   # [S, H, N, P] float32


class _Projection8:
    """A projection of 8-bit rows with a scale each: the weight in 8 bits with a scale an output, laid out once."""

    def __init__(self, weight: torch.Tensor) -> None:
        scale = weight.float().abs().amax(-1, keepdim=True).clamp(min=1e-12) / _FP8_MAX       # weight [out, in]
        self.weight = (weight.float() / scale).to(torch.float8_e4m3fn)
        self.scale = scale.t().contiguous()

    def __call__(self, codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
        rows = codes.reshape(-1, codes.shape[-1])
        y = torch._scaled_mm(rows, self.weight.t(), scale_a=scales.reshape(-1, 1), scale_b=self.scale,
                             out_dtype=torch.bfloat16)
        return y.view(*codes.shape[:-1], -1)

    def plain(self) -> torch.Tensor:
        """The weight [out, in] that the codes stand for."""
        return self.weight.float() * self.scale.t()


@dataclass
class SsmLayer:
    norm_w: torch.Tensor        # [D]
    in_w: torch.Tensor          # [D, 2 H P + 2 G N + H]: z, x, B, C, dt
    conv_w: torch.Tensor        # [H P + 2 G N, K]
    conv_b: torch.Tensor
    A: torch.Tensor             # [H] float32, negative
    D: torch.Tensor
    dt_bias: torch.Tensor
    gate_w: torch.Tensor        # [H P]
    out: _Projection8
    H: int
    P: int
    G: int
    N: int

    def cache(self, slots: int) -> LayerCache:
        dev, (W, K) = self.conv_w.device, self.conv_w.shape
        return LayerCache(torch.zeros(slots, K - 1, W, device=dev, dtype=self.conv_w.dtype),
                          torch.zeros(slots, self.H, self.N, self.P, device=dev))

    def _split(self, row):
        """z, x B C and dt of projected rows [..., W]; then x, B and C of convolved ones."""
        inner, shared = self.H * self.P, 2 * self.G * self.N
        return row.split([inner, inner + shared, self.H], dim=-1)

    def _operands(self, xbc):
        x, b, c = xbc.split([self.H * self.P, self.G * self.N, self.G * self.N], dim=-1)
        return x.unflatten(-1, (self.H, self.P)), b.unflatten(-1, (self.G, self.N)), c.unflatten(-1, (self.G, self.N))

    def _project(self, y):
        codes, scales, _ = add_rms_norm_fp8(y, self.gate_w)
        return self.out(codes, scales)

    def prefill(self, hidden: torch.Tensor, residual: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, LayerCache]:
        """hidden, residual [B,T,D] -> (output [B,T,D], the residual stream, the states after each prompt)."""
        y, stream = add_rms_norm(hidden, self.norm_w, residual)
        z, xbc, dt = self._split(y @ self.in_w)
        xbc, conv = causal_conv(xbc, self.conv_w, self.conv_b, lengths=lengths)
        x, b, c = (t.transpose(1, 2) for t in self._operands(xbc))
        y, state = ssm_chunk_forward(x, dt.transpose(1, 2), self.A, b, c, self.D,
                                     z=z.unflatten(-1, (self.H, self.P)).transpose(1, 2), dt_bias=self.dt_bias,
                                     dt_softplus=True, lengths=lengths)
        out = self._project(y.transpose(1, 2).flatten(-2))
        return out, hidden if stream is None else stream, LayerCache(conv, state)

    def step(self, hidden: torch.Tensor, residual: Optional[torch.Tensor], cache: LayerCache,
             slots: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """One token of each sequence: hidden, residual [B,D]; the states named by ``slots`` move on."""
        y, stream = add_rms_norm(hidden, self.norm_w, residual)
        z, xbc, dt = self._split(y @ self.in_w)
        xbc = causal_conv_step(xbc, cache.conv, self.conv_w, self.conv_b, slots=slots)
        x, b, c = self._operands(xbc)
        y = ssm_step(cache.state, x, dt, self.A, b, c, self.D, z=z.unflatten(-1, (self.H, self.P)), dt_bias=self.dt_bias,
                     dt_softplus=True, slots=slots)
        return self._project(y.flatten(-2)), hidden if stream is None else stream


@dataclass
class GdnLayer:
    norm_w: torch.Tensor        # [D]
    in_w: torch.Tensor          # [D, 3 H 128 + 2 H]: q, k, v, beta's and g's logits
    conv_w: torch.Tensor        # [3 H 128, K]
    out_norm_w: torch.Tensor    # [H 128] float32, as the recurrence's output is
    out: _Projection8
    H: int
    gate_scale: float = 0.1

    HEAD = 128

    def cache(self, slots: int) -> LayerCache:
        dev, (W, K) = self.conv_w.device, self.conv_w.shape
        return LayerCache(torch.zeros(slots, K - 1, W, device=dev, dtype=self.conv_w.dtype),
                          torch.zeros(slots, self.H, self.HEAD, self.HEAD, device=dev))

    def _operands(self, qkv, gates):
        """q, k of unit length, v [..., H, 128]; beta, g [..., H] float32."""
        q, k, v = (t.unflatten(-1, (self.H, self.HEAD)) for t in qkv.chunk(3, dim=-1))
        unit = torch.nn.functional.normalize
        beta, g = gates.float().chunk(2, dim=-1)
        return unit(q, dim=-1), unit(k, dim=-1), v, torch.sigmoid(beta), -self.gate_scale * torch.nn.functional.softplus(g)

    def _project(self, o):
        codes, scales, _ = add_rms_norm_fp8(o, self.out_norm_w)
        return self.out(codes, scales)

    def prefill(self, hidden: torch.Tensor, residual: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, LayerCache]:
        """hidden, residual [B,T,D] -> (output [B,T,D], the residual stream, the states after each prompt).  The chunked
        forward takes whole chunks: the rest, and what follows a prompt's end, is filled with tokens that leave the state
        alone (k = 0, beta = 0, g = 0)."""
        T = hidden.shape[1]
        y, stream = add_rms_norm(hidden, self.norm_w, residual)
        qkv, gates = (y @ self.in_w).split([3 * self.H * self.HEAD, 2 * self.H], dim=-1)
        qkv, conv = causal_conv(qkv, self.conv_w, lengths=lengths)
        q, k, v, beta, g = self._operands(qkv, gates)
        if lengths is not None:
            live = (torch.arange(T, device=hidden.device) < lengths[:, None])[..., None]
            beta, g = torch.where(live, beta, 0.0), torch.where(live, g, 0.0)
        heads = [torch.nn.functional.pad(t.transpose(1, 2), (0, 0, 0, -T % 64)).contiguous() for t in (q, k, v)]
        gate = [torch.nn.functional.pad(t.transpose(1, 2), (0, -T % 64)).contiguous() for t in (beta, g)]
        o, state = gdn_chunk_forward(*heads, *gate)
        out = self._project(o[:, :, :T].transpose(1, 2).flatten(-2))
        return out, hidden if stream is None else stream, LayerCache(conv, state)

    def step(self, hidden: torch.Tensor, residual: Optional[torch.Tensor], cache: LayerCache,
             slots: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """One token of each sequence: hidden, residual [B,D]; the states named by ``slots`` move on."""
        y, stream = add_rms_norm(hidden, self.norm_w, residual)
        qkv, gates = (y @ self.in_w).split([3 * self.H * self.HEAD, 2 * self.H], dim=-1)
        qkv = causal_conv_step(qkv, cache.conv, self.conv_w, slots=slots)
        q, k, v, beta, g = self._operands(qkv, gates)
        o = gdn_step(cache.state, q, k, v, beta.contiguous(), g.contiguous(), slots=slots)
        return self._project(o.flatten(-2)), hidden if stream is None else stream


def make_ssm_layer(D: int, H: int, P: int = 64, G: int = 1, N: int = 128, K: int = 4, *, seed: int = 0,
                   device="cuda") -> SsmLayer:
    """Seeded weights with the usual scales: steps between 1e-3 and 1e-1, A between -16 and -1."""
    gen = torch.Generator().manual_seed(seed)
    randn, rand = (lambda *s: torch.randn(*s, generator=gen)), (lambda *s: torch.rand(*s, generator=gen))
    inner, W = H * P, H * P + 2 * G * N
    step = torch.exp(-6.9 + 4.6 * rand(H))
    bf = lambda t: t.to(device, torch.bfloat16)  # noqa: E731
    return SsmLayer(bf(1 + 0.1 * randn(D)), bf(randn(D, inner + W + H) * D ** -0.5), bf((2 * rand(W, K) - 1) * K ** -0.5),
                    bf(0.1 * randn(W)), (-1 - 15 * rand(H)).to(device), (1 + 0.1 * randn(H)).to(device),
                    (step + torch.log(-torch.expm1(-step))).to(device), bf(1 + 0.1 * randn(inner)),
                    _Projection8((randn(D, inner) * inner ** -0.5).to(device)), H, P, G, N)


def make_gdn_layer(D: int, H: int, K: int = 4, *, seed: int = 0, device="cuda") -> GdnLayer:
    gen = torch.Generator().manual_seed(seed)
    randn, rand = (lambda *s: torch.randn(*s, generator=gen)), (lambda *s: torch.rand(*s, generator=gen))
    inner = H * GdnLayer.HEAD
    bf = lambda t: t.to(device, torch.bfloat16)  # noqa: E731
    return GdnLayer(bf(1 + 0.1 * randn(D)), bf(randn(D, 3 * inner + 2 * H) * D ** -0.5), bf((2 * rand(3 * inner, K) - 1) * K ** -0.5),
                    (1 + 0.1 * randn(inner)).to(device), _Projection8((randn(D, inner) * inner ** -0.5).to(device)), H)
