"""Every form of the state space scan: both types, states of up to 64 and up to 128 rows, workgroups of 64, 128 and 256
columns, whole sequences and segments, with and without z, a state in and lengths, against the recurrence in float64 (on
the device), value by value.

float32: the operations that the scan's other tests count.  bfloat16 has 8 bits, the first of them implied: rounding to the
nearest is off by u = 2^-8 of a value at most (1 + 2^-8 lies between 1 and 1 + 2^-7).  y = rn(v) with v off by d is then off by
u |want| + (1 + u) d.  d is float32's, and for each term at most u^2 = 2^-16 where the entering state or the decayed score is
taken in two such terms (u left of the first, u of that of the second), and as much where the state of a segment was made of
such: 2^-15 of the terms' magnitudes.
"""
import pytest
import torch

import serving_refs as ref
from conftest import announce
from test_gpu_serving import BF, DEV, F32, NAN, _ssm_case, _ssm_ops, pf_ssm

pytestmark = pytest.mark.gpu

# type, B, H, T, P, N: the columns of a workgroup that the plan gives them, and segments
FORMS = [(F32, 2, 3, 65, 32, 32, 64, False), (F32, 2, 3, 130, 32, 32, 64, True), (F32, 3, 48, 65, 128, 32, 128, False),
         (F32, 3, 48, 200, 32, 32, 128, True), (F32, 2, 3, 65, 32, 112, 64, False), (F32, 2, 3, 130, 32, 112, 64, True),
         (F32, 3, 48, 65, 128, 112, 128, False), (F32, 3, 48, 200, 32, 112, 128, True),
         (BF, 2, 3, 65, 32, 32, 64, False), (BF, 2, 3, 130, 32, 32, 64, True), (BF, 3, 48, 65, 128, 32, 128, False),
         (BF, 3, 48, 200, 32, 32, 128, True), (BF, 24, 48, 65, 32, 32, 256, False), (BF, 3, 48, 200, 64, 32, 256, True),
         (BF, 2, 3, 65, 32, 112, 64, False), (BF, 2, 3, 130, 32, 112, 64, True), (BF, 3, 48, 65, 128, 112, 128, False),
         (BF, 3, 48, 200, 32, 112, 128, True), (BF, 24, 48, 65, 32, 112, 256, False), (BF, 2, 64, 520, 32, 112, 256, True)]


@pytest.mark.parametrize("full", [True, False])
@pytest.mark.parametrize("dtype,B,H,T,P,N,columns,segments", FORMS)
def test_ssm_forms(dtype, B, H, T, P, N, columns, segments, full):
    from pto_fuser_amd import _hip
    announce(f"ssm_chunk_forward {dtype} B{B} H{H} T{T} P{P} N{N}: {columns} columns, segments={segments}, full={full}")
    assert (_hip.load().pf_ssm_workspace_bytes(B, H, 1, T, N, P, int(dtype is BF)) > 0) == segments
    s = _ssm_case(T + N, dtype, B, H, T, P, 1, N, z=full, h0=full, D=full)
    lengths = [max(0, T - 37 * b) for b in range(B)] if full else None
    a = {k: None if v is None else v.double() for k, v in s.items()}
    with torch.device(DEV):
        want, mag, S, M = ref.ssm(a["x"], a["dt"], a["A"], a["B"], a["C"], a["D"], a["z"], a["dt_bias"], True, a["h0"], lengths)
    if full:
        for b, n in enumerate(lengths):
            for k in ("x", "dt", "B", "C", "z"):
                s[k][b, :, n:] = NAN
    y, final = pf_ssm(s, lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV))
    small = _ssm_ops(T) * ref.EPS32
    assert torch.isfinite(y).all() and torch.isfinite(final).all()
    assert ((final.double() - S).abs() <= small * (M + S.abs()) + 1e-30).all()
    tol = small * (mag + want.abs()) + 1e-30
    if dtype is BF:
        u = 2.0 ** -8
        tol = u * want.abs() + (1 + u) * (tol + 2.0 ** -15 * mag)
    error = (y.double() - want).abs()
    print(f"of its tolerance {(error / tol).max().item():.3f}, of y's norm {(error.norm() / want.norm()).item():.3e}")
    assert (error <= tol).all()
