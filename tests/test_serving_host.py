"""Refusals of the serving operators, without a GPU: the C entry points' statuses, the argument structs' sizes, and the
Python operators' checks (device tensors are stood in for by CPU ones where a check comes after the device's)."""
import os
import subprocess

import pytest
import torch

import pto_fuser_amd as pf
from pto_fuser_amd import _build, _hip, ops, serving

STRUCTS = {"pf_conv_args": serving._CONV_SIZE, "pf_conv_step_args": serving._CONV_STEP_SIZE, "pf_step_args": serving._STEP_SIZE,
           "pf_ssm_args": serving._SSM_SIZE, "pf_norm_args": serving._NORM_SIZE}


@pytest.fixture(scope="module")
def lib():
    _build.ensure_built()
    return _hip.load()


@pytest.fixture
def on_cpu(monkeypatch):
    """CPU tensors pass for device ones, and a launch is recorded."""
    made = []
    on = lambda t, name: t.device  # noqa: E731
    monkeypatch.setattr(serving, "_device_of", on)
    monkeypatch.setattr(serving, "_exec", lambda name, dev, layout, *fields: made.append((name, layout.pack(*fields))))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: None)
    return made


def test_struct_sizes_are_the_header_s(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "pto_fuser_hip.h"\nint main(void) {' +
                   "".join(f'printf("{n} %zu\\n", sizeof({n}));' for n in STRUCTS) + "return 0; }\n")
    subprocess.run(["gcc", "-I", _build.INCLUDE, str(src), "-o", str(tmp_path / "sizes")], check=True)
    out = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout
    assert dict((n, int(s)) for n, s in (line.split() for line in out.splitlines())) == STRUCTS


def _conv(**kw):
    f = dict(size=serving._CONV_SIZE, x=64, w=64, bias=0, state_in=0, lengths=0, y=64, state_out=0, x_b=0, x_t=0, y_b=0, y_t=0,
             si=0, so=0, B=1, T=4, W=8, K=4, dtype=1, w_f32=0, act=1)
    assert not set(kw) - set(f)
    return serving._CONV.pack(*{**f, **kw}.values())


@pytest.mark.parametrize("bad", [dict(size=8), dict(dtype=2), dict(K=1), dict(K=5), dict(W=0), dict(T=-1), dict(B=-1), dict(w=0),
                                 dict(x=0), dict(y=0), dict(x_t=-1), dict(B=2 ** 31 - 1, W=2 ** 24, T=2 ** 20)])
def test_conv_statuses(lib, bad):
    assert lib.pf_conv_exec(_conv(**bad), None) == _hip.PF_ERR_ARG


def test_empty_calls_launch_nothing(lib):
    assert lib.pf_conv_exec(_conv(B=0, x=0, y=0), None) == _hip.PF_OK
    assert lib.pf_conv_exec(None, None) == _hip.PF_ERR_ARG
    assert lib.pf_norm_exec(_norm(rows=0, x=0, y=0), None) == _hip.PF_OK
    assert lib.pf_ssm_step_exec(_step(B=0), None) == _hip.PF_OK
    assert lib.pf_gdn_step_exec(_step(B=0, G=2, beta=64), None) == _hip.PF_OK
    assert lib.pf_conv_step_exec(_conv_step(B=0), None) == _hip.PF_OK


def _conv_step(**kw):
    f = dict(size=serving._CONV_STEP_SIZE, x=64, w=64, bias=0, state=64, slots=0, y=64, x_b=0, y_b=0, s_b=0, B=1, S=1, W=8, K=4,
             dtype=1, w_f32=0, act=1)
    return serving._CONV_STEP.pack(*{**f, **kw}.values())


@pytest.mark.parametrize("bad", [dict(size=0), dict(dtype=-1), dict(K=1), dict(K=5), dict(W=0), dict(state=0), dict(B=2), dict(x_b=-1)])
def test_conv_step_statuses(lib, bad):
    assert lib.pf_conv_step_exec(_conv_step(**bad), None) == _hip.PF_ERR_ARG


def _step(**kw):
    f = dict(size=serving._STEP_SIZE, state=64, slots=0, v=64, k=64, q=64, y=64, dt=64, z=0, a=64, d=0, dt_bias=0, beta=0, g=0)
    f.update({f"s{i}": 0 for i in range(13)})
    f.update(B=1, S=1, H=2, G=1, N=16, P=8, dtype=1, dt_f32=0, softplus=0, g_rows=0, scale=1.0)
    return serving._STEP.pack(*{**f, **kw}.values())


@pytest.mark.parametrize("bad", [dict(size=4), dict(dtype=3), dict(H=3, G=2), dict(N=257), dict(N=0), dict(P=6), dict(P=0), dict(dt=0),
                                 dict(a=0), dict(state=0), dict(B=2), dict(s0=-1), dict(G=0)])
def test_step_statuses(lib, bad):
    assert lib.pf_ssm_step_exec(_step(**bad), None) == _hip.PF_ERR_ARG


@pytest.mark.parametrize("bad", [dict(beta=0, G=2), dict(beta=64, G=1), dict(beta=64, G=2, N=300)])
def test_gdn_step_statuses(lib, bad):
    assert lib.pf_gdn_step_exec(_step(**bad), None) == _hip.PF_ERR_ARG


def _ssm(**kw):
    f = dict(size=serving._SSM_SIZE, x=64, dt=64, b=64, c=64, z=0, a=64, d=0, dt_bias=0, h0=0, lengths=0, y=64, h_final=0, ws=0,
             ws_bytes=0)
    f.update({f"s{i}": 64 for i in range(18)})
    f.update(B=1, H=4, G=2, T=100, N=64, P=64, dtype=1, dt_f32=0, softplus=0)
    assert not set(kw) - set(f)
    return serving._SSM.pack(*{**f, **kw}.values())


@pytest.mark.parametrize("bad", [dict(size=0), dict(dtype=2), dict(H=3), dict(H=0), dict(G=0), dict(N=144), dict(N=24), dict(N=0),
                                 dict(P=48), dict(P=288), dict(P=0), dict(T=-1), dict(B=-1), dict(x=0), dict(dt=0), dict(b=0), dict(c=0),
                                 dict(y=0), dict(a=0), dict(s0=-1), dict(s17=-1), dict(s2=63),
                                 dict(s8=0), dict(s11=1 << 23), dict(z=64, s14=8), dict(B=1 << 30, H=1 << 20, G=1)])
def test_ssm_statuses(lib, bad):
    assert lib.pf_ssm_exec(_ssm(**bad), None) == _hip.PF_ERR_ARG


def test_ssm_workspace_sizes(lib):
    """Whole sequences need none; segments a state and a decay each, never more than a generation of workgroups' worth;
    an unsupported shape, or one past any memory, reports 0."""
    size = lib.pf_ssm_workspace_bytes
    assert lib.pf_ssm_exec(_ssm(B=0), None) == _hip.PF_OK
    assert size(1, 4, 1, 64, 128, 64, 1) == 0 and size(64, 64, 1, 8192, 128, 64, 1) == 0
    assert size(1, 4, 1, 8192, 100, 64, 1) == 0 and size(1 << 20, 1 << 20, 1, 8192, 128, 64, 1) == 0
    for H, G, T, N, P in ((4, 1, 8192, 128, 64), (32, 1, 32768, 128, 64), (32, 32, 4096, 64, 128), (64, 2, 1 << 30, 64, 64)):
        one = H * (N * P + 1) * 4
        for dtype in (0, 1):
            n = size(1, H, G, T, N, P, dtype)
            assert n and n % one == 0 and 2 <= n // one <= 512
    assert 0 < size(1, 1, 1, 1 << 30, 16, 32, 1) <= 256 * 256 * 64 * 4 + 1024      # narrow states: padded blocks


@pytest.mark.parametrize("B,H,T,P,dtype,segments", [
    (1, 4, 256, 64, 1, 4), (1, 4, 512, 64, 1, 8), (1, 32, 1024, 64, 1, 16), (1, 32, 4096, 64, 1, 32), (2, 32, 8192, 64, 1, 16),
    (4, 32, 2048, 64, 1, 8), (4, 32, 512, 64, 1, 4), (16, 32, 256, 64, 1, 0), (16, 32, 1024, 64, 1, 0), (16, 64, 512, 64, 1, 0),
    (8, 64, 192, 64, 1, 0), (1, 4, 512, 64, 0, 8), (8, 32, 256, 64, 0, 0), (2, 32, 1024, 64, 0, 8)])
def test_ssm_plans_where_they_were_measured(lib, B, H, T, P, dtype, segments):
    """The number of segments (0: whole sequences) at shapes measured every way; the times are beside the rule."""
    n, one = lib.pf_ssm_workspace_bytes(B, H, 1, T, 128, P, dtype), B * H * (128 * P + 1) * 4
    assert n == segments * one


def _norm(**kw):
    f = dict(size=serving._NORM_SIZE, x=64, residual=0, w=64, y=64, scales=0, h=0, x_row=8, r_row=8, y_row=8, h_row=8, rows=1, D=256,
             dtype=1, y_dtype=1, r_f32=0, w_f32=0, block=0, eps=1e-6)
    return serving._NORM.pack(*{**f, **kw}.values())


@pytest.mark.parametrize("bad", [dict(size=1), dict(dtype=2), dict(D=0), dict(D=32769), dict(y_dtype=0), dict(y_dtype=2), dict(block=128),
                                 dict(y_dtype=2, scales=64, block=64), dict(y_dtype=2, scales=64, block=128, D=200), dict(h=64),
                                 dict(x=0), dict(rows=-1), dict(x_row=-1)])
def test_norm_statuses(lib, bad):
    assert lib.pf_norm_exec(_norm(**bad), None) == _hip.PF_ERR_ARG


def test_operators_want_a_device():
    x = torch.zeros(1, 4, 8)
    with pytest.raises(ValueError, match="HIP device"):
        pf.causal_conv(x, torch.zeros(8, 4))
    with pytest.raises(ValueError, match="HIP device"):
        pf.causal_conv_step(x[0], torch.zeros(4, 3, 8), torch.zeros(8, 4))
    with pytest.raises(ValueError, match="HIP device"):
        pf.ssm_step(torch.zeros(1, 4, 2, 8), x, torch.zeros(1, 4), torch.zeros(4), x[:, :1, :2], x[:, :1, :2])
    with pytest.raises(ValueError, match="HIP device"):
        pf.gdn_step(torch.zeros(1, 4, 8, 8), x, x, x, torch.zeros(1, 4))
    with pytest.raises(ValueError, match="HIP device"):
        pf.add_rms_norm(x, torch.zeros(8))


def test_conv_refusals(on_cpu):
    x, w = torch.zeros(2, 4, 8), torch.zeros(8, 4)
    pf.causal_conv(x, w, torch.zeros(8), initial_state=torch.zeros(2, 3, 8))
    assert on_cpu.pop()[0] == "pf_conv_exec"
    for match, call in (
            (r"\[B,T,W\]", lambda: pf.causal_conv(x[0], w)),
            ("taps", lambda: pf.causal_conv(x, torch.zeros(8, 5))),
            ("dtype", lambda: pf.causal_conv(x.half(), w)),
            ("weight has shape", lambda: pf.causal_conv(x, torch.zeros(7, 4))),
            ("weight has dtype", lambda: pf.causal_conv(x, w.double())),
            ("bias has dtype", lambda: pf.causal_conv(x.bfloat16(), w, torch.zeros(8, dtype=torch.bfloat16))),
            ("last dimension", lambda: pf.causal_conv(torch.zeros(2, 8, 4).transpose(1, 2), w)),
            ("initial_state has shape", lambda: pf.causal_conv(x, w, initial_state=torch.zeros(2, 4, 8))),
            ("lengths has dtype", lambda: pf.causal_conv(x, w, lengths=torch.zeros(2, dtype=torch.int64))),
            ("activation", lambda: pf.causal_conv(x, w, activation="gelu")),
            ("out may not be x", lambda: pf.causal_conv(x, w, out=x)),
            ("state holds 3", lambda: pf.causal_conv_step(x[0, :2], torch.zeros(3, 3, 8), w)),
            ("slots has dtype", lambda: pf.causal_conv_step(x[0, :2], torch.zeros(3, 3, 8), w, slots=torch.zeros(2))),
            ("state has shape", lambda: pf.causal_conv_step(x[0, :2], torch.zeros(2, 2, 8), w))):
        with pytest.raises(ValueError, match=match):
            call()
    assert not on_cpu


def test_step_refusals(on_cpu):
    x, b, S = torch.zeros(2, 4, 8), torch.zeros(2, 2, 16), torch.zeros(2, 4, 16, 8)
    dt, A = torch.zeros(2, 4), torch.zeros(4)
    pf.ssm_step(S, x, dt, A, b, b)
    pf.gdn_step(S, torch.zeros(2, 4, 16), torch.zeros(2, 4, 16), x, dt, torch.zeros(2, 4, 16))
    assert [n for n, _ in on_cpu] == ["pf_ssm_step_exec", "pf_gdn_step_exec"]
    on_cpu.clear()
    q = torch.zeros(2, 4, 16)
    for match, call in (
            ("multiple of G", lambda: pf.ssm_step(S, x, dt, A, torch.zeros(2, 3, 16), b)),
            ("multiple of 4", lambda: pf.ssm_step(S, torch.zeros(2, 4, 6), dt, A, b, b)),
            ("up to 256", lambda: pf.ssm_step(S, x, dt, A, torch.zeros(2, 2, 257), b)),
            ("C has shape", lambda: pf.ssm_step(S, x, dt, A, b, b[:, :1])),
            ("dt is", lambda: pf.ssm_step(S, x, dt[:1], A, b, b)),
            ("dt has dtype", lambda: pf.ssm_step(S, x, dt.double(), A, b, b)),
            ("A must", lambda: pf.ssm_step(S, x, dt, None, b, b)),
            ("state has shape", lambda: pf.ssm_step(S[:, :, :8], x, dt, A, b, b)),
            ("state has dtype", lambda: pf.ssm_step(S.bfloat16(), x, dt, A, b, b)),
            ("z has shape", lambda: pf.ssm_step(S, x, dt, A, b, b, z=x[:1])),
            ("beta", lambda: pf.gdn_step(S, q, q, x, None)),
            ("g has shape", lambda: pf.gdn_step(S, q, q, x, dt, dt[:1])),
            ("k has shape", lambda: pf.gdn_step(S, q, q[:, :2], x, dt)),
            ("out has dtype", lambda: pf.gdn_step(S, q.bfloat16(), q.bfloat16(), x.bfloat16(), dt, out=x.bfloat16()))):
        with pytest.raises(ValueError, match=match):
            call()
    assert not on_cpu


def test_ssm_refusals(on_cpu):
    x, b = torch.zeros(2, 4, 9, 32), torch.zeros(2, 2, 9, 16)
    dt, A, h0 = torch.zeros(2, 4, 9), torch.zeros(4), torch.zeros(2, 4, 16, 32)
    pf.ssm_chunk_forward(x, dt, A, b, b, A, z=x, dt_bias=A, h0=h0)
    assert on_cpu.pop()[0] == "pf_ssm_exec"
    for match, call in (
            (r"\[B,H,T,P\]", lambda: pf.ssm_chunk_forward(x[0], dt, A, b, b)),
            ("multiple of G", lambda: pf.ssm_chunk_forward(x, dt, A, torch.zeros(2, 3, 9, 16), b)),
            ("P of 32", lambda: pf.ssm_chunk_forward(x[..., :16], dt, A, b, b)),
            ("N of 16", lambda: pf.ssm_chunk_forward(x, dt, A, torch.zeros(2, 2, 9, 144), b)),
            ("dtype", lambda: pf.ssm_chunk_forward(x.half(), dt, A, b, b)),
            ("B has shape", lambda: pf.ssm_chunk_forward(x, dt, A, b[:, :, :8], b)),
            ("C has dtype", lambda: pf.ssm_chunk_forward(x, dt, A, b, b.bfloat16())),
            ("dt is", lambda: pf.ssm_chunk_forward(x, dt[:, :, :8], A, b, b)),
            ("A has shape", lambda: pf.ssm_chunk_forward(x, dt, A[:2], b, b)),
            ("last dimension", lambda: pf.ssm_chunk_forward(torch.zeros(2, 4, 32, 9).transpose(2, 3), dt, A, b, b)),
            ("z has shape", lambda: pf.ssm_chunk_forward(x, dt, A, b, b, z=x[:1])),
            ("h0 has shape", lambda: pf.ssm_chunk_forward(x, dt, A, b, b, h0=h0.transpose(2, 3))),
            ("lengths has dtype", lambda: pf.ssm_chunk_forward(x, dt, A, b, b, lengths=torch.zeros(2))),
            ("final_out has shape", lambda: pf.ssm_chunk_forward(x, dt, A, b, b, final_out=h0[:1])),
            ("out has dtype", lambda: pf.ssm_chunk_forward(x, dt, A, b, b, out=x.bfloat16()))):
        with pytest.raises(ValueError, match=match):
            call()
    assert not on_cpu


def test_norm_refusals(on_cpu):
    x, w = torch.zeros(3, 256), torch.zeros(256)
    pf.add_rms_norm(x, w, x)
    assert on_cpu.pop()[0] == "pf_norm_exec"
    for match, call in (
            (r"\[\.\.\., D\]", lambda: pf.add_rms_norm(torch.zeros(2, 32769), w)),
            ("weight has shape", lambda: pf.add_rms_norm(x, w[:8])),
            ("residual is", lambda: pf.add_rms_norm(x, w, x[:2])),
            ("residual has dtype", lambda: pf.add_rms_norm(x, w, x.half())),
            ("without a residual", lambda: pf.add_rms_norm(x, w, residual_out=x)),
            ("evenly spaced", lambda: pf.add_rms_norm(torch.zeros(256, 3).t(), w)),
            ("out_dtype", lambda: pf.add_rms_norm(x.bfloat16(), w, out_dtype=torch.float32)),
            ("scale_block", lambda: pf.add_rms_norm_fp8(x, w, scale_block=64)),
            ("scale_block", lambda: pf.add_rms_norm_fp8(torch.zeros(3, 200), w[:200], scale_block=128)),
            ("scales_out has shape", lambda: pf.add_rms_norm_fp8(x, w, scales_out=torch.zeros(3)))):
        with pytest.raises(ValueError, match=match):
            call()
    assert not on_cpu


def test_sizes_past_32_bits_are_refused(monkeypatch):
    """A size that does not fit its field is a ValueError, not a struct's."""
    monkeypatch.setattr(serving, "_FUNCTIONS", {"pf_norm_exec": None})
    with pytest.raises(ValueError, match="past what pf_norm_exec takes"):
        serving._exec("pf_norm_exec", torch.device("cuda", 0), serving._NORM, serving._NORM_SIZE, *[0] * 10, 1 << 31, *[0] * 6, 0.0)


def test_outputs_that_share_memory_are_refused(on_cpu):
    """A workgroup may not write what another still reads; the very view that its writer reads may be written, and slices that
    lie side by side in one buffer are apart."""
    x, w = torch.zeros(2, 4, 8), torch.zeros(8, 4)
    buf, state = torch.zeros(2, 5, 8), torch.zeros(2, 3, 8)
    q, S, dt, A = torch.zeros(2, 4, 8), torch.zeros(2, 4, 8, 8), torch.zeros(2, 4), torch.zeros(4)
    v, b = torch.zeros(2, 4, 8), torch.zeros(2, 2, 8)
    px, pb, h0 = torch.zeros(2, 4, 9, 32), torch.zeros(2, 2, 9, 16), torch.zeros(2, 4, 16, 32)
    pdt, pool = torch.zeros(2, 4, 9), torch.zeros(3, 4, 16, 32)
    rows, nw = torch.zeros(6, 256), torch.zeros(256)
    scales = torch.zeros(6, 1)
    for match, call in (
            ("out may not be x", lambda: pf.causal_conv(buf[:, :4], w, out=buf[:, 1:])),
            ("out may not be initial_state", lambda: pf.causal_conv(x[:, :3], w, initial_state=state, out=state)),
            ("final_out may not be x", lambda: pf.causal_conv(x, w, final_out=x.view(-1)[:48].view(2, 3, 8))),
            ("final_out may not be initial_state", lambda: pf.causal_conv(x, w, initial_state=buf.view(-1)[:48].view(2, 3, 8),
                                                                          final_out=buf.view(-1)[8:56].view(2, 3, 8))),
            ("final_out may not be out", lambda: pf.causal_conv(x[:, :3], w, out=state, final_out=state)),
            ("out may not be state", lambda: pf.causal_conv_step(x[:, 0], state, w, out=state[:, 0])),
            ("out may not be x", lambda: pf.causal_conv_step(buf.view(-1)[:16].view(2, 8), state, w, out=buf.view(-1)[8:24].view(2, 8))),
            ("out may not be q", lambda: pf.gdn_step(S, q, v, v, dt, out=q)),
            ("out may not be k", lambda: pf.gdn_step(S, q, v, q + 1, dt, out=v)),
            ("out may not be state", lambda: pf.gdn_step(S, q, q, v, dt, out=S[:, :, 0])),
            ("out may not be B", lambda: pf.ssm_step(S, v, dt, A, q, q, out=q)),
            ("out may not be x", lambda: pf.ssm_step(S, v, dt, A, b, b, out=v.view(4, 2, 8).transpose(0, 1))),
            ("out may not be x", lambda: pf.ssm_chunk_forward(px, pdt, A, pb, pb, out=px)),
            ("out may not be z", lambda: pf.ssm_chunk_forward(px + 1, pdt, A, pb, pb, z=px, out=px)),
            ("final_out may not be h0", lambda: pf.ssm_chunk_forward(px, pdt, A, pb, pb, h0=pool[:2], final_out=pool[1:])),
            ("out may not be x", lambda: pf.add_rms_norm(rows[:5], nw, out=rows[1:])),
            ("out may not be x", lambda: pf.add_rms_norm(rows, nw, out_dtype=torch.bfloat16, out=rows.view(torch.bfloat16)[:, :256])),
            ("residual_out may not be out", lambda: pf.add_rms_norm(rows + 1, nw, rows, out=rows, residual_out=rows)),
            ("residual_out may not be residual", lambda: pf.add_rms_norm(rows[:5] + 1, nw, rows[:5], residual_out=rows[1:])),
            ("scales_out may not be x", lambda: pf.add_rms_norm_fp8(rows, nw, scales_out=rows.view(-1)[:6].view(6, 1)))):
        with pytest.raises(ValueError, match=match):
            call()
    assert not on_cpu
    wide = torch.zeros(2, 4, 24)
    pf.causal_conv(wide[..., :8], w, out=wide[..., 8:16], initial_state=state, final_out=state)
    pf.causal_conv_step(x[:, 0], state, w, out=x[:, 0])
    pf.gdn_step(S, q, q, v, dt, out=v)
    pf.ssm_step(S, v, dt, A, b, b, z=q, out=q)
    pf.ssm_step(S, v, dt, A, b, b, out=v)
    heads = torch.zeros(2, 9, 256)
    one, two = (heads[..., i:i + 128].unflatten(-1, (4, 32)).transpose(1, 2) for i in (0, 128))
    pf.ssm_chunk_forward(one, pdt, A, pb, pb, h0=h0, out=two, final_out=h0)
    pf.add_rms_norm(rows, nw, rows + 1, out=rows)
    pf.add_rms_norm(rows, nw, nw.expand(6, 256).contiguous(), out=rows[:, :256].view(6, 256))
    pf.add_rms_norm(rows, nw, rows + 1, residual_out=rows)
    pf.add_rms_norm_fp8(rows, nw, scales_out=scales)
    assert len(on_cpu) == 10


def test_memory_in_common_is_never_missed():
    """Random views of one buffer against their elements' addresses."""
    import random
    rng, buf, found = random.Random(1), torch.zeros(400), 0

    def view():
        shape = [rng.randint(1, 4) for _ in range(rng.randint(1, 3))]
        strides = [rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 24, 48]) for _ in shape]
        return torch.as_strided(buf, shape, strides[:-1] + [rng.choice([1, strides[-1]])], rng.randint(0, 50))

    def cells(t):
        at = {t.storage_offset()}
        for n, s in zip(t.shape, t.stride()):
            at = {o + i * s for o in at for i in range(n)}
        return at

    for _ in range(3000):
        a, b = view(), view()
        if cells(a) & cells(b):
            assert serving._share(a, b)
            found += 1
    assert found > 100


def test_outputs_over_themselves_are_refused(on_cpu):
    """An element is written by one thread: no expanded dimension, no rows closer than they are long."""
    x, w, v, S = torch.zeros(2, 4, 8), torch.zeros(8, 4), torch.zeros(2, 4, 8), torch.zeros(2, 4, 8, 8)
    dt, A, b, rows, nw = torch.zeros(2, 4), torch.zeros(4), torch.zeros(2, 2, 8), torch.zeros(6, 256), torch.zeros(256)
    px, pb, pdt = torch.zeros(2, 4, 9, 32), torch.zeros(2, 2, 9, 16), torch.zeros(2, 4, 9)
    for call in (lambda: pf.causal_conv(x, w, out=torch.zeros(4, 8).expand(2, 4, 8)),
                 lambda: pf.causal_conv(x, w, out=torch.zeros(64).as_strided((2, 4, 8), (24, 7, 1))),
                 lambda: pf.causal_conv_step(x[:, 0], torch.zeros(2, 3, 8), w, out=torch.zeros(8).expand(2, 8)),
                 lambda: pf.gdn_step(S, v, v, v, dt, out=torch.zeros(2, 1, 8).expand(2, 4, 8)),
                 lambda: pf.ssm_step(S, v, dt, A, b, b, out=torch.zeros(64).as_strided((2, 4, 8), (16, 8, 1))),
                 lambda: pf.ssm_chunk_forward(px, pdt, A, pb, pb, out=torch.zeros(2, 1, 9, 32).expand(2, 4, 9, 32)),
                 lambda: pf.ssm_chunk_forward(px, pdt, A, pb, pb, out=torch.zeros(2048).as_strided((2, 4, 9, 32), (1000, 32, 31, 1))),
                 lambda: pf.add_rms_norm(rows, nw, out=torch.zeros(256).expand(6, 256)),
                 lambda: pf.add_rms_norm(rows, nw, rows, residual_out=torch.zeros(2000).as_strided((6, 256), (255, 1)))):
        with pytest.raises(ValueError, match="overlapping rows"):
            call()
    assert not on_cpu
    pf.causal_conv(x, w, out=torch.zeros(100).as_strided((2, 4, 8), (8, 20, 1)))
    pf.causal_conv(x[:1, :1], w, out=torch.zeros(8).as_strided((1, 1, 8), (0, 0, 1)))
    assert len(on_cpu) == 2


@pytest.mark.parametrize("T", [2 ** 30 + 1, 2 ** 31 - 7, 2 ** 31 - 1])
def test_prompts_past_the_counters_are_refused(lib, T):
    """Rounded up to whole tiles they would pass 2^31."""
    assert lib.pf_conv_exec(_conv(T=T), None) == _hip.PF_ERR_ARG
    assert lib.pf_ssm_exec(_ssm(T=T), None) == _hip.PF_ERR_ARG


@pytest.mark.parametrize("P", [2 ** 30 + 4, 2 ** 31 - 4])
def test_heads_past_the_counters_are_refused(lib, P):
    assert lib.pf_ssm_step_exec(_step(P=P), None) == _hip.PF_ERR_ARG
    assert lib.pf_gdn_step_exec(_step(P=P, G=2, beta=64), None) == _hip.PF_ERR_ARG


def test_empty_batches_launch_nothing(lib):
    """Tensors of no elements have null pointers."""
    null = dict(v=0, k=0, q=0, y=0, dt=0, beta=0)
    for S, state in ((0, 0), (5, 64)):
        assert lib.pf_ssm_step_exec(_step(B=0, S=S, state=state, **null), None) == _hip.PF_OK
        assert lib.pf_gdn_step_exec(_step(B=0, S=S, state=state, G=2, **null), None) == _hip.PF_OK
        assert lib.pf_conv_step_exec(_conv_step(B=0, S=S, state=state, x=0, y=0), None) == _hip.PF_OK
    assert lib.pf_conv_exec(_conv(B=0, x=0, y=0), None) == lib.pf_ssm_exec(_ssm(B=0, x=0, dt=0, b=0, c=0, y=0), None) == _hip.PF_OK


def test_calls_that_no_launch_covers_are_value_errors(monkeypatch):
    """What an entry point does not take is refused as such; what fails in the launch is the library's error."""
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    for status, error in ((_hip.PF_ERR_ARG, ValueError), (719, _hip.HipKernelError)):
        monkeypatch.setattr(serving, "_FUNCTIONS", {"pf_norm_exec": lambda args, stream: status})
        with pytest.raises(error, match="pf_norm_exec"):
            serving._exec("pf_norm_exec", torch.device("cuda", 0), serving._NORM, serving._NORM_SIZE, *[0] * 17, 0.0)


def test_ssm_token_strides(on_cpu):
    """Operands whose tokens overlap or lie past the kernel's offsets are laid out first, an output is refused."""
    far = serving.SSM_MAX_STRIDE + 8
    buf = torch.zeros(far + 256)
    view = lambda n, stride: buf.as_strided((1, 1, 2, n), (0, 0, stride, 1))  # noqa: E731
    dt, A = torch.zeros(1, 1, 2), torch.zeros(1)
    for stride, same in ((32, True), (serving.SSM_MAX_STRIDE, True), (far, False), (0, False), (16, False)):
        pf.ssm_chunk_forward(view(32, stride), dt, A, view(16, stride), view(16, stride), z=view(32, stride))
        f = serving._SSM.unpack(on_cpu.pop()[1])
        x_t, b_t, c_t, z_t = (f[i] for i in (17, 23, 26, 29))
        want = [stride, stride, stride, stride] if same else [32, stride if stride == 16 else 16, stride if stride == 16 else 16, 32]
        assert [x_t, b_t, c_t, z_t] == want
        assert (f[1] == buf.data_ptr()) == same
    with pytest.raises(ValueError, match="elements apart"):
        pf.ssm_chunk_forward(view(32, 32) + 0, dt, A, view(16, 16) + 0, view(16, 16) + 0, out=view(32, far))
    assert not on_cpu
