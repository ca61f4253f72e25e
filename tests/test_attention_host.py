"""Refusals of the attention operators and the paged cache's, without a GPU: the C entry points' statuses, the argument
structs' sizes, and the Python operators' checks (CPU tensors stand in for device ones)."""
import subprocess

import pytest
import torch

import attention_refs as att
from pto_fuser_amd import _build, _hip, attention

STRUCTS = {"pf_attn_args": attention._ATTN_SIZE, "pf_attn_step_args": attention._ATTN_STEP_SIZE,
           "pf_assign_args": attention._ASSIGN_SIZE, "pf_release_args": attention._RELEASE_SIZE,
           "pf_store_args": attention._STORE_SIZE}
BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


@pytest.fixture(scope="module")
def lib():
    _build.ensure_built()
    return _hip.load()


@pytest.fixture
def on_cpu(monkeypatch):
    """CPU tensors pass for device ones, and a launch is recorded."""
    made = []
    monkeypatch.setattr(attention, "_device_of", lambda t, name: t.device)
    monkeypatch.setattr(attention, "_exec", lambda name, dev, layout, *fields: made.append((name, layout.unpack(layout.pack(*fields)))))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: None)
    return made


def test_struct_sizes_are_the_header_s(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "pto_fuser_hip.h"\nint main(void) {' +
                   "".join(f'printf("{n} %zu\\n", sizeof({n}));' for n in STRUCTS) + "return 0; }\n")
    subprocess.run(["gcc", "-I", _build.INCLUDE, str(src), "-o", str(tmp_path / "sizes")], check=True)
    out = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout
    assert dict((n, int(s)) for n, s in (line.split() for line in out.splitlines())) == STRUCTS


def _attn(**kw):
    f = dict(size=attention._ATTN_SIZE, q=64, k=64, v=64, o=64, cu=64, lengths=0)
    f.update({f"s{i}": 64 for i in range(8)})
    f.update(N=4, B=1, H=4, G=2, D=64, dtype=1, zero=1, scale=0.1)
    assert not set(kw) - set(f)
    return attention._ATTN.pack(*{**f, **kw}.values())


@pytest.mark.parametrize("bad", [dict(size=8), dict(dtype=2), dict(H=3), dict(H=0), dict(G=0), dict(D=12), dict(D=264), dict(D=0),
                                 dict(N=-1), dict(N=(1 << 30) + 1), dict(B=-1), dict(cu=0), dict(q=0), dict(k=0), dict(v=0), dict(o=0),
                                 dict(q=66), dict(k=72), dict(v=8), dict(s0=4), dict(s2=-8), dict(s3=12), dict(s4=1 << 23),
                                 dict(s0=1 << 23), dict(s7=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                                 dict(N=1 << 30, H=65536, G=1)])
def test_attention_statuses(lib, bad):
    assert lib.pf_attn_exec(_attn(**bad), None) == _hip.PF_ERR_ARG


def _step(**kw):
    f = dict(size=attention._ATTN_STEP_SIZE, q=64, k=64, v=64, o=64, tables=64, lengths=64, slots=0, ws=0, ws_bytes=0)
    f.update({f"s{i}": 64 for i in range(10)})
    f.update(B=1, S=1, H=4, G=2, D=64, M=9, pages=5, page=16, dtype=1, scale=0.1)
    assert not set(kw) - set(f)
    return attention._ATTN_STEP.pack(*{**f, **kw}.values())


@pytest.mark.parametrize("bad", [dict(size=8), dict(dtype=-1), dict(H=5), dict(D=20), dict(page=0), dict(page=8), dict(page=24),
                                 dict(page=1 << 17), dict(B=-1), dict(B=2), dict(S=-1), dict(M=-1), dict(pages=-1), dict(q=0), dict(o=0),
                                 dict(k=0), dict(v=0), dict(tables=0), dict(lengths=0), dict(k=72), dict(s4=4), dict(s5=-8),
                                 dict(s5=1 << 23), dict(s2=-1), dict(M=1 << 27), dict(scale=0.0),
                                 dict(B=1 << 16, S=1 << 16, M=1 << 22)])
def test_step_statuses(lib, bad):
    assert lib.pf_attn_step_exec(_step(**bad), None) == _hip.PF_ERR_ARG


def test_step_workspaces(lib):
    """A walk that is shared out needs its workspace; an unsupported shape has none."""
    size = lib.pf_attn_step_workspace_bytes
    need = size(1, 4, 2, 64, 1000, 16, 1)
    assert need > 0 and size(1, 4, 2, 64, 2, 16, 1) == 0 and size(64, 32, 8, 128, 1 << 16, 16, 0) <= 64 << 20
    assert size(1, 5, 2, 64, 1000, 16, 1) == size(1, 4, 2, 64, 1000, 24, 1) == size(1, 4, 2, 64, 1 << 27, 16, 1) == 0
    for ws, n in ((0, 0), (64, need - 1), (72, need)):
        assert lib.pf_attn_step_exec(_step(M=1000, ws=ws, ws_bytes=n), None) == _hip.PF_ERR_WORKSPACE


def _assign(**kw):
    f = dict(size=attention._ASSIGN_SIZE)
    f.update({n: 64 for n in ("tables", "lengths", "tokens", "slots", "free", "taken", "rows", "cu", "after", "taken_out")})
    f.update(B=2, S=2, M=4, F=9, capacity=5, page=16)
    assert not set(kw) - set(f)
    return attention._ASSIGN.pack(*{**f, **kw}.values())


@pytest.mark.parametrize("bad", [dict(size=0), dict(tables=0), dict(lengths=0), dict(free=0), dict(taken=0), dict(rows=0), dict(cu=0),
                                 dict(after=0), dict(taken_out=0), dict(B=-1), dict(B=3, slots=0), dict(S=-1), dict(M=-1),
                                 dict(F=-1), dict(capacity=-1), dict(page=12), dict(M=1 << 27)])
def test_assign_statuses(lib, bad):
    assert lib.pf_assign_exec(_assign(**bad), None) == _hip.PF_ERR_ARG


def _release(**kw):
    f = dict(size=attention._RELEASE_SIZE)
    f.update({n: 64 for n in ("tables", "lengths", "slots", "free", "taken", "taken_out")})
    f.update(B=2, S=2, M=4, F=9, page=16)
    return attention._RELEASE.pack(*{**f, **kw}.values())


@pytest.mark.parametrize("bad", [dict(size=0), dict(tables=0), dict(lengths=0), dict(free=0), dict(taken=0), dict(taken_out=0),
                                 dict(B=-1), dict(B=3, slots=0), dict(S=-1), dict(M=-1), dict(F=-1), dict(page=15)])
def test_release_statuses(lib, bad):
    assert lib.pf_release_exec(_release(**bad), None) == _hip.PF_ERR_ARG


def _store(**kw):
    f = dict(size=attention._STORE_SIZE, k=64, v=64, kc=64, vc=64, rows=64)
    f.update({f"s{i}": 64 for i in range(10)})
    f.update(N=3, G=2, D=64, pages=4, page=16, dtype=1)
    return attention._STORE.pack(*{**f, **kw}.values())


@pytest.mark.parametrize("bad", [dict(size=0), dict(k=0), dict(v=0), dict(kc=0), dict(vc=0), dict(rows=0), dict(s3=-1), dict(N=-1),
                                 dict(G=0), dict(D=0), dict(D=12), dict(G=1 << 17), dict(D=1 << 17), dict(pages=-1), dict(page=100),
                                 dict(dtype=2)])
def test_store_statuses(lib, bad):
    assert lib.pf_store_exec(_store(**bad), None) == _hip.PF_ERR_ARG


def test_empty_calls_launch_nothing(lib):
    assert lib.pf_attn_exec(_attn(N=0, q=0, k=0, v=0, o=0), None) == _hip.PF_OK
    assert lib.pf_attn_step_exec(_step(B=0, q=0, o=0), None) == _hip.PF_OK
    assert lib.pf_store_exec(_store(N=0), None) == _hip.PF_OK and lib.pf_store_exec(_store(pages=0), None) == _hip.PF_OK
    for fn in (lib.pf_attn_exec, lib.pf_attn_step_exec, lib.pf_assign_exec, lib.pf_release_exec, lib.pf_store_exec):
        assert fn(None, None) == _hip.PF_ERR_ARG


def test_a_cpu_tensor_is_refused():
    t = torch.zeros(4, 2, 64)
    for call in (lambda: attention.causal_attention(t, t, t, torch.zeros(2, dtype=I32)),
                 lambda: attention.attention_step(t, t[None], t[None], torch.zeros(4, 1, dtype=I32), torch.zeros(4, dtype=I32)),
                 lambda: attention.store_kv(t, t, t[None], t[None], torch.zeros(4, dtype=torch.int64)),
                 lambda: attention.assign_pages(torch.zeros(1, 1, dtype=I32), torch.zeros(1, dtype=I32), None,
                                                torch.zeros(1, dtype=I32), torch.zeros(1, dtype=I32), page_size=16)):
        with pytest.raises(ValueError, match="HIP device"):
            call()


def _attn_call(**kw):
    f = dict(q=torch.zeros(10, 4, 64, dtype=BF), k=torch.zeros(10, 2, 64, dtype=BF), v=torch.zeros(10, 2, 64, dtype=BF),
             cu_seqlens=torch.zeros(3, dtype=I32))
    f.update(kw)
    args = [f.pop(n) for n in ("q", "k", "v", "cu_seqlens")]
    return attention.causal_attention(*args, **f)


def test_attention_checks(on_cpu):
    assert _attn_call().shape == (10, 4, 64) and on_cpu[-1][0] == "pf_attn_exec"
    q = torch.zeros(10, 4, 64, dtype=BF)
    for match, kw in (("q must be", dict(q=q[0])), ("k must be", dict(k=None)), ("k has shape", dict(k=torch.zeros(9, 2, 64, dtype=BF))),
                      ("v has dtype", dict(v=torch.zeros(10, 2, 64))), ("unsupported shape", dict(q=q[:, :3])),
                      ("unsupported shape", dict(q=q[..., :60])), ("v must be a tensor", dict(v=None)),
                      ("contiguous along", dict(q=q.transpose(1, 2).contiguous().transpose(1, 2))),
                      ("cu_seqlens has dtype", dict(cu_seqlens=torch.zeros(3, dtype=torch.int64))),
                      ("an entry more", dict(cu_seqlens=torch.zeros(0, dtype=I32))), ("cu_seqlens must be", dict(cu_seqlens=None)),
                      ("lengths has shape", dict(lengths=torch.zeros(3, dtype=I32))), ("scale", dict(scale=0.0)),
                      ("scale", dict(scale=float("inf"))), ("scale", dict(scale=1e39)), ("scale", dict(scale=-0.1)), ("out has shape", dict(out=q[:9])), ("out may not be q", dict(q=q, out=q))):
        with pytest.raises(ValueError, match=match):
            _attn_call(**kw)
    with pytest.raises((ValueError, TypeError)):
        _attn_call(q=q.half(), k=q[:, :2].half(), v=q[:, :2].half())


def test_attention_copies_what_is_not_whole_vectors(on_cpu):
    buf = torch.zeros(10, 4 * 64 + 8, dtype=BF)
    aligned, off = buf[:, 8:].unflatten(1, (4, 64)), buf[:, 1:257].unflatten(1, (4, 64))
    _attn_call(q=aligned)
    assert on_cpu[-1][1][1] == aligned.data_ptr() and on_cpu[-1][1][7] == 264
    _attn_call(q=off)
    assert on_cpu[-1][1][1] != off.data_ptr() and on_cpu[-1][1][7] == 256


def _step_call(**kw):
    f = dict(q=torch.zeros(3, 4, 64), k_cache=torch.zeros(5, 16, 2, 64), v_cache=torch.zeros(5, 16, 2, 64),
             tables=torch.zeros(3, 7, dtype=I32), lengths=torch.zeros(3, dtype=I32))
    f.update(kw)
    args = [f.pop(n) for n in ("q", "k_cache", "v_cache", "tables", "lengths")]
    return attention.attention_step(*args, **f)


def test_step_checks(on_cpu):
    assert _step_call().shape == (3, 4, 64) and on_cpu[-1][0] == "pf_attn_step_exec"
    c = torch.zeros(5, 16, 2, 64)
    for match, kw in (("q must be", dict(q=c)), ("k_cache must be", dict(k_cache=c[0])), ("power of two", dict(k_cache=c[:, :8], v_cache=c[:, :8])),
                      ("v_cache has shape", dict(v_cache=c[:4])), ("k_cache has dtype", dict(k_cache=c.to(BF))),
                      ("heads of 32", dict(k_cache=c[..., :32], v_cache=c[..., :32])), ("unsupported shape", dict(q=torch.zeros(3, 5, 64))),
                      ("tables must be", dict(tables=None)), ("tables has dtype", dict(tables=torch.zeros(3, 7))),
                      ("state holds 2", dict(tables=torch.zeros(2, 7, dtype=I32))),
                      ("lengths has shape", dict(lengths=torch.zeros(2, dtype=I32))), ("lengths must be", dict(lengths=None)), ("slots has dtype", dict(slots=torch.zeros(3))),
                      ("whole 16-byte", dict(k_cache=torch.zeros(5, 16, 2, 65)[..., 1:])),
                      ("out may not be", dict(q=c[:3, 0, :].repeat(1, 2, 1), out=c[:3, :4, 0], v_cache=c))):
        with pytest.raises(ValueError, match=match):
            _step_call(**kw)
    big = torch.zeros(1, dtype=I32).expand(3, 1).contiguous()
    with pytest.raises(ValueError, match="up to"):
        attention._pool_state(torch.empty(3, (1 << 14) + 1, dtype=I32), torch.zeros(3, dtype=I32), big[:, 0], big[:1, 0], None, 65536,
                              torch.device("cpu"))


def test_pages_checks(on_cpu):
    def call(**kw):
        f = dict(tables=torch.zeros(3, 7, dtype=I32), lengths=torch.zeros(3, dtype=I32), tokens=torch.zeros(3, dtype=I32),
                 free=torch.zeros(9, dtype=I32), taken=torch.zeros(1, dtype=I32), page_size=16, capacity=20)
        f.update(kw)
        args = [f.pop(n) for n in ("tables", "lengths", "tokens", "free", "taken")]
        return attention.assign_pages(*args, **f)

    plan = call()
    assert plan.rows.shape == (20,) and plan.cu_seqlens.shape == (4,) and plan.lengths.shape == (3,) and plan.taken.shape == (1,)
    assert call(tokens=None, capacity=None).rows.shape == (3,)
    z = torch.zeros(3, dtype=I32)
    for match, kw in (("tables must be", dict(tables=z)), ("lengths must be", dict(lengths=None)), ("tokens has shape", dict(tokens=z[:2])),
                      ("free has dtype", dict(free=z.long())), ("taken has shape", dict(taken=z)), ("taken must be", dict(taken=None)), ("free must be", dict(free=None)), ("power of two", dict(page_size=48)),
                      ("capacity must be given", dict(capacity=None)), ("capacity must be 0", dict(capacity=-1)),
                      ("state holds 2", dict(tables=torch.zeros(2, 7, dtype=I32))), ("slots has shape", dict(slots=z[:2]))):
        with pytest.raises(ValueError, match=match):
            call(**kw)
    both = torch.zeros(30, dtype=I32)
    with pytest.raises(ValueError, match="tables may not be lengths"):
        call(tables=both[:21].view(3, 7), lengths=both[18:21])
    with pytest.raises(ValueError, match="free may not be tables"):
        attention.release_pages(both[:21].view(3, 7), z, both[15:], z[:1], page_size=16)


def test_store_checks(on_cpu):
    def call(**kw):
        f = dict(k=torch.zeros(4, 2, 64), v=torch.zeros(4, 2, 64), k_cache=torch.zeros(5, 16, 2, 64), v_cache=torch.zeros(5, 16, 2, 64),
                 rows=torch.zeros(4, dtype=torch.int64))
        f.update(kw)
        return attention.store_kv(*f.values())

    call()
    c = torch.zeros(5, 16, 2, 64)
    for match, kw in (("k must be", dict(k=c)), ("v has shape", dict(v=torch.zeros(3, 2, 64))), ("rows has dtype", dict(rows=torch.zeros(4, dtype=I32))),
                      ("rows has shape", dict(rows=torch.zeros(5, dtype=torch.int64))), ("rows must be", dict(rows=None)), ("v must be", dict(v=None)),
                      ("k_cache must be", dict(k_cache=None)), ("v_cache must be", dict(v_cache=None)), ("expected 2 of 64", dict(k_cache=c[:, :, :1], v_cache=c[:, :, :1])),
                      ("power of two", dict(k_cache=c[:, :12], v_cache=c[:, :12])), ("v_cache has shape", dict(v_cache=c[1:])),
                      ("k_cache may not be v_cache", dict(k_cache=c, v_cache=c)),
                      ("k_cache has overlapping rows", dict(k_cache=c[:, :1].expand(5, 16, 2, 64)))):
        with pytest.raises(ValueError, match=match):
            call(**kw)


@pytest.mark.parametrize("swap", [False, True])
def test_store_operands_that_share_memory(on_cpu, swap):
    n, rows = 2 * 16 * 2 * 64, torch.zeros(4, dtype=torch.int64)          # elements of a cache of two pages

    def call(at_k, at_v, at_first, at_second, rows=rows):
        """Operands at these elements of one buffer: keys and values are 4 tokens of 2 heads, 512 elements."""
        buf = torch.zeros(4 * n)
        k, v = (buf[at:at + 512].view(4, 2, 64) for at in (at_k, at_v))
        caches = [buf[at:at + n].view(2, 16, 2, 64) for at in (at_first, at_second)]
        return attention.store_kv(k, v, *(caches[::-1] if swap else caches), rows)

    for k, v, first, second in ((0, 512, 1024, 1024 + n), (0, n + 512, 512, n + 1024), (n, n + 512, 0, n + 1024),
                                (3 * n, 2 * n, 0, n), (0, 0, 512, 512 + n)):
        call(k, v, first, second)
    assert len(on_cpu) == 5
    for k, v, first, second in ((0, 511, 512, 512 + n), (1022, 0, 1024, 1024 + n), (n - 1, n + 511, 0, n + 1023), (n, n + 512, 0, n + 511),
                                (2 * n - 1, 3 * n, 0, n), (3 * n, 0, 0, n), (3 * n, 2 * n + 8, 0, n + 16), (3 * n, 3 * n, 0, n - 1)):
        with pytest.raises(ValueError, match="may not be"):
            call(k, v, first, second)
    # Views whose ends cross but whose elements do not: two halves of one cache's heads.
    both = torch.zeros(2, 16, 4, 64)
    call_views = lambda k, v: attention.store_kv(k, v, both[:, :, :2], both[:, :, 2:], rows)
    call_views(torch.zeros(4, 2, 64), torch.zeros(4, 2, 64))
    with pytest.raises(ValueError, match="k_cache may not be k"):
        call_views(both[0, :4, :2], torch.zeros(4, 2, 64))
    with pytest.raises(ValueError, match="v_cache may not be rows"):
        words = torch.zeros(2 * 16 * 2 * 64)
        attention.store_kv(torch.zeros(4, 2, 64), torch.zeros(4, 2, 64), torch.zeros(2, 16, 2, 64), words.view(2, 16, 2, 64),
                           words.view(torch.int64)[-4:])


def test_pages_by_hand():
    """The definitions that the device is held to, at sizes worked out by hand."""
    rows, cu, after, taken, tables = att.assign([[7, -1, -1], [-1] * 3, [5, 6, -1]], [15, 0, 32], [3, 2, 1], [0, 0, 0, 9, 4, 2], 3, 16, 7)
    assert tables == [[7, 9, -1], [4, -1, -1], [5, 6, 2]] and after == [18, 2, 33] and taken == 6 and cu == [0, 3, 5, 6]
    assert rows == [7 * 16 + 15, 9 * 16, 9 * 16 + 1, 4 * 16, 4 * 16 + 1, 2 * 16, -1]
    # one page left: the first that needs more lacks it, and no later one that needs any gets it
    rows, cu, after, taken, tables = att.assign([[-1] * 3, [-1] * 3, [1, -1, -1]], [0, 0, 3], [17, 4, 1], [9], 0, 16, 22)
    assert rows == [-1] * 21 + [19] and after == [0, 0, 4] and taken == 0
    assert att.release([[7, 9], [4, 0]], [18, 3], [0] * 6, 4, 16) == ([0, 4, 9, 7, 0, 0], 1)


@pytest.mark.parametrize("seed", range(4))
def test_plain_forms_agree_with_the_definitions(seed):
    """The reference's own two ways: a paged sequence is a prompt's last row."""
    gen = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(9, h, 16, generator=gen, dtype=torch.float64) for h in (4, 2, 2))
    whole, mag, size = att.attention(q, k, v)
    last, lmag, lsize = att.attention(q[8:], k, v, causal=False)
    for a, b in ((whole, last), (mag, lmag), (size, lsize)):
        assert torch.allclose(a[8:], b, atol=1e-14)
