"""Refusals of the entry point that marks requests which hold tokens, without a GPU: statuses, the struct's size, Python's checks."""
import subprocess

import pytest
import torch

from pto_fuser_amd import _build, _hip, attention
from pto_fuser_amd.attention import PagePlan
from test_attention_host import lib, on_cpu  # noqa: F401

I32 = torch.int32


def test_struct_size_is_the_header_s(tmp_path):
    src = tmp_path / "size.c"
    src.write_text('#include <stdio.h>\n#include "pto_fuser_hip.h"\nint main(void) { printf("%zu", sizeof(pf_refuse_args)); return 0; }\n')
    subprocess.run(["gcc", "-I", _build.INCLUDE, str(src), "-o", str(tmp_path / "size")], check=True)
    out = subprocess.run([str(tmp_path / "size")], capture_output=True, text=True, check=True).stdout
    assert int(out) == attention._REFUSE_SIZE


def _refuse(**kw):
    f = dict(size=attention._REFUSE_SIZE, cu=64, lengths=64, rows=64, k=64, k_t=64, k_h=64, N=4, B=2, G=2, dtype=1)
    assert not set(kw) - set(f)
    return attention._REFUSE.pack(*{**f, **kw}.values())


@pytest.mark.parametrize("bad", [dict(size=8), dict(cu=0), dict(lengths=0), dict(rows=0), dict(k=0), dict(k_t=-1), dict(k_h=-8),
                                 dict(N=-1), dict(B=-1), dict(B=2 ** 31 - 1), dict(G=0), dict(G=1 << 17), dict(dtype=2)])
def test_statuses(lib, bad):  # noqa: F811
    assert lib.pf_refuse_exec(_refuse(**bad), None) == _hip.PF_ERR_ARG


def test_empty_calls_launch_nothing(lib):  # noqa: F811
    assert lib.pf_refuse_exec(_refuse(N=0, k=0, rows=0), None) == _hip.PF_OK
    assert lib.pf_refuse_exec(_refuse(B=0, lengths=0), None) == _hip.PF_OK
    assert lib.pf_refuse_exec(None, None) == _hip.PF_ERR_ARG


def test_checks(on_cpu):  # noqa: F811
    k = torch.zeros(10, 2, 64)
    plan = PagePlan(torch.zeros(10, dtype=torch.int64), torch.zeros(4, dtype=I32), torch.zeros(3, dtype=I32), torch.zeros(1, dtype=I32))
    attention.refuse_held(k, plan)
    assert on_cpu[-1][0] == "pf_refuse_exec" and on_cpu[-1][1][5:] == (128, 64, 10, 3, 2, 0)
    for match, key, new in (("k must be", k[0], plan), ("rows has shape", k[:9], plan), ("contiguous along", k.transpose(1, 2), plan),
                            ("rows must be", k, plan._replace(rows=None)), ("cu_seqlens has shape", k, plan._replace(cu_seqlens=plan.cu_seqlens[:3])),
                            ("lengths must be", k, plan._replace(lengths=None)), ("lengths has dtype", k, plan._replace(lengths=torch.zeros(3))),
                            ("k may not be rows", k.view(-1)[:640].view(10, 1, 64), plan._replace(rows=k.view(-1).view(torch.int64)[:10]))):
        with pytest.raises(ValueError, match=match):
            attention.refuse_held(key, new)
