"""Single tokens on both sides of the bounds between a workgroup a row and a walk that is shared out: the tables' width, and
the number of rows (sequences times heads of keys times blocks of 16 query heads).  Which one a call takes shows in its workspace."""
import pytest
import torch

from conftest import announce
from pto_fuser_amd import _build, _hip, attention_step
from test_gpu_attention import BF, DEV, F32, _check_step, _ints, _paged, _rand

CODE = {BF: _hip.PF_DTYPE_BF16, F32: _hip.PF_DTYPE_F32}


def _shared(B, H, G, D, tokens, dtype, page=16):
    _build.ensure_built()
    return _hip.load().pf_attn_step_workspace_bytes(B, H, G, D, tokens // page, page, CODE[dtype]) > 0


@pytest.mark.parametrize("dtype,least", [(BF, 256), (F32, 128)])
@pytest.mark.parametrize("D,rows", [(64, 256), (80, 128), (128, 128), (256, 64)])
def test_which_walks_are_shared(dtype, least, D, rows):
    """Few rows from a few hundred tokens on, a table of exactly 512 as one of 528; many rows past 512 tokens only."""
    for B, H, G in ((1, 4, 4), (rows // 4, 4, 4), (rows // 8, 68, 4)):
        assert not _shared(B, H, G, D, least, dtype) and _shared(B, H, G, D, least + 16, dtype)
    assert _shared(1, 4, 4, D, 512, dtype) and _shared(1, 4, 4, D, 528, dtype)
    assert _shared(rows, 1, 1, D, 512, dtype) and not _shared(rows + 1, 1, 1, D, 512, dtype) and _shared(rows + 1, 1, 1, D, 528, dtype)
    assert _shared(rows // 2, 17, 1, D, 512, dtype) and not _shared(rows // 2 + 1, 17, 1, D, 512, dtype)      # two blocks a row


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,G,D", [(4, 2, 64), (4, 4, 128), (20, 1, 80), (2, 1, 256)])
@pytest.mark.parametrize("tokens", [112, 128, 144, 240, 256, 272, 496, 512, 528])
def test_rows_of_every_width(dtype, H, G, D, tokens):
    """Tables that end where their longest row does, beside rows of none, one and a few tokens."""
    announce(f"attention_step {dtype} H{H} G{G} D{D} tables of {tokens} shared={_shared(5, H, G, D, tokens, dtype)}")
    lens = [tokens, 0, 1, tokens - 15, 63]
    (k, v), tables, rows = _paged(lens, G, D, 16, dtype, tokens + D)
    tables = tables[:, :tokens // 16].contiguous()
    q = _rand(D)(len(lens), H, D).to(DEV, dtype)
    _check_step(attention_step(q, k, v, tables, _ints(lens)), q, rows, lens, "o")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B", [63, 64, 65])
def test_numbers_of_rows(dtype, B):
    """At the largest number of rows that is shared, below it and above, 512 tokens."""
    announce(f"attention_step {dtype} B{B} shared={_shared(B, 4, 2, 128, 512, dtype)}")
    assert _shared(B, 4, 2, 128, 512, dtype) == (B <= 64)
    lens = [(512, 300, 0, 17, 511)[b % 5] for b in range(B)]
    (k, v), tables, rows = _paged(lens, 2, 128, 16, dtype, B)
    tables = tables[:, :32].contiguous()
    q = _rand(B)(B, 4, 128).to(DEV, dtype)
    _check_step(attention_step(q, k, v, tables, _ints(lens)), q, rows, lens, "o")
