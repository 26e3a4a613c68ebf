"""Refusals of the drafted-token step's entry points that need no GPU: every call here is answered before a
CUDA call (the addresses are never dereferenced)."""

import pytest

from gemmagemini4hackathon2026_10_2425_b200 import _lib
from test_draft_step import P, attn_args, qk_args

WS = dict(ws=P, wsb=1 << 40)


@pytest.mark.parametrize("kw", [
    dict(),  # out is q
    dict(out=P + 128, ldo=128),  # half a row further on
    dict(out=P + 7 * 256 + 240, ldo=136),  # q's last row
    dict(q=P + 8 * 256 - 16),  # out's last row
    dict(q=P + 8 * 512 - 16, odt=0),  # out is fp32
    dict(q=P + 2 * 8 * 256 - 16, odt=4),  # out's lo plane
    dict(q=P + 256, ldq=256, ldo=256 + 8),  # rows between q's at first, not to the end
])
def test_attn_out_shares_memory_with_q(kw):
    assert _lib.lib().b2d_paged_tree_attn(*attn_args(**WS, **kw)) == _lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("kw", [
    dict(ldq=64),  # qkv itself, its rows closer together
    dict(odt=1, ldq=384),  # another type
    dict(out=P + 256, ldq=192),  # k's place
    dict(out=P + 3 * 768 - 16, ldq=192),  # the last row's v
    dict(qkv=P + 2 * 768 + 256 - 16, ldq=192),  # out's last row
])
def test_qk_out_shares_memory_with_qkv(kw):
    assert _lib.lib().b2d_qk_norm_rope_append(*qk_args(rows=3, **kw)) == _lib.ERR_UNSUPPORTED
