"""CPU side of the drafted-token step: refusals of the four entry points (no kernel runs: every bad
argument is answered before a CUDA call), and known answers of the oracle the GPU tests use."""

import numpy as np
import pytest
import torch

from gemmagemini4hackathon2026_10_2425_b200 import _lib, ops
from oracle import ops as O

P = 1 << 20  # a non-NULL, 16-byte aligned address that nothing dereferences


def plan_args(**kw):
    a = dict(ctx=P, q=P, parents=None, table=P, mb=4, n_pages=P, stack=P, cap=8, n_free=P, B=2, R=8, words=0, cu=P,
             slots=P, pos=P, mask=None, status=P, npo=P, nfo=P)
    a.update(kw)
    return [*a.values(), None]


@pytest.mark.parametrize("name", ["ctx", "q", "table", "n_pages", "stack", "n_free", "cu", "slots", "pos", "status", "npo", "nfo"])
def test_plan_null(name):
    assert _lib.lib().b2d_paged_plan(*plan_args(**{name: None})) == _lib.ERR_NULL


@pytest.mark.parametrize("kw", [dict(B=0), dict(B=8193), dict(R=0), dict(R=(1 << 24) + 1), dict(mb=0), dict(mb=(1 << 17) + 1),
                                dict(cap=0), dict(words=1), dict(parents=P, mask=P), dict(parents=P, mask=P, words=9)])
def test_plan_shapes(kw):
    assert _lib.lib().b2d_paged_plan(*plan_args(**kw)) == _lib.ERR_SHAPE


def test_plan_mask_missing():
    assert _lib.lib().b2d_paged_plan(*plan_args(parents=P, words=1)) == _lib.ERR_NULL


def qk_args(**kw):
    a = dict(qkv=P, dt=0, ld=192, qg=None, kg=None, eps=1e-6, vn=0, pos=P, slots=P, nr=None, invf=P, out=P, odt=0, ldq=64,
             k=P, v=P, nb=1, hq=1, hk=1, hd=64, rows=1)
    a.update(kw)
    return [*a.values(), None]


@pytest.mark.parametrize("kw,status", [
    (dict(qkv=None), "NULL"), (dict(pos=None), "NULL"), (dict(invf=None), "NULL"), (dict(out=None), "NULL"),
    (dict(k=None), "NULL"), (dict(v=None), "NULL"),
    (dict(rows=0), "SHAPE"), (dict(hq=0), "SHAPE"), (dict(hk=0), "SHAPE"), (dict(nb=0), "SHAPE"), (dict(ld=188), "SHAPE"),
    (dict(ldq=60), "SHAPE"), (dict(hd=96), "UNSUPPORTED"), (dict(dt=2), "UNSUPPORTED"), (dict(odt=4), "UNSUPPORTED"),
    (dict(qkv=P + 8), "ALIGN"), (dict(out=P + 4), "ALIGN"), (dict(k=P + 2), "ALIGN"), (dict(qg=P + 4), "ALIGN"),
    (dict(ld=194), "ALIGN"), (dict(dt=1, ld=196), "ALIGN"), (dict(ldq=66), "ALIGN"),
])
def test_qk_refusals(kw, status):
    assert _lib.lib().b2d_qk_norm_rope_append(*qk_args(**kw)) == getattr(_lib, "ERR_" + status)


def attn_args(**kw):
    a = dict(q=P, dt=1, ldq=128, k=P, v=P, table=P, mb=4, nb=8, ctx=P, cu=P, mask=None, words=0, pos=None, hq=2, hk=1, hd=64,
             B=1, R=8, max_q=8, max_ctx=64, scale=0.0, window=0, out=P, odt=1, ldo=128, ws=None, wsb=0)
    a.update(kw)
    return [*a.values(), None]


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), "NULL"), (dict(k=None), "NULL"), (dict(v=None), "NULL"), (dict(table=None), "NULL"),
    (dict(ctx=None), "NULL"), (dict(cu=None), "NULL"), (dict(out=None), "NULL"), (dict(mask=P, words=1, window=4), "NULL"),
    (dict(B=0), "SHAPE"), (dict(B=65536), "SHAPE"), (dict(R=0), "SHAPE"), (dict(hq=3, hk=2), "SHAPE"), (dict(hq=0), "SHAPE"),
    (dict(max_q=0), "SHAPE"), (dict(max_ctx=0), "SHAPE"), (dict(max_q=65), "SHAPE"), (dict(max_ctx=65), "SHAPE"),
    (dict(nb=0), "SHAPE"), (dict(window=-1), "SHAPE"), (dict(words=1), "SHAPE"), (dict(mask=P), "SHAPE"),
    (dict(mask=P, words=9), "SHAPE"), (dict(ldq=120), "SHAPE"), (dict(ldo=120), "SHAPE"), (dict(hq=130, hk=2), "SHAPE"),
    (dict(hd=80), "UNSUPPORTED"), (dict(dt=4), "UNSUPPORTED"), (dict(odt=3), "UNSUPPORTED"),
    (dict(q=P + 2), "ALIGN"), (dict(out=P + 8), "ALIGN"), (dict(k=P + 2), "ALIGN"), (dict(ldq=132), "ALIGN"), (dict(ldo=132), "ALIGN"),
    (dict(nb=1 << 30), "SHAPE"),
])
def test_attn_refusals(kw, status):
    assert _lib.lib().b2d_paged_tree_attn(*attn_args(**kw)) == getattr(_lib, "ERR_" + status)


def test_attn_workspace_is_asked_for():
    lib = _lib.lib()
    need = lib.b2d_paged_tree_attn_workspace_bytes(1, 8, 2, 1, 64, 8, 65536)
    assert need > 0
    big = dict(max_ctx=65536, mb=4096)
    assert lib.b2d_paged_tree_attn(*attn_args(**big)) == _lib.ERR_WORKSPACE
    assert lib.b2d_paged_tree_attn(*attn_args(**big, ws=P, wsb=need - 1)) == _lib.ERR_WORKSPACE
    assert lib.b2d_paged_tree_attn(*attn_args(**big, ws=P + 4, wsb=need)) == _lib.ERR_ALIGN
    assert lib.b2d_paged_tree_attn_workspace_bytes(0, 8, 2, 1, 64, 8, 64) == 0


def score_args(**kw):
    a = dict(x=P, dt=0, ld=100, V=100, R=1, nr=None, t=P, nt=1, k=1, lp=P, ent=P, ids=P, tlp=P)
    a.update(kw)
    return [*a.values(), None]


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), "NULL"), (dict(t=None), "NULL"), (dict(lp=None), "NULL"), (dict(ids=None), "NULL"), (dict(tlp=None), "NULL"),
    (dict(R=0), "SHAPE"), (dict(V=0), "SHAPE"), (dict(ld=99), "SHAPE"), (dict(k=33), "SHAPE"), (dict(k=-1), "SHAPE"),
    (dict(nt=-1), "SHAPE"), (dict(V=20, k=21), "SHAPE"), (dict(dt=4), "UNSUPPORTED"), (dict(x=P + 2), "ALIGN"),
    (dict(dt=1, x=P + 1), "ALIGN"),
])
def test_score_refusals(kw, status):
    assert _lib.lib().b2d_token_logprobs(*score_args(**kw)) == getattr(_lib, "ERR_" + status)


def test_python_entry_points_refuse_cpu_tensors():
    i = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    pages = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        ops.paged_plan(i(2), i(2), i(2, 4), i(2), i(8), i(1), 8)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_append(torch.zeros(1, 192), i(1), i(1).long(), torch.zeros(32), pages, pages, 1, 1, 64)
    with pytest.raises(ValueError):
        ops.paged_tree_attn(torch.zeros(1, 64), pages, pages, i(1, 2), i(1), i(2), 1, 1, 64, 1, 32)
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.zeros(1, 10))


def test_oracle_plan_known_answer():
    """Two requests and an ended one: 3 pages are released, 2 taken from the stack's end."""
    r = O.paged_plan(
        np.array([15, 40, 16]), np.array([2, -1, 1]), np.array([[7, -1], [4, 5], [9, -1]], np.int32),
        np.array([1, 2, 1]), np.array([1, 0, 0, 0], np.int32), 1, 5,
    )
    assert r["stack"].tolist() == [1, 4, 5, 0] and r["n_free"].tolist() == [1]
    assert r["table"].tolist() == [[7, 5], [4, 5], [9, 4]]
    assert r["cu_q"].tolist() == [0, 2, 2, 3] and r["n_pages"].tolist() == [2, 0, 2]
    assert r["slots"].tolist() == [7 * 16 + 15, 5 * 16, 4 * 16, -9, -9]


def test_oracle_tree_known_answer():
    bits, depth = O.tree_bits([-1, 0, 0, 1, -1, 9])
    assert depth.tolist() == [0, 1, 1, 2, 0, 0]
    assert O.pack_bits(bits, 1)[:, 0].tolist() == [1, 3, 5, 11, 16, 32]


def test_oracle_logprobs_known_answer():
    tl, ent, ids, tlp = O.token_logprobs(np.array([[0.0, 0.0, -np.inf, 0.0]]), np.array([[1, 2, 9]]), 3)
    np.testing.assert_allclose(tl, [[-np.log(3), -np.inf, -np.inf]])
    np.testing.assert_allclose(ent, [np.log(3)])
    assert ids.tolist() == [[0, 1, 3]]
