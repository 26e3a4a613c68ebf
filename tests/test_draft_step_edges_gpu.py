"""The drafted-token step's operators at the edges of their ranges: finite bans and large logits,
non-finite values in hidden places, weak keys beside a strong one, large scores, refused requests.
Helpers and the oracle's tolerances are test_draft_step_gpu.py's."""

import numpy as np
import pytest
import torch

from gemmagemini4hackathon2026_10_2425_b200 import _lib, ops
from oracle import ops as O
from test_draft_step_gpu import (
    DEV, E16, E32, TINY16, attn_bound, attn_case, check_attn, check_plan, check_qk, check_score, gpu, i32, qk_case, run_attn,
    run_plan, same, tree_clean,
)

pytestmark = pytest.mark.gpu

# -- token_logprobs -----------------------------------------------------------------------------

BANS = [-1e4, -1.6e7, -(2.0**24), -2.0e7, -1e9, -2e9, -1e10, -1e12, -1e20, -1e30, -3e38]


def logits(R, V, seed=0):
    return 3 * torch.randn(R, V, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def score_targets(R, V):
    return np.tile([0, V // 2, V - 1], (R, 1))


@pytest.mark.parametrize("V,copies", [(1000, 1), (128256, 1), (9001, 30)])
def test_score_finite_bans(V, copies):
    """Tokens banned with a finite constant, most of a row and all of it, one CTA (300 rows) and eight per row."""
    part = logits(len(BANS) * copies, V)
    for i in range(len(part)):
        part[i, : 9 * V // 10] = BANS[i % len(BANS)]
    check_score(part, score_targets(len(part), V), 20)
    part[:, 9 * V // 10 :] = part[:, :1]
    check_score(part, score_targets(len(part), V), 20)


@pytest.mark.parametrize("V,copies", [(1000, 1), (128256, 1), (9001, 40)])
def test_score_large_logits(V, copies):
    """A single large logit, two of them, and rows of nothing else."""
    big = [1.6e7, 2.0**24, 2.1e7, 2e9, 1e10, 1e20, 1e30, 2.5e38]
    x = logits(len(big) * copies, V, 1)
    for i in range(len(x)):
        x[i, V // 2] = big[i % len(big)]
    check_score(x, score_targets(len(x), V), 7)
    x[:, V - 1] = x[:, V // 2]
    check_score(x, score_targets(len(x), V), 7)
    for s in (-1, 1):
        y = s * torch.tensor(big * copies, device=DEV)[:, None] * (1 + 0.1 * logits(len(big) * copies, V, 2).abs().clamp(max=5))
        check_score(y.clamp(-3e38, 3e38), score_targets(len(y), V), 7)


def test_score_around_the_floor():
    """Rows whose maximum lies near -2^24, the smallest value that counts as itself in the sums."""
    x = torch.full((6, 5000), -(2.0**24) - 64, device=DEV)
    for i, m in enumerate([-300, 0, 100, 254, 258, 1000]):
        x[i, 17] = -(2.0**24) + m
        x[i, 99] = -(2.0**24) + m - 2
    check_score(x, score_targets(6, 5000), 5)


# -- paged_tree_attn ----------------------------------------------------------------------------


def spoil(c, b, places, part, fill, heads=slice(None)):
    for j in places:
        c[part][c["table"][b, j // 16], heads, j % 16, 5] = fill


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("fill", [np.nan, np.inf])
def test_attn_hidden_rows_of_many_tiles(hd, fill):
    """Every tile of a wide tree holds places that some rows must not see, and in most of them v (every
    other tile: none, one or several rows) is not finite."""
    for T, ctx in ((256, 40), (200, 0)):
        c = attn_case(hd + T, [ctx, 9], [T, 3], 4, 2, hd, True)
        for tile in (0, 1, 3):
            spoil(c, 0, ctx + 64 * tile + np.arange(5, 5 + 3 * (tile + 1), 3), "vp", fill, tile % 2)
        spoil(c, 0, [ctx + 130], "kp", fill)
        check_attn(c, torch.float16)
        check_attn(c, torch.float32)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attn_window_of_many_tiles(hd):
    """Chunks whose window cuts through every tile that they read; what left it, and every page's unused
    part, is not finite."""
    for window in (30, 200):
        c = attn_case(hd + window, [700, 90], [150, 70], 4, 2, hd, False)
        spoil(c, 0, range(700 - window), "vp", np.inf)
        spoil(c, 0, range(700 - window), "kp", np.nan)
        spoil(c, 0, [701, 790, 840], "vp", np.nan, 1)
        check_attn(c, torch.float16, window=window)
        check_attn(c, torch.float32, window=window)


def check_exact_scores(c, out_dtype, scale, lost=0.0, got=None):
    """Rows whose scores are exact in fp32 and the largest of a row's far weights 2^-64 or nothing.  A weight
    is off by the roundings of z = (s - m) c, |z| <= 64: the difference, the product and c, 2^-24 each (times
    ln 2), and the exponential's 2^-22; then by E16 where it is an fp16 number, 2^-21 as two; `lost` is what
    places of small weight may lose.  Sums over n places: one step per 16."""
    hq, hk, hd = c["dims"]
    got = run_attn(c, out_dtype, scale=scale) if got is None else got
    got = got.float().cpu().numpy().astype(np.float64).reshape(-1, hq, hd)
    want, mag = O.tree_attention(c["q"], c["kp"], c["vp"], c["table"], c["ctx"], c["cu"], hq, hk, hd, c["bits"], c["pos"], scale)
    fp16, out16 = c["q"].dtype == np.float16 and out_dtype == torch.float16, out_dtype == torch.float16
    err_p = 3 * 64 * E32 * 0.7 + 2.0**-22 + (E16 if fp16 else 2.0**-21)
    lim = (2 * err_p + (c["max_ctx"] / 16 + 8) * 2.0**-23) * mag + (E16 if out16 else 4 * E32) * np.abs(want) + (TINY16 if out16 else 0)
    lim = lim + lost
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    err = np.abs(got - want)
    assert np.all((err <= lim)[ok]), (np.max((err / lim)[ok]), np.argwhere(~(err <= lim) & ok)[:4])
    tree_clean()


@pytest.mark.parametrize("hd,T", [(64, 3), (64, 40), (128, 5), (128, 70), (256, 4)])
@pytest.mark.parametrize("dt", [np.float16, np.float32])
def test_attn_large_scores(hd, T, dt):
    """Scores of one large number and small multiples of its last places: +-2^e + d u, u = 2^max(0, e - 21),
    d in 0 .. 15, exact in fp32.  Up to 2^22 the weights differ by less than e^15; beyond, the scale brings
    the differences to that, or leaves the rows with the largest (one or several) alone."""
    r = np.random.default_rng(hd + T)
    c = attn_case(hd + T, [900, 3, 2000], [T, 2, 1], 4, 2, hd, False, dt=dt)
    c["vp"] = np.nan_to_num(c["vp"])
    for e, sign, scale in [(12, 1, 1.0), (20, -1, 0.7), (22, 1, 1.0), (22, -1, 0.9), (25, 1, 0.06), (28, -1, 0.007), (30, 1, 0.0019),
                           (25, 1, 1.0), (29, -1, 0.3), (30, 1, 0.77), (30, -1, 53.0)]:
        a = (e + 1) // 2
        q = np.zeros((c["R"], 4, hd))
        q[..., 3], q[..., 40] = sign * 2.0**a, 2.0 ** max(0, e - 21)
        c["q"] = q.reshape(c["R"], -1).astype(dt)
        c["kp"][:] = 0
        c["kp"][..., 3] = 2.0 ** (e - a)
        c["kp"][..., 40] = r.integers(0, 16, c["kp"].shape[:-1])
        for out in (torch.float16, torch.float32):
            check_exact_scores(c, out, scale)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attn_scores_that_grow(hd):
    """The running maximum passes from small scores to ones past 2^22 and on, within one CTA and over several
    (to 2^27 for 2300 places; 2500 end in an infinite key, whose rows are NaN)."""
    for ctx, q in (([2300], [9]), ([2500], [9]), ([700] * 80, [1] * 80)):
        c = attn_case(hd, ctx, q, 2, 1, hd, False)
        c["vp"] = np.nan_to_num(c["vp"])
        n = int(c["ctx"][0])
        c["q"] = np.zeros((c["R"], 2, hd), np.float16)
        c["q"][:, 0, 1], c["q"][:, 1, 1] = 2.0**12, -(2.0**12)
        c["q"] = c["q"].reshape(c["R"], -1)
        c["kp"][:] = 0
        for b in range(len(ctx)):
            for j in range(n + q[b]):
                c["kp"][c["table"][b, j // 16], :, j % 16, 1] = 2.0 ** (j // 100 - 8) if j % 100 == 7 else 0
        for scale in (1.0, 30.0):
            check_exact_scores(c, torch.float16, scale)
            check_exact_scores(c, torch.float32, scale)


@pytest.mark.parametrize("hd,T,dt,out", [(64, 1, np.float32, torch.float32), (64, 1, np.float16, torch.float16), (128, 1, np.float32, torch.float16),
                                         (64, 70, np.float16, torch.float16), (128, 70, np.float16, torch.float16),
                                         (256, 1, np.float32, torch.float32), (256, 2, np.float16, torch.float16)])
def test_attn_weak_keys_beside_a_strong_one(hd, T, dt, out):
    """One key 8 to 21 above thousands of others, whose values alone make the output: their weights are small
    numbers of fp16 (or of fp16 pairs), none of which may be lost.  A weight is off by 2^-25 at most where
    fp16 has no smaller step, and the row's largest weight is 2^7 or more: 2^-32 of |v| per place.  More
    sequences than SMs (of the same pages), so that a CTA sees the strong key and many others."""
    B, ctx = 160, 8191 if T > 2 else 32767
    r = np.random.default_rng(hd + T)
    c = attn_case(hd, [ctx], [T], 2, 1, hd, False, dt=dt)
    at = lambda j: (c["table"][0, j // 16], slice(None), j % 16)  # noqa: E731
    c["kp"][:], c["vp"][:] = 0, np.abs(r.standard_normal(c["vp"].shape))
    c["kp"][..., 1] = r.integers(-8, 9, c["kp"].shape[:-1]) / 16
    c["kp"][at(100)], c["vp"][at(100)] = 0, 0
    c["kp"][at(100)][..., 0] = 16
    strong = np.linspace(8, 21, B * T * 2).reshape(-1, 2)
    q = np.zeros((B * T, 2, hd))
    q[..., 0], q[..., 1] = strong * hd**0.5 / 16, hd**0.5
    few = [0, B // 2, B - 1]
    for name, n in (("many", B), ("few", len(few))):
        c[name] = dict(c, table=np.repeat(c["table"], n, 0), ctx=np.repeat(c["ctx"], n), cu=(np.arange(n + 1) * T).astype(np.int32),
                       pos=np.tile(c["pos"], n), R=n * T)
    c["many"]["q"] = q.reshape(B * T, -1).astype(dt)
    c["few"]["q"] = np.concatenate([c["many"]["q"][b * T : (b + 1) * T] for b in few])
    got = run_attn(c["many"], out)
    got = torch.cat([got[b * T : (b + 1) * T] for b in few])
    check_exact_scores(c["few"], out, 0.0, lost=c["vp"].astype(np.float64).sum((0, 2)).max() * 2.0**-32, got=got)


# -- refused requests -----------------------------------------------------------------------------


def test_plan_refused_rows_have_no_stale_pages():
    """Table rows that still name an earlier request's pages: a refused request's places there have none,
    whatever it was refused for; served and ended requests keep theirs."""
    stale = np.arange(50, 50 + 7 * 8, dtype=np.int32).reshape(7, 8)
    c = dict(ctx=np.array([20, 100, -3, 5, 10, 0, 3]), q=np.array([30, 60, 2, 40, 1, -1, 90]), table=stale, n_pages=np.array([2, 3, 0, 1, 1, 0, 0]),
             stack=np.arange(200, 230, dtype=np.int32), n_free=1, R=140, parents=np.full(140, -1, np.int32), words=1)
    w = check_plan(c)
    assert w["status"].tolist() == [_lib.PLAN_PAGES, _lib.PLAN_TABLE, _lib.PLAN_TABLE, _lib.PLAN_TREE, 0, 0, _lib.PLAN_ROWS]
    assert w["table"][0].tolist() == [50, 51, -1, -1, 54, 55, 56, 57] and w["table"][1, 3:].tolist() == [-1] * 5
    assert w["table"][3, 1:4].tolist() == [-1, -1, 77] and w["table"][6, 0] == -1
    for b in (2, 4, 5):
        assert w["table"][b].tolist() == stale[b].tolist()
    c["words"], c["parents"] = 0, None
    check_plan(c)


def test_refused_rows_see_no_other_request():
    """A slot whose table row still holds an ended request's pages, given to a request that is refused: its
    rows attend to nothing there (the pages hold NaN), the served request beside it is untouched."""
    hq, hk, hd = 4, 2, 64
    table = np.array([[3, 4, 5, 6], [0, 1, -1, -1]], np.int32)
    c = dict(ctx=np.array([0, 20]), q=np.array([40, 5]), table=table, n_pages=np.array([0, 2]), stack=np.zeros(4, np.int32), n_free=0, R=45,
             parents=None, words=0)
    plan, dev = run_plan(c)
    same(plan.status, [_lib.PLAN_PAGES, 0])
    a = attn_case(5, [20], [5], hq, hk, hd, False)
    kp = torch.full((8, hk, 16, hd), float("nan"), dtype=torch.float16, device=DEV)
    vp = kp.clone()
    for src, dst in ((a["kp"], kp), (a["vp"], vp)):
        dst[:2] = gpu(src)[gpu(a["table"][0]).long()]
    q = torch.randn(45, hq * hd, device=DEV)
    q[40:] = gpu(a["q"])
    got = ops.paged_tree_attn(q, kp, vp, dev["table"], i32(c["ctx"]), plan.cu_q, hq, hk, hd, 40, 64)
    assert got[:40].eq(0).all()
    a["q"] = a["q"].astype(np.float32)
    want, mag = O.tree_attention(a["q"], a["kp"], a["vp"], a["table"], a["ctx"], a["cu"], hq, hk, hd)
    assert np.all(np.abs(got[40:].cpu().numpy().reshape(want.shape) - want) <= attn_bound(a, want, mag, False, False, 0))


# -- buffers that overlap, or lie close together ----------------------------------------------------


def test_qk_rows_of_q_out_between_rows_of_qkv():
    hq, hk, hd, R = 6, 2, 64, 21
    c, n = qk_case(2, R, hq, hk, hd, np.float16), (hq + 2 * hk) * hd
    wide = torch.zeros(R, n + hq * hd, dtype=torch.float16, device=DEV)
    wide[:, :n] = gpu(c["x"])
    check_qk(c, torch.float16, x_dev=wide[:, :n], q_out=wide[:, n:])
    same(wide[:, :n], c["x"])
    for q_out in (wide[:, 8 : hq * hd + 8], wide[:, n - 8 : -8]):
        with pytest.raises(ValueError, match="overlap"):
            check_qk(c, torch.float16, x_dev=wide[:, :n], q_out=q_out)
    one = gpu(c["x"])[:1].contiguous()  # a single row in place
    c.update({k: c[k][:1] for k in ("x", "pos", "slots")})
    check_qk(c, torch.float16, x_dev=one, q_out=one[:, : hq * hd])


def test_attn_rows_of_out_between_rows_of_q():
    hq, hk, hd = 8, 2, 64
    c = attn_case(10, [50, 20], [6, 2], hq, hk, hd, True)
    want = run_attn(c, torch.float16)
    wide = torch.zeros(c["R"], 2 * hq * hd, dtype=torch.float16, device=DEV)
    wide[:, : hq * hd] = gpu(c["q"])
    run_attn(c, q=wide[:, : hq * hd], out=wide[:, hq * hd :])
    assert torch.equal(wide[:, hq * hd :], want) and torch.equal(wide[:, : hq * hd], gpu(c["q"]))
    for out in (wide[:, : hq * hd], wide[:, 64 : hq * hd + 64], wide[:, hq * hd - 8 : -8]):
        with pytest.raises(ValueError, match="overlap"):
            run_attn(c, q=wide[:, : hq * hd], out=out)


# -- nothing to do ------------------------------------------------------------------------------------


def test_empty_batches_and_rows():
    """No requests, or no rows: every call returns, outputs of the sizes asked for, buffers untouched."""
    z = lambda *n, t=torch.int32: torch.zeros(*n, dtype=t, device=DEV)  # noqa: E731
    kp, vp = z(3, 2, 16, 64, t=torch.float16), z(3, 2, 16, 64, t=torch.float16)
    stack, n_free = i32([4, 5, 6]), i32([2])
    p = ops.paged_plan(z(0), z(0), z(0, 7), z(0), stack, n_free, 5)
    assert p.cu_q.tolist() == [0] and p.n_free.tolist() == [2] and p.status.numel() == 0 and p.slots.shape == (5,)
    p = ops.paged_plan(z(0), z(0), z(0, 7), z(0), stack, n_free, 5, out=ops.PagedPlan(p.cu_q.fill_(9), p.slots, p.positions, None, z(0), z(0), n_free))
    assert p.cu_q.tolist() == [0] and n_free.tolist() == [2] and stack.tolist() == [4, 5, 6]
    with pytest.raises(ValueError, match="max_tokens"):
        ops.paged_plan(z(2), z(2), z(2, 7), z(2), stack, n_free, 0)
    out = torch.full((5, 256), 3.0, device=DEV)
    for rows in (5, 0):
        got = ops.paged_tree_attn(z(rows, 256, t=torch.float32), kp, vp, z(0, 7), z(0), z(1), 4, 2, 64, 2, 32, out=out[:rows])
        assert got.shape == (rows, 256)
    assert out.eq(3).all()
    assert ops.qk_norm_rope_append(z(0, 512, t=torch.float32), z(0), z(0, t=torch.int64), z(32, t=torch.float32), kp, vp, 4, 2, 64).shape == (0, 256)
    assert ops.token_logprobs(z(0, 50, t=torch.float32), z(0), 3).top_ids.shape == (0, 3)


# -- arguments that the C interface cannot carry -----------------------------------------------------------


def test_integers_and_strides_past_32_bits_are_refused():
    """ctypes keeps the low 32 bits of an int: window = 2^32 + 5 would have been 5, a row stride another row."""
    c = attn_case(1, [20], [3], 4, 2, 64, True)
    for kw in (dict(window=2**32 + 5), dict(max_q=2**32 + 3), dict(max_ctx=2**32 + 23)):
        with pytest.raises(ValueError, match="32 bits"):
            run_attn(c, **kw)
    x = logits(2, 100)
    with pytest.raises(ValueError, match="32 bits"):
        ops.token_logprobs(x, None, 2**32 + 3)
    z = lambda *n: torch.zeros(*n, dtype=torch.int32, device=DEV)  # noqa: E731
    with pytest.raises(ValueError, match="32 bits"):
        ops.paged_plan(z(1), z(1), z(1, 2), z(1), z(4), z(1), 2, parents=z(2), mask_words=2**32 + 1)
    wide = torch.empty(2**32 + 8192, dtype=torch.float16, device=DEV)
    far = wide.as_strided((2, 256), (2**32 + 4096, 1))
    far.copy_(gpu(attn_case(2, [9], [2], 4, 2, 64, False)["q"]))
    a = attn_case(2, [9], [2], 4, 2, 64, False)
    with pytest.raises(ValueError, match="32 bits"):
        run_attn(a, q=far)
    with pytest.raises(ValueError, match="32 bits"):
        run_attn(a, out=far)
    q = qk_case(3, 2, 2, 1, 64, np.float16)
    for kw in (dict(x_dev=far), dict(x_dev=gpu(q["x"]), q_out=far[:, :128])):
        with pytest.raises(ValueError, match="32 bits"):
            check_qk(q, torch.float16, **kw)
    check_score(far, np.zeros((2, 1), int), 3)  # this one takes 64 bits


def test_a_single_row_of_any_stride():
    """One row's stride says nothing, whatever it is."""
    a = attn_case(2, [9], [1], 4, 2, 64, False)
    row = gpu(a["q"]).as_strided((1, 256), (3, 1))
    assert torch.equal(run_attn(a, q=row), run_attn(a))
    q = qk_case(3, 1, 2, 1, 64, np.float16)
    check_qk(q, torch.float16, x_dev=gpu(q["x"]).as_strided((1, 256), (5, 1)))


def test_tables_and_masks_without_two_dimensions_are_refused():
    c = attn_case(1, [20], [3], 4, 2, 64, True)
    z = lambda *n: torch.zeros(*n, dtype=torch.int32, device=DEV)  # noqa: E731
    with pytest.raises(ValueError):
        run_attn(dict(c, table=c["table"][:, 0]))
    with pytest.raises(ValueError):
        run_attn(c, mask=gpu(c["mask"])[:, 0].contiguous())
    with pytest.raises(ValueError):
        run_attn(c, q=gpu(c["q"])[0])
    with pytest.raises(ValueError):
        ops.paged_plan(z(3), z(3), z(3), z(3), z(4), z(1), 2)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_append(torch.zeros((), device=DEV), z(1), z(1).long(), torch.zeros(32, device=DEV), gpu(c["kp"]), gpu(c["vp"]), 4, 2, 64)
