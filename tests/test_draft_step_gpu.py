"""The drafted-token step's operators against the 64-bit oracle: page plan (exact), Q/K norm + rotation
+ append, tree attention, token log probabilities, and a run of them together.

Tolerances are bounds on the kernels' own roundings, written where they are used: eps32 = 2^-24 and
eps16 = 2^-11 are half a step of fp32 and fp16, relative to the value.
"""

import numpy as np
import pytest
import torch

from gemmagemini4hackathon2026_10_2425_b200 import _lib, ops
from oracle import ops as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
E32, E16 = 2.0**-24, 2.0**-11
TINY16 = 2.0**-25  # half a step of the smallest fp16 numbers


def gpu(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV, dtype)


def i32(a):
    return gpu(np.asarray(a, np.int32))


def same(got, want, what=""):
    np.testing.assert_array_equal(got.cpu().numpy(), want, err_msg=what)


# -- paged_plan ---------------------------------------------------------------------------------


def plan_case(seed, B, ctx_hi, q_hi, ended=0.1, spare=8, words=0, short=False):
    r = np.random.default_rng(seed)
    ctx, q = r.integers(0, ctx_hi + 1, B), r.integers(0, q_hi + 1, B)
    q[r.random(B) < ended] = -1
    have = -(-ctx // 16) + r.integers(0, 2, B)
    mb = int((ctx + q_hi).max()) // 16 + 2
    need = int(np.where(q >= 0, np.maximum(0, -(-(ctx + q) // 16) - have), 0).sum())
    free = need // 2 if short else need + spare
    ids = r.permutation(int(have.sum()) + free).astype(np.int32)
    table = np.full((B, mb), -1, np.int32)
    table[np.arange(mb)[None] < have[:, None]] = ids[: have.sum()]
    stack = np.full(free + int(have.sum()) + 1, -1, np.int32)
    stack[:free] = ids[have.sum() :]
    R = int(np.maximum(q, 0).sum()) + 3
    par = np.concatenate([np.concatenate([r.integers(-1, max(1, i), 1) for i in range(max(0, k))] or [np.zeros(0, int)])
                          for k in q] + [np.full(3, 5)]).astype(np.int32)
    return dict(ctx=ctx, q=q, table=table, n_pages=have, stack=stack, n_free=free, R=R, parents=par if words else None, words=words)


def run_plan(c, out=None, R=None):
    R = c["R"] if R is None else R
    dev = {k: i32(c[k]) for k in ("ctx", "q", "table", "n_pages", "stack")}
    n_free = i32([c["n_free"]])
    B, w = len(c["ctx"]), c["words"]
    full = lambda n, t=torch.int32: torch.full(n if isinstance(n, tuple) else (n,), -9, dtype=t, device=DEV)  # noqa: E731
    out = ops.PagedPlan(full(B + 1), full(R, torch.int64), full(R), full((R, w)) if w else None, full(B), full(B), full(1))
    par = None if not w else i32(c["parents"][:R])
    ops.paged_plan(dev["ctx"], dev["q"], dev["table"], dev["n_pages"], dev["stack"], n_free, R, parents=par, mask_words=w, out=out)
    return out, dev


def check_plan(c, R=None):
    out, dev = run_plan(c, R=R)
    w = O.paged_plan(c["ctx"], c["q"], c["table"], c["n_pages"], c["stack"], c["n_free"], c["R"] if R is None else R,
                     c["parents"], c["words"])
    for k in ("cu_q", "slots", "positions", "status", "n_pages", "n_free"):
        same(getattr(out, k), w[k], k)
    if c["words"]:
        same(out.mask, w["mask"], "mask")
    same(dev["table"], w["table"], "table")
    same(dev["stack"], w["stack"], "stack")
    return w


@pytest.mark.parametrize("B,ctx_hi,q_hi", [(1, 0, 1), (1, 40, 1), (5, 100, 3), (33, 500, 40), (513, 300, 2), (700, 60, 65), (2000, 17, 1), (8192, 40, 2)])
@pytest.mark.parametrize("short", [False, True])
def test_plan(B, ctx_hi, q_hi, short):
    check_plan(plan_case(B + q_hi, B, ctx_hi, q_hi, short=short))


@pytest.mark.parametrize("B,q_hi,words", [(1, 1, 1), (7, 32, 1), (40, 64, 2), (9, 100, 4), (3, 256, 8), (300, 5, 3)])
def test_plan_trees(B, q_hi, words):
    check_plan(plan_case(B * 7 + q_hi, B, 200, q_hi, words=words))


def test_plan_deepest_chain_and_bad_parents():
    c = plan_case(3, 2, 50, 256, ended=0, words=8)
    c["q"] = np.array([256, 100])
    c["table"] = np.full((2, 32), -1, np.int32)
    c["n_pages"] = np.array([0, 0])
    c["ctx"] = np.array([0, 7])
    c["stack"], c["n_free"], c["R"] = np.arange(64, dtype=np.int32), 60, 356
    c["parents"] = np.concatenate([np.arange(256) - 1, np.where(np.arange(100) % 7 == 3, 1000, np.arange(100) - 1)]).astype(np.int32)
    c["parents"][300] = -50
    w = check_plan(c)
    assert w["positions"][255] == 255


def test_plan_refusals_reported_per_request():
    """Too many pages for the table row, a negative context, a tree too wide, rows past max_tokens and an
    empty stack: each request says why, its rows have no slots, the others are served."""
    c = dict(ctx=np.array([100, -3, 5, 0, 40, 3]), q=np.array([30, 2, 40, 1, 2, 9]), table=np.full((6, 8), -1, np.int32),
             n_pages=np.array([0, 0, 1, 0, 3, 0]), stack=np.arange(100, 130, dtype=np.int32), n_free=20, R=80,
             parents=np.full(80, -1, np.int32), words=1)
    c["table"][2, 0], c["table"][4, :3] = 3, [4, 5, 6]
    w = check_plan(c)
    assert w["status"].tolist() == [_lib.PLAN_TABLE, _lib.PLAN_TABLE, _lib.PLAN_TREE, 0, 0, _lib.PLAN_ROWS]
    c["n_free"] = 0
    assert check_plan(c)["status"].tolist()[3] == _lib.PLAN_PAGES


def test_plan_none_and_all_ended():
    c = plan_case(11, 20, 100, 4, ended=0)
    c["q"][:] = 0
    check_plan(c)
    c["q"][:] = -1
    w = check_plan(c)
    assert w["cu_q"].max() == 0 and w["n_free"][0] == c["n_free"] + c["n_pages"].sum()


def test_plan_pushes_past_the_stacks_end_are_dropped():
    c = plan_case(12, 10, 300, 2, ended=0.6)
    c["stack"] = c["stack"][: c["n_free"] + 5]
    check_plan(c)


def test_plan_in_place_over_steps():
    """Steps that update n_pages and n_free in place, as a serving loop does; no page is ever lost."""
    r = np.random.default_rng(5)
    B, mb, pool = 12, 40, 200
    ctx, have, table = np.zeros(B, int), np.zeros(B, int), np.full((B, mb), -1, np.int32)
    stack, n_free = np.arange(pool, dtype=np.int32), pool
    t_dev, s_dev, h_dev, f_dev = i32(table), i32(stack), i32(have), i32([n_free])
    full = lambda n, t=torch.int32: torch.zeros(n, dtype=t, device=DEV)  # noqa: E731
    out = ops.PagedPlan(full(B + 1), full(400, torch.int64), full(400), None, full(B), h_dev, f_dev)
    for _ in range(12):
        q = r.integers(0, 30, B)
        q[r.random(B) < 0.2] = -1
        w = O.paged_plan(ctx, q, table, have, stack, n_free, 400)
        ops.paged_plan(i32(ctx), i32(q), t_dev, h_dev, s_dev, f_dev, 400, out=out)
        table, stack, have, n_free = w["table"], w["stack"], w["n_pages"], int(w["n_free"][0])
        same(t_dev, table), same(s_dev, stack), same(h_dev, have), same(f_dev, [n_free])
        assert n_free + have.sum() == pool
        kept = np.maximum(q - r.integers(0, 5, B), 0)  # some drafted tokens are rejected
        ctx = np.where(q < 0, 0, np.where(w["status"] == 0, ctx + kept, ctx))


# -- qk_norm_rope_append ------------------------------------------------------------------------


def qk_case(seed, R, hq, hk, hd, dt, far=5000):
    r = np.random.default_rng(seed)
    blocks = R // 16 + 3
    x = r.standard_normal((R, (hq + 2 * hk) * hd)).astype(dt)
    return dict(x=x, pos=r.integers(0, far, R).astype(np.int32), slots=r.permutation(blocks * 16)[:R].astype(np.int64),
                invf=O.inv_freq(hd, 10000.0), qg=(1 + 0.2 * r.standard_normal(hd)).astype(np.float32),
                kg=(1 + 0.2 * r.standard_normal(hd)).astype(np.float32), blocks=blocks, dims=(hq, hk, hd))


def qk_bound(hd, parts, dt):
    """|error| of a rotated, normalized value from the magnitudes of the pair it comes from: the mean of
    squares is a sum of hd terms over hd/8 lanes of 8 (hd/8 + 8 roundings), the rest (rsqrt, three products,
    sine and cosine of 2 steps, the angle in [-pi, pi] rounded to fp32: 2^-23, two products and a sum) is
    under 24 half steps; then the output's rounding."""
    lo, hi = np.split(np.abs(parts), 2, axis=-1)
    pair = np.concatenate([lo + hi, lo + hi], -1)
    return (hd / 8 + 32) * E32 * pair + (E16 * pair + TINY16 if dt == np.float16 else 0)


def check_qk(c, dt_out, *, norm=True, v_norm=False, n_rows=None, x_dev=None, q_out=None, live=None):
    hq, hk, hd = c["dims"]
    R = len(c["x"])
    kp = torch.full((c["blocks"], hk, 16, hd), -3.25, dtype=torch.float16, device=DEV)
    vp = torch.full_like(kp, -3.25)
    x_dev = gpu(c["x"]) if x_dev is None else x_dev
    if q_out is None:
        q_out = torch.full((R, hq * hd), 7.0, dtype=dt_out, device=DEV)
    q = ops.qk_norm_rope_append(x_dev, gpu(c["pos"]), gpu(c["slots"]), gpu(c["invf"]), kp, vp, hq, hk, hd,
                                q_gamma=gpu(c["qg"]) if norm else None, k_gamma=gpu(c["kg"]) if norm else None,
                                v_norm=v_norm, n_rows=n_rows, q_out=q_out)
    g = dict(q_gamma=c["qg"], k_gamma=c["kg"]) if norm else {}
    wq, wk, wv = O.qk_norm_rope(c["x"], c["pos"], c["invf"], hq, hk, hd, v_norm=v_norm, **g)
    live = np.ones(R, bool) if live is None else live
    got = q.float().cpu().numpy().reshape(R, hq, hd).astype(np.float64)
    # the rotation keeps a pair's length, so the rotated pair bounds its parts up to sqrt 2
    out_dt = np.float16 if q.dtype == torch.float16 else np.float32
    assert np.all(np.abs(got - wq)[live] <= 1.5 * qk_bound(hd, wq, out_dt)[live])
    rk, rv = kp.cpu().numpy().astype(np.float64), vp.cpu().numpy().astype(np.float64)
    touched = np.zeros((c["blocks"], 16), bool)
    for i in np.flatnonzero(live):
        s = int(c["slots"][i])
        if 0 <= s < c["blocks"] * 16:
            touched[s // 16, s % 16] = True
            assert np.all(np.abs(rk[s // 16, :, s % 16] - wk[i]) <= 1.5 * qk_bound(hd, wk[i], np.float16))
            assert np.all(np.abs(rv[s // 16, :, s % 16] - wv[i]) <= ((hd / 8 + 12) * E32 + E16) * np.abs(wv[i]) + TINY16)
    for p in (rk, rv):
        assert np.all(p.transpose(0, 2, 1, 3)[~touched] == -3.25)
    return q


@pytest.mark.parametrize("hq,hk,hd", [(32, 8, 64), (32, 8, 128), (8, 1, 256), (3, 1, 64), (5, 5, 128)])
@pytest.mark.parametrize("dt", [np.float32, np.float16])
@pytest.mark.parametrize("R", [1, 2, 37])
def test_qk(hq, hk, hd, dt, R):
    c = qk_case(R + hd, R, hq, hk, hd, dt)
    for dt_out in (torch.float32, torch.float16):
        check_qk(c, dt_out)
    check_qk(c, torch.float32, norm=False, v_norm=True)
    check_qk(c, torch.float16, norm=True, v_norm=True)


def test_qk_far_positions():
    """Angles of positions near 2^24: exact to fp32, where an fp32 product would be off by up to a radian."""
    c = qk_case(1, 9, 4, 2, 64, np.float32)
    c["pos"][:] = (1 << 24) - 1 - np.arange(9) * 977
    check_qk(c, torch.float32)


def test_qk_strided_rows_and_in_place():
    hq, hk, hd, R = 6, 2, 64, 21
    c = qk_case(2, R, hq, hk, hd, np.float16)
    wide = torch.zeros(R, (hq + 2 * hk) * hd + 40, dtype=torch.float16, device=DEV)
    x = wide[:, 8 : 8 + (hq + 2 * hk) * hd]
    x.copy_(gpu(c["x"]))
    q = check_qk(c, torch.float16, x_dev=x, q_out=x[:, : hq * hd])
    assert q.data_ptr() == x.data_ptr()
    same(x[:, hq * hd :], c["x"][:, hq * hd :])
    assert wide[:, :8].eq(0).all() and wide[:, 8 + (hq + 2 * hk) * hd :].eq(0).all()


def test_qk_padding_is_left_alone():
    c = qk_case(4, 30, 4, 2, 128, np.float32)
    c["pos"][[3, 29]] = -1
    c["slots"][5], c["slots"][6], c["slots"][7] = -1, c["blocks"] * 16, 1 << 40
    live = np.arange(30) < 22
    live[3] = False
    q = check_qk(c, torch.float32, n_rows=i32([22]), live=live)
    assert q.cpu().numpy()[~live].min() == 7.0 and q.cpu().numpy()[~live].max() == 7.0


# -- paged_tree_attn ----------------------------------------------------------------------------


def attn_case(seed, ctx, q, hq, hk, hd, tree, dt=np.float16, holes=0.0, extra_rows=0):
    r = np.random.default_rng(seed)
    ctx, q = np.asarray(ctx), np.asarray(q)
    B = len(ctx)
    pages = -(-(ctx + q) // 16)
    mb, blocks = max(1, int(pages.max())), int(pages.sum()) + 3
    table = np.full((B, mb), -1, np.int32)
    table[np.arange(mb)[None] < pages[:, None]] = r.permutation(blocks)[: pages.sum()]
    cu = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
    R = int(cu[-1]) + extra_rows
    # every place that holds no token is NaN: none of it may reach an output
    kp = np.full((blocks, hk, 16, hd), np.nan, np.float16)
    vp = np.full((blocks, hk, 16, hd), np.nan, np.float16)
    for b in range(B):
        for j in range(int(ctx[b] + q[b])):
            kp[table[b, j // 16], :, j % 16] = r.standard_normal((hk, hd))
            vp[table[b, j // 16], :, j % 16] = r.standard_normal((hk, hd))
    bits, pos = None, np.concatenate([c + np.arange(n) for c, n in zip(ctx, q)] + [np.full(extra_rows, -1)]).astype(np.int32)
    if tree:
        bits = []
        for b in range(B):
            t, depth = O.tree_bits([int(r.integers(-1, max(1, i))) for i in range(q[b])])
            t[r.random(q[b]) < holes] = False
            bits += list(t)
            pos[cu[b] : cu[b + 1]] = ctx[b] + depth
    words = max(1, -(-int(q.max()) // 32))
    mask = None
    if tree:
        mask = np.full((R, words), -1, np.int32)
        for i, t in enumerate(bits):
            mask[i] = O.pack_bits(t[None], words)[0]
    return dict(q=r.standard_normal((R, hq * hd)).astype(dt), kp=kp, vp=vp, table=table, ctx=ctx.astype(np.int32), cu=cu,
                bits=bits, mask=mask, pos=pos, dims=(hq, hk, hd), max_q=int(q.max()), max_ctx=int((ctx + q).max()), R=R)


def run_attn(c, out_dtype=torch.float32, window=0, scale=0.0, **kw):
    args = dict(mask=None if c["mask"] is None else gpu(c["mask"]), positions=gpu(c["pos"]), scale=scale, window=window,
                out_dtype=out_dtype)
    args.update(kw)
    q = args.pop("q", None)
    return ops.paged_tree_attn(gpu(c["q"]) if q is None else q, gpu(c["kp"]), gpu(c["vp"]), gpu(c["table"]), gpu(c["ctx"]),
                               gpu(c["cu"]), *c["dims"], args.pop("max_q", c["max_q"]), args.pop("max_ctx", c["max_ctx"]), **args)


def attn_bound(c, o, mag, fp16, out16, scale):
    """A score is a sum of hd exact products in fp32 (tensor cores drop bits below the running sum: one
    step, 2^-23, per 16 terms), then a product and the exponential's argument: relative error of a weight
    err_p <= scale * |q||k| * (hd/16 + 4) * 2^-23 + |s| 2^-22.  Weights in fp16 add eps16 each (22 bits
    otherwise), sums over n places one step per 16, and the output its own rounding."""
    hq, hk, hd = c["dims"]
    n = c["max_ctx"]
    live = c["q"][: c["cu"][-1]].astype(np.float64).reshape(-1, hq, hd)
    qn = np.linalg.norm(live, axis=-1).max()
    K = c["kp"].astype(np.float64)
    kn = np.sqrt(np.nanmax(np.where(np.isfinite(K).all(-1), (K * K).sum(-1), 0)))
    sc = scale if scale > 0 else hd**-0.5
    err_p = sc * qn * kn * ((hd / 16 + 4) * 2.0**-23 + 2.0**-22 + (0 if fp16 else 2.0**-21)) + 2.0**-21
    err_p += E16 if fp16 else 2.0**-21
    return (2 * err_p + (n / 16 + 8) * 2.0**-23) * mag + (E16 if out16 else 4 * E32) * np.abs(o) + (TINY16 if out16 else 0)


def check_attn(c, out_dtype=torch.float32, window=0, scale=0.0, **kw):
    hq, hk, hd = c["dims"]
    got = run_attn(c, out_dtype, window, scale, **kw).float().cpu().numpy().astype(np.float64).reshape(-1, hq, hd)
    want, mag = O.tree_attention(c["q"], c["kp"], c["vp"], c["table"], c["ctx"], c["cu"], hq, hk, hd, c["bits"], c["pos"], scale, window)
    n = int(c["cu"][-1])
    got, want, mag = got[:n], want[:n], mag[:n]
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    ok = np.isfinite(want)
    np.testing.assert_array_equal(got[~ok & ~np.isnan(want)], want[~ok & ~np.isnan(want)])
    fp16 = c["q"].dtype == np.float16 and out_dtype == torch.float16
    err, lim = np.abs(got - want), attn_bound(c, want, mag, fp16, out_dtype == torch.float16, scale)
    assert np.all(err[ok] <= lim[ok]), (np.max((err / lim)[ok]), np.argwhere((err > lim) & ok)[:4])
    tree_clean()


def tree_clean():
    ops.tree_attn_check()


HEADS = [(32, 8, 64), (4, 4, 64), (16, 2, 128), (8, 2, 128), (8, 1, 256), (3, 1, 64), (20, 4, 128)]


@pytest.mark.parametrize("hq,hk,hd", HEADS)
@pytest.mark.parametrize("tree", [True, False])
def test_attn_ragged(hq, hk, hd, tree):
    c = attn_case(hq + hd, [0, 15, 200, 64, 33], [1, 17, 5, 1, 40], hq, hk, hd, tree)
    check_attn(c, torch.float16)
    check_attn(c, torch.float32)
    c["q"] = c["q"].astype(np.float32) + np.float32(1e-4)
    check_attn(c, torch.float32)
    check_attn(c, torch.float16)


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100])
def test_attn_row_counts(T):
    check_attn(attn_case(T, [70, 0], [T, max(1, T - 1)], 8, 2, 64, T % 2 == 0), torch.float16)


@pytest.mark.parametrize("ctx", [0, 1, 15, 16, 63, 64, 65, 127, 128, 129, 511])
def test_attn_context_ends(ctx):
    check_attn(attn_case(ctx, [ctx], [3], 4, 1, 128, True), torch.float32)


@pytest.mark.parametrize("hd,T,tree", [(64, 3, True), (128, 40, True), (128, 130, False), (256, 5, False)])
def test_attn_long_context_many_chunks(hd, T, tree):
    c = attn_case(hd + T, [5000, 130], [T, 2], 4, 1, hd, tree)
    assert ops.tree_attn_workspace_bytes(2, c["R"], 4, 1, hd, c["max_q"], c["max_ctx"]) > 0
    check_attn(c, torch.float16)
    check_attn(c, torch.float32)


@pytest.mark.parametrize("hq,hk,hd,q", [(8, 8, 64, 9), (16, 4, 64, 70), (8, 4, 128, 7), (8, 4, 128, 90), (4, 2, 256, 5)])
def test_attn_many_sequences(hq, hk, hd, q):
    """More (sequence, KV head) pairs than SMs, of 1 to several key tiles: a CTA works on several of them."""
    r = np.random.default_rng(q)
    c = attn_case(q, r.integers(0, 700, 40), r.integers(0, q + 1, 40), hq, hk, hd, q % 2 == 1)
    check_attn(c, torch.float16)
    check_attn(c, torch.float32)


@pytest.mark.parametrize("hd", [64, 128])
def test_attn_large_batch(hd):
    """More sequences than prefix sums are kept for, many of them without rows."""
    r = np.random.default_rng(hd)
    c = attn_case(hd, r.integers(0, 40, 900), r.integers(0, 3, 900), 2, 1, hd, False)
    check_attn(c, torch.float16)


def test_attn_two_calls_at_once():
    """Two streams, each with its own call in flight: nothing is shared between them."""
    cases = [attn_case(20 + i, [4000, 900], [30, 9], 8, 2, 128, True) for i in range(2)]
    want = [run_attn(c, torch.float16) for c in cases]
    args = [(gpu(c["q"]), gpu(c["kp"]), gpu(c["vp"]), gpu(c["table"]), gpu(c["ctx"]), gpu(c["cu"]), *c["dims"], c["max_q"], c["max_ctx"])
            for c in cases]
    masks = [gpu(c["mask"]) for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.paged_tree_attn(*args[i], mask=masks[i], out_dtype=torch.float16))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_attn_fp16_rows_to_planes():
    c = attn_case(16, [300, 2], [9, 70], 16, 4, 64, True)
    want = run_attn(c)
    x2 = torch.zeros(2, c["R"], 16 * 64, dtype=torch.float16, device=DEV)
    run_attn(c, out=x2)
    err = (ops.from_f16x2(x2) - want).abs()
    assert torch.all(err <= 2.0**-21 * want.abs() + 2.0**-24)


def test_attn_positions_are_held_to_the_tree():
    """Given positions below the context or past a row's own place count as those."""
    c = attn_case(17, [60, 7], [12, 5], 4, 2, 64, True)
    c["pos"] = np.where(np.arange(c["R"]) % 2 == 0, -5, 10**6).astype(np.int32)
    got = run_attn(c, window=30)
    own = np.concatenate([np.arange(12), np.arange(5)])
    c["pos"] = np.where(np.arange(c["R"]) % 2 == 0, np.repeat(c["ctx"], [12, 5]), np.repeat(c["ctx"], [12, 5]) + own).astype(np.int32)
    assert torch.equal(got, run_attn(c, window=30))
    check_attn(c, torch.float32, window=30)


def test_attn_widest_tree():
    check_attn(attn_case(8, [37], [256], 4, 2, 64, True), torch.float16)


@pytest.mark.parametrize("window", [1, 7, 64, 100, 1000])
@pytest.mark.parametrize("tree", [True, False])
def test_attn_window(window, tree):
    c = attn_case(window, [300, 5, 900], [20, 33, 3], 8, 2, 64, tree)
    check_attn(c, torch.float16, window=window)
    check_attn(c, torch.float32, window=window, scale=0.5)


def test_attn_rows_that_see_nothing():
    c = attn_case(6, [0, 0, 20], [6, 33, 4], 8, 2, 128, True, holes=0.5)
    for dt in (torch.float16, torch.float32):
        check_attn(c, dt)
    empty = [i for i in range(39) if not c["bits"][i].any()]
    assert empty and run_attn(c)[empty].eq(0).all()


@pytest.mark.parametrize("fill", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("T,ctx", [(9, 40), (40, 0), (40, 100)])
def test_attn_hidden_rows_hold_anything(fill, T, ctx):
    """A drafted token whose k and v are not finite: the branches that do not pass through it are clean,
    its own branch gets what the formula gives."""
    for dt in (np.float16, np.float32):
        c = attn_case(T, [ctx], [T], 8, 2, 64, True, dt=dt)
        for node, part in ((T // 2, "kp"), (T // 3, "vp")):
            j = ctx + node
            c[part][c["table"][0, j // 16], 1, j % 16, 5] = fill
        check_attn(c, torch.float32 if dt == np.float32 else torch.float16)


def test_attn_window_hides_what_left_it():
    c = attn_case(3, [400], [4], 8, 2, 64, False)
    for j in range(330):  # every place at or below 404 - 1 - 64 has left every row's window
        c["vp"][c["table"][0, j // 16], :, j % 16] = np.inf
        c["kp"][c["table"][0, j // 16], :, j % 16] = np.nan
    check_attn(c, torch.float16, window=64)
    c["table"][0, :20] = -1
    check_attn(c, torch.float16, window=64)


def test_attn_pages_outside_the_pool_are_hidden():
    c = attn_case(9, [100, 40], [3, 3], 8, 2, 64, True)
    c["table"][0, 2], c["table"][1, 1] = 10**6, -7
    check_attn(c, torch.float16)
    c["table"][:] = -1
    assert run_attn(c).eq(0).all()


def test_attn_strided_rows_and_planes():
    hq, hk, hd = 8, 2, 64
    c = attn_case(10, [50, 20], [6, 2], hq, hk, hd, True, dt=np.float32)
    wide = torch.zeros(c["R"], hq * hd + 64, device=DEV)
    wide[:, 32 : 32 + hq * hd] = gpu(c["q"])
    want = run_attn(c)
    out = torch.full((c["R"], hq * hd + 16), 5.0, device=DEV)
    run_attn(c, q=wide[:, 32 : 32 + hq * hd], out=out[:, : hq * hd])
    assert torch.equal(out[:, : hq * hd], want) and out[:, hq * hd :].eq(5).all()
    x2 = torch.zeros(2, c["R"], hq * hd, dtype=torch.float16, device=DEV)
    run_attn(c, out=x2)
    err = (ops.from_f16x2(x2) - want).abs()
    assert torch.all(err <= 2.0**-21 * want.abs() + 2.0**-24)


def test_attn_rows_behind_the_last_sequence():
    c = attn_case(12, [50, 20], [6, 2], 8, 2, 64, True, extra_rows=7)
    out = torch.full((c["R"], 8 * 64), 9.0, dtype=torch.float16, device=DEV)
    run_attn(c, out=out)
    assert out[8:].eq(9).all() and out[:8].ne(9).all()
    # a sequence past max_ctx, and rows past max_q, are left as they were
    out.fill_(9)
    run_attn(c, out=out, max_ctx=30)
    assert out[:6].eq(9).all() and out[6:8].ne(9).all()
    out.fill_(9)
    run_attn(c, out=out, max_q=4)
    assert out[4:6].eq(9).all() and out[:4].ne(9).all() and out[6:8].ne(9).all()


def test_attn_empty_sequences():
    c = attn_case(13, [50, 0, 20, 9], [0, 3, 0, 2], 8, 2, 64, True)
    check_attn(c, torch.float16)


def test_attn_one_row_matches_decode():
    """One row per sequence: the decode step's attention on the same cache."""
    c = attn_case(14, [100, 3000, 0], [1, 1, 1], 32, 8, 64, False)
    c["kp"], c["vp"] = np.nan_to_num(c["kp"]), np.nan_to_num(c["vp"])
    got = run_attn(c)
    qkv = torch.zeros(3, 48 * 64, dtype=torch.float16, device=DEV)
    qkv[:, : 32 * 64] = gpu(c["q"])
    want = ops.paged_decode_attn(qkv, gpu(c["kp"]), gpu(c["vp"]), gpu(c["table"]), gpu(c["ctx"]), None, 32, 8, 64, c["max_ctx"], append=False)
    assert torch.allclose(got, want, rtol=1e-4, atol=1e-5)


def test_attn_is_deterministic():
    c = attn_case(15, [3000, 700], [20, 9], 8, 2, 128, True)
    a = run_attn(c, torch.float16)
    for _ in range(3):
        assert torch.equal(a, run_attn(c, torch.float16))


# -- token_logprobs -----------------------------------------------------------------------------


def check_score(x, t, k, **kw):
    """The row's sum is formed from partial sums of at most V/512 + 60 terms, each weight within
    2^-22 (the exponential) + |z| 2^-24 (its argument, |z| <= 64 where the weight counts): a logprob is
    off by at most that, its own rounding and the fp32 log2(e)'s 2^-25 relative; the entropy likewise,
    relative to 1 + H."""
    r = ops.token_logprobs(x, None if t is None else i32(t), k, **kw)
    tl, ent, ids, tlp = O.token_logprobs(x.float().cpu().numpy(), t, k)
    V = x.shape[1]
    rel = (V / 512 + 60) * E32 + 2.0**-22 + 64 * E32

    def near(got, want, slack):
        got = got.cpu().numpy().astype(np.float64).reshape(want.shape)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        f = np.isfinite(want)
        np.testing.assert_array_equal(got[~f & ~np.isnan(want)], want[~f & ~np.isnan(want)])
        assert np.all(np.abs(got - want)[f] <= slack(np.abs(want[f])))

    if t is not None:
        near(r.logprobs, tl, lambda w: rel + 2 * 2.0**-24 * w)
    near(r.entropy, ent, lambda w: 2 * rel * (1 + w))
    if k:
        same(r.top_ids, ids)
        near(r.top_logprobs, tlp, lambda w: rel + 2 * 2.0**-24 * w)
    return r


@pytest.mark.parametrize("V", [1, 2, 7, 33, 1000, 4097, 32003, 128256])
@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
def test_score(V, dt):
    g = torch.Generator(device=DEV).manual_seed(V)
    for R in (1, 3):
        x = (3 * torch.randn(R, V, generator=g, device=DEV)).to(dt)
        t = np.random.default_rng(V).integers(0, V, (R, 3))
        for k in {0, min(1, V), min(5, V), min(32, V)}:
            check_score(x, t, k)
    check_score(x, None, min(2, V))


@pytest.mark.parametrize("R", [148, 700, 1500])
def test_score_many_rows(R):
    g = torch.Generator(device=DEV).manual_seed(R)
    check_score(torch.randn(R, 2049, generator=g, device=DEV).half(), np.zeros((R, 1), int), 20)


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
def test_score_any_alignment(dt):
    """Rows that start at every place of a 16-byte vector, and a row stride that is not V."""
    g = torch.Generator(device=DEV).manual_seed(0)
    wide = torch.randn(9, 5003, generator=g, device=DEV).to(dt)
    for o in range(9):
        check_score(wide[:, o : o + 4000 + o], np.full((9, 2), 17), 7)


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
def test_score_ties_take_the_lowest_index(dt):
    x = torch.zeros(4, 9001, dtype=dt, device=DEV)
    x[1, ::3] = 1.0
    x[2, 5000:] = -0.0
    x[3] = -2.0
    x[3, 8990:] = torch.linspace(1, 2, 11, device=DEV).to(dt)
    check_score(x, np.zeros((4, 1), int), 32)


def test_score_largest_values_in_one_threads_vectors():
    """All of the row's largest values where one thread reads them: more candidates than are ranked at once."""
    x = torch.randn(2, 128256, device=DEV)
    for ranks in (1, 2, 4, 8):
        stride = ranks * 512 * 4
        for j in range(4):
            x[0, j::stride] += 50
    x[1] = torch.linspace(0, 30, 128256, device=DEV)
    check_score(x, np.zeros((2, 1), int), 32)


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
def test_score_extremes(dt):
    """Rows of -inf, the type's lowest, a single finite value, NaN, +inf and large finite values."""
    lowest, big = torch.finfo(dt).min, torch.finfo(dt).max
    x = torch.randn(12, 3001, device=DEV).to(dt)
    x[0] = -np.inf
    x[1] = lowest
    x[2] = -np.inf
    x[2, 77] = 3.0
    x[3, 100:] = lowest
    x[4, 5:] = -np.inf
    x[5, 9] = np.nan
    x[6, 9] = np.inf
    x[7] = np.nan
    x[8, 50] = big
    x[9] = big
    x[10, :3000] = np.nan
    x[11] = -np.inf
    x[11, 9] = lowest
    check_score(x, np.tile([9, 77, 3000, -1, 3001], (12, 1)), 32)


def test_score_rows_in_use():
    x = torch.randn(6, 1000, device=DEV)
    f = lambda *n: torch.full(n, 8.0, device=DEV)  # noqa: E731
    out = ops.TokenLogprobs(f(6), f(6), torch.full((6, 3), 8, dtype=torch.int32, device=DEV), f(6, 3))
    ops.token_logprobs(x, i32(np.zeros(6)), 3, n_rows=i32([4]), out=out)
    want = ops.token_logprobs(x, i32(np.zeros(6)), 3)
    for a, b in zip((out.logprobs, out.entropy, out.top_ids, out.top_logprobs),
                    (want.logprobs, want.entropy, want.top_ids, want.top_logprobs)):
        assert torch.equal(a[:4], b[:4]) and a[4:].eq(8).all()


# -- refusals of the Python entry points ----------------------------------------------------------


def test_wrong_arguments_are_refused():
    c = attn_case(1, [20], [3], 4, 2, 64, True)
    for kw in (dict(mask=gpu(c["mask"]).long()), dict(mask=gpu(c["mask"])[:2]), dict(positions=gpu(c["pos"])[:1]),
               dict(q=gpu(c["q"]).double()), dict(q=gpu(c["q"])[:, :128]), dict(max_q=0), dict(max_q=40), dict(max_ctx=1000),
               dict(positions=None, window=4), dict(q=gpu(c["q"]).T.contiguous().T),
               dict(out=torch.empty(3, 128, device=DEV)), dict(out=torch.empty(3, 256, device="cpu"))):
        with pytest.raises(ValueError):
            run_attn(c, **kw)
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.zeros(2, 10, device=DEV), i32([0]), 0)
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.zeros(2, 10, device=DEV), None, 11)
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.zeros(2, 10, device=DEV).long())
    p = plan_case(1, 2, 20, 2)
    with pytest.raises(ValueError):
        ops.paged_plan(i32(p["ctx"]), i32(p["q"]), i32(p["table"]), i32(p["n_pages"]), i32(p["stack"]), i32([1]), p["R"], mask_words=1)


# -- a step of them together ------------------------------------------------------------------------


class Step:
    """Two layers' worth of a verification step over preallocated buffers: plan, append, attention, logits,
    scores.  run() uses device data alone, so it can be captured."""

    HQ, HK, HD, B, R, W, V = 8, 2, 64, 6, 96, 1, 1001
    POOL, MB = 64, 12

    def __init__(self, seed):
        r = np.random.default_rng(seed)
        n = (self.HQ + 2 * self.HK) * self.HD
        self.h = dict(qkv=r.standard_normal((2, self.R, n)).astype(np.float16), kg=np.ones(self.HD, np.float32) * 1.1,
                      qg=np.ones(self.HD, np.float32) * 0.9, head=(r.standard_normal((self.V, self.HQ * self.HD)) * 0.05).astype(np.float16))
        self.d = {k: gpu(v) for k, v in self.h.items()}
        self.invf = gpu(O.inv_freq(self.HD, 10000.0))
        z = lambda *n, t=torch.int32: torch.zeros(*n, dtype=t, device=DEV)  # noqa: E731
        self.ctx, self.q, self.n_pages, self.n_free = z(self.B), z(self.B), z(self.B), z(1)
        self.table, self.stack, self.parents = z(self.B, self.MB) - 1, z(self.POOL), z(self.R) - 1
        self.targets = z(self.R, 2)
        self.kp = torch.full((2, self.POOL, self.HK, 16, self.HD), float("nan"), dtype=torch.float16, device=DEV)
        self.vp = self.kp.clone()
        self.plan = ops.PagedPlan(z(self.B + 1), z(self.R, t=torch.int64), z(self.R), z(self.R, self.W), z(self.B), self.n_pages, self.n_free)

    def load(self, seed):
        """New requests' state: lengths, pages and cache contents."""
        r = np.random.default_rng(seed)
        ctx = r.integers(0, 120, self.B)
        q = r.integers(1, 14, self.B)
        have = -(-ctx // 16)
        ids = r.permutation(self.POOL).astype(np.int32)
        table = np.full((self.B, self.MB), -1, np.int32)
        table[np.arange(self.MB)[None] < have[:, None]] = ids[: have.sum()]
        stack = np.zeros(self.POOL, np.int32)
        free = self.POOL - int(have.sum())
        stack[:free] = ids[have.sum() :]
        par = np.concatenate([[int(r.integers(-1, max(1, i))) for i in range(k)] for k in q] + [np.zeros(self.R - q.sum(), int)])
        kv = r.standard_normal((2, 2, self.POOL, self.HK, 16, self.HD)).astype(np.float16)
        t = r.integers(0, self.V, (self.R, 2))
        self.now = dict(ctx=ctx, q=q, have=have, table=table, stack=stack, free=free, par=par, kv=kv, t=t)
        for dst, a in ((self.ctx, ctx), (self.q, q), (self.n_pages, have), (self.table, table), (self.stack, stack),
                       (self.parents, par), (self.targets, t)):
            dst.copy_(torch.from_numpy(np.asarray(a, np.int32)))
        self.n_free.fill_(free)
        self.kp.copy_(torch.from_numpy(kv[0])), self.vp.copy_(torch.from_numpy(kv[1]))

    def run(self):
        p = ops.paged_plan(self.ctx, self.q, self.table, self.n_pages, self.stack, self.n_free, self.R, parents=self.parents,
                           mask_words=self.W, out=self.plan)
        o = None
        self.attn = []
        for layer in range(2):
            q = ops.qk_norm_rope_append(self.d["qkv"][layer], p.positions, p.slots, self.invf, self.kp[layer], self.vp[layer], self.HQ,
                                        self.HK, self.HD, q_gamma=self.d["qg"], k_gamma=self.d["kg"], n_rows=p.n_rows, out_dtype=torch.float16)
            o = ops.paged_tree_attn(q, self.kp[layer], self.vp[layer], self.table, self.ctx, p.cu_q, self.HQ, self.HK, self.HD, 16,
                                    self.MB * 16, mask=p.mask, positions=p.positions, out_dtype=torch.float16)
            self.attn.append(o)
        logits = ops.gemv(self.d["head"], o)
        self.score = ops.token_logprobs(logits, self.targets, 5, n_rows=p.n_rows)
        self.logits = logits
        return self

    def check(self):
        s = self.now
        w = O.paged_plan(s["ctx"], s["q"], s["table"], s["have"], s["stack"], s["free"], self.R, s["par"], self.W)
        n = int(w["cu_q"][-1])
        assert w["status"].max() == 0
        for k in ("cu_q", "status", "n_pages", "n_free"):
            same(getattr(self.plan, k), w[k], k)
        for k in ("slots", "positions", "mask"):
            same(getattr(self.plan, k)[:n], w[k][:n], k)
        bits = []
        for b in range(self.B):
            bits += list(O.tree_bits(s["par"][w["cu_q"][b] : w["cu_q"][b + 1]])[0])
        for layer in range(2):
            wq, wk, wv = O.qk_norm_rope(self.h["qkv"][layer], w["positions"], self.invf.cpu().numpy(), self.HQ, self.HK, self.HD,
                                        self.h["qg"], self.h["kg"])
            kp, vp = s["kv"][0, layer].copy(), s["kv"][1, layer].copy()
            for i in range(n):
                kp[w["slots"][i] // 16, :, w["slots"][i] % 16] = wk[i]
                vp[w["slots"][i] // 16, :, w["slots"][i] % 16] = wv[i]
            o, mag = O.tree_attention(wq[:n].reshape(n, -1), kp, vp, w["table"], s["ctx"], w["cu_q"], self.HQ, self.HK, self.HD, bits, w["positions"])
            # rounded q and k: scores off by 2 eps16 |q||k| scale <= 2 eps16 * 8 * 1.5 (normalized heads,
            # gammas 0.9 * 1.1), so weights by e^that - 1; weights and output rounded to fp16
            err = np.abs(self.attn[layer].cpu().numpy()[:n].reshape(o.shape) - o)
            assert np.all(err <= (2 * 2 * E16 * 12 + 2 * E16) * mag + E16 * np.abs(o) + TINY16)
        x = self.logits[:n]
        tl, ent, ids, tlp = O.token_logprobs(x.cpu().numpy(), s["t"][:n], 5)
        same(self.score.top_ids[:n], ids)
        for got, want in ((self.score.logprobs, tl), (self.score.entropy, ent), (self.score.top_logprobs, tlp)):
            np.testing.assert_allclose(got[:n].cpu().numpy(), want, atol=2e-5, rtol=1e-6)


def test_step_together():
    s = Step(1)
    for seed in (2, 3):
        s.load(seed)
        s.run().check()


def test_step_on_another_stream():
    s = Step(4)
    s.load(5)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        s.run()
    side.synchronize()
    s.check()


def test_two_captured_steps_replayed_together():
    """Two captured graphs on two streams: they share no scratch, and replay with new lengths."""
    steps = [Step(6), Step(7)]
    graphs = []
    for i, s in enumerate(steps):
        s.load(8 + i)
        s.run()  # first launches outside the capture
        torch.cuda.synchronize()
        s.load(8 + i)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.run()
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for round_ in range(3):
        for i, s in enumerate(steps):
            s.load(20 + 2 * round_ + i)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s in steps:
            s.check()
    del graphs


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_other_device_than_the_current_one():
    x = torch.randn(3, 500, device="cuda:1")
    r = ops.token_logprobs(x, None, 3)
    assert r.top_ids.device.index == 1
    same(r.top_ids, torch.sort(x, dim=1, descending=True, stable=True).indices[:, :3].cpu().numpy())
