"""What the operators of a drafted-token step are measured on.

A step that verifies drafted tokens (or prefills chunks of several requests at once) over the paged KV
cache has four operators: paged_plan (pages, slots, positions and tree masks from the requests' lengths),
qk_norm_rope_append (per-head norms, rotation, append), paged_tree_attn (several query rows per sequence
over the cache) and token_logprobs (log probabilities, entropy and top alternatives of the logits).

Each case is a dict of plain values.  `run` computes an operator in its plain form (elementary torch
operations in 32 bits), or with `own` set through this package's entry points.
"""

import math
import random

import numpy as np
import torch

own = False

PAGE = 16
DEV = "cuda"
_LOWEST = {"f16": -65504.0, "f32": -3.4028234663852886e38}
_DT = {"f16": torch.float16, "f32": torch.float32}


# -- cases ------------------------------------------------------------------------------------


def listed():
    return [
        # One serving step's plan: 32 running requests (the batch of the 1B decode workload), each with a
        # drafted tree of 16 to 40 nodes, two requests just ended.
        dict(name="plan_draft_32", op="plan", batch=32, ended=2, chunks=0, chunk=1, tree=True, q_lo=16, q_hi=40,
             ctx_lo=64, ctx_hi=4096, short=False),
        # A large mixed step: 512 requests, most with one token, 24 with a 509-token prefill chunk, 40 ended.
        dict(name="plan_mixed_512", op="plan", batch=512, ended=40, chunks=24, chunk=509, tree=False, q_lo=1, q_hi=1,
             ctx_lo=1, ctx_hi=32768, short=False),
        # A single token of the 1B model in the step's own fp32 activations: pure latency.
        dict(name="qk_token", op="qk", rows=1, hq=32, hk=8, hd=64, dt="f32", norm=True, v_norm=False, far=4096),
        # The drafted rows of a batch, fp16, head_dim 128 (the attention workload's heads).
        dict(name="qk_draft_777", op="qk", rows=777, hq=32, hk=8, hd=128, dt="f16", norm=True, v_norm=False, far=8192),
        # A prefill chunk of many requests, fp32 projections: bound by memory bandwidth.
        dict(name="qk_prefill_8191", op="qk", rows=8191, hq=32, hk=8, hd=128, dt="f32", norm=True, v_norm=False,
             far=131072),
        # One sequence, a short draft, the 1B model's heads in fp32: latency.
        dict(name="tree_one", op="attn", batch=1, q_lo=8, q_hi=8, ctx_lo=1021, ctx_hi=1021, hq=32, hk=8, hd=64, dt="f32",
             tree=True, holes=False, window=0),
        # The 1B decode workload's batch (32 contexts in 512..4096) with trees of 5 to 24 nodes.
        dict(name="tree_batch_32", op="attn", batch=32, q_lo=5, q_hi=24, ctx_lo=512, ctx_hi=4096, hq=32, hk=8, hd=64,
             dt="f16", tree=True, holes=False, window=0),
        # Wide trees over long contexts: 64 nodes a sequence, head_dim 128.
        dict(name="tree_long_8", op="attn", batch=8, q_lo=61, q_hi=64, ctx_lo=8192, ctx_hi=32768, hq=32, hk=8, hd=128,
             dt="f16", tree=True, holes=False, window=0),
        # Chunked prefill of four requests: 509 to 512 causal rows each, bound by the tensor cores.
        dict(name="chunk_causal_4", op="attn", batch=4, q_lo=509, q_hi=512, ctx_lo=0, ctx_hi=8192, hq=32, hk=8, hd=128,
             dt="f16", tree=False, holes=False, window=0),
        # The sampled token's log probability with 5 alternatives, one row of fp32 logits: latency.
        dict(name="score_one", op="score", rows=1, vocab=128256, dt="f32", targets=1, k=5, banned=False),
        # Scores of a batch's drafted rows, fp16 logits, four children a row, 20 alternatives.
        dict(name="score_draft_771", op="score", rows=771, vocab=128256, dt="f16", targets=4, k=20, banned=True),
        # Scoring prompts: 2048 rows of fp32 logits, bound by memory bandwidth.
        dict(name="score_prompt_2048", op="score", rows=2048, vocab=128256, dt="f32", targets=1, k=8, banned=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(32, 8, 64), (32, 8, 128), (16, 4, 64), (8, 8, 64), (8, 2, 128), (8, 1, 128), (8, 1, 256), (4, 1, 64), (16, 2, 128)]


def draw(rng):
    op = rng.choice(["plan", "qk", "attn", "attn", "score"])
    if op == "plan":
        batch = _log_int(rng, 1, 1024)
        tree = rng.random() < 0.5
        chunks = 0 if tree else min(batch, rng.randint(0, 24))
        q_hi = rng.randint(1, 64) if tree else rng.randint(1, 8)
        return dict(op=op, batch=batch, ended=rng.randint(0, (batch - chunks) // 4), chunks=chunks,
                    chunk=rng.randint(17, 512), tree=tree, q_lo=rng.randint(0, q_hi), q_hi=q_hi, ctx_lo=rng.randint(0, 64),
                    ctx_hi=_log_int(rng, 64, 32768), short=rng.random() < 0.25)
    if op == "qk":
        hq, hk, hd = rng.choice(_HEADS)
        return dict(op=op, rows=_log_int(rng, 1, 8191), hq=hq, hk=hk, hd=hd, dt=rng.choice(["f16", "f32"]),
                    norm=rng.random() < 0.75, v_norm=rng.random() < 0.3, far=_log_int(rng, 64, 131072))
    if op == "attn":
        hq, hk, hd = rng.choice(_HEADS)
        tree = rng.random() < 0.6
        q_hi = _log_int(rng, 1, 96 if tree else 512)
        ctx_hi = _log_int(rng, 1, 32768)
        # the costliest draw stays below tree_long_8 and chunk_causal_4 in rows x keys x heads
        room = 8 * 32768 * 64 * 32 * 128 // ((ctx_hi + q_hi) * q_hi * hq * hd)
        batch = _log_int(rng, 1, max(1, min(64, room, 262144 // (ctx_hi + q_hi))))
        return dict(op=op, batch=batch, q_lo=rng.randint(1, q_hi), q_hi=q_hi, ctx_lo=rng.randint(0, ctx_hi),
                    ctx_hi=ctx_hi, hq=hq, hk=hk, hd=hd, dt=rng.choice(["f16", "f16", "f32"]), tree=tree,
                    holes=tree and rng.random() < 0.3, window=rng.choice([0, 0, 0, 128, 1000]))
    vocab = _log_int(rng, 1000, 256000)
    rows = _log_int(rng, 1, max(1, min(2048, 2048 * 128256 // vocab)))
    return dict(op=op, rows=rows, vocab=vocab, dt=rng.choice(["f16", "f32"]), targets=rng.randint(1, 8),
                k=rng.choice([0, 1, 5, 20, 32]), banned=rng.random() < 0.5)


# -- lengths of a case (the case alone decides them; seeds change values, pages and tree shapes) --------------


def _spread(lo, hi, n, salt):
    """n whole numbers over [lo, hi], evenly spaced and shuffled."""
    v = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]
    random.Random(salt).shuffle(v)
    return np.array(v, dtype=np.int64)


def _plan_lens(c):
    n = c["batch"]
    ctx, q = _spread(c["ctx_lo"], c["ctx_hi"], n, 1), _spread(c["q_lo"], c["q_hi"], n, 2)
    order = np.random.RandomState(3).permutation(n)
    q[order[: c["chunks"]]] = c["chunk"]
    q[order[c["chunks"] : c["chunks"] + c["ended"]]] = -1
    return ctx, q


def _parents(rs, n):
    """A drafted tree of n nodes: each hangs below an earlier one (-1: below the last cached token)."""
    p = rs.randint(-1, np.maximum(np.arange(n), 1))
    return np.where(rs.rand(n) < 0.5, np.arange(n) - 1, p)


def _ancestors(parents):
    """Truth values [n, n]: row i has its own bit and its ancestors'.  Also the nodes' depths."""
    n = len(parents)
    a = np.eye(n, dtype=bool)
    for i in range(n):
        if parents[i] >= 0:
            a[i] |= a[parents[i]]
    return a, a.sum(1) - 1


def _pack(bits, words):
    """Truth values [n, m] -> int32 words [n, words], bit j of the row in word j / 32."""
    out = np.zeros((bits.shape[0], 32 * words), dtype=np.uint8)
    out[:, : bits.shape[1]] = bits
    return np.packbits(out, axis=1, bitorder="little").view(np.int32)


# -- inputs --------------------------------------------------------------------------------------


def _gpu(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV, dtype)


def _i32(a):
    return _gpu(np.asarray(a, dtype=np.int32))


def _inv_freq(hd):
    return (10000.0 ** (-np.arange(0, hd, 2, dtype=np.float64) / hd)).astype(np.float32)


def _prepare_plan(c, seed):
    rs = np.random.RandomState(seed)
    ctx, q = _plan_lens(c)
    n = c["batch"]
    have = -(-ctx // PAGE) + np.random.RandomState(6).randint(0, 2, n)  # some kept a page from a longer draft
    mb = int((-(-(ctx + np.maximum(q, 0)) // PAGE)).max()) + 1
    have = np.minimum(have, mb)
    need = np.where(q < 0, 0, np.maximum(0, -(-(ctx + np.maximum(q, 0)) // PAGE) - have))
    back = int(have[q < 0].sum())
    free = max(0, int(need.sum()) - back) + (0 if c["short"] else 64)
    free = free // 2 if c["short"] else free
    ids = rs.permutation(int(have.sum()) + free).astype(np.int32)
    table = np.full((n, mb), -1, np.int32)
    table[np.arange(mb)[None] < have[:, None]] = ids[: have.sum()]
    stack = np.full(free + back + 1, -1, np.int32)
    stack[:free] = ids[have.sum() :]
    total = int(np.maximum(q, 0).sum())
    rows = total + 5  # a padded token buffer: the rows behind the last request stay as they are
    words = -(-max(1, c["q_hi"]) // 32) if c["tree"] else 0
    par = np.full(rows, -1, np.int32)
    if c["tree"]:
        par[:total] = np.concatenate([_parents(rs, max(0, int(k))) for k in q] + [np.zeros(0, np.int64)])
    return dict(op="plan", ctx=_i32(ctx), q=_i32(q), table=_i32(table), n_pages=_i32(have), stack=_i32(stack),
                n_free=_i32([free]), parents=_i32(par) if c["tree"] else None, rows=rows, words=words,
                nodes=int(max(1, c["q_hi"])), cu=_i32(np.full(n + 1, -9)), slots=_gpu(np.full(rows, -9, np.int64)),
                positions=_i32(np.full(rows, -9)), mask=_i32(np.full((rows, words), 9)) if c["tree"] else None,
                status=_i32(np.full(n, -9)), n_pages_out=_i32(np.full(n, -9)), n_free_out=_i32([-9]))


def _prepare_qk(c, seed):
    rs = np.random.RandomState(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows, hq, hk, hd = c["rows"], c["hq"], c["hk"], c["hd"]
    blocks = -(-rows // PAGE) + 2
    slots = rs.permutation(blocks * PAGE)[:rows].astype(np.int64)
    if rows > 8:
        slots[rs.randint(0, rows, rows // 8)] = -1  # rows that get no page: q only
    qkv = torch.randn(rows, (hq + 2 * hk) * hd, generator=g, device=DEV).to(_DT[c["dt"]])
    gam = (1 + 0.1 * rs.randn(2, hd)).astype(np.float32)
    kv = torch.randn(2, blocks, hk, PAGE, hd, generator=g, device=DEV, dtype=torch.float16)
    return dict(op="qk", hq=hq, hk=hk, hd=hd, qkv=qkv, positions=_i32(rs.randint(0, c["far"], rows)), slots=_gpu(slots),
                inv_freq=_gpu(_inv_freq(hd)), qg=_gpu(gam[0]) if c["norm"] else None,
                kg=_gpu(gam[1]) if c["norm"] else None, v_norm=c["v_norm"], k=kv[0], v=kv[1], eps=1e-6)


def _attn_lens(c):
    return _spread(c["ctx_lo"], c["ctx_hi"], c["batch"], 4), _spread(c["q_lo"], c["q_hi"], c["batch"], 5)


def _prepare_attn(c, seed):
    rs = np.random.RandomState(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    ctx, q = _attn_lens(c)
    n, hq, hk, hd = c["batch"], c["hq"], c["hk"], c["hd"]
    if c["holes"]:
        ctx[0] = 0  # a sequence without context: a row with an empty mask then has no key at all
    pages = -(-(ctx + q) // PAGE)
    mb, blocks = int(pages.max()), int(pages.sum()) + 2
    table = np.full((n, mb), -1, np.int32)
    table[np.arange(mb)[None] < pages[:, None]] = rs.permutation(blocks)[: pages.sum()]
    cu = np.concatenate([[0], np.cumsum(q)])
    words = -(-int(q.max()) // 32) if c["tree"] else 0
    masks, depths = [], []
    for k in q if c["tree"] else []:
        bits, depth = _ancestors(_parents(rs, int(k)))
        if c["holes"]:
            bits[rs.rand(int(k)) < 0.2] = False
        masks.append(_pack(bits, words))
        depths.append(depth)
    pos = np.concatenate([x + (depths[b] if c["tree"] else np.arange(q[b])) for b, x in enumerate(ctx)])
    kv = torch.randn(2, blocks, hk, PAGE, hd, generator=g, device=DEV, dtype=torch.float16)
    qs = torch.randn(int(cu[-1]), hq * hd, generator=g, device=DEV).to(_DT[c["dt"]])
    # a flat [sequence, node] index of the rows, kept with the step's plan
    seq = np.repeat(np.arange(n), q)
    node = np.arange(cu[-1]) - cu[seq]
    return dict(op="attn", hq=hq, hk=hk, hd=hd, q=qs, k=kv[0], v=kv[1], table=_i32(table), ctx=_i32(ctx), cu=_i32(cu),
                mask=_gpu(np.concatenate(masks)) if c["tree"] else None, positions=_i32(pos), max_q=int(q.max()),
                max_ctx=int((ctx + q).max()), window=c["window"], seq=_gpu(seq), node=_gpu(node))


def _prepare_score(c, seed):
    rs = np.random.RandomState(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows, vocab = c["rows"], c["vocab"]
    x = (torch.randn(rows, vocab, generator=g, device=DEV) * 2.5).to(_DT[c["dt"]])
    top = torch.randint(0, vocab, (rows, 4), generator=g, device=DEV)
    x.scatter_add_(1, top, (10 * torch.rand(rows, 4, generator=g, device=DEV)).to(x.dtype))  # a few likely tokens
    if c["banned"]:  # guided decoding: most of a row forbidden, with -inf or the type's lowest value
        some = torch.rand(rows, generator=g, device=DEV) < 0.25
        ban = (torch.rand(vocab, generator=g, device=DEV) < 0.9)[None] & some[:, None]
        x.masked_fill_(ban, -math.inf if seed % 2 else _LOWEST[c["dt"]])
    t = rs.randint(0, vocab, (rows, c["targets"]))
    t[:, 0] = top[:, 0].cpu().numpy()
    return dict(op="score", logits=x, targets=_i32(t), k=c["k"])


def prepare(case, seed):
    return {"plan": _prepare_plan, "qk": _prepare_qk, "attn": _prepare_attn, "score": _prepare_score}[case["op"]](case, seed)


# -- the plain forms -------------------------------------------------------------------------------


def _plan(s):
    ctx, q, table, have = s["ctx"].long(), s["q"].long(), s["table"], s["n_pages"].long()
    n, mb = table.shape
    rows, dev = s["rows"], table.device
    ended, add = q < 0, q.clamp(min=0)
    # pages of ended requests go onto the stack in order, then new ones come off its top
    col = torch.arange(mb, device=dev)
    back = torch.where(ended, have, 0)
    start = s["n_free"].long() + back.cumsum(0) - back
    at = torch.where(col[None] < back[:, None], start[:, None] + col[None], len(s["stack"]))
    stack = torch.cat([s["stack"], s["stack"].new_zeros(1)]).scatter(0, at.reshape(-1), table.reshape(-1))[:-1]
    top = s["n_free"].long() + back.sum()
    need = torch.where(ended, 0, ((ctx + add + PAGE - 1) // PAGE - have).clamp(min=0))
    end = need.cumsum(0)
    ok = (end <= top) | (need == 0)
    got = torch.where(ok, need, 0)
    j = col[None] - have[:, None]
    take = (top - 1 - (end - need)[:, None] - j).clamp(0, max(0, len(stack) - 1))
    fresh = (j >= 0) & (j < got[:, None])
    new_table = torch.where(fresh, stack[take], table)
    cu = torch.cat([add.new_zeros(1), add.cumsum(0)])
    # rows of tokens; those behind the last request keep what they held
    row = torch.arange(rows, device=dev)
    live = row < cu[-1]
    seq = torch.searchsorted(cu[1:].contiguous(), row, right=True).clamp(max=n - 1)
    i = row - cu[seq]
    at = ctx[seq] + i
    page = new_table[seq, (at // PAGE).clamp(0, mb - 1)].long()
    slots = torch.where(live, torch.where(ok[seq] & (page >= 0), page * PAGE + at % PAGE, -1), s["slots"])
    depth, mask = i, s["mask"]
    if mask is not None:
        m = s["nodes"]
        here = torch.arange(m, device=dev)
        flat = (cu[:-1, None] + here[None]).clamp(max=rows - 1)
        par = torch.where(here[None] < add[:, None], s["parents"].long()[flat], -1)
        reach = (here[None, None] == here[None, :, None]) | (here[None, None] == par[:, :, None])
        reach = reach.float()
        for _ in range(max(1, (m - 1).bit_length())):  # paths of twice the length each time
            reach = (reach @ reach > 0).float()
        mine = reach[seq, i.clamp(0, m - 1)]
        depth = mine.sum(1).long() - 1
        wide = torch.zeros(rows, 32 * s["words"], dtype=torch.long, device=dev)
        wide[:, :m] = mine.long()
        word = (wide.view(rows, -1, 32) << torch.arange(32, device=dev)).sum(2)
        word = torch.where(word >= 2**31, word - 2**32, word).int()
        mask = torch.where(live[:, None], word, mask)
    positions = torch.where(live, (ctx[seq] + depth).int(), s["positions"])
    out = dict(cu_q=cu.int(), slots=slots, positions=positions, status=torch.where(ok, 0, 1).int(),
               n_pages=torch.where(ended, 0, have + got).int(), n_free=(top - got.sum()).int().view(1), table=new_table,
               stack=stack)
    return out if mask is None else out | dict(mask=mask)


def _rms(x, gamma, eps):
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    return x if gamma is None else x * gamma


def _qk(s):
    hq, hk, hd = s["hq"], s["hk"], s["hd"]
    x = s["qkv"].float().view(len(s["qkv"]), hq + 2 * hk, hd)
    q, k, v = x[:, :hq], x[:, hq : hq + hk], x[:, hq + hk :]
    if s["qg"] is not None:
        q, k = _rms(q, s["qg"], s["eps"]), _rms(k, s["kg"], s["eps"])
    if s["v_norm"]:
        v = _rms(v, None, s["eps"])
    a = s["positions"].double()[:, None] * s["inv_freq"].double()[None]
    cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]

    def turn(t):
        lo, hi = t[..., : hd // 2], t[..., hd // 2 :]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)

    put = s["slots"] >= 0
    page, at = s["slots"][put] // PAGE, s["slots"][put] % PAGE
    s["k"][page, :, at] = turn(k)[put].half()
    s["v"][page, :, at] = v[put].half()
    return dict(q=turn(q).to(s["qkv"].dtype).reshape(len(x), hq * hd), k=s["k"], v=s["v"])


def _attn(s):
    hq, hk, hd, t = s["hq"], s["hk"], s["hd"], s["max_q"]
    n, keys = len(s["ctx"]), s["max_ctx"]
    seq, node, dev = s["seq"], s["node"], s["q"].device
    pages = s["table"][:, : -(-keys // PAGE)].long().clamp(min=0)
    k = s["k"][pages].transpose(1, 2).reshape(n, hk, -1, hd)[:, :, :keys].float()
    v = s["v"][pages].transpose(1, 2).reshape(n, hk, -1, hd)[:, :, :keys].float()
    q = torch.zeros(n, t, hq, hd, device=dev)
    q[seq, node] = s["q"].float().view(-1, hq, hd)
    q = q.view(n, t, hk, hq // hk, hd).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, hd)
    # which keys a row sees: all of the context, and of the step's own tokens those of its mask
    ctx, key = s["ctx"].long(), torch.arange(keys, device=dev)
    other = key[None] - ctx[:, None]  # the key's number among the step's tokens
    if s["mask"] is None:
        sees = (other[seq] <= node[:, None]) & (key[None] < (ctx + s["cu"][1:] - s["cu"][:-1])[seq][:, None])
    else:
        j = other[seq].clamp(0, 32 * s["mask"].shape[1] - 1)
        bit = (s["mask"].gather(1, j >> 5) >> (j & 31).int()) & 1
        count = (s["cu"][1:] - s["cu"][:-1])[seq][:, None]
        sees = (other[seq] < 0) | ((other[seq] < count) & (bit == 1))
    if s["window"]:
        flat = (s["cu"].long()[:-1, None] + other.clamp(min=0)).clamp(max=len(node) - 1)
        where = torch.where(other < 0, key[None], s["positions"].long()[flat])  # positions of the keys
        sees = sees & (where[seq] > s["positions"].long()[:, None] - s["window"])
    allow = torch.zeros(n, t, keys, dtype=torch.bool, device=dev)
    allow[seq, node] = sees
    allow = allow[:, None, None].expand(n, 1, hq // hk, t, keys).reshape(n, 1, -1, keys)
    p = (q @ k.transpose(2, 3)) / math.sqrt(hd)
    p = p.masked_fill_(~allow, -math.inf)
    p = (p - p.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total > 0, total, 1)
    o = o.view(n, hk, hq // hk, t, hd).permute(0, 3, 1, 2, 4).reshape(n, t, hq * hd)
    return o[seq, node].to(s["q"].dtype)


def _score(s):
    x, t, k = s["logits"].float(), s["targets"].long(), s["k"]
    top = x.amax(1, keepdim=True)
    z = x - top
    e = z.exp()
    total = e.sum(1, keepdim=True)
    mean = torch.where(e > 0, z * e, 0).sum(1, keepdim=True) / total
    lse = total.log()
    out = dict(logprobs=z.gather(1, t) - lse, entropy=(lse - mean)[:, 0])
    if k:
        # one whole number per entry that grows with the value and, among equals, falls with the index
        b = (x + 0.0).view(torch.int32).long()
        order = torch.where(b < 0, -(b & 0x7FFFFFFF), b)
        order = (order << 32) + (0x7FFFFFFF - torch.arange(x.shape[1], device=x.device))
        ids = 0x7FFFFFFF - (order.topk(k, 1).values & 0xFFFFFFFF)
        out |= dict(top_ids=ids.int(), top_logprobs=z.gather(1, ids) - lse)
    return out


# -- the framework's operators ------------------------------------------------------------------------


def _own(s):
    from gemmagemini4hackathon2026_10_2425_b200 import ops

    if s["op"] == "plan":
        out = ops.PagedPlan(s["cu"], s["slots"], s["positions"], s["mask"], s["status"], s["n_pages_out"], s["n_free_out"])
        ops.paged_plan(s["ctx"], s["q"], s["table"], s["n_pages"], s["stack"], s["n_free"], s["rows"],
                       parents=s["parents"], mask_words=s["words"], out=out)
        out = dict(cu_q=s["cu"], slots=s["slots"], positions=s["positions"], status=s["status"],
                   n_pages=s["n_pages_out"], n_free=s["n_free_out"], table=s["table"], stack=s["stack"])
        return out if s["mask"] is None else out | dict(mask=s["mask"])
    if s["op"] == "qk":
        q = ops.qk_norm_rope_append(s["qkv"], s["positions"], s["slots"], s["inv_freq"], s["k"], s["v"], s["hq"], s["hk"],
                                    s["hd"], q_gamma=s["qg"], k_gamma=s["kg"], eps=s["eps"], v_norm=s["v_norm"],
                                    out_dtype=s["qkv"].dtype)
        return dict(q=q, k=s["k"], v=s["v"])
    if s["op"] == "attn":
        return ops.paged_tree_attn(s["q"], s["k"], s["v"], s["table"], s["ctx"], s["cu"], s["hq"], s["hk"], s["hd"],
                                   s["max_q"], s["max_ctx"], mask=s["mask"], positions=s["positions"], window=s["window"],
                                   out_dtype=s["q"].dtype)
    r = ops.token_logprobs(s["logits"], s["targets"], s["k"])
    out = dict(logprobs=r.logprobs, entropy=r.entropy)
    return out | dict(top_ids=r.top_ids, top_logprobs=r.top_logprobs) if s["k"] else out


def run(state):
    if own:
        return _own(state)
    return {"plan": _plan, "qk": _qk, "attn": _attn, "score": _score}[state["op"]](state)


# -- what a pass cannot do without -------------------------------------------------------------------


def work(case):
    c = case
    if c["op"] == "plan":
        ctx, q = _plan_lens(c)
        add = np.maximum(q, 0)
        pages = int((-(-(ctx + add) // PAGE) - ctx // PAGE)[q > 0].sum()) + int((-(-ctx // PAGE))[q < 0].sum())
        per_token = 12 + (4 + 4 * -(-max(1, c["q_hi"]) // 32) if c["tree"] else 0)
        return {"bytes": 24 * c["batch"] + 8 * pages + per_token * int(add.sum()), "flops": max(1, int(add.sum()))}
    if c["op"] == "qk":
        size = 4 if c["dt"] == "f32" else 2
        q, kv = c["hq"] * c["hd"], 2 * c["hk"] * c["hd"]
        return {"bytes": c["rows"] * (size * (2 * q + kv) + 2 * kv + 12), "flops": c["rows"] * 8 * (q + kv)}
    if c["op"] == "attn":
        ctx, q = _attn_lens(c)
        if c["holes"]:
            ctx[0] = 0
        size = 4 if c["dt"] == "f32" else 2
        low = np.maximum(0, ctx - c["window"] + 1) if c["window"] else np.zeros_like(ctx)
        kv = int((ctx + q - low).sum()) * 2 * c["hk"] * c["hd"] * 2
        # rows x keys: the context (within the window), and half of the step's own tokens (a tree's rows see fewer)
        seen = int((q * np.minimum(ctx, c["window"] or ctx) + (0 if c["tree"] else q * (q + 1) // 2)).sum())
        return {"bytes": kv + int(q.sum()) * 2 * c["hq"] * c["hd"] * size, "flops": max(1, seen) * 4 * c["hq"] * c["hd"]}
    n = c["rows"] * c["vocab"]
    return {"bytes": n * (4 if c["dt"] == "f32" else 2) + c["rows"] * (8 * c["k"] + 8 * c["targets"] + 4), "flops": 4 * n}


# -- the definitions in 64 bits -----------------------------------------------------------------------


def _exact_plan(c, s):
    h = {k: v.cpu().numpy().copy() for k, v in s.items() if torch.is_tensor(v)}
    stack, table = h["stack"], h["table"]
    top = int(h["n_free"][0])
    for b in np.flatnonzero(h["q"] < 0):
        stack[top : top + h["n_pages"][b]] = table[b, : h["n_pages"][b]]
        top += int(h["n_pages"][b])
    cu, status, owned, asked, given = [0], [], [], 0, 0
    for b, q in enumerate(h["q"]):
        x, have = int(h["ctx"][b]), int(h["n_pages"][b])
        want = max(0, -(-(x + int(q)) // PAGE) - have) if q >= 0 else 0
        fits = want == 0 or asked + want <= top
        if fits:
            table[b, have : have + want] = stack[top - asked - want : top - asked][::-1]
            given += want
        asked += want
        status.append(0 if fits else 1)
        owned.append(0 if q < 0 else have + (want if fits else 0))
        n, r = max(0, int(q)), cu[-1]
        at = x + np.arange(n)
        if n:
            h["slots"][r : r + n] = table[b, at // PAGE] * PAGE + at % PAGE if fits else -1
            h["positions"][r : r + n] = at
            if c["tree"]:
                bits, depth = _ancestors(h["parents"][r : r + n])
                h["positions"][r : r + n] = x + depth
                h["mask"][r : r + n] = _pack(bits, s["words"])
        cu.append(r + n)
    i32 = lambda v: np.array(v, np.int32)  # noqa: E731
    out = dict(cu_q=i32(cu), slots=h["slots"], positions=h["positions"], status=i32(status), n_pages=i32(owned),
               n_free=i32([top - given]), table=table, stack=stack)
    return out | dict(mask=h["mask"]) if c["tree"] else out


def _exact_qk(c, s):
    hq, hk, hd = s["hq"], s["hk"], s["hd"]
    x = s["qkv"].double().view(-1, hq + 2 * hk, hd)
    scale = (x.square().sum(-1, keepdim=True) / hd + s["eps"]).pow(-0.5)
    qk, v = x[:, : hq + hk], x[:, hq + hk :]
    if s["v_norm"]:
        v = v * scale[:, hq + hk :]
    if s["qg"] is not None:
        gam = torch.cat([s["qg"].expand(hq, hd), s["kg"].expand(hk, hd)]).double()
        qk = qk * scale[:, : hq + hk] * gam
    turn = torch.polar(torch.ones(len(x), hd // 2, dtype=torch.double, device=x.device),
                       torch.outer(s["positions"].double(), s["inv_freq"].double()))
    z = torch.complex(qk[..., : hd // 2].contiguous(), qk[..., hd // 2 :].contiguous()) * turn[:, None]
    qk = torch.cat([z.real, z.imag], -1)
    pages = []
    for pool, new in ((s["k"], qk[:, hq:]), (s["v"], v)):
        flat = pool.double().transpose(1, 2).reshape(-1, hk, hd)
        flat[s["slots"][s["slots"] >= 0]] = new[s["slots"] >= 0]
        pages.append(flat.view(-1, PAGE, hk, hd).transpose(1, 2))
    return dict(q=qk[:, :hq].reshape(len(x), -1), k=pages[0], v=pages[1])


def _exact_attn(c, s):
    hq, hk, hd = s["hq"], s["hk"], s["hd"]
    ctx, q = _attn_lens(c)
    if c["holes"]:
        ctx[0] = 0
    if float((ctx + q) @ q) * hq * hd > 4e11:
        return None
    out = torch.zeros(len(s["q"]), hq, hd, dtype=torch.double, device=s["q"].device)
    r = 0
    for b in range(len(ctx)):
        n, t = int(ctx[b] + q[b]), int(q[b])
        ids = s["table"][b, : -(-n // PAGE)].long()
        k = s["k"][ids].double().permute(0, 2, 1, 3).reshape(-1, hk, hd)[:n]
        v = s["v"][ids].double().permute(0, 2, 1, 3).reshape(-1, hk, hd)[:n]
        see = torch.ones(t, n, dtype=torch.bool, device=out.device)
        pos = s["positions"][r : r + t].long()
        if c["tree"]:
            words = s["mask"][r : r + t].cpu().numpy().view(np.uint8)
            see[:, int(ctx[b]) :] = _gpu(np.unpackbits(words, axis=1, bitorder="little")[:, :t].astype(bool))
        else:
            see = see.tril(int(ctx[b]))
        if c["window"]:
            at = torch.cat([torch.arange(int(ctx[b]), device=out.device), pos])
            see &= at[None] > pos[:, None] - c["window"]
        for h in range(hk):
            rows = s["q"][r : r + t].double().view(t, hq, hd)[:, h * (hq // hk) : (h + 1) * (hq // hk)].transpose(0, 1)
            w = (rows @ k[:, h].T * hd**-0.5).masked_fill(~see[None], -math.inf)
            w = torch.nan_to_num(torch.softmax(w, -1), nan=0.0)
            out[r : r + t, h * (hq // hk) : (h + 1) * (hq // hk)] = (w @ v[:, h]).transpose(0, 1)
        r += t
    return out.view(len(out), -1)


def _exact_score(c, s):
    parts = []
    for x, t in zip(s["logits"].split(128), s["targets"].split(128)):
        lp = torch.log_softmax(x.double(), 1)
        r = dict(logprobs=lp.gather(1, t.long()), entropy=-torch.special.xlogy(lp.exp(), lp.exp()).sum(1))
        if s["k"]:
            ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, : s["k"]]
            r |= dict(top_ids=ids.int(), top_logprobs=lp.gather(1, ids))
        parts.append(r)
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "qk": _exact_qk, "attn": _exact_attn, "score": _exact_score}[case["op"]](case, s)
