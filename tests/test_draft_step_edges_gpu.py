"""The drafted-token step's operators at the edges of their ranges: finite bans and large logits,
non-finite values in hidden places, weak keys beside a strong one, large scores, refused requests.
Helpers and the oracle's tolerances are test_draft_step_gpu.py's."""

import numpy as np
import pytest
import torch

from test_draft_step_gpu import DEV, attn_case, check_attn, check_score

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
