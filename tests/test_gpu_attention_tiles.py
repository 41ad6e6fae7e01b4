"""The forms of the attention that share the cache between waves, in tiles of 64 and 128 rows: several query heads a token, so
that a tile, a wave's 32 rows and a token's heads end in different places. And the join in the same launch, on any workspace."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aklr_amd
from aklr_amd import workspace
from tests.helpers import say
from tests.test_gpu_attention import call, i32, problem, tree
from tests.test_gpu_attention_weights import FORMS, FORMS_OF, check, exact, lost, reach
from tests.test_gpu_kv_cache import BF16, DEV, F16

pytestmark = pytest.mark.gpu

# head_dim, kv heads, group, query tokens and positions of each sequence, page: rows of a tile
TILES = [
    (64, 64, 7, [19, 7], [1500, 7], 16, 128),  # 133 rows: a second tile of 5; no context
    (64, 64, 4, [20, 10], [900, 333], 48, 64),
    (128, 32, 4, [33, 1, 0, 28], [2100, 40, 5, 700], 64, 64),  # 132 rows: a third tile of 4
    (128, 64, 5, [60, 40], [64, 1111], 16, 128),
    (128, 16, 7, [50, 3, 37, 1, 0, 2, 19, 40], [50, 900, 300, 1, 0, 260, 129, 1000], 32, 128),
    (256, 16, 7, [25, 5, 0, 12], [777, 6, 300, 1024], 48, 128),
    (256, 32, 4, [16, 12], [1300, 12], 64, 64),
    (256, 64, 3, [41, 90], [128, 90], 16, 128),
]


def some(rng, t):
    return rng.random((t, t)) < 0.2


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("mask", [None, tree, some])
@pytest.mark.parametrize("d,h,group,counts,lens,page,rows", TILES)
def test_several_heads_of_a_token(d, h, group, counts, lens, page, rows, mask, dtype):
    say(f"tiles {d} {h} {group} {counts} {rows} {mask and mask.__name__} {dtype}")
    p = problem(lens, counts, h, group, d, page, dtype, seed=31, mask=mask, extra_q=2)
    check(p, rows)
    out = torch.full_like(p["q"], 7.0)
    call(p, out=out)
    assert bool((out[sum(counts):] == 7).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,form", FORMS_OF)
def test_a_score_is_an_fp32_sum_in_every_form(d, form, dtype):
    # Every token sees one position, itself: the log of its sum is its score. d exact products, summed with a rounding of at
    # most 2^-24 of their size each, three scalings; with the score x in powers of two, a reference of at most |x| + 20, four
    # roundings of that size around the exponential and the logarithm of a weight between 2^-20 and 2^20.
    say(f"scores {d} {form} {dtype}")
    b, t, h, group = FORMS[form]
    p = problem([t] * b, [t] * b, h, group, d, 16, dtype, seed=29, mask=lambda rng, n: np.eye(n, dtype=bool))
    reach(p, form)
    out, lse = call(p, return_lse=True)
    want, wl, weighed, size, _ = exact(p, d ** -0.5)
    assert bool(((lse.double() - wl).abs() <= 2**-24 * ((d + 3) * size + 4 * wl.abs() / np.log(2) + 128)).all())
    tol = want.abs() * (torch.finfo(dtype).eps / 2 + lost(form, dtype)) * 1.01 + 2**-25
    assert bool(((out.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("d,h,b,group,page,rows", [(64, 64, 64, 35, 16, 128), (128, 64, 128, 20, 32, 64), (256, 32, 32, 31, 64, 128)])
def test_one_piece_of_each_tile(d, h, b, group, page, rows):
    # no more than 128 positions: nothing to join, and no workspace
    say(f"one piece {d} {rows}")
    counts = [[3, 1, 0, 5, 2][i % 5] for i in range(b)]
    p = problem([128 if i == 0 else c + 13 * i % 120 for i, c in enumerate(counts)], counts, h, group, d, page, BF16, seed=33, mask=tree)
    assert p["table"].shape[1] * page == 128
    check(p, rows, joined=False)
    p["mask"] = None
    check(p, rows, joined=False)


@pytest.mark.parametrize("d,h,group,counts,lens,page,rows", [TILES[0], TILES[2], TILES[5]])
def test_lengths_below_the_counts_and_missing_pages(d, h, group, counts, lens, page, rows):
    say(f"short and missing {d} {rows}")
    p = problem(lens, counts, h, group, d, page, BF16, seed=35)
    p["lens"] = i32([n if i else max(0, counts[0] - 6) for i, n in enumerate(lens)])
    check(p, rows)
    p = problem(lens, counts, h, group, d, page, BF16, seed=36, mask=tree)
    p["table"][0, 3], p["table"][0, 8], p["table"][-1, 0] = -1, p["cache"][0].shape[0], 2**31 - 1
    check(p, rows)
    p["mask"] = torch.zeros_like(p["mask"])
    p["lens"] = p["starts"][1:] - p["starts"][:-1]  # no context, and nothing of the drafts
    check(p, rows)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("d,h,group,counts,lens,page,rows", [TILES[0], TILES[2], TILES[4], TILES[5], TILES[6]])
def test_nothing_unseen_reaches_a_row(d, h, group, counts, lens, page, rows, masked):
    say(f"NaN and infinities not seen {d} {rows} {masked}")
    p = problem(lens, counts, h, group, d, page, BF16, seed=37, mask=tree if masked else None)
    reach(p, rows)
    want = call(p, return_lse=True)
    used = torch.zeros(p["cache"][2].shape[0], page, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        at = torch.arange(n, device=DEV)
        used[p["table"][b].long()[at // page], at % page] = True
    for c in p["cache"][:2]:
        c.view(torch.uint8).masked_fill_(~used[:, None, :, None], 0x7F)
    for c, bad in zip(p["cache"][2:], (float("inf"), float("nan"))):
        c.masked_fill_(~used[:, None, :], bad)
    assert all(torch.equal(a, b) for a, b in zip(call(p, return_lse=True), want))
    b = int(np.argmax(counts))
    t, first = counts[b] // 2, sum(counts[:b])
    pos = lens[b] - counts[b] + t
    place = (p["table"][b, pos // page].long(), slice(None), pos % page)
    p["cache"][0].view(torch.uint8)[place + (3,)] = 0xFF
    p["cache"][1].view(torch.uint8)[place + (5,)] = 0x7F
    out, lse = call(p, return_lse=True)
    tokens = torch.arange(p["q"].shape[0], device=DEV)
    sees = (tokens >= first) & (tokens < first + counts[b])
    sees &= p["mask"][:, t] if masked else tokens >= first + t
    assert bool(out[sees].isnan().all()) and bool(lse[sees].isnan().all())
    assert torch.equal(out[~sees], want[0][~sees]) and torch.equal(lse[~sees], want[1][~sees])


@pytest.mark.parametrize("d,h,group,counts,lens", [(64, 1, 4, [1, 1], [300, 310]), (128, 8, 4, [1], [900]), (256, 2, 8, [2, 1, 1], [200, 1, 390])])
def test_the_last_workgroup_joins_on_any_workspace(d, h, group, counts, lens):
    say(f"arrival words {d} {h} {lens}")
    p = problem(lens, counts, h, group, d, 16, BF16, seed=39)
    check(p, 16, joined=False)
    want = call(p, return_lse=True)
    args = (p["q"], *p["cache"], p["table"], p["lens"], p["starts"], p["mask"])
    real, asked = workspace.get, []
    for fill in (0xFF, 0x7F, 0x80, 0x01, 0x00):
        def filled(device, nbytes):
            asked.append(nbytes)
            t = real(device, nbytes)
            return t if t is None else t.fill_(fill)
        try:
            workspace.get = filled
            got = [aklr_amd.tree_attention_fp8.general(*args, return_lse=True) for _ in range(3)]
        finally:
            workspace.get = real
        assert all(torch.equal(a, b) for g in got for a, b in zip(g, want)), fill
    assert min(asked) > 0  # several pieces


def test_a_workspace_of_an_earlier_call_serves():
    # words and partial results that an earlier call of another shape left
    say("used workspace")
    big = problem([900, 700], [1, 1], 8, 4, 128, 16, BF16, seed=41)
    small = problem([300, 310], [1, 1], 8, 2, 128, 16, BF16, seed=42)
    memory = torch.empty(64 << 20, dtype=torch.uint8, device=DEV)
    want = [call(p, return_lse=True) for p in (big, small)]
    real = workspace.get
    try:
        workspace.get = lambda device, nbytes: memory[:nbytes]
        for _ in range(3):
            for p, w in zip((big, small), want):
                got = aklr_amd.tree_attention_fp8.general(p["q"], *p["cache"], p["table"], p["lens"], p["starts"], p["mask"], return_lse=True)
                assert all(torch.equal(a, b) for a, b in zip(got, w))
    finally:
        workspace.get = real
