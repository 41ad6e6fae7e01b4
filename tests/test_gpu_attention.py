"""Attention over the FP8 cache on the GPU, against the 64-bit oracle.

Tolerance. A score's products are exact in fp32 (8 by 4, or 11 by 4, bits), their sum and the two scalings round at most
head_dim + 2 times by 2^-24 of scale * sum |q_d k_d| =: size, at head_dim <= 256 under 2^-15 * size; exp2 and its
argument add under 2^-20. So a weight is off by a factor of 1 + e, e <= 2^-15 * size + 2^-20 (and its rounding to bf16
before the second product, 2^-8), the sum of weights by 1 + e, and an output by at most (2^-8 + 2e + 2^-18) times the
weighted sum of |v|, plus half a step of its type. The log of the sum is off by e + 2^-21 * (1 + |lse|).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aklr_amd
from oracle import cache as oc
from tests.helpers import say, u8
from tests.test_gpu_kv_cache import BF16, DEV, F16, gen, new_cache, normal

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)


def problem(lens, counts, h, group, d, page, dtype=BF16, seed=0, mask=None, spare=2, extra_q=0, extra_cols=0):
    """q, a cache of quantized random keys and values on shuffled pages, block table, lens, starts, mask."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    cache = new_cache(pages, h, d, page)
    every = torch.arange(pages * page, device=DEV)
    aklr_amd.kv_cache_write_fp8(normal((pages * page, h, d), BF16, seed + 1), normal((pages * page, h, d), BF16, seed + 2), *cache, every)
    order = torch.randperm(pages, generator=gen(seed + 3), device=DEV).to(torch.int32)
    table = torch.zeros((len(lens), max([1] + need) + extra_cols), dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    q = normal((sum(counts) + extra_q, h * group, d), torch.float32, seed + 4).mul(2).to(dtype)
    starts = np.r_[0, np.cumsum(counts)]
    m = None
    if mask is not None:
        m = torch.zeros((q.shape[0], max([1] + counts)), dtype=torch.bool, device=DEV)
        rng = np.random.default_rng(seed)
        for b, t in enumerate(counts):
            m[starts[b]:starts[b] + t, :t] = torch.from_numpy(mask(rng, t)).to(DEV)
    return {"q": q, "cache": cache, "table": table, "lens": i32(lens), "starts": i32(starts), "mask": m}


def tree(rng, t):
    m = np.zeros((t, t), bool)
    for i in range(t):
        if i and (parent := rng.integers(-1, i)) >= 0:
            m[i] = m[parent]
        m[i, i] = True
    return m


def call(p, **kw):
    return aklr_amd.tree_attention_fp8(p["q"], *p["cache"], p["table"], p["lens"], p["starts"], p["mask"], **kw)


def check(p, got, lse, scale=None, what=""):
    d = p["q"].shape[2]
    scale = d ** -0.5 if scale is None else scale
    end = int(p["starts"][-1])
    want, wl, weighed, size = oc.attention(
        p["q"].double().cpu().numpy()[:end], u8(p["cache"][0]), u8(p["cache"][1]), *(t.cpu().numpy() for t in p["cache"][2:]),
        p["table"].cpu().numpy(), p["lens"].cpu().numpy(), p["starts"].cpu().numpy(),
        None if p["mask"] is None else p["mask"].cpu().numpy(), scale)
    e = 2**-15 * size + 2**-20
    out = got.double().cpu().numpy()[:end]
    assert np.array_equal(np.isnan(out), np.isnan(want)), what
    tol = weighed * (2**-8 + 2 * e[..., None] + 2**-18)
    tol = tol + np.abs(want) * torch.finfo(p["q"].dtype).eps / 2 * 1.01 + 2**-25
    far = np.abs(out - want) - tol
    assert (far[~np.isnan(want)] <= 0).all(), f"{what}: {np.nanmax(far)} past the tolerance"
    empty = wl == -np.inf
    assert (out[empty] == 0).all()
    if lse is not None:
        l = lse.double().cpu().numpy()[:end]
        assert lse.dtype == torch.float32 and (l[empty] == -np.inf).all()
        ok = ~empty & ~np.isnan(wl)
        assert np.array_equal(np.isnan(l), np.isnan(wl))
        assert (np.abs(l[ok] - wl[ok]) <= e[ok] + 2**-21 * (1 + np.abs(wl[ok]))).all(), what


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens,h,group,page", [([1], 1, 1, 16), ([17, 128, 129], 2, 4, 16), ([700, 1, 0, 33], 1, 7, 48),
                                               ([2049], 8, 16, 64), ([300, 31], 3, 24, 128)])
def test_decode(lens, h, group, page, d, dtype):
    say(f"decode {lens} {h} {group} {page} {d} {dtype}")
    p = problem(lens, [1] * len(lens), h, group, d, page, dtype)
    out, lse = call(p, return_lse=True)
    assert out.dtype == dtype and out.shape == p["q"].shape
    check(p, out, lse)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("lens,counts,h,group,d,page", [
    ([5], [5], 1, 1, 64, 16),  # no context
    ([40, 300, 64], [8, 1, 33], 2, 4, 128, 16),  # drafts on both sides of a page's and a step's end
    ([130, 16, 900, 47], [3, 0, 64, 47], 1, 5, 128, 48),
    ([513, 100], [9, 100], 2, 1, 256, 64),
    ([2000], [70], 1, 8, 64, 32),  # more drafts than 64
    ([260], [257], 1, 3, 128, 16)])
def test_trees_and_chains(lens, counts, h, group, d, page, masked, dtype):
    say(f"trees {lens} {counts} {h} {group} {d} {page} {masked} {dtype}")
    p = problem(lens, counts, h, group, d, page, dtype, mask=tree if masked else None)
    out, lse = call(p, return_lse=True, softmax_scale=0.11)
    check(p, out, lse, scale=0.11)
    assert torch.equal(out, call(p, softmax_scale=0.11))  # and the same every time


def test_many_sequences_and_ragged_counts():
    say("200 sequences")
    rng = np.random.default_rng(3)
    counts = [int(c) for c in rng.integers(0, 4, 200)]
    lens = [int(c + x) for c, x in zip(counts, rng.integers(0, 90, 200))]
    p = problem(lens, counts, 1, 2, 64, 16, mask=tree)
    check(p, *call(p, return_lse=True))


def test_rows_that_see_nothing_and_rows_behind_the_last_sequence():
    say("empty rows, padded rows")
    p = problem([9, 0, 3, 40], [4, 2, 3, 3], 2, 2, 128, 16, mask=lambda rng, t: rng.random((t, t)) < 0.3, extra_q=5)
    p["mask"][4:6] = True  # a sequence of no positions
    p["mask"][6] = False  # no context and no draft seen
    out = torch.full_like(p["q"], 7.0)
    got, lse = call(p, return_lse=True, out=out)
    assert got is out
    check(p, got, lse)
    assert (lse[6] == float("-inf")).all() and not out[6].any() and not out[4:6].any()
    assert (out[12:] == 7).all()
    # fewer positions than query tokens: the first ones have none
    p = problem([3], [5], 1, 2, 64, 16)
    check(p, *call(p, return_lse=True))
    # a mask narrower than the drafts: what it does not hold is not seen
    p = problem([30], [6], 1, 2, 64, 16, mask=tree)
    p["mask"] = p["mask"][:, :2].contiguous()
    check(p, *call(p, return_lse=True))
    # no column at all in the block table
    p = problem([0], [2], 1, 2, 64, 16)
    p["table"], p["lens"] = p["table"][:, :0], i32([50])
    out, lse = call(p, return_lse=True)
    assert not out.any() and (lse == float("-inf")).all()


@pytest.mark.parametrize("d,page", [(64, 16), (128, 48), (256, 64)])
def test_nothing_unseen_reaches_a_row(d, page):
    say(f"NaN and infinities in places that are not seen, {d} {page}")
    counts, lens = [7, 40], [page + 20, 200]
    p = problem(lens, counts, 2, 3, d, page, mask=tree, extra_cols=2)
    clean = call(p, return_lse=True)
    used = torch.zeros(p["cache"][2].shape[0], page, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        for pos in range(n):
            used[p["table"][b, pos // page], pos % page] = True
    for c in p["cache"][:2]:
        c.view(torch.uint8).masked_fill_(~used[:, None, :, None], 0x7F)
    for c, bad in zip(p["cache"][2:], (float("inf"), float("nan"))):
        c.masked_fill_(~used[:, None, :], bad)
    for got, want in zip(call(p, return_lse=True), clean):
        assert torch.equal(got, want)
    # a draft that is itself all NaN: only rows that see it turn NaN
    for codes_bad in (True, False):
        q = {**p, "cache": tuple(c.clone() for c in p["cache"])}
        pos = lens[1] - counts[1] + 3
        page_id, off = int(p["table"][1, pos // page]), pos % page
        if codes_bad:
            q["cache"][0].view(torch.uint8)[page_id, :, off, 3] = 0x7F
            q["cache"][1].view(torch.uint8)[page_id, :, off] = 0xFF
        else:
            q["cache"][2][page_id, :, off] = float("nan")
            q["cache"][3][page_id, :, off] = float("inf")
        out, lse = call(q, return_lse=True)
        sees = p["mask"][7:, 3]
        assert out[7:][sees].isnan().all() and lse[7:][sees].isnan().all()
        for got, want in zip((out, lse), clean):
            assert torch.equal(got[7:][~sees], want[7:][~sees]) and torch.equal(got[:7], want[:7])


def test_pages_the_cache_does_not_have():
    say("pages outside the cache, lengths past the table")
    p = problem([100, 90, 64], [3, 1, 2], 2, 2, 128, 16)
    p["table"][0, 2], p["table"][1, 0], p["table"][2, 3] = -1, p["cache"][0].shape[0], 2**31 - 1
    check(p, *call(p, return_lse=True))
    p = problem([100, 90], [3, 1], 2, 2, 128, 16)
    p["lens"] = i32([100, 2**31 - 1])
    p["table"] = p["table"][:, :6].contiguous()  # 96 positions of each
    out, lse = call(p, return_lse=True)
    check(p, out, lse)
    # lengths and starts that make no sense read nothing outside: 4 rows, whatever comes
    for lens, starts in (([-5, 3], [0, 2, 4]), ([10, 10], [3, 1, 2]), ([10, 10], [-2, 9, 100])):
        p["lens"], p["starts"] = i32(lens), i32(starts)
        call(p)
    torch.cuda.synchronize()


def test_strides_kv_pairs_and_streams():
    say("strided q, keys and values in one allocation, a padded table, another stream")
    h, d, page = 2, 128, 32
    p = problem([150, 61], [2, 5], h, 4, d, page, mask=tree)
    want = call(p)
    rows = torch.zeros((7, (8 + 4) * d), dtype=BF16, device=DEV)
    rows[:, :8 * d] = p["q"].view(7, -1)
    pages = p["cache"][0].shape[0]
    codes = torch.zeros((pages, 2, h, page, d), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    scales = torch.zeros((pages, 2, h, page), device=DEV)
    for i in (0, 1):
        codes.view(torch.uint8)[:, i] = p["cache"][i].view(torch.uint8)
        scales[:, i] = p["cache"][2 + i]
    wide = torch.full((2, 64), -1, dtype=torch.int32, device=DEV)
    wide[:, :p["table"].shape[1]] = p["table"]
    mask = torch.ones((7, 90), dtype=torch.uint8, device=DEV)
    mask[:, :p["mask"].shape[1]] = p["mask"]
    other = {**p, "q": rows[:, :8 * d].view(7, 8, d), "cache": (codes[:, 0], codes[:, 1], scales[:, 0], scales[:, 1]),
             "table": wide, "mask": mask[:, :33]}
    got = call(other)  # a wider table cuts the work into other pieces: within the tolerance, not the same bits
    check(other, got, None)
    assert (got.float() - want.float()).abs().max() < 0.05
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        there = call(other)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(there, got)


def test_a_decode_layer_captured_and_replayed_on_new_lengths():
    """Rotation, write and attention of a step as one graph, replayed as the sequences grow; every replay equals the
    eager run. Two graphs at once on two streams own their workspaces."""
    say("graph")
    h, group, d, page, pages = 2, 4, 128, 16, 40
    f = aklr_amd.rotary_frequencies(d, device=DEV)
    q, k, v = normal((2, h * group, d), BF16, 1), normal((2, h, d), BF16, 2), normal((2, h, d), BF16, 3)
    table = torch.randperm(pages, generator=gen(4), device=DEV).to(torch.int32).view(2, 20)
    pos, slots = torch.zeros(2, dtype=torch.int64, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    lens, starts = i32([0, 0]), i32([0, 1, 2])
    caches = [new_cache(pages, h, d, page) for _ in range(3)]

    def step(cache):
        turned = aklr_amd.rotary_kv_cache_write_fp8(q, k, v, pos, f, *cache, slots)
        return aklr_amd.tree_attention_fp8(turned, *cache, table, lens, starts)

    def to(n):
        at = torch.tensor([n, 3 * n], device=DEV)
        pos.copy_(at)
        slots.copy_(table[torch.arange(2, device=DEV), at // page] * page + at % page)
        lens.copy_((at + 1).to(torch.int32))
        for i, x in enumerate((q, k, v)):
            x.copy_(normal(x.shape, BF16, 100 * n + i))

    to(0)
    step(caches[0])
    graphs, outs = [], []
    for c in caches[1:]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for n in range(0, 100, 7):
        to(n)
        want = step(caches[0])
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, want), n


def test_any_workspace_content():
    say("workspace content")
    from aklr_amd import workspace

    p = problem([3000, 100, 1500], [3, 1, 20], 2, 4, 128, 16, mask=tree)
    want = call(p, return_lse=True)
    real = workspace.get
    for fill in (0xFF, 0x7F, 0x00):
        def filled(device, nbytes):
            t = real(device, nbytes)
            return t if t is None else t.fill_(fill)
        try:
            workspace.get = filled
            got = aklr_amd.tree_attention_fp8.general(p["q"], *p["cache"], p["table"], p["lens"], p["starts"], p["mask"],
                                                      return_lse=True)
        finally:
            workspace.get = real
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits():
    say("a cache of more than 4 GiB a side")
    h, d, page, pages = 1, 256, 1024, 17000
    cache = tuple(torch.zeros((pages, h, page, d), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in "kv") + tuple(
        torch.zeros((pages, h, page), device=DEV) for _ in "kv")
    table = i32([[pages - 1, 3], [16999, 16384]])
    slots = torch.cat([table[0, 0].long() * page + torch.arange(1024, device=DEV), table[1, 1].long() * page + torch.arange(300, device=DEV)])
    aklr_amd.kv_cache_write_fp8(normal((1324, h, d), BF16, 1), normal((1324, h, d), BF16, 2), *cache, slots)
    q = normal((2, 4, d), BF16, 3)
    out = aklr_amd.tree_attention_fp8(q, *cache, table, i32([1000, 1324]), i32([0, 1, 2]))
    small = tuple(t[torch.tensor([pages - 1, 16384], device=DEV)] if t.dtype != torch.float8_e4m3fn
                  else t.view(torch.uint8)[torch.tensor([pages - 1, 16384], device=DEV)].view(t.dtype) for t in cache)
    want = aklr_amd.tree_attention_fp8(q, *small, i32([[0, 0], [0, 1]]), i32([1000, 1324]), i32([0, 1, 2]))
    assert torch.equal(out, want) and out.float().abs().max() > 0.01


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t", [3, 30, 50, 100])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_score_is_an_fp32_sum(t, d, dtype):
    # Every token sees one position, itself, so the log of its sum is its score. The products are exact, d of them are
    # summed with a rounding of at most 2^-24 of their size each, and three scalings round as much. With the score x in
    # powers of two the reference is at most |x| + 20: four roundings of that size around the exponential, and the
    # logarithm of a weight between 2^-20 and 2^20: under 2^-24 * (4 |x| + 128) together.
    say(f"scores {t} {d} {dtype}")
    p = problem([t], [t], 2, 1, d, 16, dtype, seed=7, mask=lambda rng, n: np.eye(n, dtype=bool))
    out, lse = call(p, return_lse=True)
    _, want, _, size = oc.attention(
        p["q"].double().cpu().numpy(), u8(p["cache"][0]), u8(p["cache"][1]), *(x.cpu().numpy() for x in p["cache"][2:]),
        p["table"].cpu().numpy(), p["lens"].cpu().numpy(), p["starts"].cpu().numpy(), p["mask"].cpu().numpy(), d ** -0.5)
    tol = 2**-24 * ((d + 3) * size + 4 * np.abs(want) / np.log(2) + 128)
    far = np.abs(lse.double().cpu().numpy() - want) - tol
    assert (far <= 0).all(), far.max()
    # and its value, whatever the weight: quotient and type round, and the weight: to fp16 (2^-11) or bf16 (2^-8);
    # up to 16 rows a bf16 one is two, and what the first leaves, at most 2^-8, is off by 2^-8 of that
    at = p["table"][0].long()
    v = (p["cache"][1].double() * p["cache"][3].double()[..., None])[at].transpose(1, 2).reshape(-1, 2, d)[:t]
    few = 2**-11 if dtype == F16 else 2**-16 if t <= 16 else 2**-8
    assert ((out.double() - v).abs() <= v.abs() * (torch.finfo(dtype).eps / 2 + few) * 1.01 + 2**-25).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lens,counts,h,group,d,page", [
    ([9000], [1], 1, 16, 128, 16), ([9000], [1], 8, 1, 64, 64), ([9000], [1], 1, 3, 256, 16), ([5000], [33], 2, 4, 128, 32),
    ([5000, 0, 4000], [5, 3, 9], 1, 8, 64, 16), ([6000, 130, 1], [20, 1, 1], 2, 4, 256, 48), ([7000], [7], 1, 4, 128, 16),
    ([40 + 90 * i for i in range(70)], [1 + i % 3 for i in range(70)], 1, 5, 128, 16),
    ([90 * i for i in range(70)], [i % 2 for i in range(70)], 1, 2, 64, 16)])
def test_many_splits(lens, counts, h, group, d, page, dtype):
    say(f"splits {lens[:3]} {counts[:3]} {h} {group} {d} {page} {dtype}")
    p = problem(lens, counts, h, group, d, page, dtype, seed=11)
    out, lse = call(p, return_lse=True)
    check(p, out, lse, what="splits")
    for _ in range(3):  # always in the same order
        again = call(p, return_lse=True)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("counts", [[130, 7], [40, 50], [0, 129], [33, 33]])
@pytest.mark.parametrize("d,h,page", [(64, 65, 16), (128, 65, 48), (256, 17, 64)])
def test_tiles_of_many_rows(d, h, page, counts, masked, dtype):
    say(f"tiles {d} {h} {page} {counts} {masked} {dtype}")
    lens = [counts[0] + 5, 1400]
    p = problem(lens, counts, h, 1, d, page, dtype, seed=5, mask=tree if masked else None, extra_q=2)
    out = torch.full_like(p["q"], 7.0)
    call(p, out=out)
    _, lse = call(p, return_lse=True, out=out)
    check(p, out, lse)
    assert (out[sum(counts):] == 7).all()
    clean = out.clone()
    # nothing that is not seen reaches a row: NaN and infinities behind the lengths, and in pages of no sequence
    used = torch.zeros(p["cache"][2].shape[0], page, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        at = torch.arange(n, device=DEV)
        used[p["table"][b].long()[at // page], at % page] = True
    for c in p["cache"][:2]:
        c.view(torch.uint8).masked_fill_(~used[:, None, :, None], 0x7F)
    for c, bad in zip(p["cache"][2:], (float("inf"), float("nan"))):
        c.masked_fill_(~used[:, None, :], bad)
    call(p, out=out)
    assert torch.equal(out, clean)
    # a query token's own position all NaN: only rows that see it turn NaN
    t, b = counts[1] // 2, 1
    pos, first = lens[1] - counts[1] + t, counts[0]
    p["cache"][0].view(torch.uint8)[p["table"][b, pos // page].long(), :, pos % page, 3] = 0xFF
    p["cache"][1].view(torch.uint8)[p["table"][b, pos // page].long(), :, pos % page, 5] = 0x7F
    call(p, out=out)
    rows = torch.arange(counts[1], device=DEV)
    sees = p["mask"][first:first + counts[1], t] if masked else rows >= t
    mine, before = out[first:first + counts[1]], clean[first:first + counts[1]]
    assert mine[sees].isnan().all() and torch.equal(mine[~sees], before[~sees]) and torch.equal(out[:first], clean[:first])
    # pages that the cache does not have are as if not there
    p = problem(lens, counts, h, 1, d, page, dtype, seed=6, mask=tree if masked else None)
    p["table"][1, 2], p["table"][1, 5] = -1, p["cache"][0].shape[0]
    check(p, *call(p, return_lse=True))


def test_tiles_of_rows_that_see_nothing():
    say("tiles: rows that see nothing, lengths below the counts")
    for counts, lens in (([100, 90], [20, 0]), ([40, 44], [44, 3])):
        p = problem(lens, counts, 65, 1, 64, 16, mask=lambda rng, t: rng.random((t, t)) < 0.02)
        check(p, *call(p, return_lse=True))
        p["mask"] = None
        check(p, *call(p, return_lse=True))
