"""Pages of the FP8 cache on the GPU against the oracle: bytes and whole numbers, equal or wrong."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aklr_amd
from oracle import requests as oq
from tests.helpers import say, u8
from tests.test_gpu_kv_cache import DEV, E4M3, new_cache

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device=DEV)


def held(cache):
    return [u8(t) if t.dtype == E4M3 else t.cpu().numpy().view(np.uint32) for t in cache]


def same(cache, want, what=""):
    for i, (got, w) in enumerate(zip(held(cache), want)):
        bad = np.argwhere(got != w)
        assert not len(bad), f"{what}: tensor {i}, {len(bad)} differ, first {bad[:2].tolist()}"


def one_allocation(pages, heads, dim, page):
    codes = torch.zeros((pages, 2, heads, page, dim), dtype=torch.uint8, device=DEV)
    codes.random_(0, 256)
    scales = torch.rand((pages, 2, heads, page), device=DEV)
    codes = codes.view(E4M3)
    return codes[:, 0], codes[:, 1], scales[:, 0], scales[:, 1]


@pytest.mark.parametrize("pages,h,d,page,n", [(2, 1, 64, 16, 1), (40, 3, 64, 48, 17), (60, 8, 128, 16, 25), (9, 2, 256, 1024, 3),
                                              (700, 8, 128, 64, 300), (5, 40, 256, 16, 2), (3000, 1, 64, 16, 1400)])
def test_copy(pages, h, d, page, n):
    say(f"copy {pages} {h} {d} {page} {n}")
    pick = np.random.RandomState(n)
    for cache in (new_cache(pages, h, d, page, 1), one_allocation(pages, h, d, page)):
        for dtype in (torch.int32, torch.int64):
            order = pick.permutation(pages)
            dst = order[:n]
            src = order[n + pick.randint(0, pages - n, n)]
            want = oq.copy_pages(held(cache), src, dst)
            got = aklr_amd.kv_cache_copy_pages_fp8(*cache, torch.tensor(src, dtype=dtype, device=DEV), torch.tensor(dst, dtype=dtype, device=DEV))
            assert all(a is b for a, b in zip(got, cache))
            same(cache, want, str(dtype))


def test_copy_skips():
    say("copy: pairs of which one is no page, a page onto itself, none")
    cache = new_cache(6, 2, 64, 16, 2)
    src = torch.tensor([0, -1, 6, 1, 2, 1 << 40, 3, -(1 << 40)], device=DEV)
    dst = torch.tensor([4, 5, 5, -1, 6, 5, 3, 5], device=DEV)
    want = oq.copy_pages(held(cache), src.tolist(), dst.tolist())
    aklr_amd.kv_cache_copy_pages_fp8(*cache, src, dst)
    same(cache, want)
    aklr_amd.kv_cache_copy_pages_fp8(*cache, src.clamp(-(1 << 31), (1 << 31) - 1).to(torch.int32), dst.to(torch.int32))
    same(cache, want)
    aklr_amd.kv_cache_copy_pages_fp8(*cache, src[:0], dst[:0])
    same(cache, want)


def compaction(pick, batch, most, page, cols, pages, dense):
    """Sequences with paths of several kinds, their pages all different."""
    order, at = pick.permutation(pages), 0
    table, lens, drafts = np.full((batch, cols), -1), np.zeros(batch, int), np.zeros(batch, int)
    path, counts = np.full((batch, most), -1), np.zeros(batch, int)
    for b in range(batch):
        lens[b] = pick.randint(0, cols * page + 1)
        need = -(-lens[b] // page)
        table[b, :need] = order[at:at + need]
        at += need
        t = drafts[b] = pick.randint(0, lens[b] + 1)
        k = min(t, most, pick.randint(0, most + 1))
        kind = pick.randint(0, 5)
        if kind == 0 and t > k:  # one left out near the beginning: every place is the next item's source
            path[b, :k] = np.arange(k) + (np.arange(k) >= min(k, 2))
        elif kind == 1:
            path[b, :k] = np.arange(t - k, t)
        elif kind == 2 and 2 * k <= t:
            path[b, :k] = 2 * np.arange(k)
        else:
            path[b, :k] = np.sort(pick.choice(t, k, replace=False)) if k else []
        counts[b] = k + (pick.randint(0, 9) if k == most else 0)
    return table, lens, drafts, path, counts


@pytest.mark.parametrize("most", [1, 3, 8, 9, 33, 64, 65, 100, 1000])
@pytest.mark.parametrize("h,d,page", [(2, 64, 16), (5, 128, 48), (1, 256, 64)])
def test_compact(most, h, d, page):
    say(f"compact {most} {h} {d} {page}")
    pick = np.random.RandomState(most + d)
    cols = -(-2 * most // page) + 2
    for batch in (1, 6):
        pages = batch * cols + 3
        for cache in (new_cache(pages, h, d, page, 3), one_allocation(pages, h, d, page)):
            for _ in range(4):
                table, lens, drafts, path, counts = compaction(pick, batch, most, page, cols, pages, False)
                starts = np.r_[0, np.cumsum(drafts)]
                want = oq.compact(held(cache), table, lens, starts, path, counts)
                got = aklr_amd.kv_cache_compact_fp8(*cache, i32(table), i32(lens), i32(starts), i32(path), i32(counts))
                assert all(a is b for a, b in zip(got, cache))
                same(cache, want)


def test_compact_shifts_by_one():
    # the longest chain of places that are sources: each item's place is the one before its source
    say("compact: everything moves by one, by 31, 32, 33")
    for n in (64, 65, 500, 4000):
        for by in (1, 31, 32, 33):
            cols = -(-(n + by) // 16)
            cache = new_cache(cols, 1, 64, 16, 4)
            table = np.arange(cols)[None, ::-1].copy()
            path = np.arange(by, n + by)[None]
            want = oq.compact(held(cache), table, [n + by], [0, n + by], path, [n])
            aklr_amd.kv_cache_compact_fp8(*cache, i32(table), i32([n + by]), i32([0, n + by]), i32(path), i32([n]))
            same(cache, want, f"{n} {by}")


def test_compact_in_windows():
    # 1024 heads of 256: 252 items are all that is copied aside at once, so 600 go in three windows, sequence by sequence
    say("compact in windows")
    h, d, page, n = 1024, 256, 16, 600
    cols = -(-(n + 50) // page)
    cache = new_cache(cols + 2, h, d, page, 5)
    assert 2 * n * 2 * h * (d + 4) > 128 << 20
    for path in (np.arange(50, n + 50), np.arange(1, n + 1), np.sort(np.random.RandomState(1).choice(n + 50, n, replace=False))):
        table = np.stack([np.arange(cols), np.full(cols, -1)])
        table[1, :2] = [cols, cols + 1]
        paths = np.stack([path, np.r_[[1, 3, 30], np.full(n - 3, -1)]])
        args = table, [n + 50, 31], [0, n + 50, n + 81], paths, [n, 3]
        a = held(cache)
        sample = [t[:, [0, 511, 1023]] for t in a]  # the oracle on three of the heads, the others by their own bytes
        want = oq.compact(sample, *[np.asarray(x) for x in args])
        first = cache[0].view(torch.uint8).clone()
        aklr_amd.kv_cache_compact_fp8(*cache, *map(i32, args))
        got = held(cache)
        for g, w in zip(got, want):
            assert np.array_equal(g[:, [0, 511, 1023]], w)
        flat = torch.arange(n, device=DEV)
        src = torch.from_numpy(path).to(DEV)
        assert torch.equal(cache[0].view(torch.uint8)[flat // page, :, flat % page], first[src // page, :, src % page])


def test_compact_skips():
    say("compact: numbers outside, pages the cache does not have, lengths past the table, nothing to do")
    for most in (7, 70):
        cache = new_cache(8, 2, 64, 16, 6)
        table = np.array([[0, 1, -1], [2, 8, 3], [4, 5, 6], [7, 7, 7]])
        path = np.full((4, most), -1)
        path[0, :4], path[1, :7], path[2, :5], path[3, :3] = [1, 20, 33, 90], [0, 2, 17, 18, 19, 33, 40], [-4, 3, 5, 1 << 30, 6], [0, 1, 2]
        for lens, counts in (([40, 44, 48, 10], [4, 7, 5, 3]), ([40, 44, 60, -5], [1000, 7, 5, 3]), ([3, 0, 0, 0], [-1, 0, 5, 3])):
            starts = np.r_[0, np.cumsum([40, 41, 48, 10])]
            want = oq.compact(held(cache), table, lens, starts, path, counts)
            aklr_amd.kv_cache_compact_fp8(*cache, i32(table), i32(lens), i32(starts), i32(path), i32(counts))
            same(cache, want, str(lens))
    before = held(cache)
    aklr_amd.kv_cache_compact_fp8(*cache, i32(table)[:0], i32([]), i32([0]), i32(path)[:0], i32([]))
    aklr_amd.kv_cache_compact_fp8(*cache, i32(table)[:, :0], i32([9] * 4), i32([0, 9, 18, 27, 36]), i32(path), i32([4] * 4))
    # paths that do not ascend move something, and touch nothing outside
    pick = np.random.RandomState(2)
    for most in (20, 90):
        aklr_amd.kv_cache_compact_fp8(*cache, i32(table[:1]), i32([32]), i32([0, 32]), i32(pick.randint(-5, 40, (1, most))), i32([most]))
    torch.cuda.synchronize()
    for g, w in zip(held(cache), before):
        assert np.array_equal(g[2:], w[2:])


def books(pick, batch, cols, page, pages, spare=None):
    """A block table whose sequences share first pages, its page counts, and lengths."""
    table, refs, lens = np.full((batch, cols), -1), np.zeros(pages, int), np.zeros(batch, int)
    free = iter(pick.permutation(pages).tolist())
    for b in range(batch):
        lens[b] = pick.randint(0, cols * page + 1)
        need = -(-lens[b] // page)
        share = pick.randint(0, need + 1) if b and pick.rand() < 0.7 else 0
        old = table[pick.randint(0, b)] if share else None
        for c in range(need):
            if share and c < share and old[c] >= 0:
                table[b, c] = old[c]
            else:
                share = 0
                table[b, c] = next(free, -1)
        full = (table[b, :need] >= 0).all()
        lens[b] = lens[b] if full else int(np.argmax(table[b, :need] < 0)) * page
        table[b, -(-lens[b] // page):] = -1
    np.add.at(refs, table[table >= 0], 1)
    refs[pick.rand(pages) < 0.1] += 1  # somebody else holds them
    if spare is not None:
        left = np.flatnonzero(refs == 0)
        refs[left[spare:]] = 1
    return table, refs, lens


def update(refs, table, lens, wants, page, parents=None):
    """The operator and the oracle on the same; the operator's outputs."""
    r = i32(refs)
    got = aklr_amd.kv_cache_update_pages(r, i32(table), i32(lens), i32(wants), page, None if parents is None else i32(parents))
    want = oq.update_pages(refs, table, lens, wants, page, parents)
    for name, g, w in zip(("table", "granted", "src", "dst", "refs"), (*got, r), want):
        assert g.dtype == torch.int32 and np.array_equal(g.cpu().numpy(), np.asarray(w)), f"{name}: {g.tolist()} instead of {np.asarray(w).tolist()}"
    return [t.cpu().numpy() for t in (*got, r)]


@pytest.mark.parametrize("batch,cols,page,pages,spare", [(1, 1, 16, 1, None), (1, 3, 16, 9, 1), (4, 5, 16, 60, None), (9, 7, 48, 200, 4),
                                                         (64, 33, 16, 3000, None), (64, 9, 64, 900, 20), (300, 12, 16, 9000, None),
                                                         (1025, 4, 16, 20000, None), (2049, 3, 32, 9000, 50), (5000, 5, 16, 40000, None),
                                                         (40, 300, 1, 20000, 300)])
def test_update(batch, cols, page, pages, spare):
    say(f"update {batch} {cols} {page} {pages} {spare}")
    pick = np.random.RandomState(batch + cols)
    for i in range(6 if batch < 1000 else 3):
        table, refs, lens = books(pick, batch, cols, page, pages, spare)
        for step in range(3):
            parents = None if (i + step) % 3 == 0 else np.where(pick.rand(batch) < 0.1, pick.choice([-1, batch, 1 << 30, -(1 << 31)], batch),
                                                                   np.where(pick.rand(batch) < 0.4, np.arange(batch), pick.randint(0, batch, batch)))
            grown = pick.randint(-2 * page, 2 * page + 1, batch) + (lens if parents is None else lens[np.clip(parents, 0, batch - 1)])
            wants = np.where(pick.rand(batch) < 0.1, pick.choice([0, -7, cols * page + 5, 1 << 30], batch), grown)
            table, lens, _, _, refs = update(refs, table, lens, wants, page, parents)


def test_update_of_one_parent():
    say("update: all go on from one, with a page in part, whole, and none left")
    pick = np.random.RandomState(3)
    for n in (2, 65, 1500):
        for length in (16, 17, 40, 48):
            table, refs = np.full((n, 4), -1), np.zeros(n + 8, int)
            table[1, : -(-length // 16)] = pick.permutation(n + 8)[: -(-length // 16)]
            refs[table[1][table[1] >= 0]] = 1
            lens = np.zeros(n, int)
            lens[1] = length
            update(refs, table, lens, np.full(n, length + 1), 16, np.ones(n, int))
            update(refs, table, lens, np.full(n, length), 16, np.ones(n, int))
            update(refs, table, lens, np.arange(n) % 64, 16, np.ones(n, int))


def test_update_oddities():
    say("update: entries that name no page, no columns, a wide table's rows, counts that are wrong")
    pick = np.random.RandomState(4)
    for _ in range(20):
        table, refs, lens = books(pick, 12, 6, 16, 80)
        table[pick.rand(12, 6) < 0.1] = pick.choice([-1, 80, 1 << 30, -(1 << 31)])
        update(refs, table, lens, lens + pick.randint(-20, 20, 12), 16, pick.randint(-1, 12, 12))
    got = aklr_amd.kv_cache_update_pages(i32([0, 0]), i32(np.zeros((3, 0))), i32([5, 0, 1]), i32([9, 9, 9]), 16)
    assert got[0].shape == (3, 0) and got[1].tolist() == [0, 0, 0] and got[2].tolist() == got[3].tolist() == [-1] * 3
    got = aklr_amd.kv_cache_update_pages(i32([0, 0]), i32(np.zeros((0, 4))), i32([]), i32([]), 16)
    assert [t.shape[0] for t in got] == [0] * 4
    wide = i32(np.full((3, 9), -1))
    wide[:, 2:6] = i32([[0, 1, -1, -1], [2, -1, -1, -1], [-1] * 4])
    refs = i32([1, 1, 1, 0, 0])
    table, granted, _, _ = aklr_amd.kv_cache_update_pages(refs, wide[:, 2:6], i32([20, 9, 0]), i32([33, 16, 5]), 16)
    assert table.tolist() == [[0, 1, 3, -1], [2, -1, -1, -1], [4, -1, -1, -1]] and granted.tolist() == [33, 16, 5] and refs.tolist() == [1] * 5
    # counts below 0, and claims that were never taken back, give out nothing and touch nothing outside
    refs = i32([-5, -(1 << 31), -(1 << 31) + 1, 0, 7])
    table, granted, _, _ = aklr_amd.kv_cache_update_pages(refs, i32([[0, 1], [2, 3]]), i32([20, 20]), i32([20, 20]), 16, i32([1, 0]))
    assert (table >= -1).all() and (table < 5).all()


def test_far_pages():
    say("copy and compact past 2^32 bytes")
    h, d, page, pages = 1, 256, 1024, 17000  # 4.46e9 bytes of codes a side
    cache = tuple(torch.empty(s, dtype=torch.uint8, device=DEV).view(E4M3) for s in [(pages, h, page, d)] * 2) + tuple(
        torch.empty((pages, h, page), device=DEV) for _ in "kv")
    for t in cache:
        t.view(torch.uint8)[[0, 5, pages - 2, pages - 1]] = torch.randint(0, 255, (4, *t.view(torch.uint8).shape[1:]), dtype=torch.uint8, device=DEV)
    at = torch.tensor([0, 5, pages - 2, pages - 1], device=DEV)
    before = [t.view(torch.uint8)[at].clone() for t in cache]
    aklr_amd.kv_cache_copy_pages_fp8(*cache, torch.tensor([pages - 1], device=DEV), torch.tensor([pages - 2], device=DEV))
    for t, w in zip(cache, before):
        assert torch.equal(t.view(torch.uint8)[at], w[[0, 1, 3, 3]])
    for n in (5, 700):
        path = torch.arange(300, 300 + n, dtype=torch.int32, device=DEV)[None]
        was = [t.view(torch.uint8)[pages - 1].clone() for t in cache]
        aklr_amd.kv_cache_compact_fp8(*cache, i32([[pages - 1]]), i32([1024]), i32([0, 1024]), path, i32([n]))
        for t, w in zip(cache, was):
            got = t.view(torch.uint8)[pages - 1]
            size = got.shape[-1] // page if got.dim() == 2 else 1  # scales: bytes of a row
            got, w = (x.view(page, -1) for x in (got, w))
            assert size >= 1 and torch.equal(got[:n], w[300:300 + n]) and torch.equal(got[n:], w[n:])


def test_captured():
    say("pages: captured and replayed with other values between eager calls")
    pick = np.random.RandomState(6)
    batch, cols, page, pages = 24, 9, 16, 400
    cases = []
    for _ in range(4):
        table, refs, lens = books(pick, batch, cols, page, pages)
        cases.append([i32(x) for x in (refs, table, lens, lens + pick.randint(-9, 20, batch), pick.randint(-1, batch, batch))])
    cache, other = new_cache(pages, 2, 64, page, 7), new_cache(pages, 2, 64, page, 7)
    long_path = torch.arange(8, 108, dtype=torch.int32, device=DEV).expand(batch, 100).contiguous()
    held_ = [x.clone() for x in cases[0]]
    alone = i32(np.arange(batch * cols).reshape(batch, cols))  # what is compacted is nobody else's: the update's tables share pages

    def run(c, refs, table, lens, wants, parents):
        new, granted, src, dst = aklr_amd.kv_cache_update_pages(refs, table, lens, wants, page, parents)
        aklr_amd.kv_cache_copy_pages_fp8(*c, src, dst)
        starts = torch.zeros(batch + 1, dtype=torch.int32, device=DEV)
        starts[1:] = granted.cumsum(0)
        aklr_amd.kv_cache_compact_fp8(*c, alone, granted, starts, long_path, (granted - 8).clamp(0, 100).int())
        aklr_amd.kv_cache_compact_fp8(*c, alone, granted, starts, long_path[:, :9], (granted - 108).clamp(0, 9).int())
        return new, granted, src, dst

    run(other, *[x.clone() for x in cases[0]])
    for t, o in zip(cache, other):
        o.view(torch.uint8).copy_(t.view(torch.uint8))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(cache, *held_)
    for case in cases + cases[:2]:
        for a, b in zip(held_, case):
            a.copy_(b)
        graph.replay()
        mine = [x.clone() for x in case]
        want = run(other, *mine)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(held_[0], mine[0])
        for t, o in zip(cache, other):
            assert torch.equal(t.view(torch.uint8), o.view(torch.uint8))
