"""Paths of a compaction with entries that are passed over, on the GPU against the oracle: bytes, equal or wrong. What an entry
that is none does to the others: nothing. Items behind it still move, and those behind one at the front have their source
before their place."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aklr_amd
from oracle import requests as oq
from tests.helpers import say
from tests.test_gpu_kv_cache import new_cache
from tests.test_gpu_kv_pages import held, i32, same

pytestmark = pytest.mark.gpu
FAR = 1 << 30  # no position of any sequence


def compacted(h, d, page, paths, positions, seed, what):
    """All sequences' paths on private pages in one call, against the oracle."""
    paths = np.asarray(paths)
    batch, cols = len(paths), -(-positions // page)
    cache = new_cache(batch * cols + 1, h, d, page, seed)
    table = np.random.RandomState(seed).permutation(batch * cols).reshape(batch, cols)
    lens, starts, counts = [positions] * batch, np.arange(batch + 1) * positions, [paths.shape[1]] * batch
    want = oq.compact(held(cache), table, lens, starts, paths, counts)
    aklr_amd.kv_cache_compact_fp8(*cache, i32(table), i32(lens), i32(starts), i32(paths), i32(counts))
    same(cache, want, what)


@pytest.mark.parametrize("most", [40, 64, 70, 97, 1000])
def test_entries_past_the_sequence_at_any_place(most):
    say(f"compact: entries past the sequence, {most}")
    paths = []
    for at in (0, 1, 31, 32, 33, 63, 64, 65, 96):
        if at < most:
            path = np.arange(1, most + 1)
            path[at] = FAR
            paths.append(path)
    path = np.arange(1, most + 1)
    path[::32] = FAR
    paths.append(path)
    path = np.arange(1, most + 1)
    path[::32] = -1
    paths.append(path)
    compacted(2, 64, 16, paths, most + 5, most, str(most))


@pytest.mark.parametrize("most,first", [(most, first) for most in (9, 12, 33, 64, 65, 70, 300, 2000)
                                        for first in (1, 2, 7, 8, 9, 31, 40, 150) if first < most])
def test_sources_before_their_places(most, first):
    say(f"compact: {first} entries that are none before the rest, {most}")
    pick = np.random.RandomState(most + first)
    paths = []
    for kind in range(5):
        path = np.full(most, -1)
        rest = most - first
        if kind == 0:  # everything moves up
            path[first:] = np.arange(rest)
        elif kind == 1:  # up, then stays, then down
            path[first:] = np.sort(pick.choice(most + 30, rest, replace=False))
        elif kind == 2:  # up, with holes between
            path[first:] = np.where(pick.rand(rest) < 0.2, pick.choice([-1, -7, FAR], rest), np.arange(rest))
        elif kind == 3:  # any entries none, the others from anywhere, in order: down, up and down again
            on = np.sort(pick.choice(most, max(1, rest - rest // 4), replace=False))
            path[on] = np.sort(pick.choice(most + 30, len(on), replace=False))
        else:
            path[first:] = np.arange(rest) + first + 1
        paths.append(path)
    compacted(2, 64, 16, paths, most + 33, most + first, f"{most} {first}")


@pytest.mark.parametrize("first", [1, 40, 230])
def test_sources_before_their_places_in_windows(first):
    # 1024 heads of 256: some 250 items are a window
    say(f"compact in windows: {first} entries that are none before the rest")
    n = 600
    up, mixed, holes = np.full(n, -1), np.full(n, -1), np.full(n, -1)
    up[first:] = np.arange(n - first)
    mixed[first:] = np.sort(np.random.RandomState(first).choice(n + 20, n - first, replace=False))
    holes[first:] = np.where(np.arange(n - first) % 32 == 0, FAR, np.arange(n - first))
    for path in (up, mixed, holes):
        h, d, page = 1024, 256, 16
        cols = -(-(n + 20) // page)
        cache = new_cache(cols, h, d, page, first)
        table = np.arange(cols)[None, ::-1].copy()
        sample = [t[:, [0, 511, 1023]] for t in held(cache)]  # the oracle on three of the heads, the keys of all by their bytes
        want = oq.compact(sample, table, [n + 20], [0, n + 20], path[None], [n])
        before = cache[0].view(torch.uint8).clone()
        aklr_amd.kv_cache_compact_fp8(*cache, i32(table), i32([n + 20]), i32([0, n + 20]), i32(path[None]), i32([n]))
        for g, w in zip(held(cache), want):
            assert np.array_equal(g[:, [0, 511, 1023]], w)
        at, src = np.arange(n), path.copy()
        on = (src >= 0) & (src < n + 20)
        at, src = torch.from_numpy(at[on]).cuda(), torch.from_numpy(src[on]).cuda()
        assert torch.equal(cache[0].view(torch.uint8)[cols - 1 - at // page, :, at % page], before[cols - 1 - src // page, :, src % page])


def test_windows_captured():
    # what one replay says of its path, that items move up, is not the next one's
    say("compact in windows: captured, replayed with paths that move up and down")
    n, h, d, page = 600, 1024, 256, 16
    cols = -(-(n + 20) // page)
    up, down = np.r_[-1, np.arange(n - 1)], np.arange(9, n + 9)
    table, lens, starts, counts = i32(np.arange(2 * cols).reshape(2, cols)), i32([n + 20] * 2), i32([0, n + 20, 2 * n + 40]), i32([n, n])
    cache, other = new_cache(2 * cols, h, d, page, 1), new_cache(2 * cols, h, d, page, 1)
    path = i32(np.stack([down, down]))
    for c in (cache, other):
        aklr_amd.kv_cache_compact_fp8(*c, table, lens, starts, path, counts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        aklr_amd.kv_cache_compact_fp8(*cache, table, lens, starts, path, counts)
    for paths in ((up, down), (down, down), (down, up), (up, up), (down, down)):
        path.copy_(i32(np.stack(paths)))
        before = other[0].view(torch.uint8).clone()
        graph.replay()
        aklr_amd.kv_cache_compact_fp8(*other, table, lens, starts, path, counts)
        torch.cuda.synchronize()
        for t, o in zip(cache, other):
            assert torch.equal(t.view(torch.uint8), o.view(torch.uint8))
        for b, src in enumerate(paths):
            at = torch.arange(n, device="cuda")[torch.from_numpy(src >= 0)]
            src = torch.from_numpy(src[src >= 0]).cuda()
            assert torch.equal(other[0].view(torch.uint8)[b * cols + at // page, :, at % page], before[b * cols + src // page, :, src % page])
