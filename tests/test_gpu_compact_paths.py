"""Paths of a compaction with entries that are passed over, on the GPU against the oracle: bytes, equal or wrong. What an entry
that is none does to the others: nothing."""
from __future__ import annotations

import numpy as np
import pytest

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
