"""Writes of more tokens than one launch has workgroups for."""
from __future__ import annotations

import pytest
import torch

import aklr_amd
from tests.helpers import say
from tests.test_gpu_kv_cache import BF16, DEV, new_cache, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rotary", [False, True])
def test_more_tokens_than_a_launch_has_workgroups(rotary):
    # 8 heads of 256: a workgroup a token. The tokens are one, read again and again; all but six of its slots are skipped
    say(f"2^24 tokens and more, {rotary}")
    h, d, page, tokens = 8, 256, 16, 2**24 + 3
    k, v = normal((1, h, d), BF16, 1), normal((1, h, d), BF16, 2)
    at = torch.tensor([0, 2**23 - 1, 2**23, 2**24 - 1, 2**24, tokens - 1], device=DEV)
    slots = torch.full((tokens,), -1, dtype=torch.int32, device=DEV)
    slots[at] = torch.tensor([5, 17, 0, 31, 8, 30], dtype=torch.int32, device=DEV)
    cache, want = new_cache(2, h, d, page), new_cache(2, h, d, page)
    if rotary:
        f = aklr_amd.rotary_frequencies(d, device=DEV)
        pos = torch.arange(tokens, dtype=torch.int32, device=DEV)
        q = torch.zeros((tokens, 1, 256), dtype=BF16, device=DEV)
        q[at] = normal((6, 1, 256), BF16, 3)
        small = aklr_amd.rotary_kv_cache_write_fp8(q[at], k.expand(6, h, d), v.expand(6, h, d), pos[at], f, *want, slots[at])
        got = aklr_amd.rotary_kv_cache_write_fp8(q, k.expand(tokens, h, d), v.expand(tokens, h, d), pos, f, *cache, slots, out=q)
        assert got is q and torch.equal(got[at], small) and int(got.any(-1).sum()) == 6
    else:
        aklr_amd.kv_cache_write_fp8(k.expand(6, h, d), v.expand(6, h, d), *want, slots[at])
        aklr_amd.kv_cache_write_fp8(k.expand(tokens, h, d), v.expand(tokens, h, d), *cache, slots)
    for x, y in zip(cache, want):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)) and bool(x.view(torch.uint8).any())
