"""Adapters with fp16: a token's small values of x a^T beside a large one keep their bits.

Tolerances: none. v has one large value, which b leaves out, and one of 11 bits some powers of two below it: its products, and
its sums with zeros, are exact, and the result is fp16's own."""
from __future__ import annotations

import pytest
import torch

import aklr_amd
from tests.helpers import say

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("below", [10, 14, 20, 28])
@pytest.mark.parametrize("t,n,r", [(1, 24, 8), (17, 264, 32), (250, 520, 128), (300, 72, 8), (3000, 136, 40), (7200, 72, 16), (7300, 2056, 128)])
def test_small_values_beside_a_large_one(t, n, r, below):
    say(f"lora small beside large {t} {n} {r} {below}")
    g = torch.Generator(device=DEV).manual_seed(t + r + below)
    count, k = 3, 24
    x, base = (torch.zeros(s, dtype=torch.float16, device=DEV) for s in ((t, k), (t, n)))
    a, b = (torch.zeros(s, dtype=torch.float16, device=DEV) for s in ((count, r, k), (count, n, r)))
    bits = torch.randint(1024, 2048, (t,), generator=g, device=DEV).double()  # 11 bits
    x[:, 1], a[:, 0, 1] = 2.0**5, 2.0**5
    x[:, 17], a[:, r - 1, 17] = (bits * 2.0**-14).half(), 2.0 ** (14 - below)  # 2^(10 - below) to twice that
    b[:, :, r - 1] = 2.0 ** (below - 14)
    ids = torch.randint(0, count, (t,), generator=g, device=DEV)
    got = aklr_amd.lora_project(x, a, b, ids, base)
    want = (bits * 2.0**-14).half()
    assert torch.equal(want.double(), bits * 2.0**-14)
    assert torch.equal(got, want[:, None].expand(t, n))
