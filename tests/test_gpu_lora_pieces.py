"""Adapters: what lies between the two products keeps all that fp32 holds of it. Where a token's values of x a^T cancel in the
second product, what is left is their last bits.

Tolerances: none. v is h + m + l of 8, 8 and 6 bits (1 down to 2^-21), b is 1, -1 and 0: every product is exact, every sum of
any of them in any order is a multiple of 2^-21 below 4, which fp32 holds, and so is each piece of v; the result is rounded
once."""
from __future__ import annotations

import pytest
import torch

import aklr_amd
from tests.helpers import say

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t,n,r", [(1, 24, 8), (5, 72, 16), (17, 264, 32), (250, 520, 128), (300, 72, 8), (700, 2056, 64), (3000, 136, 40),
                                   (7200, 72, 16), (7300, 2048, 128), (7300, 2056, 128)])
def test_what_cancels_leaves_its_last_bits(t, n, r, dtype):
    say(f"lora pieces {t} {n} {r} {dtype}")
    g = torch.Generator(device=DEV).manual_seed(t + r)
    count, k, at, rows = 3, 40, (0, 13, 39), (0, r // 2, r - 1)
    draw = lambda lo, hi: torch.randint(lo, hi, (t,), generator=g, device=DEV).double()  # noqa: E731
    sign = 2 * draw(0, 2) - 1
    h, m, l = sign * draw(128, 256) * 2.0**-7, sign * draw(0, 256) * 2.0**-15, sign * draw(0, 64) * 2.0**-21
    x, base = torch.zeros((t, k), dtype=torch.float64, device=DEV), torch.zeros((t, n), dtype=dtype, device=DEV)
    a, b = (torch.zeros(s, dtype=dtype, device=DEV) for s in ((count, r, k), (count, n, r)))
    for i, part in zip(at, (h, m, l)):
        x[:, i] = part
    a[:, rows[0], list(at)], a[:, rows[1], at[0]], a[:, rows[2], at[1]] = 1, 1, 1  # h + m + l, h, m
    b[:, :, rows[0]], b[:, :, rows[1]], b[:, ::2, rows[2]] = 1, -1, -1  # l, and m + l
    ids = torch.randint(0, count, (t,), generator=g, device=DEV)
    got = aklr_amd.lora_project(x.to(dtype), a, b, ids, base)
    assert torch.equal(x.to(dtype).double(), x)
    assert torch.equal(got[:, ::2], l.to(dtype)[:, None].expand(t, (n + 1) // 2))
    assert torch.equal(got[:, 1::2], (m + l).to(dtype)[:, None].expand(t, n // 2))


@pytest.mark.parametrize("t", [3, 300, 7300])
def test_values_past_the_largest_bf16(t):
    # v = 2^127 * (2 - 2^-8) is fp32's and not bf16's; times 2^-100 and 2^-120 it is a number again
    say(f"lora past bf16 {t}")
    x, a = torch.zeros((t, 16), dtype=BF16, device=DEV), torch.zeros((1, 8, 16), dtype=BF16, device=DEV)
    x[:, 1], x[:, 9] = 2.0**127 * (2 - 2.0**-7), 2.0**119
    a[0, 3, [1, 9]] = 1
    b, base = torch.zeros((1, 24, 8), dtype=BF16, device=DEV), torch.zeros((t, 24), dtype=BF16, device=DEV)
    b[0, :12, 3], b[0, 12:, 3] = 2.0**-100, -(2.0**-120)
    got = aklr_amd.lora_project(x, a, b, torch.zeros(t, dtype=torch.int32, device=DEV), base)
    want = 2.0**127 * (2 - 2.0**-8)
    assert torch.equal(got[:, :12].float(), torch.full((t, 12), want * 2.0**-100, device=DEV).bfloat16().float())
    assert torch.equal(got[:, 12:].float(), torch.full((t, 12), -want * 2.0**-120, device=DEV).bfloat16().float())
