"""Adapters added to the very rows they read: x, base and out in one place, on both call paths, against the call with three."""
from __future__ import annotations

import pytest
import torch

import aklr_amd
from tests import test_gpu_cache_host as cache_host
from tests.helpers import say
from tests.test_gpu_lora import BF16, F16, check, problem
from tests.test_gpu_requests_host import OPS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t,n,r,count", [(1, 264, 8, 2), (40, 520, 16, 3), (250, 264, 128, 9), (300, 72, 24, 5), (2100, 520, 64, 4),
                                         (7300, 264, 32, 3), (7300, 2048, 128, 3)])
def test_x_base_and_out_in_one_place(t, n, r, count, dtype, monkeypatch):
    say(f"lora in place {t} {n} {r} {count} {dtype}")
    monkeypatch.setattr(cache_host, "OPS", OPS)
    p = problem(t, n, n, r, count, dtype, t + n)
    x = p["x"]
    want = aklr_amd.lora_project(x, p["a"], p["b"], p["ids"], x.clone(), scales=p["scales"])
    if t < 1000:
        check(want, {**p, "base": x})
    args, kw = (x, p["a"], p["b"], p["ids"], x), {"scales": p["scales"]}
    assert torch.equal(aklr_amd.lora_project(*args, **kw), want)  # read twice, written nowhere
    for base, out in ((x, x), (x.view(x.shape), x), (x, x[:])):
        cache_host.both("lora", (*args[:4], base), {**kw, "out": out}, True)
    wide = torch.zeros((t, n + 40), dtype=dtype, device=x.device)
    rows = wide[:, 16:16 + n]
    rows.copy_(x)
    assert aklr_amd.lora_project(rows, *args[1:4], rows, **kw, out=rows) is rows
    assert torch.equal(rows, want) and not wide[:, :16].any() and not wide[:, 16 + n:].any()
    cache_host.both("lora", (*args[:4], torch.zeros_like(x)), {**kw, "out": x}, False, False)
