"""Where ``lora_project`` may put its result, without a GPU: by the place of what it reads, not by which tensor names it."""
from __future__ import annotations

import pytest
import torch

import aklr_amd
from aklr_amd.dispatch import FallbackReason, KernelInfo
from tests.test_cache_ops_host import BF16
from tests.test_requests_host import anywhere, lora_args  # noqa: F401

OOC = FallbackReason.OUT_OF_CONTRACT


@pytest.mark.parametrize("tokens", [1, 3, 300])
def test_out_where_x_and_base_are(anywhere, tokens):  # noqa: F811
    serving = aklr_amd.lora_project.serving
    a = lora_args(t=tokens, k=24)
    x = a["x"]
    both = {**a, "base": x}
    for base in (x, x.view(x.shape), x[:]):
        for out in (x, x.view(x.shape), x[:]):
            assert isinstance(serving(**{**a, "base": base}, out=out), KernelInfo)
    assert isinstance(serving(**both), KernelInfo) and isinstance(serving(**both, out=torch.zeros_like(x)), KernelInfo)
    assert serving(**a, out=x) is OOC and serving(**a, out=x.view(x.shape)) is OOC  # base elsewhere
    memory = torch.zeros(tokens * 24 + 8, dtype=BF16)
    first, second = memory[:-8].view(tokens, 24), memory[8:].view(tokens, 24)
    for x, base, out in ((first, first, second), (first, second, first), (second, first, first)):
        assert serving(**{**a, "x": x, "base": base}, out=out) is OOC


def test_out_apart_from_the_adapters(anywhere):  # noqa: F811
    serving = aklr_amd.lora_project.serving
    a = lora_args(t=8, k=24, count=1)
    for name in ("a", "b"):
        assert serving(**{**a, "base": torch.zeros((8, 24), dtype=BF16)}, out=a[name].view(8, 24)) is OOC
        assert serving(**{**a, "base": a[name].view(8, 24)}, out=a[name].view(8, 24)) is OOC
