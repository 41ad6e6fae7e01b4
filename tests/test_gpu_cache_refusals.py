"""What the cache operators refuse, on the GPU: the native path leaves it to the plan, and the call returns the reason."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import aklr_amd
from aklr_amd import _lib
from aklr_amd.dispatch import FallbackReason
from tests.helpers import say
from tests.test_gpu_attention import i32
from tests.test_gpu_kv_cache import BF16, DEV, new_cache, normal

pytestmark = pytest.mark.gpu
OOC = FallbackReason.OUT_OF_CONTRACT


def calls():
    """{op: (function, native name, args, the places of what can have a gradient, the name of an output, its value)}"""
    q, k, v = normal((3, 4, 64), BF16, 1), normal((3, 2, 64), BF16, 2), normal((3, 2, 64), BF16, 3)
    pos, f, slots = torch.arange(3, device=DEV), aklr_amd.rotary_frequencies(64, device=DEV), torch.arange(3, device=DEV)
    cache = new_cache(2, 2, 64, 16)
    table = i32([[0, 1]])
    return {
        "rotary": (aklr_amd.rotary_embedding, "rotary", (q, k, pos, f), (0, 1, 3), "out_q", torch.zeros_like(q)),
        "write": (aklr_amd.kv_cache_write_fp8, "kv_write", (k, v, *cache, slots), (0, 1, 4, 5), None, None),
        "both": (aklr_amd.rotary_kv_cache_write_fp8, "rotary_kv_write", (q, k, v, pos, f, *cache, slots), (0, 1, 2, 4, 7), "out", torch.zeros_like(q)),
        "read": (aklr_amd.kv_cache_read_fp8, "kv_read", (*cache, table, i32([0, 3]), 3), (2, 3), "out_v", torch.zeros_like(k)),
        "attend": (aklr_amd.tree_attention_fp8, "tree_attention", (q, *cache, table, i32([3]), i32([0, 3])), (0, 3, 4), "out", torch.zeros_like(q)),
    }


@pytest.mark.parametrize("op", ["rotary", "write", "both", "read", "attend"])
def test_gradients_tangents_and_transforms(op):
    say(f"refusals {op}")
    fn, native, args, places, out, value = calls()[op]
    host = _lib.host_function(native)

    def refused(*a, **kw):
        return host(a, kw) is None and fn(*a, **kw) is OOC

    assert not isinstance(fn(*args), FallbackReason) and host(args, {}) is not None
    for i in places:
        t = args[i]
        assert refused(*args[:i], t.clone().requires_grad_(), *args[i + 1:])
        with forward_ad.dual_level():
            assert refused(*args[:i], forward_ad.make_dual(t, torch.ones_like(t)), *args[i + 1:])
        answers = []

        def ask(x):
            answers.append(refused(*args[:i], x, *args[i + 1:]))
            return x.float().sum()

        torch.vmap(ask)(torch.stack([t, t]))
        torch.func.jvp(ask, (t,), (torch.ones_like(t),))
        torch.func.grad(ask)(t)
        assert answers == [True] * len(answers) and answers
    if out:
        assert refused(*args, **{out: value.clone().requires_grad_()})
        with forward_ad.dual_level():
            assert refused(*args, **{out: forward_ad.make_dual(value, torch.ones_like(value))})
        with torch.no_grad():
            assert not isinstance(fn(*args, **{out: value.clone().requires_grad_()}), FallbackReason)
    assert not isinstance(fn(*args), FallbackReason)


def test_numbers_and_one_tensor_twice():
    say("numbers past fp32, one tensor as queries and keys")
    c = calls()
    for op, name in (("rotary", "magnitude"), ("both", "magnitude"), ("attend", "softmax_scale")):
        fn, native, args = c[op][:3]
        for bad in (1e39, 10**400, float("inf"), float("nan")):
            assert _lib.host_function(native)(args, {name: bad}) is None and fn(*args, **{name: bad}) is OOC
    x = normal((3, 4, 64), BF16, 5)
    pos, f = c["rotary"][2][2:]
    want = aklr_amd.rotary_embedding(x, x, pos, f)
    assert torch.equal(want[0], want[1])
    for kw in ({"out_q": x}, {"out_k": x}, {"out_q": x, "out_k": x}):
        assert _lib.host_function("rotary")((x, x, pos, f), kw) is None and aklr_amd.rotary_embedding(x, x, pos, f, **kw) is OOC


def test_more_workgroups_than_a_launch_has_room_for():
    say("65536 sequences, 256 kv heads")
    cache = new_cache(1, 256, 64, 16)
    n = 65536
    q = torch.zeros((1, 256, 64), dtype=BF16, device=DEV).expand(n, 256, 64)
    args = (q, *cache, torch.zeros((n, 1), dtype=torch.int32, device=DEV), i32([1] * n), torch.arange(n + 1, dtype=torch.int32, device=DEV))
    assert _lib.host_function("tree_attention")(args, {}) is None and aklr_amd.tree_attention_fp8(*args) is OOC
