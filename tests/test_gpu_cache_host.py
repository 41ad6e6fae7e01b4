"""The native host path of the cache operators against their Python path: the same bits where it serves a call, None
exactly where the Python path decides (which then serves or refuses). Also what a call may not do: wait for the GPU."""
from __future__ import annotations

import pytest
import torch

import aklr_amd
from aklr_amd import _lib
from aklr_amd.dispatch import FallbackReason
from tests.helpers import say
from tests.test_gpu_attention import call, problem, tree
from tests.test_gpu_kv_cache import BF16, DEV, F16, new_cache, normal

pytestmark = pytest.mark.gpu
OPS = {"rotary": aklr_amd.rotary_embedding, "kv_write": aklr_amd.kv_cache_write_fp8,
       "rotary_kv_write": aklr_amd.rotary_kv_cache_write_fp8, "kv_read": aklr_amd.kv_cache_read_fp8,
       "tree_attention": aklr_amd.tree_attention_fp8}


def same(a, b):
    if isinstance(a, tuple):
        return isinstance(b, tuple) and len(a) == len(b) and all(same(x, y) for x, y in zip(a, b))
    if not isinstance(a, torch.Tensor):
        return a is b
    if a.dtype != b.dtype or a.shape != b.shape or a.stride() != b.stride():
        return False
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def both(name, args, kw, native, served=True):
    """Runs a call on each path, on cloned buffers that are written."""
    say(f"{name} {sorted(kw)} {native} {served}")

    def fresh():  # every tensor of the call again, with its strides, and one for one
        made = {}

        def again(x):
            if not isinstance(x, torch.Tensor):
                return x
            if id(x) not in made:
                base = x._base if x._base is not None else x
                if id(base) not in made:
                    made[id(base)] = base.detach().clone() if base.dtype != torch.float8_e4m3fn else base.view(torch.uint8).clone().view(base.dtype)
                y = made[id(base)]
                if base is not x:
                    y = y.view(x.dtype) if y.dtype != x.dtype else y
                    y = torch.as_strided(y, x.shape, x.stride(), x.storage_offset() - base.storage_offset() + y.storage_offset())
                made[id(x)] = y
            return made[id(x)]
        return tuple(again(x) for x in args), {k: again(x) for k, x in kw.items()}

    a1, k1 = fresh()
    a2, k2 = fresh()
    got = _lib.host_function(name)(a1, k1)
    want = OPS[name].general(*a2, **k2)
    assert (got is not None) == native and isinstance(want, FallbackReason) != served
    if native:
        assert same(got, want)
        for x, y in zip(a1 + tuple(k1[k] for k in sorted(k1)), a2 + tuple(k2[k] for k in sorted(k2))):
            if isinstance(x, torch.Tensor):
                assert same(x, y)  # what was written
    a3, k3 = fresh()
    assert same(OPS[name](*a3, **k3), want)


def test_rotary():
    f = aklr_amd.rotary_frequencies(64, device=DEV)
    q, k = normal((5, 4, 64), BF16, 1), normal((5, 2, 64), BF16, 2)
    pos = torch.arange(5, device=DEV) * 77
    for kw in ({}, {"interleaved": True, "magnitude": 2}, {"magnitude": 1.5}, {"out_q": torch.zeros_like(q)}, {"out_q": q, "out_k": k},
               {"out_k": torch.zeros((2, 5, 64), dtype=BF16, device=DEV).transpose(0, 1)}):
        both("rotary", (q, k, pos, f), kw, True)
    both("rotary", (q, None, pos.to(torch.int32), f), {}, True)
    both("rotary", (q,), {"k": k, "positions": pos, "frequencies": f}, True)
    both("rotary", (q[:0], k[:0], pos[:0], f), {}, False)
    rows = normal((5, 6 * 64), BF16, 3)
    both("rotary", (rows[:, :256].view(5, 4, 64), rows[:, 256:].view(5, 2, 64), pos, f), {}, True)
    for args, kw in [((q.double(), k, pos, f), {}), ((q, k.half(), pos, f), {}), ((q, k, pos.float(), f), {}), ((q, k, pos, f.float()), {}),
                     ((q, k, pos, f[:9]), {}), ((q, k, pos[:4], f), {}), ((q, k, pos, f), {"magnitude": float("nan")}),
                     ((q, k, pos, f), {"interleaved": 3}), ((q, k, pos, f), {"out_q": q[:, :2]}), ((q, None, pos, f), {"out_k": k}),
                     ((q[..., :40], k[..., :40], pos, f[:16]), {}), ((q, k, pos, f), {"out_q": q.view(-1)[:640].view(5, 2, 64)}),
                     ((q.view(-1)[1:257].view(1, 4, 64), None, pos[:1], f), {})]:
        both("rotary", args, kw, False, False)
    wants = q.clone().requires_grad_()
    assert _lib.host_function("rotary")((wants, k, pos, f), {}) is None
    assert aklr_amd.rotary_embedding(wants, k, pos, f) is FallbackReason.OUT_OF_CONTRACT
    with torch.no_grad():
        assert same(aklr_amd.rotary_embedding(wants, k, pos, f), aklr_amd.rotary_embedding(q, k, pos, f))


def test_writes_and_read():
    f = aklr_amd.rotary_frequencies(128, device=DEV)
    q, k, v = normal((5, 4, 128), BF16, 1), normal((5, 2, 128), BF16, 2), normal((5, 2, 128), BF16, 3)
    cache = new_cache(3, 2, 128, 32)
    slots, pos = torch.tensor([3, -1, 95, 96, 40], device=DEV), torch.arange(5, device=DEV)
    both("kv_write", (k, v, *cache, slots), {}, True)
    both("kv_write", (k.float(), v.float(), *cache), {"slots": slots.to(torch.int32)}, True)
    both("kv_write", (k[:0], v[:0], *cache, slots[:0]), {}, False)
    both("rotary_kv_write", (q, k, v, pos, f, *cache, slots), {}, True)
    both("rotary_kv_write", (q, k, v, pos, f, *cache, slots), {"interleaved": True, "magnitude": 1.2, "out": q}, True)
    both("rotary_kv_write", (q, k, v, pos, f, *cache, slots), {"out": torch.zeros_like(q)}, True)
    for args in [(k.double(), v, *cache, slots), (k, v[:, :1], *cache, slots), (k, v, cache[0], cache[0], *cache[2:], slots),
                 (k, v, *cache, slots.float()), (k, v, *cache[:2], cache[2].half(), cache[3], slots), (k, v, *cache, slots[:3]),
                 (k, v, cache[0].view(torch.uint8), *cache[1:], slots), (k[..., :64], v[..., :64], *cache, slots)]:
        both("kv_write", args, {}, False, False)
    both("rotary_kv_write", (q, k, v, pos, f, *cache, slots), {"out": k}, False, False)
    both("rotary_kv_write", (q[..., :64], k, v, pos, f, *cache, slots), {}, False, False)
    aklr_amd.kv_cache_write_fp8(k, v, *cache, slots)
    table, starts = torch.tensor([[0, 1], [2, 7]], dtype=torch.int32, device=DEV), torch.tensor([0, 40, 80], dtype=torch.int32, device=DEV)
    both("kv_read", (*cache, table, starts, 80), {}, True)
    both("kv_read", (*cache, table, starts, 80), {"out_dtype": F16, "out_k": None}, True)
    both("kv_read", (*cache, table, starts, 80), {"out_k": torch.zeros((80, 2, 128), dtype=BF16, device=DEV)}, False)
    for args, kw in [((*cache, table, starts, -1), {}), ((*cache, table, starts, 1 << 31), {}), ((*cache, table, starts, 80.0), {}),
                     ((*cache, table, starts, 1 << 70), {}), ((*cache, table.long(), starts, 80), {}), ((*cache, table, starts[:2], 80), {}),
                     ((*cache, table, starts, 80), {"out_dtype": torch.float32})]:
        both("kv_read", args, kw, False, False)


def test_attention():
    p = problem([90, 33], [3, 2], 2, 3, 128, 32, mask=tree)
    args = (p["q"], *p["cache"], p["table"], p["lens"], p["starts"])
    for kw in ({}, {"tree_mask": p["mask"]}, {"return_lse": True}, {"softmax_scale": 0.3, "out": torch.zeros_like(p["q"])},
               {"return_lse": True, "out": torch.zeros_like(p["q"]), "tree_mask": p["mask"].to(torch.uint8)}):
        both("tree_attention", args, kw, True)
    both("tree_attention", (*args, p["mask"]), {"softmax_scale": 1}, True)
    both("tree_attention", (p["q"][:0], *args[1:]), {}, False)
    for at, bad in ((0, p["q"].float()), (0, p["q"][:, :5]), (0, p["q"][..., :64]), (5, p["table"][:1]), (5, p["table"].long()),
                    (6, p["lens"].long()), (7, p["starts"][:2]), (2, p["cache"][0].view(torch.uint8))):
        both("tree_attention", (*args[:at], bad, *args[at + 1:]), {}, False, False)
    for kw in ({"tree_mask": p["mask"].float()}, {"tree_mask": p["mask"][:2]}, {"softmax_scale": float("inf")}, {"out": p["q"]},
               {"return_lse": "yes"}):
        both("tree_attention", args, kw, False, False)


def test_calls_wait_for_nothing_and_follow_the_stream():
    say("a call behind a long queue returns, and runs on the current stream")
    p = problem([500], [1], 2, 4, 128, 16)
    want = call(p)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    q = torch.zeros_like(p["q"])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        a = torch.ones((4096, 4096), device=DEV)
        for _ in range(40):
            b = a @ a
        q.copy_(p["q"])
        got = call({**p, "q": q})
        done = side.query()
    side.synchronize()
    assert not done and torch.equal(got, want) and b is not None
