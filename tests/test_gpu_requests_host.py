"""The native host path of draft verification, the page operators and the adapters against their Python path, their refusals on
the GPU, and what a call may not do: wait for the GPU, or use another stream than the current one."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import aklr_amd
from aklr_amd import _lib
from aklr_amd.dispatch import FallbackReason
from tests import test_gpu_cache_host as cache_host
from tests.helpers import say
from tests.test_gpu_kv_cache import BF16, DEV, new_cache
from tests.test_gpu_lora import problem as lora_problem
from tests.test_gpu_verify import problem as verify_problem

pytestmark = pytest.mark.gpu
OOC = FallbackReason.OUT_OF_CONTRACT
OPS = {"verify": aklr_amd.verify_drafts, "kv_copy": aklr_amd.kv_cache_copy_pages_fp8, "kv_compact": aklr_amd.kv_cache_compact_fp8,
       "kv_update": aklr_amd.kv_cache_update_pages, "lora": aklr_amd.lora_project}


@pytest.fixture(autouse=True)
def _ops(monkeypatch):
    monkeypatch.setattr(cache_host, "OPS", OPS)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def verify_args():
    p = verify_problem([4, 3, 5], 300, 1)
    return (p["target"], p["tokens"], p["starts"], p["u"], p["v"], 5), {"draft_probs": p["draft"], "parents": p["parents"]}


def lora_args(t=9):
    p = lora_problem(t, 72, 40, 16, 3, BF16, 2)
    return (p["x"], p["a"], p["b"], p["ids"], p["base"]), {"scales": p["scales"], "ranks": i32(16, 3, 0)}


def compact_args(most=4):
    cache = new_cache(6, 2, 64, 16, 3)
    path = torch.arange(1, most + 1, dtype=torch.int32, device=DEV).expand(2, most).contiguous()
    return (*cache, i32([0, 1, 2, 3, 4, 5], [5, 4, 3, 2, 1, 0])[:, :3], i32(40, 33), i32(0, 30, 50), path, i32(most, 2))


def test_verify():
    args, kw = verify_args()
    both = cache_host.both
    both("verify", args, kw, True)
    both("verify", args, {}, True)
    both("verify", args[:4], {"sample_uniforms": args[4], "most": 3, "parents": kw["parents"]}, True)
    both("verify", (args[0].half(), args[1].int(), *args[2:]), {"draft_probs": kw["draft_probs"].half()}, True)
    both("verify", (args[0][:0], args[1][:0], i32(0, 0), args[3][:0], args[4][:1], 2), {}, False)
    both("verify", (*args[:2], args[2][:1], args[3], args[4][:0], 2), {}, False)
    for at, bad in ((0, args[0].double()), (0, args[0][:, ::2]), (1, args[1].short()), (1, args[1][:3]), (2, args[2].long()), (3, args[3].double()),
                    (4, args[4][:2]), (5, 0), (5, 1025), (5, 3.0), (5, True), (5, 1 << 70), (5, -(1 << 70))):
        both("verify", (*args[:at], bad, *args[at + 1:]), kw, False, False)
    for bad in ({"draft_probs": kw["draft_probs"].half()}, {"draft_probs": kw["draft_probs"][:3]}, {"parents": kw["parents"].long()}, {"parents": 1}):
        both("verify", args, {**kw, **bad}, False, False)


def test_pages():
    both = cache_host.both
    cache = new_cache(6, 2, 64, 16, 3)
    both("kv_copy", (*cache, i32(0, 1, -1), i32(4, 5, 2)), {}, True)
    both("kv_copy", cache, {"src": torch.tensor([0, 9], device=DEV), "dst": torch.tensor([4, 5], device=DEV)}, True)
    both("kv_copy", (*cache, i32(), i32()), {}, False)
    for args in ((*cache, i32(0, 1), i32(2)), (*cache, i32(0), torch.tensor([1], device=DEV)), (cache[0], cache[0], *cache[2:], i32(0), i32(1)),
                 (*cache, i32([0]), i32([1])), (*cache, torch.zeros(2, device=DEV), i32(1, 2)), (*cache[:3], cache[3][:, :, ::2], i32(0), i32(1))):
        both("kv_copy", args, {}, False, False)
    for most in (4, 70):
        args = compact_args(most)
        both("kv_compact", args, {}, True)
        both("kv_compact", args[:7], {"path": args[7], "counts": args[8]}, True)
        for at, bad in ((4, args[4][:1]), (4, args[4].long()), (5, args[5][:1]), (6, args[6][:2]), (7, args[7].long()), (7, args[7].t()), (8, args[8].long()),
                        (0, args[0].view(torch.uint8))):
            both("kv_compact", (*args[:at], bad, *args[at + 1:]), {}, False, False)
    both("kv_compact", (*args[:7], args[7][:, :0], args[8]), {}, False)
    refs, table, lens, wants = i32(1, 1, 0, 0, 1), i32([0, 1], [4, -1]), i32(20, 7), i32(32, 9)
    both("kv_update", (refs, table, lens, wants, 16), {}, True)
    both("kv_update", (refs, table, lens, wants, 16, i32(1, 0)), {}, True)
    both("kv_update", (refs, table, lens, wants), {"page_size": 16, "parents": i32(1, 1)}, True)
    for args in ((refs.long(), table, lens, wants, 16), (refs, table[:1], lens, wants, 16), (refs, table, lens.long(), wants, 16), (refs, table, lens, wants, 0),
                 (refs, table, lens, wants, 16.0), (refs, table, lens, wants, 1 << 70), (refs, table, refs[:2], wants, 16), (refs, table, lens, wants, 1 << 30),
                 (refs[1:], table, lens, wants, 16), (refs, table, lens, wants, 16, i32(0))):
        both("kv_update", args, {}, False, False)


def test_lora():
    both = cache_host.both
    for t in (9, 300):
        args, kw = lora_args(t)
        both("lora", args, kw, True)
        both("lora", args, {}, True)
        both("lora", args[:3], {"adapters": args[3].int(), "base": args[4], "out": torch.zeros_like(args[4])}, True)
        both("lora", args, {**kw, "out": args[4]}, True)
        both("lora", tuple(x.half() if x.dtype == BF16 else x for x in args), kw, True)
    both("lora", (args[0][:0], *args[1:3], args[3][:0], args[4][:0]), {}, False)
    for at, bad in ((0, args[0].float()), (0, args[0][:, :36]), (1, args[1][:, :8]), (2, args[2][:2]), (3, args[3].float()), (3, args[3][:5]), (4, args[4].half()),
                    (2, args[2].transpose(1, 2)), (0, args[0].t())):
        both("lora", (*args[:at], bad, *args[at + 1:]), {}, False, False)
    for bad in ({"scales": kw["scales"].double()}, {"ranks": kw["ranks"].long()}, {"ranks": kw["ranks"][:2]}, {"out": args[4][:, :8]}, {"out": args[0]}):
        both("lora", args, {**kw, **bad}, False, False)


def test_gradients_tangents_and_transforms():
    say("refusals: gradients, tangents, transforms")
    args, kw = verify_args()
    largs, lkw = lora_args()
    cache = new_cache(6, 2, 64, 16, 3)
    for name, a, k, places in (("verify", args, kw, (0, 3, 4)), ("lora", largs, lkw, (0, 1, 2, 4)), ("kv_copy", (*cache, i32(0), i32(1)), {}, (2, 3))):
        host, fn = _lib.host_function(name), OPS[name]

        def refused(*x):
            return host(x, k) is None and fn(*x, **k) is OOC

        assert not isinstance(fn(*a, **k), FallbackReason) and host(a, k) is not None
        for i in places:
            assert refused(*a[:i], a[i].clone().requires_grad_(), *a[i + 1:])
            with forward_ad.dual_level():
                assert refused(*a[:i], forward_ad.make_dual(a[i], torch.ones_like(a[i])), *a[i + 1:])
            answers = []

            def ask(x):
                answers.append(refused(*a[:i], x, *a[i + 1:]))
                return x.float().sum()

            torch.vmap(ask)(torch.stack([a[i], a[i]]))
            torch.func.grad(ask)(a[i])
            assert answers == [True] * len(answers) and answers
    out = torch.zeros_like(largs[4]).requires_grad_()
    assert OPS["lora"](*largs, out=out) is OOC
    with torch.no_grad():
        assert OPS["lora"](*largs, out=out) is out


def test_disabled_and_traced(monkeypatch):
    say("disabled and traced")
    args, kw = lora_args()
    want = aklr_amd.lora_project(*args, **kw)
    monkeypatch.setenv("AKLR_DISABLE", "lora_project@1.0")
    assert aklr_amd.lora_project(*args, **kw) is FallbackReason.DISABLED
    assert not isinstance(aklr_amd.verify_drafts(*verify_args()[0]), FallbackReason)
    monkeypatch.setenv("AKLR_DISABLE", "0")
    monkeypatch.setenv("AKLR_TRACE", "op")
    assert torch.equal(aklr_amd.lora_project(*args, **kw), want)


def test_calls_wait_for_nothing_and_follow_the_stream():
    say("calls behind a long queue return, and run on the current stream")
    args, kw = lora_args()
    vargs, vkw = verify_args()
    uargs = (i32([0, 1], [4, -1]), i32(20, 7), i32(32, 9), 16)
    cargs = compact_args()
    before = [t.clone() if t.dtype != torch.float8_e4m3fn else t.view(torch.uint8).clone() for t in cargs[:4]]
    want = aklr_amd.lora_project(*args, **kw), aklr_amd.verify_drafts(*vargs, **vkw), aklr_amd.kv_cache_update_pages(i32(1, 1, 0, 0, 1), *uargs)
    aklr_amd.kv_cache_compact_fp8(*cargs)
    wanted = [t.view(torch.uint8).clone() for t in cargs[:4]]
    late = [torch.zeros_like(args[0]), torch.zeros_like(vargs[0]), i32(0, 0, 0, 0, 0)]
    given = i32(1, 1, 0, 0, 1)
    a = torch.ones((4096, 4096), device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(60):
            b = a @ a
        late[0].copy_(args[0])
        late[1].copy_(vargs[0])
        late[2].copy_(given)
        for t, w in zip(cargs[:4], before):
            t.view(torch.uint8).copy_(w.view(torch.uint8))
        got = aklr_amd.lora_project(late[0], *args[1:], **kw), aklr_amd.verify_drafts(late[1], *vargs[1:], **vkw), aklr_amd.kv_cache_update_pages(late[2], *uargs)
        aklr_amd.kv_cache_compact_fp8(*cargs)
        done = side.query()
    side.synchronize()
    assert not done and b is not None
    assert cache_host.same(got, want) and all(torch.equal(t.view(torch.uint8), w) for t, w in zip(cargs[:4], wanted))
