"""Adapters on the GPU against the oracle in 64 bits.

Tolerances. Products of bf16 (8 x 8 bits) and fp16 (11 x 11) values are exact in fp32. The sum over K of n terms in fp32 is off
by at most n * 2^-24 of the sum of their magnitudes in any order; K + 64 covers the parts' joins. v enters the second product as
two pieces, off by 2^-17 of it (bf16: half a step of what the first left) or 2^-23 of the token's largest (fp16, scaled to 0.5
to 1, half a step of the least subnormal 2^-25), which the sum over the rank multiplies by |b|; that product's own sum has 2 R
terms. The sum with base and the scale round twice in fp32, then half a step of the type. The oracle gives the sums of
magnitudes."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aklr_amd
from oracle import requests as oq
from tests.helpers import say
from tests.test_gpu_kv_cache import half_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16 = torch.bfloat16, torch.float16


def problem(t, k, n, r, count, dtype, seed, kind="mixed"):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x, base = (torch.randn(s, generator=g, device=DEV).to(dtype) for s in ((t, k), (t, n)))
    a = (torch.randn((count, r, k), generator=g, device=DEV) * k**-0.5).to(dtype)
    b = (torch.randn((count, n, r), generator=g, device=DEV) * r**-0.5).to(dtype)
    if kind == "mixed":
        ids = torch.randint(-1, count, (t,), generator=g, device=DEV)
    elif kind == "runs":
        ids = (torch.arange(t, device=DEV) // max(1, t // 5)) % (count + 1) - 1
    elif kind == "one":
        ids = torch.full((t,), count - 1, device=DEV)
    else:
        ids = torch.full((t,), -1, device=DEV)
    return {"x": x, "a": a, "b": b, "ids": ids, "base": base, "scales": torch.randn(count, generator=g, device=DEV), "ranks": None}


def call(p, **kw):
    return aklr_amd.lora_project(p["x"], p["a"], p["b"], p["ids"], p["base"], scales=p["scales"], ranks=p["ranks"], **kw)


def check(got, p, what=""):
    d = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    a, b = d(p["a"]), d(p["b"])
    want, terms, size = oq.lora(d(p["x"]), a, b, p["ids"].cpu().numpy(), d(p["base"]), d(p["scales"]), d(p["ranks"]))
    dtype, k, r = p["x"].dtype, a.shape[2], a.shape[1]
    piece = 2**-17 if dtype == BF16 else 2**-23
    tol = half_step(want, dtype) * (1 + 2**-10) + terms * (k + 64) * 2**-24 + size * (piece + (2 * r + 64) * 2**-24)
    tol += 2**-23 * (np.abs(d(p["base"])) + np.abs(want - d(p["base"])))
    far = np.abs(got.double().cpu().numpy() - want) - tol
    assert got.dtype == dtype and got.shape == want.shape and (far <= 0).all(), f"{what}: {far.max()} past its tolerance at {np.argwhere(far > 0)[:3].tolist()}"


SIZES = [(1, 8, 8, 8, 1), (2, 64, 64, 16, 1), (5, 40, 24, 24, 3), (16, 72, 40, 8, 2), (17, 264, 136, 16, 2), (64, 520, 1032, 40, 9),
         (65, 512, 256, 128, 3), (129, 1000, 72, 32, 200), (200, 1032, 520, 64, 50), (256, 264, 328, 56, 4), (257, 136, 264, 16, 5),
         (300, 72, 264, 128, 5), (700, 520, 136, 24, 300), (1999, 264, 72, 64, 9), (2048, 8, 8, 8, 2), (2053, 136, 328, 8, 4),
         (3001, 1032, 264, 128, 7), (2500, 264, 520, 32, 3), (2200, 2056, 72, 64, 33)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t,k,n,r,count", SIZES)
def test_sizes(t, k, n, r, count, dtype):
    say(f"lora {t} {k} {n} {r} {count} {dtype}")
    for kind in ("mixed", "runs"):
        p = problem(t, k, n, r, count, dtype, t + k, kind)
        check(call(p), p, kind)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t,k,n,r,count", [(7168, 72, 40, 16, 3), (7301, 136, 2056, 128, 5), (7200, 264, 2048, 128, 9), (9000, 1032, 4104, 64, 2),
                                           (4000, 512, 4096, 128, 3), (8000, 136, 72, 24, 4000), (7999, 2056, 520, 8, 1), (16400, 72, 4096, 32, 7)])
def test_many_tokens(t, k, n, r, count, dtype):
    # the oracle on some of the rows; all rows of tokens without an adapter
    say(f"lora many {t} {k} {n} {r} {count} {dtype}")
    for kind in ("mixed", "runs"):
        p = problem(t, k, n, r, count, dtype, t + k, kind)
        p["ranks"] = torch.arange(count, dtype=torch.int32, device=DEV) % (r + 1)
        p["ranks"][-1] = r
        got = call(p)
        none = (p["ids"] < 0) | (p["ranks"][p["ids"].clamp(min=0)] == 0)
        assert torch.equal(got[none], p["base"][none])
        rows = torch.from_numpy(np.r_[0, t - 1, np.random.RandomState(1).choice(t, 250, replace=False)]).to(DEV)
        check(got[rows], {**p, "x": p["x"][rows], "ids": p["ids"][rows], "base": p["base"][rows]}, kind)
        assert bool(got.isfinite().all()) and torch.equal(call({**p, "base": p["base"].clone()}, out=p["base"]), got)


@pytest.mark.parametrize("t", [3, 40, 250, 600, 2300])
def test_who_has_which(t):
    say(f"lora adapters {t}")
    for kind in ("one", "none"):
        p = problem(t, 136, 72, 16, 3, BF16, 5, kind)
        got = call(p)
        check(got, p, kind)
        if kind == "none":
            assert torch.equal(got, p["base"])
    p = problem(t, 136, 72, 16, 3, BF16, 6)
    p["ids"][::4] = torch.tensor([3, -(1 << 40), 1 << 32, (1 << 32) + 1, 1 << 62, -1, (1 << 31) - 1, -(1 << 31)], device=DEV).repeat(t)[: len(p["ids"][::4])]
    got = call(p)
    check(got, p, "numbers of no adapter")
    small = p["ids"].clamp(-(1 << 31), (1 << 31) - 1)
    assert torch.equal(call({**p, "ids": small.to(torch.int32)}), got)
    assert torch.equal(call({**p, "scales": None}), call({**p, "scales": torch.ones(3, device=DEV)}))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t,k,n,r,count", [(300, 4104, 4104, 64, 3), (700, 2056, 4360, 128, 6), (2600, 4096, 4096, 40, 2), (257, 4360, 8200, 104, 40)])
def test_many_ranges_of_columns(t, k, n, r, count, dtype):
    say(f"lora ranges {t} {k} {n} {r} {count} {dtype}")
    for kind in ("mixed", "runs"):
        p = problem(t, k, n, r, count, dtype, t + n, kind)
        got = call(p)
        check(got, p, kind)
        assert torch.equal(call(p), got)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t,r", [(9, 8), (70, 24), (200, 128), (400, 64), (2300, 16), (2100, 128), (7200, 64)])
def test_ranks_and_what_lies_behind_them(t, r, dtype):
    say(f"lora ranks {t} {r} {dtype}")
    p = problem(t, 264, 136, r, 12, dtype, 7)
    p["ranks"] = torch.tensor(([0, 1, 7, r - 1, r, 3, r // 2, r // 2 + 1, r - 8, 4, r, 2])[:12], dtype=torch.int32, device=DEV)
    want = call(p)
    check(want, p)
    for i, n in enumerate(p["ranks"].tolist()):
        p["a"][i, n:], p["b"][i, :, n:] = float("nan"), float("inf")
    assert torch.equal(call(p), want)
    odd = p["ranks"].clone()
    odd[odd == r] = r + 1000  # counts as r
    odd[odd == 0] = -5
    assert torch.equal(call({**p, "ranks": odd}), want)


@pytest.mark.parametrize("t", [20, 200, 500, 2100, 7300])
def test_views_and_places(t):
    say(f"lora views {t}")
    k, n, r, count = 136, 72, 16, 4
    p = problem(t, k, n, r, count, BF16, 8)
    want = call(p)
    g = torch.Generator(device=DEV).manual_seed(9)
    wide_x = torch.randn((t, k + 24), generator=g, device=DEV).bfloat16()
    wide_x[:, 16:16 + k] = p["x"]
    stack_a, stack_b = torch.full((count, 3 * r, k), float("nan"), dtype=BF16, device=DEV), torch.full((count, 2 * n, r), float("nan"), dtype=BF16, device=DEV)
    stack_a[:, r:2 * r], stack_b[:, n:] = p["a"], p["b"]
    rows = torch.randn((t, 3 * n), generator=g, device=DEV).bfloat16()
    rows[:, n:2 * n] = p["base"]
    keep = rows.clone()
    q = {**p, "x": wide_x[:, 16:16 + k], "a": stack_a[:, r:2 * r], "b": stack_b[:, n:], "base": rows[:, n:2 * n]}
    assert torch.equal(call(q), want) and torch.equal(rows, keep)
    assert call(q, out=rows[:, 2 * n:]) is not None and torch.equal(rows[:, 2 * n:], want) and torch.equal(rows[:, :2 * n], keep[:, :2 * n])
    view = rows[:, n:2 * n]
    assert call(q, out=view) is view and torch.equal(view, want) and torch.equal(rows[:, :n], keep[:, :n])
    out = torch.full((t, n), 7.0, dtype=BF16, device=DEV)
    assert call(p, out=out) is out and torch.equal(out, want)
    assert torch.equal(call({**p, "x": p["x"][:1].expand(t, k)})[:1], want[:1])
    few = {**p, "x": p["x"][:0], "ids": p["ids"][:0], "base": p["base"][:0]}
    assert call(few).shape == (0, n)


def test_a_result_does_not_hang_on_its_place():
    say("lora: tokens in another order, among others, twice")
    for t in (60, 250, 700, 2600, 7400):
        p = problem(t, 520, 264, 32, 6, BF16, 10)
        want = call(p)
        assert torch.equal(call(p), want)
        order = torch.randperm(t, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
        assert torch.equal(call({**p, "x": p["x"][order], "ids": p["ids"][order], "base": p["base"][order]}), want[order])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t", [20, 300, 7300])
def test_values_that_are_not_finite_stay_with_their_token(t, dtype):
    say(f"lora values {t} {dtype}")
    p = problem(t, 136, 72, 24, 3, dtype, 11, "one")
    want = call(p)
    x = p["x"].clone()
    x[3, 5], x[7, 0], x[11, 135] = float("nan"), float("inf"), -float("inf")
    got = call({**p, "x": x})
    bad = torch.zeros(t, dtype=torch.bool, device=DEV)
    bad[[3, 7, 11]] = True
    assert torch.equal(got[~bad], want[~bad]) and not got[bad].isfinite().any()
    base = p["base"].clone()
    base[2, 9] = float("inf")
    got = call({**p, "base": base})
    want2 = want.clone()
    want2[2, 9] = float("inf")
    assert torch.equal(got, want2)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t", [20, 300, 7300])
def test_an_infinite_weight_beside_large_values(t, dtype):
    say(f"lora infinite weight {t} {dtype}")
    p = problem(t, 136, 72, 24, 3, dtype, 15)
    p["x"], p["a"][1] = p["x"] * 2.0**12, p["a"][1] * 2.0**12  # v of 2^24, past fp16
    p["x"][p["x"] == 0], p["b"][p["b"] == 0], p["scales"][1] = 1, 1, 0.5
    want = call(p)
    hit = p["ids"] == 1
    p["a"][1, 7, 5] = float("inf")
    got = call(p)
    assert hit.any() and torch.equal(got[~hit], want[~hit])
    assert torch.equal(got[hit], (p["x"][hit][:, 5:6].sign() * p["b"][1, :, 7].sign() * float("inf")).to(dtype))


@pytest.mark.parametrize("t", [20, 300])
def test_large_and_small_values(t):
    # products of 2^15 and more in a row: v of 2^36, past fp16; weights of fp16's subnormals
    say(f"lora large and small {t}")
    p = problem(t, 264, 40, 16, 2, F16, 12, "one")
    p["x"] *= 2.0**12
    p["a"] *= 2.0**10
    p["b"] = (p["b"].float() * 2.0**-20).half()
    check(call(p), p, "large")
    p = problem(t, 264, 40, 16, 2, F16, 13, "one")
    p["a"] = (p["a"].float() * 2.0**-18).half()
    p["b"] = (p["b"].float() * 2.0**8).half()
    p["base"].zero_()
    check(call(p), p, "small")
    p = problem(t, 264, 40, 16, 2, BF16, 14, "one")
    p["x"], p["a"], p["b"] = p["x"] * 2.0**40, p["a"] * 2.0**30, p["b"] * 2.0**-70
    check(call(p), p, "bf16")


def test_offsets_past_32_bits():
    say("lora: weights and rows behind 2^31 values")
    count, r, k, n, t = 300, 128, 65536, 64, 4
    a = torch.zeros((count, r, k), dtype=BF16, device=DEV)
    b = torch.zeros((count, n, r), dtype=BF16, device=DEV)
    a[count - 1, 5, 65535], b[count - 1, 63, 5] = 2, 3
    x = torch.ones((t, k), dtype=BF16, device=DEV)
    base = torch.ones((t, n), dtype=BF16, device=DEV)
    want = base.clone()
    want[2, 63] = 7
    ids = torch.tensor([0, 1, count - 1, -1], device=DEV)
    assert torch.equal(aklr_amd.lora_project(x, a, b, ids, base), want)
    del a
    wide = torch.zeros((1100, 1 << 21), dtype=BF16, device=DEV)
    x = wide[:, :64]
    x[1099, 7] = 4
    a = torch.zeros((2, 8, 64), dtype=BF16, device=DEV)
    a[1, 3, 7] = 2
    b = torch.zeros((2, 16, 8), dtype=BF16, device=DEV)
    b[1, 9, 3] = 1
    out = wide[:, 128:144]
    aklr_amd.lora_project(x, a, b, torch.ones(1100, dtype=torch.int64, device=DEV), wide[:, 64:80], out=out)
    assert out[1099, 9] == 8 and out.sum() == 8


def test_captured_and_on_streams():
    say("lora: captured, replayed with other values between eager calls; two streams at once")
    for t in (40, 250, 700, 7200):
        ps = [problem(t, 264, 136, 32, 5, BF16, s) for s in range(30, 33)]
        p = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in ps[0].items()}
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call(p)
        for q in ps + ps[:2]:
            for k, v in q.items():
                if isinstance(v, torch.Tensor):
                    p[k].copy_(v)
            graph.replay()
            want = call(q)
            torch.cuda.synchronize()
            assert torch.equal(got, want)
        want = [call(q) for q in ps]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in ps]
        for _ in range(4):
            outs = []
            for s, q in zip(streams, ps):
                with torch.cuda.stream(s):
                    outs.append(call(q))
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
