"""How exactly the attention over the FP8 cache weighs values: every form of the kernel, both types, against 64 bits.

Tolerance. A score's products are exact in fp32 (8 by 4, or 11 by 4, bits), their sum and the scalings round at most
head_dim + 2 times by 2^-24 of scale * sum |q_d k_d| =: size; the exponential and its argument, in powers of two below
|x| + 64, by 2^-24 of (8 |x| + 128). So a weight is off by a factor of 1 + e with e = 2^-24 * ((head_dim + 3) * size +
8 |x| / ln 2 + 128). Before the second product it is rounded to bf16, half a step of which is 2^-8: W of it is lost, 2^-8
where one bf16 holds it, 2^-16 where a second holds what the first leaves. A sum over n positions, of the weights or of a
dimension, is at most n + 64 roundings of 2^-24 of the weighted sum of |v|. So an output is off by at most (W + 2 e +
2 (n + 64) 2^-24) times that, and by half a step of its type: 2^-25 where fp16 has no more bits.
"""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import aklr_amd
from aklr_amd import _lib
from tests.helpers import say
from tests.test_gpu_attention import call, i32, problem, tree
from tests.test_gpu_kv_cache import BF16, DEV, F16, new_cache, normal

pytestmark = pytest.mark.gpu

# sequences, query tokens each, kv heads, group: as many rows a tile as the form takes (d: 64 and 128, or 256)
FORMS = {16: (64, 1, 8, 4), 32: (64, 6, 8, 4), 64: (8, 12, 16, 4), 128: (4, 33, 16, 4)}
FORMS_OF = [(d, r) for d in (64, 128, 256) for r in FORMS if (d, r) != (256, 32)]


def rows_of(p):
    """(rows of a tile, workgroups a tile's pieces are joined by) of a problem's call."""
    joiners = ctypes.c_int(-1)
    t, hq, d = p["q"].shape
    cache = p["cache"][0]
    rows = _lib.lib().aklr_tree_attention_fp8_rows(t, p["lens"].numel(), hq, cache.shape[1], d,
                                                   p["table"].shape[1] * cache.shape[2], ctypes.byref(joiners))
    return rows, joiners.value


def reach(p, rows):
    """Widens the block table, whose room the choice of a form goes by, until the call takes tiles of `rows` rows."""
    page = p["cache"][0].shape[2]
    while rows_of(p)[0] != rows and p["table"].shape[1] * page < 2**18:
        p["table"] = torch.cat([p["table"], torch.full_like(p["table"], -1)], 1)
    assert rows_of(p)[0] == rows, (rows_of(p), rows)


def lost(rows, dtype):
    return 2**-16 if rows <= 32 or dtype == F16 else 2**-8


def exact(p, scale):
    """out, lse, weighted |v|, size, n in 64 bits."""
    kc, vc, ks, vs = p["cache"]
    heads, page, d = kc.shape[1:]
    hq = p["q"].shape[1]
    starts, lens = p["starts"].tolist(), p["lens"].tolist()
    outs = [torch.zeros(p["q"].shape, dtype=torch.float64, device=DEV) for _ in range(2)]
    rows = [torch.zeros(p["q"].shape[:2], dtype=torch.float64, device=DEV) for _ in range(2)]
    for b, n in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        pages = p["table"][b, : -(-n // page)].long()
        there = ((pages >= 0) & (pages < kc.shape[0])).repeat_interleave(page)[:n]
        pages = pages.clamp(0, kc.shape[0] - 1)
        k, v = ((c.view(torch.uint8)[pages].view(c.dtype).float().double() * s[pages].double()[..., None]).permute(1, 0, 2, 3).reshape(heads, -1, d)[:, :n].contiguous()
                for c, s in ((kc, ks), (vc, vs)))
        t, group = hi - lo, hq // heads
        q = p["q"][lo:hi].double().view(t, heads, group, d).transpose(0, 1).reshape(heads, t * group, d)
        if not t or not n:
            rows[0][lo:hi] = -float("inf")
            continue
        j = torch.arange(n, device=DEV) - (n - t)
        if p["mask"] is None:
            sees = j <= torch.arange(t, device=DEV)[:, None]
        else:
            sees = (j < 0) | p["mask"][lo:hi, j.clamp(0, t - 1)].bool()
        sees = (sees & there).repeat_interleave(group, 0)

        def place(x):  # [heads, t * group, ...] -> [t, hq, ...]
            return x.view(heads, t, group, *x.shape[2:]).transpose(0, 1).reshape(t, hq, *x.shape[2:])

        x = (torch.matmul(q, k.transpose(1, 2).contiguous()) * scale).masked_fill(~sees, -float("inf"))
        end = x.logsumexp(-1)
        w = (x - end[..., None]).exp().masked_fill(~sees, 0)
        outs[0][lo:hi], outs[1][lo:hi], rows[0][lo:hi] = place(torch.matmul(w, v)), place(torch.matmul(w, v.abs())), place(end)
        size = torch.matmul(q.abs(), k.abs().transpose(1, 2).contiguous()).masked_fill(~sees, 0).amax(-1) * abs(scale)
        rows[1][lo:hi] = place(size)
    return outs[0], rows[0], outs[1], rows[1], max(lens)


def check(p, rows=None, scale=None, joined=None):
    if rows is not None:
        reach(p, rows)
    got_rows, joiners = rows_of(p)
    assert joined is None or bool(joiners) == joined
    d, dtype = p["q"].shape[2], p["q"].dtype
    scale = d ** -0.5 if scale is None else scale
    out, lse = call(p, return_lse=True, softmax_scale=scale)
    want, wl, weighed, size, n = exact(p, scale)
    top = size.clamp_min(1) / np.log(2)
    e = 2**-24 * ((d + 3) * size + 8 * top + 128)
    end, empty = int(p["starts"][-1]), wl == -float("inf")
    assert torch.equal(lse[:end] == -float("inf"), empty[:end]) and not bool(out[:end][empty[:end]].any())
    out, lse, want, wl, weighed, e, empty = (x[:end] for x in (out, lse, want, wl, weighed, e, empty))
    assert bool(((lse.double() - wl).abs() <= e + (n + 64) * 2**-24 + 2**-23 * wl.abs())[~empty].all())
    tol = weighed * (lost(got_rows, dtype) + 2 * e[..., None] + 2 * (n + 64) * 2**-24)
    tol = tol + want.abs() * torch.finfo(dtype).eps / 2 * 1.01 + (2**-25 if dtype == F16 else 0)
    finite = want.abs() <= torch.finfo(dtype).max
    assert not bool(out[finite].isnan().any())
    far = ((out.double() - want).abs() - tol)[finite]
    assert bool((far <= 0).all()), f"{float(far.max())} past the tolerance"
    assert torch.equal(out, call(p, softmax_scale=scale)[:end])
    return out, lse


def built(form, d, dtype, ctx, bits, values, page=32, seed=0, alike=False):
    """Sequences whose positions p < ctx score bits[p] (in powers of two; heads that are not alike up to twice that) and
    hold `values` [ctx, d] times a kv head's factor; the query tokens' own positions score 0 and hold the first values."""
    b, t, h, group = FORMS[form]
    n = ctx + t
    scale = 0.125
    k = torch.zeros((n, h, d), device=DEV)
    k[:ctx, :, 0] = bits[:, None] / (4 * scale / np.log(2))
    v = torch.cat([values, values[:t]])[:, None] * torch.linspace(0.5, 1, h, device=DEV)[None, :, None]
    cols = -(-n // page)
    cache = new_cache(b * cols, h, d, page)
    table = torch.randperm(b * cols, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)).to(torch.int32).view(b, cols)
    at = torch.arange(n, device=DEV)
    for i in range(b):
        aklr_amd.kv_cache_write_fp8(k, v, *cache, table[i].long()[at // page] * page + at % page)
    q = torch.zeros((b * t, h * group, d), device=DEV)
    q[..., 0] = 4 * (1 + torch.arange(h * group, device=DEV) / 64 * (not alike))
    return {"q": q.to(dtype), "cache": cache, "table": table, "lens": i32([n] * b), "starts": i32(np.arange(b + 1) * t), "mask": None}, scale


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("d,form", FORMS_OF)
def test_weights_keep_their_bits(d, form, masked, dtype):
    say(f"weights {d} {form} {masked} {dtype}")
    b, t, h, group = FORMS[form]
    p = problem([300 + 37 * i for i in range(b)], [t] * b, h, group, d, 16, dtype, seed=21, mask=tree if masked else None)
    check(p, form)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,form", FORMS_OF)
def test_one_large_value_among_small_ones(d, form, dtype):
    # values from a cache that fp16 could not have written: a scale of 600 on a position whose weight, 13 powers of two
    # above what came before it, is most of the sum
    say(f"large value {d} {form} {dtype}")
    ctx = 2048
    place = torch.arange(ctx, device=DEV) % 512
    bits = torch.where((place >= 256) & (place < 320), 13.0, 0.0)
    values = normal((ctx, d), torch.float32, 5)
    values[270, 3] = 600 * 448
    values[280, 7] = -1e5
    p, scale = built(form, d, dtype, ctx, bits, values, alike=True)
    check(p, form, scale)


@pytest.mark.parametrize("gap", [17, 24, 29])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,form", FORMS_OF)
def test_positions_that_draw_all_the_weight_and_hold_nothing(d, form, dtype, gap):
    # what the others hold is the output: 2^-gap of the sum each, in every wave's and every piece's share
    say(f"sink {d} {form} {dtype} {gap}")
    ctx = 2048
    at = torch.arange(ctx, device=DEV)
    bits = torch.where(at % 16 == 0, float(gap), torch.rand(ctx, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)))
    values = normal((ctx, d), torch.float32, 6) * 2.0**8
    values[at % 16 == 0] = 0
    p, scale = built(form, d, dtype, ctx, bits, values)
    out, _ = check(p, form, scale)
    assert bool(out.any())


@pytest.mark.parametrize("power", [-6, -11, -16])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,form", [(64, 16), (128, 32), (128, 128), (256, 128)])
def test_small_values_keep_their_bits(d, form, dtype, power):
    say(f"small values {d} {form} {dtype} {power}")
    ctx = 700
    values = normal((ctx, d), torch.float32, 7) * 2.0**power
    p, scale = built(form, d, dtype, ctx, torch.zeros(ctx, device=DEV), values)
    check(p, form, scale)
