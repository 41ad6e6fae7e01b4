"""Rotary positions and the FP8 cache's write and read on the GPU, against the 64-bit oracle.

Tolerances. Rotation: cos and sin come from a fraction of a half-turn rounded to fp32 (pi * 2^-25 of angle), a sincos
of at most 4 ulps (2^-22 near 1), one rounding by the magnitude (2^-24), and two roundings of the sum (2^-23): together
under 2^-20 of magnitude * (|a| + |b|) for the pair (a, b); then half a step of the output's type. Stored keys and
values that are not rotated, and what is read back, are the oracle's fp32 steps bit for bit. A rotated key: its scale is
within 2^-20 * magnitude * max(|a| + |b|) / 448 and two roundings of the exact one, its code within half a step of e4m3
(2^-4 of the value, 2^-10 of the scale below the normal range) of the rotated value, plus the errors before it.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aklr_amd
from oracle import cache as oc
from tests.helpers import assert_same_bits, say, u8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(shape, dtype, seed):
    return torch.randn(shape, generator=gen(seed), device=DEV).to(dtype)


def half_step(y, dtype):
    return np.maximum(np.abs(y) * torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2)


def pair_size(x, rot, interleaved):
    """|a| + |b| at both places of every pair, 0 elsewhere."""
    x = np.abs(x.double().cpu().numpy())
    out = np.zeros_like(x)
    lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    out[..., lo] = out[..., hi] = x[..., lo] + x[..., hi]
    return out


def check_rotated(got, x, positions, f, interleaved, magnitude, what):
    want = oc.rotate(x.double().cpu().numpy(), positions.cpu().numpy(), f.cpu().numpy(), interleaved, magnitude)
    tol = half_step(want, x.dtype) * (1 + 2**-10) + 2**-20 * abs(magnitude) * pair_size(x, 2 * f.numel(), interleaved)
    far = np.abs(got.double().cpu().numpy() - want) - tol
    assert got.dtype == x.dtype and (far <= 0).all(), f"{what}: {far.max()} past its tolerance"
    if 2 * f.numel() < x.shape[-1]:
        assert torch.equal(got[..., 2 * f.numel():], x[..., 2 * f.numel():])


def new_cache(pages, heads, dim, page, seed=None):
    c = aklr_amd.new_kv_cache_fp8(pages, heads, dim, page, DEV)
    if seed is not None:  # anything, so that a stray write shows
        for t in c[:2]:
            t.view(torch.uint8).random_(0, 256, generator=gen(seed))
        for t in c[2:]:
            t.uniform_(0, 1, generator=gen(seed + 1))
    return c


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("t,hq,hk,d,rot", [(1, 1, 1, 16, 16), (3, 5, 2, 64, 64), (16, 128, 1, 64, 64), (33, 4, 4, 128, 64),
                                           (7, 3, 1, 96, 48), (2, 1, 1, 1024, 1024), (257, 32, 8, 128, 128), (1, 300, 2, 256, 32),
                                           (2051, 32, 8, 128, 64)])
def test_rotary(t, hq, hk, d, rot, dtype, interleaved):
    say(f"rotary {t} {hq} {hk} {d} {rot} {dtype} {interleaved}")
    q, k = normal((t, hq, d), dtype, 1), normal((t, hk, d), dtype, 2)
    pos = torch.randint(0, 1 << 24, (t,), generator=gen(3), device=DEV)
    f = aklr_amd.rotary_frequencies(rot, scaling="yarn", factor=8.0, original_length=4096, device=DEV)
    a, b = aklr_amd.rotary_embedding(q, k, pos, f, interleaved=interleaved, magnitude=1.25)
    check_rotated(a, q, pos, f, interleaved, 1.25, "q")
    check_rotated(b, k, pos, f, interleaved, 1.25, "k")


def test_rotary_places_and_forms():
    say("rotary: position 0, negative and int32 positions, no k, no tokens, views, in place, outputs given")
    f = aklr_amd.rotary_frequencies(64, device=DEV)
    q = normal((5, 6, 64), BF16, 1)
    zero = torch.zeros(5, dtype=torch.int32, device=DEV)
    out, none = aklr_amd.rotary_embedding(q, None, zero, f)
    assert none is None and torch.equal(out, q)
    pos = torch.tensor([-7, 0, 1, 2**31 - 1, -2**31], dtype=torch.int32, device=DEV)
    got, _ = aklr_amd.rotary_embedding(q[:3], None, pos[:3].contiguous(), f)
    check_rotated(got, q[:3], pos[:3], f, False, 1.0, "int32")
    # at 2^31 an angle in 64 bits is off by 2^31 * 3 * 2^-53: 2^-20 of a radian, so as much again in the tolerance
    far, _ = aklr_amd.rotary_embedding(q[3:], None, pos[3:].contiguous(), f)
    want = oc.rotate(q[3:].double().cpu().numpy(), pos[3:].cpu().numpy(), f.cpu().numpy())
    tol = half_step(want, BF16) * (1 + 2**-10) + 2**-19 * pair_size(q[3:], 64, False)
    assert (np.abs(far.double().cpu().numpy() - want) <= tol).all()
    a, b = aklr_amd.rotary_embedding(q[:0], q[:0, :2], pos[:0], f)
    assert a.shape == (0, 6, 64) and b.shape == (0, 2, 64)
    # the last 64 of 192 in a query head and of 576 in a latent row, turned where they lie
    heads, latent = normal((5, 6, 192), BF16, 4), normal((5, 576), BF16, 5)
    pos = torch.arange(5, device=DEV) * 1000
    qv, kv = heads[..., 128:], latent[:, 512:].unsqueeze(1)
    q0, k0, left = qv.clone(), kv.clone(), (heads[..., :128].clone(), latent[:, :512].clone())
    a, b = aklr_amd.rotary_embedding(qv, kv, pos, f, interleaved=True, out_q=qv, out_k=kv)
    assert a is qv and b is kv
    check_rotated(qv, q0, pos, f, True, 1.0, "q in place")
    check_rotated(kv, k0, pos, f, True, 1.0, "k in place")
    assert torch.equal(heads[..., :128], left[0]) and torch.equal(latent[:, :512], left[1])
    # queries and keys of one projection, to head-major outputs
    rows = normal((5, 8 * 64), BF16, 6)
    qv, kv = rows[:, :384].view(5, 6, 64), rows[:, 384:].view(5, 2, 64)
    oq, ok = (torch.empty((n, 5, 64), dtype=BF16, device=DEV).transpose(0, 1) for n in (6, 2))
    aklr_amd.rotary_embedding(qv, kv, pos, f, out_q=oq, out_k=ok)
    check_rotated(oq, qv, pos, f, False, 1.0, "q head-major")
    check_rotated(ok, kv, pos, f, False, 1.0, "k head-major")
    one = kv[:, :1].expand(5, 2, 64)
    _, ok = aklr_amd.rotary_embedding(qv, one, pos, f)
    check_rotated(ok, one, pos, f, False, 1.0, "one head read twice")


def place(slots, page):
    s = slots.cpu().numpy().astype(np.int64)
    return s // page, s % page


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("t,h,d,page,pages", [(1, 1, 64, 16, 1), (5, 3, 64, 48, 4), (64, 8, 128, 16, 9), (333, 2, 256, 64, 7),
                                              (257, 1, 128, 1024, 1), (19, 40, 64, 16, 3), (2051, 40, 64, 16, 129)])
def test_write_and_read(t, h, d, page, pages, dtype):
    say(f"write {t} {h} {d} {page} {dtype}")
    k, v = normal((t, h, d), dtype, 1) * 3, normal((t, h, d), dtype, 2)
    k[0, 0] = 0
    slots = torch.randperm(pages * page, generator=gen(3), device=DEV)[:t].contiguous()
    cache = new_cache(pages, h, d, page, 4)
    want = [x.clone().cpu() for x in cache]
    got = aklr_amd.kv_cache_write_fp8(k, v, *cache, slots if t % 2 else slots.to(torch.int32))
    assert all(a is b for a, b in zip(got, cache))
    at, off = place(slots, page)
    for i, x in ((0, k), (1, v)):
        q, s = oc.quantize(x.float().cpu().numpy())
        want[i].view(torch.uint8).numpy()[at, :, off] = q
        want[2 + i].numpy()[at, :, off] = s
        assert_same_bits(u8(cache[i]), u8(want[i]), f"codes {i}")
        assert_same_bits(cache[2 + i].cpu().numpy(), want[2 + i].numpy(), f"scales {i}")
    # read back what was written, a token a sequence, so that every page is somebody's first
    if page == 16 and t <= 64:
        table = torch.arange(pages, dtype=torch.int32, device=DEV).view(pages, 1)
        starts = torch.arange(0, pages * page + 1, page, dtype=torch.int32, device=DEV)
        for out_dtype in (BF16, F16):
            rk, rv = aklr_amd.kv_cache_read_fp8(*cache, table, starts, pages * page, out_dtype=out_dtype)
            for i, r in ((0, rk), (1, rv)):
                full = want[i].float() * want[2 + i][..., None]
                full = full.transpose(1, 2).reshape(pages * page, h, d).to(out_dtype)
                assert r.dtype == out_dtype and torch.equal(r.cpu().nan_to_num(7.0), full.nan_to_num(7.0))
                assert torch.equal(r.cpu().isnan(), full.isnan())


def test_write_skips_and_marks():
    say("write: slots outside the cache, values that are not finite, strided k and v, pages apart, empty")
    h, d, page, pages = 2, 128, 16, 4
    rows = normal((9, 3 * h * d), BF16, 1)
    k, v = rows[:, :h * d].view(9, h, d), rows[:, h * d:2 * h * d].view(9, h, d)
    k[1, 0, 5], k[2, 1, 127], v[3, 0, 0], v[4, 1, 64] = float("nan"), float("inf"), -float("inf"), float("nan")
    k[5, 0], v[5, 1] = 1e-30, 3e38  # below the floor of the scale; the largest magnitudes
    codes = torch.zeros((pages, 2, h, page, d), dtype=torch.uint8, device=DEV).view(E4M3)
    scales = torch.zeros((pages, 2, h, page), device=DEV)
    cache = (codes[:, 0], codes[:, 1], scales[:, 0], scales[:, 1])
    slots = torch.tensor([0, 17, 34, 51, 5, 6, -1, pages * page, 1 << 40], device=DEV)
    aklr_amd.kv_cache_write_fp8(k, v, *cache, slots)
    at, off = place(slots[:6], page)
    for i, x in ((0, k), (1, v)):
        q, s = oc.quantize(x[:6].float().cpu().numpy())
        want, ws = np.zeros((pages, h, page, d), np.uint8), np.zeros((pages, h, page), np.float32)
        want[at, :, off], ws[at, :, off] = q, s
        assert np.array_equal(u8(cache[i]), want)
        assert np.array_equal(cache[2 + i].cpu().numpy(), ws, equal_nan=True)
    assert np.isnan(cache[2][1, 0, 1].item()) and np.isnan(cache[3][0, 1, 5].item())
    before = codes.view(torch.uint8).clone()
    aklr_amd.kv_cache_write_fp8(k[:0], v[:0], *cache, slots[:0])
    aklr_amd.kv_cache_write_fp8(k[:2], v[:2], *cache, torch.tensor([-5, -(1 << 31)], dtype=torch.int32, device=DEV))
    assert torch.equal(codes.view(torch.uint8), before)
    rk, _ = aklr_amd.kv_cache_read_fp8(*cache, torch.tensor([[1]], dtype=torch.int32, device=DEV),
                                       torch.tensor([0, 2], dtype=torch.int32, device=DEV), 2)
    assert rk[1, 0].isnan().all() and not rk[1, 1].isnan().any()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,hq,h,d,rot,dtype", [(1, 1, 1, 64, 64, BF16), (8, 64, 8, 128, 128, BF16), (37, 6, 2, 256, 64, F16),
                                                (300, 4, 4, 64, 32, BF16), (12, 3, 1, 128, 96, F32),
                                                (2051, 33, 4, 128, 128, BF16), (4109, 5, 3, 256, 256, F16)])
def test_rotary_write(t, hq, h, d, rot, dtype, interleaved):
    say(f"rotary write {t} {hq} {h} {d} {rot} {dtype} {interleaved}")
    page, pages = 16, -(-t // 16) + 2
    q, k, v = normal((t, hq, d), dtype, 1), normal((t, h, d), dtype, 2), normal((t, h, d), dtype, 3)
    pos = torch.randint(0, 1 << 20, (t,), generator=gen(4), device=DEV)
    f = aklr_amd.rotary_frequencies(rot, device=DEV)
    slots = torch.randperm(pages * page, generator=gen(5), device=DEV)[:t].contiguous()
    if t > 3:
        slots[2] = -1
    cache = new_cache(pages, h, d, page, 6)
    before = [x.clone() for x in cache]
    mag = 1.1
    got = aklr_amd.rotary_kv_cache_write_fp8(q, k, v, pos, f, *cache, slots, interleaved=interleaved, magnitude=mag)
    check_rotated(got, q, pos, f, interleaved, mag, "q")
    apart = aklr_amd.rotary_embedding(q, None, pos, f, interleaved=interleaved, magnitude=mag)[0]
    assert torch.equal(got, apart)  # the same arithmetic
    keep = (slots >= 0).cpu().numpy()
    at, off = place(slots[slots >= 0], page)
    qv, sv = oc.quantize(v.float().cpu().numpy()[keep])
    assert_same_bits(u8(cache[1])[at, :, off], qv, "v codes")
    assert_same_bits(cache[3].cpu().numpy()[at, :, off], sv, "v scales")
    want = oc.rotate(k.double().cpu().numpy(), pos.cpu().numpy(), f.cpu().numpy(), interleaved, mag)[keep]
    slack = 2**-20 * mag * pair_size(k, rot, interleaved)[keep]
    scale = cache[2].cpu().double().numpy()[at, :, off]
    exact = np.maximum(np.abs(want).max(-1), 1e-10) / 448
    assert (np.abs(scale - exact) <= slack.max(-1) / 448 + exact * 2**-22).all()
    value = oc.E4M3[u8(cache[0])[at, :, off]] * scale[..., None]
    tol = np.maximum(np.abs(want) * 2**-4, scale[..., None] * 2**-10) * (1 + 2**-20) + slack + np.abs(want) * 2**-21
    assert (np.abs(value - want) <= tol).all()
    other = np.ones(cache[0].shape[:1] + cache[0].shape[2:3], bool)
    other[at, off] = False
    for a, b in zip(cache, before):  # no other place changed
        a, b = (u8(x) if x.dtype == E4M3 else x.cpu().numpy().view(np.uint32) for x in (a, b))
        p, o = np.nonzero(other)
        assert np.array_equal(a[p, :, o], b[p, :, o])
    again = aklr_amd.rotary_kv_cache_write_fp8(q, k, v, pos, f, *cache, slots, interleaved=interleaved, magnitude=mag, out=q)
    assert again is q and torch.equal(q, got)


@pytest.mark.parametrize("d,h,page", [(64, 2, 16), (128, 8, 48), (256, 1, 64), (128, 96, 512)])
def test_read_packs_ragged_prefixes(d, h, page):
    say(f"read {d} {h} {page}")
    pages = 12
    cache = new_cache(pages, h, d, page, 1)
    cache[0].view(torch.uint8).clamp_(max=126)  # finite codes
    cache[1].view(torch.uint8).clamp_(max=126)
    lens = [3 * page + 5, 0, 1, page, 2 * page - 1, 3 * page]
    starts = np.r_[0, np.cumsum(lens)].astype(np.int32)
    total = int(starts[-1]) + 9  # rows behind the last sequence
    table = torch.randint(0, pages, (len(lens), 5), generator=gen(2), device=DEV, dtype=torch.int32)
    table[0, 1], table[3, 0] = pages, -1  # pages the cache does not have
    sent = [torch.full((total, h, d), 3.5, dtype=BF16, device=DEV) for _ in "kv"]
    got = aklr_amd.kv_cache_read_fp8(*cache, table[:, :3], torch.from_numpy(starts).to(DEV), total, out_k=sent[0], out_v=sent[1])
    for i, (r, o) in enumerate(zip(got, sent)):
        assert r is o
        want = np.full((total, h, d), 3.5)
        for b, n in enumerate(lens):
            want[starts[b]:starts[b] + n] = oc.gather(u8(cache[i]), cache[2 + i].cpu().numpy(), table[:, :3].cpu().numpy(), b, n)[0]
        # a product rounded to fp32, then to bf16
        want = torch.from_numpy(want).float().bfloat16()
        assert torch.equal(r.cpu(), want)
    empty = aklr_amd.kv_cache_read_fp8(*cache, table[:0], torch.zeros(1, dtype=torch.int32, device=DEV), 0)
    assert empty[0].shape == (0, h, d) and empty[0].dtype == BF16
    # starts that do not ascend read nothing outside the cache and write nothing outside the rows
    aklr_amd.kv_cache_read_fp8(*cache, table, torch.tensor([5, 2, 900, -4, 7, 1, 3], dtype=torch.int32, device=DEV), 16)
    torch.cuda.synchronize()


def test_offsets_past_32_bits():
    say("a cache of more than 4 GiB of codes a side")
    h, d, page = 1, 256, 1024
    pages = 17000  # 4.46e9 bytes
    cache = tuple(torch.empty(s, dtype=torch.uint8, device=DEV).view(E4M3) for s in [(pages, h, page, d)] * 2) + tuple(
        torch.empty((pages, h, page), device=DEV) for _ in "kv")
    slots = torch.tensor([pages * page - 1, 0, 16777216, 12345678], device=DEV)
    k, v = normal((4, h, d), BF16, 1), normal((4, h, d), BF16, 2)
    aklr_amd.kv_cache_write_fp8(k, v, *cache, slots)
    table = torch.tensor([[pages - 1], [0], [16777216 // page], [12345678 // page]], dtype=torch.int32, device=DEV)
    lens = (slots % page + 1).cpu().numpy()
    starts = torch.from_numpy(np.r_[0, np.cumsum(lens)].astype(np.int32)).to(DEV)
    rk, rv = aklr_amd.kv_cache_read_fp8(*cache, table, starts, int(lens.sum()))
    at = starts[1:].long() - 1
    for r, x in ((rk, k), (rv, v)):
        q, s = oc.quantize(x.float().cpu().numpy())
        want = torch.from_numpy(oc.E4M3[q] * s[..., None].astype(np.float64)).float().bfloat16()
        assert torch.equal(r[at].cpu(), want)
