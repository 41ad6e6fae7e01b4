"""Calls of the cache operators that are refused with a reason where they used to raise, or to be served wrongly. The plans
are asked on CPU tensors in the place of GPU ones."""
from __future__ import annotations

import ctypes

import pytest
import torch

import aklr_amd
from aklr_amd.dispatch import FallbackReason, KernelInfo
from tests.test_cache_ops_host import BF16, OPS, anywhere, attend_args, both_args, cache_args, rot_args, write_args  # noqa: F401

OOC = FallbackReason.OUT_OF_CONTRACT


def i32(n):
    return torch.zeros(n, dtype=torch.int32)


def test_more_workgroups_than_a_launch_has_room_for(anywhere, native_lib):
    # 65536 sequences of one token, 256 kv heads of one query head: 65536 / 16 + 65536 tiles a head, 17.8 million workgroups
    c = {n: t for n, t in cache_args(h=256).items()}
    q = torch.zeros((1, 1, 64), dtype=BF16)
    for batch, served in ((65536, False), (60000, True)):
        args = {"q": q.expand(batch, 256, 64), **c, "block_table": i32((batch, 1)), "seq_lens": i32(batch),
                "starts": i32(batch + 1)}
        assert isinstance(aklr_amd.tree_attention_fp8.serving(**args), KernelInfo) == served
        assert bool(native_lib.aklr_tree_attention_fp8_rows(batch, batch, 256, 256, 64, 16, None)) == served


def test_attention_workspace_is_for_what_is_split(native_lib):
    # partial results: at most as many pieces as twice the chip runs at once and half as many again (512 workgroups of 128
    # rows: 1536), whatever the number of query tokens; beside them a word a tile
    size, rows = native_lib.aklr_tree_attention_fp8_workspace_bytes, native_lib.aklr_tree_attention_fp8_rows
    last = 0
    for tokens in (1, 100, 1000, 8192, 65536, 1 << 20):
        got = size(tokens, 2, 64, 8, 128, 1 << 17)
        r = rows(tokens, 2, 64, 8, 128, 1 << 17, None)
        tiles = 8 * (tokens * 8 // r + 2)
        assert last <= got <= 1536 * r * (128 + 4) * 4 + 8 * tiles + 16
        last = got
    assert last < 120 << 20


def test_attention_rows_query(native_lib):
    rows = native_lib.aklr_tree_attention_fp8_rows
    join = ctypes.c_int(-1)
    assert rows(1, 1, 8, 8, 128, 4096, None) == 16 and rows(20, 1, 8, 8, 128, 4096, None) == 32
    assert rows(4096, 2, 32, 8, 128, 16384, ctypes.byref(join)) == 128 and join.value > 0
    assert rows(2, 2, 4, 1, 64, 320, ctypes.byref(join)) == 16 and join.value == 0  # the last workgroup joins
    assert rows(1, 1, 8, 8, 96, 4096, None) == 0 and rows(1, 1, 8, 3, 64, 4096, None) == 0 and rows(0, 1, 8, 8, 64, 4096, None) == 0


def test_one_tensor_as_queries_and_keys_is_not_rotated_in_place(anywhere):
    # written in place as q while it is read as k, the keys would be rotated once or twice, as the workgroups come
    serving = aklr_amd.rotary_embedding.serving
    a = rot_args(hq=2, hk=2)
    x = a["q"]
    assert serving(**{**a, "k": x}, out_q=x) is OOC and serving(**{**a, "k": x}, out_k=x) is OOC
    assert serving(**{**a, "k": x}, out_q=x, out_k=x) is OOC
    assert isinstance(serving(**{**a, "k": x}), KernelInfo)  # into new memory
    assert isinstance(serving(**{**a, "k": x}, out_q=a["k"]), KernelInfo)
    assert isinstance(serving(**a, out_q=x, out_k=a["k"]), KernelInfo)


@pytest.mark.parametrize("op,name,good", [("rotary", "magnitude", 1e38), ("both", "magnitude", -2), ("attend", "softmax_scale", 0.0)])
def test_numbers_an_fp32_does_not_hold(anywhere, op, name, good):
    fn, make = OPS[op]
    assert isinstance(fn.serving(**make(), **{name: good}), KernelInfo)
    for bad in (10**400, -(10**400), 1e300, -1e39, float("nan"), torch.ones(2)):
        assert fn.serving(**make(), **{name: bad}) is OOC, bad


@pytest.mark.parametrize("op,name", [("rotary", "interleaved"), ("both", "interleaved"), ("attend", "return_lse")])
def test_flags_that_are_none(anywhere, op, name):
    fn, make = OPS[op]
    assert isinstance(fn.serving(**make(), **{name: True}), KernelInfo) and isinstance(fn.serving(**make(), **{name: 0}), KernelInfo)
    for bad in (torch.zeros(2), torch.zeros(1), None, "1", 2):
        assert fn.serving(**make(), **{name: bad}) is OOC, bad


@pytest.mark.parametrize("op", OPS)
def test_tensors_of_a_function_transform_are_refused(anywhere, op):
    fn, make = OPS[op]
    args = make()
    for name, t in args.items():
        if not isinstance(t, torch.Tensor) or t.dtype == torch.float8_e4m3fn:
            continue
        answers = []

        def ask(x):
            answers.append(fn.serving(**{**args, name: x}))
            return x.float().sum()

        torch.vmap(ask)(torch.stack([t, t]))
        if t.is_floating_point():
            torch.func.jvp(ask, (t,), (torch.ones_like(t),))
            torch.func.grad(ask)(t)
        assert answers and all(a is OOC for a in answers), (name, answers)


@pytest.mark.parametrize("op,name", [("rotary", "q"), ("rotary", "k"), ("rotary", "frequencies"), ("write", "k"), ("write", "v"),
                                     ("write", "v_scale"), ("both", "q"), ("both", "v"), ("both", "frequencies"), ("read", "k_scale"),
                                     ("attend", "q"), ("attend", "k_scale")])
def test_tangents_are_refused_not_lost(anywhere, op, name):
    fn, make = OPS[op]
    args = make()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        assert fn.serving(**{**args, name: dual}) is OOC
        with torch.no_grad():
            assert fn.serving(**{**args, name: dual}) is OOC
        assert isinstance(fn.serving(**args), KernelInfo)
    assert isinstance(fn.serving(**args), KernelInfo)


OUTS = {"rotary": ("out_q", "q"), "both": ("out", "q"), "read": ("out_k", None), "attend": ("out", "q")}


@pytest.mark.parametrize("op", OUTS)
def test_an_output_that_wants_gradients_or_has_a_tangent_is_refused(anywhere, op):
    fn, make = OPS[op]
    args, (name, like) = make(), OUTS[op]
    out = torch.zeros_like(args[like]) if like else torch.zeros((args["total"], 2, 64), dtype=BF16)
    assert isinstance(fn.serving(**args, **{name: out}), KernelInfo)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(out, torch.ones_like(out))
        assert fn.serving(**args, **{name: dual}) is OOC
    out.requires_grad_()
    assert fn.serving(**args, **{name: out}) is OOC
    with torch.no_grad():
        assert isinstance(fn.serving(**args, **{name: out}), KernelInfo)
