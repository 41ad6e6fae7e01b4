"""The contracts of draft verification, the page operators and the adapters without a GPU: what their plans accept, refuse and
name, and what the C entry points reject before any launch. CPU tensors stand in for GPU ones where only the plan is asked."""
from __future__ import annotations

import ctypes

import pytest
import torch

import aklr_amd
from aklr_amd import drafts, kv_cache, kv_pages, lora
from aklr_amd.dispatch import FallbackReason, KernelInfo
from tests.test_cache_ops_host import BF16, F16, F32, cache_args

OOC = FallbackReason.OUT_OF_CONTRACT
I32, I64 = torch.int32, torch.int64


@pytest.fixture
def anywhere(monkeypatch, native_lib):
    for module in (drafts, kv_pages, lora, kv_cache):
        monkeypatch.setattr(module, "on_gpu", lambda *t: True)


def i32(*v):
    return torch.tensor(v, dtype=I32)


def verify_args(t=5, v=40, b=2, dtype=F32):
    return {"target_probs": torch.zeros((t, v), dtype=dtype), "draft_tokens": torch.zeros(t, dtype=I64),
            "starts": torch.linspace(0, t, b + 1).to(I32), "accept_uniforms": torch.zeros(t), "sample_uniforms": torch.zeros(b),
            "most": 3, "draft_probs": torch.zeros((t, v), dtype=dtype), "parents": torch.zeros(t, dtype=I32)}


def copy_args(**kw):
    return {**cache_args(**kw), "src": i32(0, 1), "dst": i32(2, 2)}


def compact_args(b=2, most=3, **kw):
    return {**cache_args(**kw), "block_table": torch.zeros((b, 2), dtype=I32), "seq_lens": torch.zeros(b, dtype=I32),
            "starts": torch.zeros(b + 1, dtype=I32), "path": torch.zeros((b, most), dtype=I32), "counts": torch.zeros(b, dtype=I32)}


def update_args(b=2, pages=8):
    return {"page_refs": torch.zeros(pages, dtype=I32), "block_table": torch.zeros((b, 2), dtype=I32),
            "lens": torch.zeros(b, dtype=I32), "new_lens": torch.zeros(b, dtype=I32), "page_size": 16,
            "parents": torch.zeros(b, dtype=I32)}


def lora_args(t=3, k=32, n=24, r=8, count=2, dtype=BF16):
    return {"x": torch.zeros((t, k), dtype=dtype), "a": torch.zeros((count, r, k), dtype=dtype),
            "b": torch.zeros((count, n, r), dtype=dtype), "adapters": torch.zeros(t, dtype=I32),
            "base": torch.zeros((t, n), dtype=dtype), "scales": torch.zeros(count), "ranks": torch.zeros(count, dtype=I32)}


OPS = {"verify": (aklr_amd.verify_drafts, verify_args), "copy": (aklr_amd.kv_cache_copy_pages_fp8, copy_args),
       "compact": (aklr_amd.kv_cache_compact_fp8, compact_args), "update": (aklr_amd.kv_cache_update_pages, update_args),
       "lora": (aklr_amd.lora_project, lora_args)}
OPTIONAL = {("verify", "draft_probs"), ("verify", "parents"), ("update", "parents"), ("lora", "scales"), ("lora", "ranks")}


def variants(args):
    """The call with each tensor in a form its own check has to refuse."""
    for name, t in args.items():
        if not isinstance(t, torch.Tensor):
            continue
        yield name, "none", {**args, name: 3}
        yield name, "dtype", {**args, name: t.to(torch.int16)}
        yield name, "double", {**args, name: t.double()}
        yield name, "dims", {**args, name: t.unsqueeze(0)}
        if t.shape[0] > 1:
            yield name, "short", {**args, name: t[:-1]}
        wide = torch.zeros(t.shape[:-1] + (2 * t.shape[-1],), dtype=torch.uint8 if t.element_size() == 1 else t.dtype).view(t.dtype)
        if t.shape[-1] > 1:
            yield name, "strided", {**args, name: wide[..., ::2]}


@pytest.mark.parametrize("op", OPS)
def test_a_call_is_served_and_each_bad_form_refused(anywhere, op):
    fn, make = OPS[op]
    args = make()
    info = fn.serving(**args)
    assert isinstance(info, KernelInfo) and info.kernel_ref.startswith("aklr_") and fn.fallback_reason(**args) is None
    for name, what, bad in variants(args):
        if what == "short" and name == "page_refs":
            continue  # fewer pages is another cache
        assert fn.serving(**bad) is OOC, (name, what)
    for op_, name in OPTIONAL:
        if op_ == op:
            assert isinstance(fn.serving(**{**args, name: None}), KernelInfo)


@pytest.mark.parametrize("op", OPS)
def test_cpu_tensors_and_disabled_ops_are_not_served(op, monkeypatch):
    fn, make = OPS[op]
    assert fn(**make()) is OOC
    monkeypatch.setenv("AKLR_DISABLE", fn.contract_id)
    assert fn(**make()) is FallbackReason.DISABLED


@pytest.mark.parametrize("op", OPS)
def test_no_call_raises(anywhere, op):
    fn, make = OPS[op]
    args = make()
    for name in args:
        for value in (None, "x", object(), 1.5, [1], torch.zeros(0), torch.tensor(3), torch.zeros(2, 2).to_sparse(), 1 << 70):
            got = fn.serving(**{**args, name: value})
            assert isinstance(got, (FallbackReason, KernelInfo)), (name, value)
            if (op, name) not in OPTIONAL or value is not None:
                assert got is OOC, (name, value)


FLOATS = [("verify", n) for n in ("target_probs", "draft_probs", "accept_uniforms", "sample_uniforms")] + [
    ("copy", "k_scale"), ("compact", "v_scale"), ("lora", "x"), ("lora", "a"), ("lora", "b"), ("lora", "base"), ("lora", "scales")]


@pytest.mark.parametrize("op,name", FLOATS)
def test_gradients_and_tangents_are_refused_not_lost(anywhere, op, name):
    fn, make = OPS[op]
    args = make()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        assert fn.serving(**{**args, name: dual}) is OOC
        with torch.no_grad():
            assert fn.serving(**{**args, name: dual}) is OOC
    args[name].requires_grad_()
    assert fn.serving(**args) is OOC
    with torch.no_grad():
        assert isinstance(fn.serving(**args), KernelInfo)


@pytest.mark.parametrize("op,name", FLOATS + [("verify", "draft_tokens"), ("copy", "src"), ("compact", "path"), ("update", "page_refs")])
def test_tensors_of_a_function_transform_are_refused(anywhere, op, name):
    fn, make = OPS[op]
    args, answers = make(), []

    def ask(x):
        answers.append(fn.serving(**{**args, name: x}))
        return x.float().sum()

    torch.vmap(ask)(torch.stack([args[name], args[name]]))
    assert answers == [OOC] * len(answers) and answers


def test_verify_forms(anywhere):
    serving = aklr_amd.verify_drafts.serving
    a = verify_args()
    assert serving(**a).variant == "tree" and serving(**{**a, "parents": None}).variant == "chain"
    assert serving(**{**a, "parents": None, "draft_probs": None}).variant == "chain_certain"
    for good in ({"dtype": BF16}, {"dtype": F16}, {"v": 8}, {"v": 9}, {"t": 0, "b": 1}, {"b": 0}, {"t": 1, "b": 1}):
        assert isinstance(serving(**verify_args(**good)), KernelInfo), good
    for good in ({"most": 1}, {"most": 1024}, {"draft_tokens": a["draft_tokens"].to(I32)},
                 {"target_probs": torch.zeros((5, 50))[:, 3:43]}, {"draft_probs": torch.zeros((9, 40))[::2]}):
        assert isinstance(serving(**{**a, **good}), KernelInfo), good
    for bad in ({"most": 0}, {"most": 1025}, {"most": True}, {"most": 3.0}, {"draft_probs": torch.zeros((5, 40), dtype=BF16)},
                {"draft_probs": torch.zeros((5, 41))}, {"target_probs": torch.zeros((1, 40)).expand(5, 40)},
                {"starts": i32()}, {"sample_uniforms": torch.zeros(3)}, {"target_probs": torch.zeros((5, 80))[:, ::2]}):
        assert serving(**{**a, **bad}) is OOC, bad
    assert serving(**verify_args(v=7)) is OOC
    bytes_ = torch.zeros(5 * 40 * 2 + 1, dtype=torch.uint8)
    if hasattr(torch, "frombuffer"):
        odd = torch.frombuffer(bytearray(bytes_.numpy().tobytes()), dtype=BF16, offset=1, count=200).view(5, 40)
        assert odd.data_ptr() % 2 == 0 or serving(**{**verify_args(dtype=BF16), "target_probs": odd}) is OOC


def test_copy_and_compact_forms(anywhere):
    a = copy_args()
    serving = aklr_amd.kv_cache_copy_pages_fp8.serving
    assert isinstance(serving(**{**a, "src": a["src"].long(), "dst": a["dst"].long()}), KernelInfo)
    assert isinstance(serving(**{**a, "src": i32(), "dst": i32()}), KernelInfo)
    assert serving(**{**a, "src": a["src"].long()}) is OOC and serving(**{**a, "v_cache": a["k_cache"]}) is OOC
    memory = torch.zeros(3 * 2 * 16, dtype=I32)
    meets = memory.view(F32).view(3, 2, 16)
    assert serving(**{**a, "k_scale": meets, "src": memory[:2]}) is OOC
    a = compact_args()
    serving = aklr_amd.kv_cache_compact_fp8.serving
    assert serving(**a).variant == "short" and serving(**compact_args(most=65)).variant == "long"
    for good in (compact_args(b=0), compact_args(most=0), {**a, "block_table": torch.zeros((2, 0), dtype=I32)},
                 {**a, "path": torch.zeros((2, 9), dtype=I32)[:, 2:5]}):
        assert isinstance(serving(**good), KernelInfo)
    for bad in ({"path": torch.zeros((2, 3), dtype=I64)}, {"path": torch.zeros((3, 3), dtype=I32)}, {"path": torch.zeros((1, 3), dtype=I32).expand(2, 3)},
                {"counts": torch.zeros(3, dtype=I32)}, {"starts": i32(0, 1)}, {"seq_lens": torch.zeros((2, 1), dtype=I32)},
                {"path": torch.zeros((3, 2), dtype=I32).t()}):
        assert serving(**{**a, **bad}) is OOC, bad
    wide = torch.zeros((1, 1), dtype=I32).expand(1, 1)
    big = compact_args(b=1)
    assert isinstance(serving(**{**big, "block_table": wide}), KernelInfo)
    huge = torch.empty((1, (1 << 24) + 1), dtype=I32)
    assert serving(**{**big, "block_table": huge}) is OOC and isinstance(serving(**{**big, "block_table": huge[:, 1:]}), KernelInfo)


def test_update_forms(anywhere):
    serving = aklr_amd.kv_cache_update_pages.serving
    a = update_args()
    assert serving(**a).variant == "fork" and serving(**{**a, "parents": None}).variant == "grow"
    for good in ({"page_size": 1}, {"page_size": 1 << 27}, {"block_table": torch.zeros((2, 5), dtype=I32)[:, 1:3]},
                 {"block_table": torch.zeros((2, 0), dtype=I32)}):
        assert isinstance(serving(**{**a, **good}), KernelInfo), good
    assert isinstance(serving(**update_args(b=0)), KernelInfo)
    for bad in ({"page_size": 0}, {"page_size": True}, {"page_size": 16.0}, {"page_size": 1 << 28}, {"page_refs": torch.zeros(0, dtype=I32)},
                {"page_refs": torch.zeros(9, dtype=I32)[1:]}, {"lens": torch.zeros(3, dtype=I32)}, {"parents": torch.zeros(2, dtype=I64)},
                {"block_table": torch.zeros((1, 2), dtype=I32).expand(2, 2)}):
        assert serving(**{**a, **bad}) is OOC, bad
    memory = torch.zeros(16, dtype=I32)
    for name, t in (("lens", memory[2:4]), ("block_table", memory[4:8].view(2, 2)), ("parents", memory[:2])):
        assert serving(**{**a, "page_refs": memory[:8], name: t}) is OOC, name
    assert aklr_amd.new_kv_page_refs(5, "cpu").tolist() == [0] * 5


def test_lora_forms(anywhere):
    serving = aklr_amd.lora_project.serving
    a = lora_args()
    assert serving(**a).variant == "decode" and serving(**lora_args(t=257)).variant == "sorted"
    for good in ({"dtype": F16}, {"k": 8}, {"k": 65536}, {"n": 8}, {"r": 128}, {"r": 24}, {"t": 0}, {"count": 1}):
        assert isinstance(serving(**lora_args(**good)), KernelInfo), good
    for bad in ({"dtype": F32}, {"k": 12}, {"k": 65544}, {"n": 20}, {"r": 136}, {"r": 12}, {"count": 4097}, {"count": 0}):
        assert serving(**lora_args(**bad)) is OOC, bad
    assert isinstance(serving(**{**a, "adapters": a["adapters"].long()}), KernelInfo)
    assert serving(**{**a, "base": torch.zeros((3, 24), dtype=F16)}) is OOC
    stacked = torch.zeros((2, 24, 32), dtype=BF16), torch.zeros((2, 72, 8), dtype=BF16)  # what three projections stack
    rows = torch.zeros((3, 72), dtype=BF16)
    sliced = {**a, "a": stacked[0][:, 8:16], "b": stacked[1][:, 24:48], "base": rows[:, 24:48]}
    assert isinstance(serving(**sliced), KernelInfo) and isinstance(serving(**sliced, out=rows[:, 24:48]), KernelInfo)
    assert isinstance(serving(**sliced, out=rows[:, 48:72]), KernelInfo)
    assert serving(**sliced, out=rows[:, 32:56]) is OOC and serving(**sliced, out=torch.zeros((1, 24), dtype=BF16).expand(3, 24)) is OOC
    assert isinstance(serving(**{**a, "x": torch.zeros((1, 32), dtype=BF16).expand(3, 32)}), KernelInfo)  # read more than once
    flat = torch.zeros(200, dtype=BF16)
    assert serving(**{**a, "base": flat[1:73].view(3, 24)}) is OOC and serving(**{**a, "x": torch.zeros((3, 36), dtype=BF16)[:, :32]}) is OOC
    square = lora_args(k=24)
    assert serving(**square, out=square["x"]) is OOC  # what is read as x
    out = torch.zeros((3, 24), dtype=BF16)
    assert isinstance(serving(**a, out=out), KernelInfo)
    out.requires_grad_()
    assert serving(**a, out=out) is OOC


def test_entry_points_reject_before_any_launch(native_lib):
    L = native_lib
    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 15) & ~15

    def copy(k=p, src=p, count=0, h=1, d=64, pages=2, page=16, stride=None):
        s = stride if stride is not None else h * page * d
        return L.aklr_kv_cache_copy_pages_fp8(k, p, p, p, s, s, h * page, h * page, src, p, 0, count, h, d, pages, page, None)

    assert copy() == 0
    for bad in ({"k": None}, {"k": p + 8}, {"d": 96}, {"page": 24}, {"pages": 0}, {"pages": 1 << 28}, {"stride": 16}, {"count": -1},
                {"count": 1, "src": None}, {"h": 0}):
        assert copy(**bad) == 1, bad

    def compact(batch=0, most=1, cols=1, lens=p, path_stride=1, page=16, ws=None, nbytes=0, stride=1, k=p):
        return L.aklr_kv_cache_compact_fp8(k, p, p, p, page * 64, page * 64, page, page, p, stride, cols, lens, p, p, path_stride, most, p,
                                           batch, 1, 64, 2, page, ws, nbytes, None)

    assert compact() == 0 and compact(batch=1, most=0) == 0 and compact(batch=1, cols=0) == 0
    for bad in ({"lens": None}, {"path_stride": 0}, {"stride": 0}, {"cols": (1 << 24) + 1, "stride": 1 << 30}, {"k": None}, {"batch": 65537},
                {"page": 20}):
        assert compact(**{"batch": 1, **bad}) == 1, bad
    size = L.aklr_kv_cache_compact_fp8_workspace_bytes
    assert size(7, 64, 8, 128) == 0 and size(1, 65, 1, 64) == 2 * 65 * 68
    assert compact(batch=1, most=65, path_stride=65) == 3 and compact(batch=1, most=65, path_stride=65, ws=p, nbytes=2 * 65 * 68 - 1) == 3
    assert compact(batch=1, most=(1 << 28) + 1, path_stride=1 << 30) == 1
    for b, most, h, d in ((1, 1 << 20, 1, 64), (65536, 100, 1, 64), (64, 8192, 8, 128), (3, 1 << 30, 1024, 256), (1, 65, 1024, 256)):
        assert 0 < size(b, most, h, d) <= 128 << 20 and size(b, most, h, d) % (2 * h * (d + 4)) == 0

    def update(refs=p, pages=4, batch=0, cols=1, stride=1, page=16, lens=p, ws=p, nbytes=1 << 12, out=p):
        return L.aklr_kv_cache_update_pages(refs, pages, p, stride, cols, lens, p, None, batch, page, out, p, p, p, ws, nbytes, None)

    assert update() == 0
    for bad in ({"refs": None}, {"pages": 0}, {"stride": 0}, {"page": 0}, {"lens": None}, {"pages": 1 << 27}, {"cols": 1 << 25, "stride": 1 << 25},
                {"batch": 65537}, {"out": None}, {"batch": -1}):
        assert update(**{"batch": 1, **bad}) == 1, bad
    assert update(batch=1, ws=None) == 3 and update(batch=1, nbytes=31) == 3

    def verify(target=p, stride=40, draft=None, dstride=0, tokens=0, vocab=40, most=3, batch=1, dtype=2, ws=p, nbytes=0, starts=p):
        return L.aklr_verify_drafts(target, stride, draft, dstride, tokens, vocab, p, 1, None, starts, p, p, batch, most, p, p, p, dtype, ws,
                                    nbytes, None)

    assert verify(batch=0) == 0 and verify(dtype=3) == 2 and verify() == 3 and verify(ws=None, nbytes=1 << 20) == 3
    for bad in ({"stride": 39}, {"draft": p, "dstride": 39}, {"vocab": 7}, {"vocab": (1 << 24) + 1, "stride": 1 << 25}, {"most": 0}, {"most": 1025},
                {"batch": 65537}, {"tokens": -1}, {"target": None, "tokens": 1}, {"starts": None}, {"batch": -1}):
        assert verify(**bad) == 1, bad
    size = L.aklr_verify_drafts_workspace_bytes
    assert size(0, 40, 3) == 0 and size(1, 7, 3) == 0 and size(2, 131072, 8) > 2 * 8 * 256

    def project(x=p, tokens=1, k=32, n=24, r=8, count=1, dtype=0, xs=32, bs=8, os=24, ws=p, nbytes=0, ids=p):
        return L.aklr_lora_project(x, xs, p, r * k, k, p, n * r, bs, ids, 0, None, None, p, 24, p, os, tokens, k, n, r, count, dtype, ws,
                                   nbytes, None)

    assert project(tokens=0) == 0 and project(dtype=2) == 2 and project() == 3 and project(ws=None, nbytes=1 << 30) == 3
    for bad in ({"x": None}, {"x": p + 2}, {"k": 12}, {"n": 12}, {"r": 12}, {"r": 136}, {"count": 0}, {"count": 4097}, {"xs": 33}, {"bs": 12},
                {"ids": None}, {"tokens": (1 << 20) + 1}, {"os": 16, "tokens": 2}, {"tokens": -1}):
        assert project(**bad) == 1, bad


def test_lora_workspace_holds_the_parts(native_lib):
    size = native_lib.aklr_lora_project_workspace_bytes
    for t in (1, 7, 256, 257, 2047, 2048, 8191, 1 << 20):
        for r in (8, 16, 24, 64, 128):
            up = 16 if r <= 16 else 32 if r <= 32 else 64 if r <= 64 else 128
            assert size(t, 8192, 10240, r, 8) >= 4 * t * up
    assert size(1, 12, 8, 8, 1) == 0 and size(0, 8, 8, 8, 1) == 0
