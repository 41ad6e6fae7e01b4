"""The cache operators' contracts without a GPU: what their plans accept, refuse and name, and what the C entry points
reject before any launch. CPU tensors stand in for GPU ones where only the plan is asked."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import aklr_amd
from aklr_amd import _lib, attention, kv_cache, rotary
from aklr_amd.dispatch import FallbackReason, KernelInfo

OOC = FallbackReason.OUT_OF_CONTRACT
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture
def anywhere(monkeypatch, native_lib):
    for module in (attention, kv_cache, rotary):
        monkeypatch.setattr(module, "on_gpu", lambda *t: True)


def rot_args(t=3, hq=4, hk=2, d=64, rot=64, dtype=BF16):
    return {"q": torch.zeros((t, hq, d), dtype=dtype), "k": torch.zeros((t, hk, d), dtype=dtype),
            "positions": torch.zeros(t, dtype=torch.int64), "frequencies": rotary.rotary_frequencies(rot)}


def cache_args(pages=3, h=2, d=64, page=16):
    return dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"), aklr_amd.new_kv_cache_fp8(pages, h, d, page, "cpu")))


def write_args(t=3, dtype=BF16, **kw):
    c = cache_args(**kw)
    h, d = c["k_cache"].shape[1], c["k_cache"].shape[3]
    return {"k": torch.zeros((t, h, d), dtype=dtype), "v": torch.zeros((t, h, d), dtype=dtype), **c,
            "slots": torch.arange(t)}


def read_args(**kw):
    return {**cache_args(**kw), "block_table": torch.zeros((2, 1), dtype=torch.int32),
            "starts": torch.tensor([0, 3, 5], dtype=torch.int32), "total": 5}


def attend_args(t=3, hq=4, dtype=BF16, **kw):
    c = cache_args(**kw)
    return {"q": torch.zeros((t, hq, c["k_cache"].shape[3]), dtype=dtype), **c,
            "block_table": torch.zeros((2, 1), dtype=torch.int32), "seq_lens": torch.tensor([2, 2], dtype=torch.int32),
            "starts": torch.tensor([0, 2, 3], dtype=torch.int32)}


def both_args(**kw):
    r, w = rot_args(d=64), write_args(**kw)
    return {"q": r["q"], "k": w["k"], "v": w["v"], "positions": r["positions"], "frequencies": r["frequencies"],
            **{n: w[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale", "slots")}}


OPS = {"rotary": (aklr_amd.rotary_embedding, rot_args), "write": (aklr_amd.kv_cache_write_fp8, write_args),
       "both": (aklr_amd.rotary_kv_cache_write_fp8, both_args), "read": (aklr_amd.kv_cache_read_fp8, read_args),
       "attend": (aklr_amd.tree_attention_fp8, attend_args)}


def variants(args):
    """The call with each tensor in a form its own check has to refuse."""
    for name, t in args.items():
        if not isinstance(t, torch.Tensor):
            continue
        yield name + " none", {**args, name: 3}
        yield name + " dtype", {**args, name: t.float() if t.dtype not in (F32, torch.float64, BF16) else t.to(torch.int16)}
        yield name + " dims", {**args, name: t.unsqueeze(0)}
        if name not in ("q", "starts", "seq_lens", "block_table", "frequencies"):
            yield name + " short", {**args, name: t[:-1] if t.shape[0] > 1 else t[:, :-1]}
        if t.dim() >= 2 and t.shape[-1] > 1:
            yield name + " strided", {**args, name: torch.zeros(t.shape[:-1] + (2 * t.shape[-1],), dtype=torch.uint8 if t.element_size() == 1 else t.dtype).view(t.dtype)[..., ::2]}
        if t.dim() >= 3:
            flat = torch.zeros(t.numel() + 16, dtype=torch.uint8 if t.element_size() == 1 else t.dtype).view(t.dtype)
            yield name + " unaligned", {**args, name: flat[1:1 + t.numel()].view(t.shape)}


@pytest.mark.parametrize("op", OPS)
def test_a_call_is_served_and_each_bad_form_refused(anywhere, op):
    fn, make = OPS[op]
    args = make()
    info = fn.serving(**args)
    assert isinstance(info, KernelInfo) and info.kernel_ref.startswith("aklr_") and fn.fallback_reason(**args) is None
    for what, bad in variants(args):
        if op == "rotary" and what == "k none":
            continue
        assert fn.serving(**bad) is OOC, what


@pytest.mark.parametrize("op", OPS)
def test_cpu_tensors_and_disabled_ops_are_not_served(op, monkeypatch):
    fn, make = OPS[op]
    assert fn(**make()) is OOC
    monkeypatch.setenv("AKLR_DISABLE", fn.contract_id)
    assert fn(**make()) is FallbackReason.DISABLED


@pytest.mark.parametrize("op,name", [("rotary", "q"), ("rotary", "k"), ("write", "k"), ("write", "v"), ("both", "q"), ("attend", "q"),
                                     ("rotary", "frequencies"), ("both", "frequencies"), ("both", "k"), ("read", "k_scale"),
                                     ("attend", "v_scale"), ("write", "k_scale")])
def test_gradients_are_refused_not_lost(anywhere, op, name):
    fn, make = OPS[op]
    args = make()
    args[name].requires_grad_()
    assert fn.serving(**args) is OOC
    with torch.no_grad():
        assert isinstance(fn.serving(**args), KernelInfo)


def test_rotary_sizes(anywhere):
    serving = aklr_amd.rotary_embedding.serving
    for kw in ({"d": 192, "rot": 64}, {"d": 16, "rot": 16}, {"d": 1024, "rot": 1024}, {"t": 0}, {"dtype": F32}, {"dtype": F16}):
        assert isinstance(serving(**rot_args(**kw)), KernelInfo), kw
    for kw in ({"d": 64, "rot": 96}, {"d": 24, "rot": 16}, {"d": 64, "rot": 24}, {"d": 1040, "rot": 16}, {"rot": 8}, {"dtype": torch.float64}):
        assert serving(**rot_args(**kw)) is OOC, kw
    assert isinstance(serving(**{**rot_args(), "k": None}), KernelInfo)
    for bad in ({"magnitude": math.inf}, {"magnitude": "1"}, {"interleaved": 2}, {"k": None, "out_k": torch.zeros((3, 2, 64), dtype=BF16)},
                {"frequencies": torch.ones(32)}, {"positions": torch.zeros(3)}):
        assert serving(**{**rot_args(), **bad}) is OOC, bad


def test_rotary_in_place_and_overlaps(anywhere):
    serving = aklr_amd.rotary_embedding.serving
    rows = torch.zeros((5, (4 + 2 + 2) * 64), dtype=BF16)  # queries, keys and values of one projection
    q, k = rows[:, :256].view(5, 4, 64), rows[:, 256:384].view(5, 2, 64)
    base = {**rot_args(t=5), "q": q, "k": k}
    assert isinstance(serving(**base, out_q=q, out_k=k), KernelInfo)
    assert serving(**base, out_q=q, out_k=rows[:, 192:320].view(5, 2, 64)) is OOC  # meets q's last head
    assert serving(**base, out_q=rows[:, 64:320].view(5, 4, 64)) is OOC  # its own input, shifted
    assert serving(**base, out_k=torch.zeros((5, 1, 64), dtype=BF16).expand(5, 2, 64)) is OOC  # one head twice
    assert isinstance(serving(**{**base, "k": k[:, :1].expand(5, 2, 64)}), KernelInfo)  # read twice is fine
    x = torch.zeros((5, 2, 64), dtype=BF16)
    assert serving(**base, out_q=torch.zeros((5, 4, 64), dtype=BF16), out_k=x[:, :1]) is OOC
    both = torch.zeros((5, 6, 64), dtype=BF16)
    assert isinstance(serving(**base, out_q=both[:, :4], out_k=both[:, 4:]), KernelInfo)
    assert serving(**base, out_q=both[:, :4], out_k=both[:, 3:5]) is OOC


def test_cache_forms(anywhere):
    serving = aklr_amd.kv_cache_write_fp8.serving
    for kw in ({"page": 48}, {"page": 1024, "pages": 1}, {"d": 128}, {"d": 256}, {"h": 1}, {"t": 0}, {"dtype": F32}, {"dtype": F16}):
        assert isinstance(serving(**write_args(**kw)), KernelInfo), kw
    for kw in ({"page": 8}, {"page": 24}, {"page": 1040}, {"d": 96}, {"d": 512}):
        assert serving(**write_args(**kw)) is OOC, kw
    a = write_args()
    codes = torch.zeros((3, 2, 2, 16, 64), dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales = torch.zeros((3, 2, 2, 16))
    one = {"k_cache": codes[:, 0], "v_cache": codes[:, 1], "k_scale": scales[:, 0], "v_scale": scales[:, 1]}
    assert isinstance(serving(**{**a, **one}), KernelInfo)  # keys and values of one allocation
    assert serving(**{**a, **one, "v_cache": codes[:, 0]}) is OOC  # the same pages twice
    assert serving(**{**a, "v_scale": a["k_scale"]}) is OOC
    assert serving(**{**a, "k_cache": a["k_cache"].transpose(1, 2).contiguous().transpose(1, 2)}) is OOC
    memory = torch.zeros(3 * 2 * 16 * 64, dtype=torch.uint8)
    meets = memory.view(torch.float8_e4m3fn).view(3, 2, 16, 64)
    assert serving(**{**a, "k_cache": meets, "k": memory[:768].view(BF16).view(3, 2, 64)}) is OOC
    assert serving(**{**a, "slots": a["slots"].to(torch.int32)}) != OOC
    assert serving(**{**a, "slots": torch.arange(6)[::2]}) is OOC


def test_read_forms(anywhere):
    serving = aklr_amd.kv_cache_read_fp8.serving
    a = read_args()
    out = torch.zeros((5, 2, 64), dtype=F16)
    assert isinstance(serving(**a, out_k=out, out_v=torch.zeros_like(out)), KernelInfo)
    for bad in ({"total": -1}, {"total": 5.0}, {"total": True}, {"out_dtype": F32}, {"out_k": out, "out_v": out},
                {"out_k": out, "out_dtype": BF16}, {"out_k": out[:4]}, {"block_table": torch.zeros((3, 1), dtype=torch.int32)},
                {"starts": torch.zeros(0, dtype=torch.int32)}, {"out_k": a["k_scale"].view(-1)[:0]}):
        assert serving(**{**a, **bad}) is OOC, bad
    wide = torch.zeros((2, 4), dtype=torch.int32)
    assert isinstance(serving(**{**a, "block_table": wide[:, :2]}), KernelInfo)
    assert isinstance(serving(**{**a, "total": 0}), KernelInfo)


def test_attention_forms(anywhere):
    serving = aklr_amd.tree_attention_fp8.serving
    a = attend_args()
    assert serving(**a).variant == "causal"
    for good in ({"tree_mask": torch.zeros((3, 2), dtype=torch.bool)}, {"tree_mask": torch.zeros((3, 9), dtype=torch.uint8)[:, :5]},
                 {"softmax_scale": 1}, {"out": torch.zeros_like(a["q"])}, {"return_lse": True}):
        assert isinstance(serving(**{**a, **good}), KernelInfo), good
    for bad in ({"tree_mask": torch.zeros((2, 2), dtype=torch.bool)}, {"tree_mask": torch.zeros((3, 2))},
                {"tree_mask": torch.zeros((3, 4), dtype=torch.bool)[:, ::2]}, {"softmax_scale": math.nan},
                {"softmax_scale": "x"}, {"return_lse": 1.5}, {"out": a["q"]}, {"out": torch.zeros((3, 4, 64), dtype=F16)},
                {"q": torch.zeros((3, 5, 64), dtype=BF16)}, {"q": torch.zeros((3, 4, 128), dtype=BF16)},
                {"q": torch.zeros((3, 4, 64), dtype=F32)}, {"starts": torch.zeros(2, dtype=torch.int32)},
                {"q": torch.zeros((3, 1, 64), dtype=BF16)}, {"block_table": torch.zeros((1, 1), dtype=torch.int32)},
                {"seq_lens": torch.zeros(4, dtype=torch.int32)[::2]}):
        assert serving(**{**a, **bad}) is OOC, bad
    assert isinstance(serving(**attend_args(t=3, hq=6)), KernelInfo)
    # pages 2^32 bytes of codes or scales apart, keys' and values' not alike, and more rows than a launch has room for
    pages = a["k_cache"].shape[0]
    shape = a["k_cache"].shape[1:]
    n = shape.numel()
    far = torch.empty((pages - 1) * 2**32 + n, dtype=torch.uint8)
    wide = torch.as_strided(far, (pages, *shape), (2**32, *a["k_cache"].stride()[1:])).view(torch.float8_e4m3fn)
    near = torch.as_strided(far, (pages, *shape), (2**32 - 16, *a["k_cache"].stride()[1:])).view(torch.float8_e4m3fn)
    assert serving(**{**a, "k_cache": wide, "v_cache": wide}) is OOC
    assert isinstance(serving(**{**a, "k_cache": near, "v_cache": near}), KernelInfo)
    assert serving(**{**a, "k_cache": near}) is OOC
    far = far[:(pages - 1) * 2**32 + n // shape[-1] * 4].view(torch.float32)
    wide = torch.as_strided(far, (pages, *shape[:2]), (2**30, shape[1], 1))
    assert serving(**{**a, "k_scale": wide, "v_scale": wide}) is OOC
    assert serving(**{**a, "k_scale": wide}) is OOC
    q = torch.zeros((1, 1, 64), dtype=BF16)
    for heads, served in ((2**14, False), (2**14 - shape[0], True)):
        big = {"q": q.expand(2**14, heads, 64), "seq_lens": a["seq_lens"], "starts": a["starts"]}
        assert (serving(**{**a, **big}) is OOC) == (not served), heads


def test_pieces_of_rows_that_do_not_meet():
    x = torch.zeros((4, 32))
    assert rotary.apart(x[:, :16], x[:, 16:]) and not rotary.apart(x[:, :17], x[:, 16:])
    assert rotary.apart(x[1:, :16], x[:3, 16:]) and not rotary.apart(x[1:, :20], x[:3, 16:])
    assert rotary.apart(x[:2], x[2:]) and not rotary.apart(x, x)
    assert not rotary.apart(x.view(-1)[:20], x[:, 16:]) and rotary.apart(x[:0], x)


def test_frequencies():
    f = rotary.rotary_frequencies(64)
    assert f.dtype == torch.float64 and f[0] == 1 and f[-1] == pytest.approx(10000 ** -(62 / 64))
    assert torch.equal(rotary.rotary_frequencies(64, scaling="linear", factor=4.0), f / 4)
    ntk = rotary.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == 1 and ntk[-1] == pytest.approx(float(f[-1]) / 4)
    yarn = rotary.rotary_frequencies(64, scaling="yarn", factor=40.0, original_length=4096)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(yarn[turns > 33], f[turns > 33]) and torch.allclose(yarn[turns < 0.9], f[turns < 0.9] / 40, rtol=1e-15)
    assert bool(((yarn <= f) & (yarn >= f / 40 * (1 - 1e-12))).all())
    assert rotary.rotary_magnitude(40.0) == pytest.approx(0.1 * math.log(40) + 1) and rotary.rotary_magnitude(1.0) == 1
    for bad in ({"rotary_dim": 7}, {"rotary_dim": 0}, {"scaling": "other"}, {"base": 0.5}, {"factor": 0.5}, {"scaling": "yarn"}):
        with pytest.raises(ValueError):
            rotary.rotary_frequencies(**{"rotary_dim": 64, **bad})


def test_entry_points_reject_before_any_launch(native_lib):
    L = native_lib
    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 15) & ~15

    def rotary_call(q=p, tokens=0, d=64, rot=64, dtype=0, stride=64, pos=p):
        return L.aklr_rotary_embedding(q, stride, 64, p, 64, 64, 1, None, 0, 0, None, 0, 0, 0, pos, 1, p, tokens, d, rot, 0, 1.0, dtype, None)

    assert rotary_call() == 0
    assert rotary_call(dtype=3) == 2
    for bad in ({"q": None}, {"q": p + 2}, {"d": 40}, {"rot": 24}, {"rot": 80}, {"stride": 60}, {"pos": None}, {"tokens": -1}):
        assert rotary_call(**bad) == 1, bad

    def write_call(k=p, slots=p, tokens=0, h=1, d=64, pages=2, page=16, stride=None, qh=0, rot=0, dtype=0):
        s = stride if stride is not None else h * page * d
        return L.aklr_kv_cache_write_fp8(None, 0, 0, None, 0, 0, qh, k, d, d, p, d, d, None, 0, None, rot, 0, 1.0, slots, 1, p, p, p,
                                         p, s, s, h * page, h * page, tokens, h, d, pages, page, dtype, None)

    assert write_call() == 0
    assert write_call(dtype=9) == 2
    for bad in ({"k": None}, {"slots": None}, {"d": 96}, {"page": 8}, {"page": 2048}, {"pages": 0}, {"pages": 1 << 28},
                {"stride": 16}, {"qh": 1}, {"rot": 64}, {"tokens": -1}, {"k": p + 8}):
        assert write_call(**bad) == 1, bad

    def read_call(table=p, starts=p, batch=0, total=4, out=p, dtype=0, cols=1, stride=1, page=16):
        return L.aklr_kv_cache_read_fp8(p, p, p, p, page * 64, page * 64, page, page, table, stride, cols, starts, batch, total, out, out,
                                        1, 64, 2, page, dtype, None)

    assert read_call() == 0 and read_call(total=0, batch=3) == 0
    assert read_call(dtype=2) == 2
    for bad in ({"table": None}, {"starts": None}, {"out": p + 4}, {"stride": 0}, {"page": 20}, {"total": -1}):
        assert read_call(**{"batch": 1, **bad}) == 1, bad

    def attend_call(q=p, total=1, batch=1, hq=2, hkv=1, d=64, page=16, cols=1, dtype=0, ws=None, nbytes=0, qs=128, lens=p):
        return L.aklr_tree_attention_fp8(q, qs, 64, p, p, p, p, hkv * page * d, hkv * page, p, cols, cols,
                                         lens, p, None, 0, 0, p, None, total, batch, hq, hkv, d, 2, page, 1.0, dtype, ws, nbytes, None)

    assert attend_call(total=0) == 0 and attend_call(batch=0) == 0
    assert attend_call(dtype=2) == 2
    for bad in ({"q": None}, {"q": p + 8}, {"hq": 3, "hkv": 2}, {"d": 80}, {"page": 12}, {"qs": 100}, {"lens": None},
                {"cols": (1 << 24) + 1}, {"cols": 1 << 24, "page": 32}):
        assert attend_call(**bad) == 1, bad
    need = L.aklr_tree_attention_fp8_workspace_bytes(1, 1, 2, 1, 64, 16 * 64)
    assert need > 0 and attend_call(cols=64) == 3 and attend_call(cols=64, ws=p, nbytes=need - 1) == 3
    assert L.aklr_tree_attention_fp8_workspace_bytes(1, 1, 2, 1, 64, 16) == 0  # one step: nothing to split


def test_attention_workspace_grows_with_what_is_asked(native_lib):
    size = native_lib.aklr_tree_attention_fp8_workspace_bytes
    for d in (64, 128, 256):
        assert size(0, 1, 8, 8, d, 4096) == 0 and size(1, 0, 8, 8, d, 4096) == 0
        last = 0
        for tokens in (1, 2, 16, 64, 1000, 5000):
            got = size(tokens, 16, 32, 8, d, 4096)
            assert got >= last
            last = got
