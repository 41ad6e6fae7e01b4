"""Draft verification on the GPU against the oracle in 64 bits: every output is a whole number and has to be the oracle's. The
kernel's sums are in 64 bits too; they differ from the oracle's by their order alone, some 2^-50 of a row's sum, and the numbers
drawn here are multiples of 2^-24: the chance that one lies that near to a border of 2^17 values is below 2^-9 in all, and of a
first run that fails for it none that a second one would mend: inputs are seeded. Rows of multiples of 1/256 have exact sums,
and their draws hit borders on purpose."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import aklr_amd
from oracle import requests as oq
from tests.helpers import say

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def problem(lens, vocab, seed, dtype=F32, form="tree", sharp=4.0, near=0.7, rows_behind=0):
    """Sequences of `lens` query tokens with drafts drawn from rows near the target's."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    pick = np.random.RandomState(seed)
    t = sum(lens) + rows_behind
    logits = sharp * torch.randn((t, vocab), generator=g, device=DEV)
    target = torch.softmax(logits, -1).to(dtype)
    draft = torch.softmax(logits + near * torch.randn(logits.shape, generator=g, device=DEV), -1).to(dtype)
    first = np.repeat(np.r_[0, np.cumsum(lens)[:-1]], lens).astype(int)
    i = np.concatenate([np.arange(n) for n in lens] + [[]]).astype(int)
    back = np.where(i > 0, pick.randint(0, 1 << 30, len(i)) % np.maximum(np.minimum(i, 4), 1), 0)
    parent = i - 1 - (0 if form == "chain" else back)
    row = torch.from_numpy(np.where(i > 0, first + parent, first)).to(DEV)
    tokens = torch.zeros(t, dtype=torch.int64, device=DEV)
    if len(i):
        tokens[: len(i)] = torch.multinomial(draft[row].float(), 1, generator=g)[:, 0]
    parents = torch.zeros(t, dtype=torch.int32, device=DEV)
    parents[: len(i)] = torch.from_numpy(parent).to(DEV).to(torch.int32)
    return {"target": target, "draft": draft if form != "certain" else None, "tokens": tokens, "parents": None if form == "chain" else parents,
            "starts": torch.tensor(np.r_[0, np.cumsum(lens)], dtype=torch.int32, device=DEV),
            "u": torch.rand(t, generator=g, device=DEV), "v": torch.rand(len(lens), generator=g, device=DEV), "most": max(max(lens, default=1), 1)}


def call(p):
    return aklr_amd.verify_drafts(p["target"], p["tokens"], p["starts"], p["u"], p["v"], p["most"], draft_probs=p["draft"],
                                  parents=p["parents"])


def check(p, what=""):
    out, path, counts = call(p)
    n = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    d = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    want = oq.verify(d(p["target"]), n(p["tokens"]), n(p["starts"]), n(p["u"]), n(p["v"]), p["most"], d(p["draft"]), n(p["parents"]))
    assert out.dtype == p["tokens"].dtype and path.dtype == counts.dtype == torch.int32
    for name, got, w in zip(("counts", "path", "tokens"), (counts, path, out), (want[2], want[1], want[0])):
        assert got.shape == w.shape and np.array_equal(got.cpu().numpy(), w), f"{what} {name}: {got.tolist()} instead of {w.tolist()}"
    return out, path, counts


@pytest.mark.parametrize("form", ["chain", "tree", "certain"])
@pytest.mark.parametrize("lens,vocab,dtype", [([1], 8, F32), ([2], 9, F32), ([4, 1, 3], 31, F32), ([5] * 7, 511, F32), ([3, 8], 512, F16),
                                              ([6, 2, 6], 513, BF16), ([9], 1024, F32), ([5, 4], 4099, F32), ([8] * 5, 50257, F32),
                                              ([7, 3], 50257, BF16), ([4, 6], 32003, F16), ([33, 20, 1], 8209, F32), ([5, 3], 131072, F32),
                                              ([4], 262144 + 5, F32), ([3], 1 << 20, BF16)])
def test_forms_types_and_vocabularies(lens, vocab, dtype, form):
    say(f"verify {lens} {vocab} {dtype} {form}")
    for seed in range(3):
        check(problem(lens, vocab, 10 * seed + len(lens), dtype, form), seed)


@pytest.mark.parametrize("form", ["chain", "tree", "certain"])
def test_many_sequences(form):
    say(f"verify many {form}")
    check(problem([5, 1, 3, 4] * 160, 300, 1, F32, form))
    check(problem([2] * 2500, 40, 2, F32, form, sharp=1.0))


@pytest.mark.parametrize("form", ["chain", "tree", "certain"])
def test_long_trees(form):
    # more nodes than a wave has lanes; children of a node lie far behind it, refused drafts are many
    say(f"verify long {form}")
    check(problem([64, 65, 200, 130], 1000, 3, F32, form, sharp=2.0, near=0.3))
    p = problem([1024, 500], 300, 4, F32, form, sharp=1.0, near=0.1)
    if form != "chain":  # bushy: the root has most of them
        pick = np.random.RandomState(5)
        i = np.r_[np.arange(1024), np.arange(500)]
        p["parents"] = torch.tensor(np.where(pick.rand(len(i)) < 0.9, 0, i // 2), dtype=torch.int32, device=DEV)
    check(p)
    if form != "chain":  # nothing stands, every one is tried
        p["u"].fill_(1.0)
        check(p)
        p["u"].fill_(0.0)
        check(p)


def test_many_rejections_of_one_node():
    say("verify: more rejections than there are rounds of launches")
    for children in (2, 3, 4, 5, 6, 9, 20):
        p = problem([children + 1] * 3, 2000, children, F32, "tree", sharp=1.0, near=2.0)
        p["parents"].zero_()
        p["u"].fill_(0.999)
        _, path, _ = check(p, children)


def test_exact_borders():
    # sums of multiples of 1/256 are exact in any order: a draw at a border belongs to the next value
    say("verify borders")
    vocab = 1400
    pick = np.random.RandomState(1)
    for seed in range(40):
        where = np.sort(pick.choice(vocab, 256, replace=False))
        p = np.zeros((4, vocab), np.float32)
        q = np.zeros((4, vocab), np.float32)
        for r in range(4):
            np.add.at(p[r], where[pick.randint(0, 256, 256)], 1 / 256)
            np.add.at(q[r], where[pick.randint(0, 256, 256)], 1 / 256)
        case = {"target": torch.from_numpy(p).to(DEV), "draft": torch.from_numpy(q).to(DEV) if seed % 3 else None,
                "tokens": torch.tensor(where[pick.randint(0, 256, 4)], device=DEV), "parents": None if seed % 2 else torch.tensor([0, 0, 0, 1], dtype=torch.int32, device=DEV),
                "starts": torch.tensor([0, 4], dtype=torch.int32, device=DEV), "u": torch.tensor(pick.randint(0, 9, 4) / 8, dtype=F32, device=DEV),
                "v": torch.tensor([pick.randint(0, 257) / 256], dtype=F32, device=DEV), "most": 4}
        check(case, seed)


def test_ends_of_the_sampling():
    say("verify: first and last values, one value, values at units' ends")
    for vocab in (8, 511, 512, 513, 1025, 70000):
        for at in {0, 7, vocab // 2, vocab - 9, vocab - 8, vocab - 2, vocab - 1} - {-1, -2}:
            at = max(at, 0)
            for v in (0.0, 0.5, 1.0, float("nan"), -3.0, 2.0):
                p = torch.zeros((1, vocab), device=DEV)
                p[0, at] = 0.3
                out = call({"target": p, "draft": None, "tokens": torch.zeros(1, dtype=torch.int32, device=DEV), "parents": None, "most": 2,
                            "starts": torch.tensor([0, 1], dtype=torch.int32, device=DEV), "u": torch.zeros(1, device=DEV), "v": torch.tensor([v], device=DEV)})
                assert out[0].tolist() == [[at, -1]] and out[1].tolist() == [[0, -1]] and out[2].tolist() == [1], (vocab, at, v)


def test_rows_of_no_probabilities():
    say("verify: NaN, infinities, negative values, zero rows, rows that do not add up to 1")
    for form in ("chain", "tree", "certain"):
        p = problem([5, 5, 5, 5], 700, 7, F32, form)
        for x in (p["target"], p["draft"]):
            if x is None:
                continue
            x[0, ::3] = float("nan")
            x[1, 1::4] = float("inf")
            x[2, ::2] *= -1
            x[5:10] *= 3.7
            x[10:12] = 0
            x[13] = float("nan")
        check(p, form)
        p["target"].zero_()
        out, _, counts = check(p, form)
        assert (out[:, 0] == -1).all() and (counts == 1).all()
    # target and draft alike: a draft with any probability stands; refused all the same (u past 1 counts as less), nothing is left
    p = problem([4, 4], 300, 8, F32, "chain", near=0.0)
    _, _, counts = check(p)
    assert counts.tolist() == [4, 4]
    p["draft"] = p["draft"] * 2
    check(p)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_probabilities_below_the_normal_range(dtype):
    say(f"verify subnormal {dtype}")
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    p = torch.zeros((3, 2000), dtype=dtype, device=DEV)
    p[:, [3, 700, 1999]] = torch.tensor([1.0, 2.0, 5.0], device=DEV).mul(tiny).to(dtype)
    q = torch.zeros_like(p)
    q[:, 700] = 3 * tiny
    for v in (0.0, 0.125, 0.374, 0.375, 0.5, 0.99):
        for u in (0.0, 0.66, 0.67):
            case = {"target": p, "draft": q, "tokens": torch.tensor([0, 700, 700], device=DEV), "parents": None, "most": 3, "v": torch.tensor([v], device=DEV),
                    "u": torch.full((3,), u, device=DEV), "starts": torch.tensor([0, 3], dtype=torch.int32, device=DEV)}
            check(case, (u, v))
            check({**case, "draft": None}, (u, v))


def test_drafts_that_are_passed_over():
    say("verify: tokens outside the vocabulary, parents that do not come before, more tokens than most, numbers that are none")
    for form in ("tree", "certain"):
        for dtype in (torch.int32, torch.int64):
            p = problem([12, 9, 10], 400, 9, F32, form)
            p["tokens"] = p["tokens"].to(dtype)
            p["tokens"][[2, 14, 25]] = torch.tensor([-1, 400, (1 << 31) - 1], dtype=dtype, device=DEV)
            if dtype == torch.int64:
                p["tokens"][[4, 15]] = torch.tensor([1 << 40, -(1 << 40)], device=DEV)
            p["parents"][[3, 6, 13, 24]] = torch.tensor([3, 9, -1, 1 << 30], dtype=torch.int32, device=DEV)
            p["u"][[1, 5, 13, 22]] = torch.tensor([float("nan"), -1.0, float("inf"), 1.5], device=DEV)
            check(p)
            for most in (1, 2, 5, 40):
                check({**p, "most": most}, most)
    for most in (1, 3):
        check({**problem([6, 6], 100, 11, F32, "chain"), "most": most})


def test_empty_sequences_and_rows_behind():
    say("verify: no tokens, sequences of none, rows behind the last, starts past the rows")
    p = problem([0, 3, 0, 2, 0], 100, 12, F32, "tree", rows_behind=4)
    check(p)
    p["most"] = 6
    _, _, counts = check(p)
    assert counts.tolist()[::2] == [0, 0, 0]
    none = problem([0, 0], 100, 13)
    assert [x.tolist() for x in call(none)] == [[[-1], [-1]], [[-1], [-1]], [0, 0]]
    out, path, counts = aklr_amd.verify_drafts(p["target"], p["tokens"], p["starts"][:1], p["u"], p["v"][:0], 3)
    assert out.shape == path.shape == (0, 3) and counts.shape == (0,)
    far = dict(p, starts=torch.tensor([0, 3, 3, 9, 2000, 4000], dtype=torch.int32, device=DEV))  # the last two reach past the rows
    check(far)
    call(dict(p, starts=torch.tensor([-5, 3, 2, -7, 5, 1 << 30], dtype=torch.int32, device=DEV)))  # none that ascend: nothing outside is read
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_anywhere(dtype):
    say(f"verify rows at any place {dtype}")
    p = problem([5, 4], 1003, 14, dtype, "tree")
    for left, right in ((1, 0), (3, 2), (0, 5)):
        def put(x):
            wide = torch.full((x.shape[0], left + 1003 + right), float("nan"), dtype=dtype, device=DEV)
            wide[:, left:left + 1003] = x
            return wide[:, left:left + 1003]
        check({**p, "target": put(p["target"]), "draft": p["draft"]})
        check({**p, "target": put(p["target"]), "draft": put(p["draft"])})
    one = {k: v for k, v in problem([1], 77, 15, dtype, "chain").items()}
    check({**one, "target": one["target"].expand(1, 77), "draft": None})


def test_offsets_past_32_bits():
    say("verify rows behind 2^31 values")
    vocab, t = 1 << 20, 2100
    target = torch.zeros((t, vocab), dtype=BF16, device=DEV)
    target[t - 2, 77], target[t - 1, vocab - 3], target[0, 5] = 1, 1, 1
    tokens = torch.zeros(t, dtype=torch.int32, device=DEV)
    tokens[t - 1] = 77
    out, path, counts = aklr_amd.verify_drafts(target, tokens, torch.tensor([0, 1, t - 2, t], dtype=torch.int32, device=DEV)[[0, 1, 3]],
                                               torch.full((t,), 0.5, device=DEV), torch.tensor([0.5, 0.5], device=DEV), 4)
    assert out[0].tolist() == [5, -1, -1, -1]
    starts = torch.tensor([t - 2, t], dtype=torch.int32, device=DEV)
    out, path, counts = aklr_amd.verify_drafts(target, tokens, starts, torch.full((t,), 0.5, device=DEV), torch.tensor([0.5], device=DEV), 4)
    assert out.tolist() == [[77, vocab - 3, -1, -1]] and counts.tolist() == [2]


def test_captured_and_on_streams():
    say("verify: captured, replayed with other values between eager calls; two streams at once")
    ps = [problem([9, 5, 9, 3], 5000, s, F32, "tree", sharp=2.0) for s in range(20, 24)]
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
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    want = [call(q) for q in ps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ps]
    for _ in range(5):
        outs = []
        for s, q in zip(streams, ps):
            with torch.cuda.stream(s):
                outs.append(call(q))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(outs, want) for a, b in zip(x, y))
