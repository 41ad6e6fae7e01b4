"""Pins of ``oracle.requests``: hand-worked cases and properties that a mistake would break."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import requests as oq


def test_chain_by_hand():
    # node 0: p(2) = 0.5 against u q = 0.5 * 0.25: stands; node 1: p(1) = 0.1, u q = 0.5 * 0.8: not; what is left of
    # p - q = [0.4 - 0.1, <0, 0.5 - 0.1] = [0.3, 0, 0.4]; 0.5 * 0.7 passes the first
    target = np.array([[0.25, 0.25, 0.5], [0.4, 0.1, 0.5], [1, 0, 0]])
    draft = np.array([[0.5, 0.25, 0.25], [0.1, 0.8, 0.1], [0, 1, 0]])
    out, path, counts = oq.verify(target, [7, 2, 1], [0, 3], [0, 0.5, 0.5], [0.5], 4, draft)
    assert out.tolist() == [[2, 2, -1, -1]] and path.tolist() == [[0, 1, -1, -1]] and counts.tolist() == [2]
    out, _, _ = oq.verify(target, [7, 2, 1], [0, 3], [0, 0.5, 0.5], [0.42], 4, draft)
    assert out.tolist() == [[2, 0, -1, -1]]
    # both stand: the next token is the last node's own
    out, path, counts = oq.verify(target, [7, 2, 1], [0, 3], [0, 0.5, 0.1], [0.9], 3, draft)
    assert out.tolist() == [[2, 1, 0]] and path.tolist() == [[0, 1, 2]] and counts.tolist() == [3]


def test_tree_by_hand():
    # two children of the root: the first is refused (0.9 * 0.5 > 0.25), which leaves [0.25 - 0.5, 0.75 - 0.5] = [0, 0.25];
    # the second, token 1: 0.4 * 0.25 * 0.5 < 0.25 stands, and its own child follows
    target, draft = np.array([[0.25, 0.75]] * 4), np.array([[0.5, 0.5]] * 4)
    args = [0, 0, 1, 1], [0, 4], [0, 0.9, 0.4, 0.5], [0.1], 4
    out, path, _ = oq.verify(target, *args, draft, [-1, 0, 0, 2])
    assert path.tolist() == [[0, 2, 3, -1]] and out.tolist() == [[1, 1, 0, -1]]
    # certain drafts: 0.9 > 0.25; then 0.4 * 0.75 < 0.75
    out, path, _ = oq.verify(target, *args, None, [-1, 0, 0, 2])
    assert path.tolist() == [[0, 2, 3, -1]] and out.tolist() == [[1, 1, 0, -1]]
    # the same token twice: once refused it weighs nothing
    out, path, _ = oq.verify(target, [0, 0, 0], [0, 3], [0, 0.9, 0.0], [0.0], 3, None, [-1, 0, 0])
    assert path.tolist() == [[0, -1, -1]] and out.tolist() == [[1, -1, -1]]


@pytest.mark.parametrize("form", ["chain", "tree", "certain"])
def test_what_comes_out_is_distributed_as_the_target(form):
    # the first token that comes out, over many draws of drafts and numbers, against the target's first row: a share of
    # 20000 is off by less than 5 * sqrt(1 / 4 / 20000) = 0.018
    rng = np.random.RandomState(1)
    vocab, n = 5, 20000
    p, q = rng.dirichlet(np.ones(vocab)), rng.dirichlet(np.ones(vocab))
    target, draft = np.stack([p] * 3), np.stack([q] * 3)
    seen = np.zeros(vocab)
    for _ in range(n):
        tokens = [0, rng.choice(vocab, p=q), rng.choice(vocab, p=q)] if form != "certain" else [0, 3, 1]
        out, _, _ = oq.verify(target, tokens, [0, 3], rng.rand(3), rng.rand(1), 3, None if form == "certain" else draft,
                              None if form == "chain" else [-1, 0, 0])
        seen[out[0, 0]] += 1
    assert np.abs(seen / n - p).max() < 0.018


def test_verify_edges():
    one = np.array([[0.0, 1.0, 0.0]])
    nan = np.array([[np.nan, -1.0, np.inf]])
    assert oq.verify(one, [5], [0, 1], [0], [1.0], 2)[0].tolist() == [[1, -1]]
    assert oq.verify(nan, [5], [0, 1], [0], [0.5], 2)[0].tolist() == [[-1, -1]]
    assert oq.verify(one, [5], [0, 0], [0], [0.5], 2)[2].tolist() == [0]
    # nothing left: the target's own row
    row = np.array([[0.5, 0.5, 0.0]] * 2)
    assert oq.verify(row, [0, 2], [0, 2], [0, 0.9], [0.6], 2, np.array([[0.6, 0.6, 0.6]] * 2))[0].tolist() == [[1, -1]]
    # a draft past `most`, or without a token of the vocabulary, is not tried
    assert oq.verify(row, [0, 0], [0, 2], [0, 0], [0.6], 1)[0].tolist() == [[1]]
    assert oq.verify(row, [0, 9], [0, 2], [0, 0], [0.6], 2)[1].tolist() == [[0, -1]]


def test_compact_and_copy_by_hand():
    t = [np.arange(2 * 1 * 4).reshape(2, 1, 4, 1).astype(float) for _ in "kv"] + [np.arange(8).reshape(2, 1, 4) * 1.0 for _ in "kv"]
    # positions 0..6 in pages 1, 0: hold 4 5 6 7 0 1 2; of the last five (2..6) keep 0, 2, 3
    for got in oq.compact(t, np.array([[1, 0]]), [7], [0, 5], np.array([[0, 2, 3]]), [3]):
        assert got.reshape(2, 4).tolist() == [[1, 1, 2, 3], [4, 5, 6, 0]]
    for got in oq.copy_pages(t, [1, 0, 5], [0, 0, 1]):
        assert got.reshape(2, 4).tolist() == [[0, 1, 2, 3], [4, 5, 6, 7]]  # the last pair for a page wins, from the old


def test_update_by_hand():
    # pages of 4; sequence 0 holds 0, 1 (6 positions), sequence 1 pages 0, 2 (5), page 0 shared
    table = np.array([[0, 1, -1], [0, 2, -1]])
    refs = [2, 1, 1, 0, 0]
    new, granted, src, dst, after = oq.update_pages(refs, table, [6, 5], [9, 3], 4)
    # 0 grows by a page; 1 falls to 3 of page 0's positions, which 0 holds too: a copy, after 0's, so page 3; page 2 is free
    assert new.tolist() == [[0, 1, 2], [3, -1, -1]] and granted == [9, 3] and (src, dst) == ([-1, 0], [-1, 3])
    assert after == [1, 1, 1, 1, 0]
    # both go on from sequence 1: the lowest takes page 2 over, the other copies it; 1's first page is shared
    new, granted, src, dst, after = oq.update_pages(refs, table, [6, 5], [6, 6], 4, [1, 1])
    assert new.tolist() == [[0, 2, -1], [0, 1, -1]] and (src, dst) == ([-1, 2], [-1, 1]) and after == [2, 1, 1, 0, 0]
    # all end; a new one begins
    new, granted, src, dst, after = oq.update_pages(refs, table, [6, 5], [0, 9], 4, [0, -1])
    assert new.tolist() == [[-1, -1, -1], [0, 1, 2]] and after == [1, 1, 1, 0, 0] and granted == [0, 9]
    # hardly a page: who asks first gets it
    new, granted, *_ , after = oq.update_pages([2, 1, 1, 1], table, [6, 5], [12, 12], 4)
    assert granted == [8, 8] and after == [2, 1, 1, 1]


def test_update_keeps_the_books():
    rng = np.random.RandomState(3)
    for _ in range(60):
        batch, cols, page, pages = rng.randint(1, 7), rng.randint(1, 6), 4, 40
        table = np.full((batch, cols), -1)
        refs = np.zeros(pages, dtype=int)
        lens = np.zeros(batch, dtype=int)
        for _ in range(6):
            parents = rng.randint(-1, batch, batch) if rng.rand() < 0.5 else None
            wants = rng.randint(0, cols * page + 3, batch)
            old = table.copy()
            table, granted, src, dst, refs = oq.update_pages(refs, table, lens, wants, page, parents)
            assert [int((table == p).sum()) for p in range(pages)] == list(refs)
            for b in range(batch):
                assert granted[b] <= wants[b] and (table[b, : -(-granted[b] // page)] >= 0).all() and (table[b, -(-granted[b] // page):] < 0).all()
                if dst[b] >= 0:
                    assert refs[dst[b]] == 1 and src[b] in old and refs[src[b]] >= 0
                # a page that will be written is nobody else's
                if granted[b] % page:
                    assert refs[table[b, granted[b] // page]] == 1
            lens = np.array(granted)


def test_lora_is_the_products():
    rng = np.random.RandomState(2)
    x, a, b, base = rng.randn(4, 6), rng.randn(3, 2, 6), rng.randn(3, 5, 2), rng.randn(4, 5)
    out, terms, _ = oq.lora(x, a, b, [2, -1, 0, 2], base, [1, 2, 3], [2, 0, 1])
    full = base + np.einsum("tnr,trk,tk->tn", b[[2, 1, 0, 2]], a[[2, 1, 0, 2]], x) * np.array([3, 0, 1, 3])[:, None]
    one = base[3] + 3 * x[3] @ a[2][0] * b[2][:, 0]
    assert np.allclose(out[1], base[1]) and np.allclose(out[2], full[2]) and np.allclose(out[3], one) and np.allclose(out[0], base[0] + 3 * x[0] @ a[2][0] * b[2][:, 0])
    assert (np.abs(out - base) <= terms + 1e-12).all()
