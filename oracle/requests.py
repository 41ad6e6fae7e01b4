"""What differs from request to request of a batch: drafted tokens verified, pages of the FP8 cache handed on, copied and
compacted, low-rank adapters. In numpy float64 and Python integers (test infrastructure; see ``oracle/__init__.py``).

The operators are not in the reference's scope of this library, so nothing of it restates them; each function is the
operator's definition, one sequence after the other, and is pinned in tests/test_oracle_requests.py by properties that a
mistake would break (hand-worked trees, the distribution that comes out, pages counted, a brute-force product).
"""
from __future__ import annotations

import numpy as np


def proper(row):
    """Probabilities with what is none (negative, infinite, NaN) as 0."""
    row = np.asarray(row, dtype=np.float64)
    return np.where(np.isfinite(row) & (row > 0), row, 0.0)


def unit(u):
    """A number cut to [0, 1 - 2^-24]."""
    return min(float(u), 1.0 - 2.0**-24) if u > 0 else 0.0


def verify(target, tokens, starts, accept, sample, most, draft=None, parents=None):
    """(tokens, path, counts) of ``verify_drafts``."""
    batch, vocab = len(sample), target.shape[1]
    out, path, counts = np.full((batch, most), -1), np.full((batch, most), -1), np.zeros(batch, dtype=np.int64)
    for b in range(batch):
        lo, hi = int(starts[b]), min(int(starts[b + 1]), len(tokens))
        n = min(hi - lo, most)
        if n <= 0:
            continue
        node, steps = 0, [0]
        while True:
            p = proper(target[lo + node])
            q = proper(draft[lo + node]) if draft is not None else None
            left, mass, found = p.copy(), 1.0, None
            for j in range(node + 1, n):
                x = int(tokens[lo + j])
                if (j - 1 if parents is None else int(parents[lo + j])) != node or not 0 <= x < vocab:
                    continue
                if unit(accept[lo + j]) * mass * (1.0 if q is None else q[x]) < left[x]:
                    found = j
                    break
                if q is None:
                    mass -= left[x]
                    left[x] = 0.0
                else:
                    left = np.maximum(left - mass * q, 0.0)
                    mass = left.sum()
            if found is None:
                break
            node = found
            steps.append(node)
        if not left.sum() > 0:
            left = p
        sums = np.cumsum(left)
        level = unit(sample[b]) * left.sum()
        over = np.flatnonzero((sums > level) & (left > 0))
        token = -1 if not sums[-1] > 0 else over[0] if len(over) else np.flatnonzero(left > 0)[-1]
        counts[b] = len(steps)
        path[b, : len(steps)] = steps
        out[b, : len(steps)] = [int(tokens[lo + j]) for j in steps[1:]] + [token]
    return out, path, counts


def copy_pages(tensors, src, dst):
    """The four tensors of a cache with pages copied; all copies read what was there before."""
    outs = [np.array(t) for t in tensors]
    pages = len(outs[0])
    for a, b in zip(src, dst):
        if 0 <= a < pages and 0 <= b < pages:
            for t, old in zip(outs, tensors):
                t[b] = old[a]
    return outs


def compact(tensors, table, lens, starts, path, counts):
    """The four tensors of a cache with the kept positions of each sequence moved together."""
    outs = [np.array(t) for t in tensors]
    pages, page = outs[0].shape[0], outs[0].shape[2]

    def place(b, pos):
        if not 0 <= pos < table.shape[1] * page or not 0 <= table[b, pos // page] < pages:
            return None
        return int(table[b, pos // page]), pos % page

    for b in range(len(lens)):
        t = int(starts[b + 1] - starts[b])
        first = int(lens[b]) - t
        for i in range(min(int(counts[b]), path.shape[1])):
            x = int(path[b, i])
            if not 0 <= x < t or x == i:
                continue
            a, z = place(b, first + x), place(b, first + i)
            if a and z:
                for new, old in zip(outs, tensors):
                    new[z[0], :, z[1]] = old[a[0], :, a[1]]
    return outs


def update_pages(refs, table, lens, wants, page, parents=None):
    """(table, granted, src, dst, refs) of ``kv_cache_update_pages``."""
    refs, (batch, cols) = [int(r) for r in refs], table.shape
    pages, room = len(refs), cols * page
    cut = [min(max(int(n), 0), room) for n in lens]
    wants = [min(max(int(n), 0), room) for n in wants]
    parents = list(range(batch)) if parents is None else [int(p) if 0 <= p < batch else None for p in parents]

    def there(p):
        return 0 <= p < pages

    for b in range(batch):
        for p in table[b, : -(-cut[b] // page)]:
            if there(p):
                refs[p] -= 1
    new = np.full((batch, cols), -1, dtype=np.int64)
    kept = [0 if parents[b] is None else min(wants[b], cut[parents[b]]) for b in range(batch)]
    for b in range(batch):
        for c in range(kept[b] // page):
            p = int(table[parents[b], c])
            if there(p):
                new[b, c] = p
                refs[p] += 1
    copies, begin = [None] * batch, [0] * batch
    for b in range(batch):
        c = kept[b] // page
        begin[b] = c
        if kept[b] % page:
            p = int(table[parents[b], c])
            if not there(p):
                begin[b] = c + 1  # a part of no page stays one
            elif refs[p] == 0:
                refs[p] = 1
                new[b, c] = p
                begin[b] = c + 1
            else:
                copies[b] = p
    free = iter([p for p in range(pages) if refs[p] == 0])
    granted, src, dst = list(wants), [-1] * batch, [-1] * batch
    for b in range(batch):
        for c in range(begin[b], -(-wants[b] // page)):
            p = next(free, None)
            if p is None:
                granted[b] = min(granted[b], c * page)
                break
            new[b, c] = p
            refs[p] += 1
            if copies[b] is not None and c == begin[b]:
                src[b], dst[b] = copies[b], p
    return new, granted, src, dst, refs


def lora(x, a, b, adapters, base, scales=None, ranks=None):
    """(out, low, size): out before its rounding; what errors are measured by: low[t] the 2-norm-free sums
    sum_r sum_k |x a| |b| (a bound of the fp32 sums' terms) and size the largest |v| of the token times sum |b|."""
    x, base = np.asarray(x, dtype=np.float64), np.asarray(base, dtype=np.float64)
    out, terms, size = base.copy(), np.zeros_like(base), np.zeros_like(base)
    for t, i in enumerate(int(i) for i in adapters):
        if not 0 <= i < len(a):
            continue
        r = len(a[i]) if ranks is None else min(max(int(ranks[i]), 0), len(a[i]))
        s = 1.0 if scales is None else float(scales[i])
        ai, bi = np.asarray(a[i][:r], dtype=np.float64), np.asarray(b[i][:, :r], dtype=np.float64)
        v = ai @ x[t]
        out[t] += s * (bi @ v)
        terms[t] = abs(s) * (np.abs(bi) @ (np.abs(ai) @ np.abs(x[t])))
        size[t] = abs(s) * np.abs(v).max(initial=0.0) * np.abs(bi).sum(1)
    return out, terms, size
