"""What differs from request to request in a batch that a served model shares, as cases that can be timed and compared.

- ``verify``: which of the drafted tokens stand, and the token that follows them (``verify_drafts``);
- ``compact``: kept positions of a paged FP8 cache moved together (``kv_cache_compact_fp8``);
- ``copy``: pages of that cache copied (``kv_cache_copy_pages_fp8``);
- ``update``: the batch's pages forked, freed and grown (``kv_cache_update_pages``);
- ``lora``: each token's low-rank adapter beside a projection that all share (``lora_project``).

The cache: e4m3 codes [pages, kv heads, page, head] and one fp32 scale for each token and head [pages, kv heads,
page]; pages lie in any order. With ``own`` false each operator is computed in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn
TYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # four sequences, four drafted tokens each, a small vocabulary: latency alone
        {"name": "verify_few", "op": "verify", "b": 4, "t": 5, "vocab": 32000, "form": "chain", "dtype": "f32"},
        # a batch's chains of drafts and a large vocabulary
        {"name": "verify_chains", "op": "verify", "b": 64, "t": 8, "vocab": 131072, "form": "chain", "dtype": "f32"},
        # trees of up to 33 drafted tokens, several for the same place
        {"name": "verify_trees", "op": "verify", "b": 16, "t": 33, "vocab": 128003, "form": "tree", "dtype": "f32"},
        # the accepted path of each of a batch's trees, behind its context
        {"name": "compact_paths", "op": "compact", "b": 64, "t": 33, "ctx": 1024, "keep": 5, "hk": 8, "d": 128, "page": 16},
        # long contexts cut to their first and last positions
        {"name": "compact_contexts", "op": "compact", "b": 8, "t": 16384, "ctx": 0, "keep": 4095, "hk": 8, "d": 128,
         "page": 64},
        # the last pages of a few forked sequences
        {"name": "copy_forks", "op": "copy", "n": 8, "hk": 8, "d": 128, "page": 16},
        # prefixes copied whole
        {"name": "copy_prefixes", "op": "copy", "n": 1024, "hk": 8, "d": 128, "page": 64},
        # a decode step of a batch: most sequences grow, a few end
        {"name": "update_step", "op": "update", "b": 64, "ctx": 8190, "page": 16, "family": 1, "forks": False, "scarce": False},
        # beams of long shared prompts choose their parents
        {"name": "update_beams", "op": "update", "b": 512, "ctx": 32749, "page": 64, "family": 8, "forks": True, "scarce": False},
        # one token of each of a few requests, every one with its own adapter
        {"name": "lora_decode", "op": "lora", "t": 8, "run": 1, "adapters": 8, "rank": 16, "k": 7168, "n": 2112, "dtype": "bf16"},
        # a decode batch of several drafted tokens a request, adapters of several ranks
        {"name": "lora_batch", "op": "lora", "t": 192, "run": 3, "adapters": 48, "rank": 64, "k": 8192, "n": 10240, "dtype": "bf16"},
        # ragged prompts
        {"name": "lora_prompts", "op": "lora", "t": 8191, "run": 1365, "adapters": 8, "rank": 32, "k": 8192, "n": 10240, "dtype": "f16"},
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = [work(c) for c in listed()]
    most = max(w["bytes"] for w in most), max(w["flops"] for w in most)
    while True:
        c = _drawn(rng)
        w = work(c)
        if w["bytes"] > most[0] or w["flops"] > most[1]:
            continue
        if c["op"] != "verify" or sum(_drafts(c["b"], c["t"])) * c["vocab"] <= 528 * 131072:
            return c


def _drawn(rng):
    op = rng.choice(["verify", "verify", "compact", "copy", "update", "lora", "lora"])
    cache = {"hk": rng.choice([1, 2, 4, 8]), "d": rng.choice([64, 128, 256]), "page": rng.choice([16, 32, 48, 64, 128])}
    if op == "verify":
        return {"op": op, "b": _spread(rng, 1, 64), "t": _spread(rng, 1, 64), "vocab": _spread(rng, 100, 160000),
                "form": rng.choice(["chain", "tree", "sure"]), "dtype": rng.choice(["f32", "f32", "bf16", "f16"])}
    if op == "compact":
        t = _spread(rng, 1, 8192)
        return {"op": op, "b": _spread(rng, 1, 64 if t <= 64 else 8), "t": t, "ctx": _spread(rng, 1, 2048),
                "keep": _spread(rng, 1, 8192) % ((t + 1) // 2 + 1), **cache}
    if op == "copy":
        return {"op": op, "n": _spread(rng, 1, 1024), **cache}
    if op == "update":
        return {"op": op, "b": _spread(rng, 1, 512), "ctx": _spread(rng, 16, 32768), "page": cache["page"],
                "family": rng.choice([1, 2, 4, 8]), "forks": rng.random() < 0.5, "scarce": rng.random() < 0.25}
    t = _spread(rng, 1, 8192)
    return {"op": op, "t": t, "run": rng.choice([1, 1, 2, 5, 33, 700]), "adapters": _spread(rng, 1, 48 if t <= 256 else 8),
            "rank": rng.choice([8, 16, 24, 32, 64, 128]), "k": 8 * _spread(rng, 32, 1024), "n": 8 * _spread(rng, 32, 1280),
            "dtype": rng.choice(["bf16", "f16"])}


def _drafts(b, t):
    """Ragged numbers of query tokens, the first the most: the last token that stands, then the drafted ones."""
    return [max(1, t - 5 * i % (t // 2 + 1)) if t <= 64 else max(1, t * (64 - 29 * i % 37) // 64) for i in range(b)]


def _contexts(b, ctx):
    """Ragged lengths, the first the longest."""
    return [max(1, ctx * (64 - 29 * i % 57) // 64) for i in range(b)] if ctx else [0] * b


def _kept(c):
    """How many positions of each sequence stay."""
    return [min(t, 1 + c["keep"] * (4 - i % 4) // 4) for i, t in enumerate(_drafts(c["b"], c["t"]))]


def _ranks(c):
    """Adapters' ranks: the largest, half of it, a quarter."""
    return [max(8, (c["rank"] >> i % 3) // 8 * 8) for i in range(c["adapters"])]


def _requests(c):
    """The adapter of each token: runs of one request's; every eleventh request has none. The runs go round the adapters."""
    run = (np.arange(c["t"]) // c["run"]).astype(np.int64)
    return np.where(run % 11 == 10, -1, run % c["adapters"])


def work(c):
    if c["op"] == "verify":
        n, rows = SIZE[c["dtype"]], 1 if c["form"] == "sure" else 2
        return {"bytes": c["b"] * (rows * c["vocab"] * n + 8 * c["t"]) + sum(_drafts(c["b"], c["t"])) * (2 * n + 16),
                "flops": c["b"] * c["vocab"] * (4 if rows == 2 else 1)}
    if c["op"] in ("compact", "copy"):
        if c["op"] == "copy":
            moved = c["n"] * c["page"]
        else:  # what is kept in its place does not move: the first sixty-fourth of long contexts, the first token of paths
            moved = sum(k - _still(k, t) for k, t in zip(_kept(c), _drafts(c["b"], c["t"])))
        return {"bytes": 4 * moved * c["hk"] * (c["d"] + 4) + 16 * c.get("b", 0) + 8 * c.get("n", 0), "flops": 0}
    if c["op"] == "update":
        return {"bytes": 8 * c["b"] * (-(-c["ctx"] // c["page"]) + 2) + 24 * c["b"], "flops": 0}
    who, ranks = _requests(c), np.array(_ranks(c))
    used = ranks[np.unique(who[who >= 0])].sum()
    return {"bytes": 2 * int(used) * (c["k"] + c["n"]) + 2 * c["t"] * (c["k"] + 2 * c["n"]) + 4 * c["t"],
            "flops": 2 * int(ranks[who[who >= 0]].sum()) * (c["k"] + c["n"])}


def _still(kept, t):
    """How many of the kept positions lie where they were; the others come from behind the kept ones' new places."""
    return kept if kept == t else max(1, kept // 64 if t > 64 else 1)


def _starts(v):
    return torch.tensor([0] + np.cumsum(v).tolist(), dtype=torch.int32, device=DEV)


def _i32(v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device=DEV)


def _cache(pages, c, g):
    """Codes of finite values and their scales."""
    got = [torch.randint(0, 254, (pages, c["hk"], c["page"], c["d"]), generator=g, device=DEV, dtype=torch.int16) for _ in "kv"]
    codes = [(x + (x >= 127)).to(torch.uint8).view(E4M3) for x in got]  # 127 and 255 are no numbers
    return codes + [torch.rand((pages, c["hk"], c["page"]), generator=g, device=DEV) + 0.01 for _ in "kv"]


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    pick = np.random.RandomState(int(seed) % (1 << 31))
    s = {"case": c}
    if c["op"] == "verify":
        _prepare_verify(s, c, g, pick)
    elif c["op"] == "compact":
        lens, drafts, kept = _contexts(c["b"], c["ctx"]), _drafts(c["b"], c["t"]), _kept(c)
        need = [-(-(x + t) // c["page"]) for x, t in zip(lens, drafts)]
        pages, at = pick.permutation(sum(need) + 3).astype(np.int32), 0
        table, path = np.zeros((c["b"], max(need)), dtype=np.int32), np.full((c["b"], max(kept)), -1, dtype=np.int32)
        for i, n in enumerate(need):
            table[i, :n] = pages[at:at + n]
            at += n
            k, t = kept[i], drafts[i]
            still = _still(k, t)
            rest = k - still
            path[i, :still] = np.arange(still)
            if t > 64:  # the last ones
                path[i, still:k] = np.arange(t - rest, t)
            else:  # a path down a tree whose levels are wide
                room = np.arange(min(max(k, still), t - rest), t)
                path[i, still:k] = np.sort(pick.choice(room, rest, replace=False))
        s["cache"] = _cache(len(pages), c, g)
        s["table"], s["lens"], s["starts"] = _i32(table), _i32([x + t for x, t in zip(lens, drafts)]), _starts(drafts)
        s["path"], s["counts"] = _i32(path), _i32(kept)
    elif c["op"] == "copy":
        order = torch.randperm(2 * c["n"] + 3, generator=g, device=DEV).to(torch.int32)
        s["cache"] = _cache(2 * c["n"] + 3, c, g)
        # some pages go to several places, as a prompt's that is forked
        s["src"] = order[torch.randint(0, c["n"] + 3, (c["n"],), generator=g, device=DEV)].contiguous()
        s["dst"] = order[c["n"] + 3:].contiguous()
    elif c["op"] == "update":
        _prepare_update(s, c, pick)
    else:
        dtype, ranks = TYPE[c["dtype"]], _ranks(c)
        names = pick.permutation(c["adapters"])  # which adapter a request has
        who, mine = _requests(c), np.zeros(c["adapters"], dtype=np.int32)
        mine[names] = ranks
        s["x"] = torch.randn((c["t"], c["k"]), generator=g, device=DEV).to(dtype)
        s["base"] = torch.randn((c["t"], c["n"]), generator=g, device=DEV).to(dtype)
        r = torch.arange(c["rank"], device=DEV)
        s["ranks"] = _i32(mine)
        there = r[None, :] < s["ranks"][:, None]
        s["a"] = (torch.randn((c["adapters"], c["rank"], c["k"]), generator=g, device=DEV) * c["k"] ** -0.5 * there[..., None]).to(dtype)
        s["b"] = (torch.randn((c["adapters"], c["n"], c["rank"]), generator=g, device=DEV) * c["rank"] ** -0.5 * there[:, None]).to(dtype)
        s["who"] = _i32(np.where(who < 0, -1, names[who]))
        s["scales"] = torch.rand(c["adapters"], generator=g, device=DEV) + 0.5
    return s


def _prepare_verify(s, c, g, pick):
    """A target's probabilities and a smaller model's near them; drafts drawn from the latter, or its likeliest ("sure")."""
    drafts = _drafts(c["b"], c["t"])
    s["starts"], s["most"] = _starts(drafts), max(drafts)
    first = np.repeat(np.cumsum([0] + drafts[:-1]), drafts)
    i = np.concatenate([np.arange(t) for t in drafts])
    parent = i - 1 if c["form"] == "chain" else np.where(i > 0, (pick.randint(0, 1 << 20, len(i)) % np.maximum(np.minimum(i, 5), 1)), 0)
    if c["form"] != "chain":  # one of the five before it
        parent = i - 1 - parent
    row = torch.from_numpy(np.where(i > 0, first + parent, first)).to(DEV)
    logits = 5 * torch.randn((len(i), c["vocab"]), generator=g, device=DEV)
    s["target"] = torch.softmax(logits, -1).to(TYPE[c["dtype"]])
    logits += 0.7 * torch.randn(logits.shape, generator=g, device=DEV)
    if c["form"] == "sure":
        seen, rank = {}, []
        for key in (first + parent).tolist():
            rank.append(seen.get(key, 0))
            seen[key] = rank[-1] + 1
        k = min(max(rank) + 1, c["vocab"])
        rank = torch.tensor(rank, device=DEV).clamp_max(k - 1)
        s["tokens"] = logits.topk(k, -1).indices[row, rank].contiguous()
        s["draft"] = None
    else:
        s["draft"] = torch.softmax(logits, -1).to(TYPE[c["dtype"]])
        noise = torch.rand(logits.shape, generator=g, device=DEV).clamp_min_(1e-30).log_().neg_().log_()
        s["tokens"] = (logits[row] - noise).argmax(-1)
    s["parents"] = None if c["form"] == "chain" else _i32(parent)
    s["u"] = torch.rand(len(i), generator=g, device=DEV)
    s["v"] = torch.rand(c["b"], generator=g, device=DEV)


def _prepare_update(s, c, pick):
    """Families of sequences that share their first pages; a prefix cache of the server's holds some pages too."""
    b, page, cols = c["b"], c["page"], -(-c["ctx"] // c["page"]) + 2
    lens = np.array(_contexts(b, c["ctx"]))
    pages = b * cols + 16
    free = iter(pick.permutation(pages).tolist())
    table, refs = np.full((b, cols), -1, dtype=np.int32), np.zeros(pages, dtype=np.int32)
    for i in range(b):
        head = i - i % c["family"]
        shared = int(min(lens[head], lens[i])) * 3 // 4 // page if i > head else 0
        table[i, :shared] = table[head, :shared]
        own_pages = range(shared, -(-int(lens[i]) // page))
        table[i, own_pages.start:own_pages.stop] = [next(free) for _ in own_pages]
    np.add.at(refs, table[table >= 0], 1)
    held = pick.permutation(np.flatnonzero(refs))
    refs[held[: len(held) // 10]] += 1
    if c["scarce"]:  # hardly a page left
        left = np.flatnonzero(refs == 0)
        refs[left[: max(0, len(left) - b // 4)]] = 1
    parents = np.arange(b)
    if c["forks"]:
        parents = parents - parents % c["family"] + pick.randint(0, c["family"], b)
        parents = np.where(pick.rand(b) < 1 / 32, -1, np.minimum(parents, b - 1))
    grown = np.where(parents >= 0, lens[parents], 0) + (1 if c["forks"] else pick.randint(-5, 9, b)) + 2 * page * c["scarce"]
    s["new"] = _i32(np.where(pick.rand(b) < 1 / 16, 0, np.maximum(grown, 0)))
    s["refs"], s["table"], s["lens"] = _i32(refs), _i32(table), _i32(lens)
    s["parents"] = _i32(parents) if c["forks"] else None


# ------------------------------------------------------------------------------------------------ plain forms
def _clean(x):
    x = x.double()
    return torch.where((x > 0) & (x < math.inf), x, 0.0)


def _plain_verify(s):
    """In 64 bits: which token is drawn hangs on sums of a whole row."""
    b, most, starts = s["case"]["b"], s["most"], s["starts"].long()
    n, i = starts[1:] - starts[:-1], torch.arange(most, device=DEV)
    at = (starts[:-1, None] + i).clamp_max(s["tokens"].numel() - 1)
    x, u = s["tokens"][at], s["u"].double()[at]
    rows = torch.arange(b, device=DEV)
    if s["parents"] is None:
        before = at[:, :-1]
        p, q = _clean(s["target"][before, x[:, 1:]]), _clean(s["draft"][before, x[:, 1:]])
        ok = (u[:, 1:] * q < p) & (i[1:] < n[:, None])
        path = torch.cat((torch.zeros((b, 1), dtype=torch.long, device=DEV), torch.where(ok.long().cumprod(1) > 0, i[1:], -1)), 1)
        count = (path >= 0).sum(1)
        last = starts[:-1] + count - 1
        refused = (count < n).double()[:, None]
        weight = (_clean(s["target"][last]) - refused * _clean(s["draft"][last])).clamp_min(0)
    else:
        parent = s["parents"].long()[at]
        cur, count = torch.zeros(b, dtype=torch.long, device=DEV), torch.ones(b, dtype=torch.long, device=DEV)
        path = torch.full((b, most + 1), -1, dtype=torch.long, device=DEV)
        path[:, 0] = 0
        scale, total = torch.zeros(b, dtype=torch.float64, device=DEV), torch.ones(b, dtype=torch.float64, device=DEV)
        gone = torch.zeros(s["target"].shape[1], dtype=torch.float64, device=DEV).repeat(b, 1)
        for j in range(1, most):  # drafts in their order: one that stands is where the search goes on
            tried = (parent[:, j] == cur) & (j < n)
            row = starts[:-1] + cur
            p, token = _clean(s["target"][row, x[:, j]]), x[:, j, None]
            if s["draft"] is not None:
                q = _clean(s["draft"][row, x[:, j]])
                w = (p - scale * q).clamp_min(0)
            else:
                q, w = torch.ones_like(p), p * (1 - gone.gather(1, token)[:, 0])
            ok, no = tried & (u[:, j] * total * q < w), tried & ~(u[:, j] * total * q < w)
            if s["draft"] is not None:
                scale = torch.where(no, scale + total, scale)
                left = (_clean(s["target"][row]) - scale[:, None] * _clean(s["draft"][row])).clamp_min(0).sum(1)
            else:
                left = total - w
                gone.scatter_(1, token, torch.where(no[:, None], 1.0, gone.gather(1, token)))
            total = torch.where(no, left, total)
            total, scale = torch.where(ok, 1.0, total), torch.where(ok, 0.0, scale)
            gone = gone * (~ok)[:, None]
            path.scatter_(1, torch.where(ok, count, most)[:, None], j)
            cur, count = torch.where(ok, j, cur), count + ok
        path = path[:, :most].where(i < count[:, None], -1)
        weight = _clean(s["target"][starts[:-1] + cur])
        if s["draft"] is not None:
            weight = (weight - scale[:, None] * _clean(s["draft"][starts[:-1] + cur])).clamp_min(0)
        else:
            weight = weight * (1 - gone)
        last = starts[:-1] + cur
    weight = torch.where((weight.sum(1) == 0)[:, None], _clean(s["target"][last]), weight)
    sums = weight.cumsum(1)
    new = torch.searchsorted(sums, (s["v"].double() * sums[:, -1])[:, None], right=True)[:, 0].clamp_max(sums.shape[1] - 1)
    out = torch.where(i[1:] < count[:, None], x.gather(1, path[:, 1:].clamp_min(0)), -1)
    out = torch.cat((out, torch.full_like(path[:, :1], -1)), 1)
    out[rows, count - 1] = torch.where(sums[:, -1] > 0, new, -1)
    return out, path.int(), count.int()


def _plain_compact(s):
    page, path = s["case"]["page"], s["path"].long()
    first = (s["lens"] - (s["starts"][1:] - s["starts"][:-1])).long()[:, None]
    i = torch.arange(path.shape[1], device=DEV)
    there = i < s["counts"][:, None]
    src, dst = first + torch.where(there, path, 0), first + torch.where(there, i, 0)  # the rest: the first onto itself
    table = s["table"].long()
    (a, ao), (b, bo) = ((table.gather(1, x // page), x % page) for x in (src, dst))
    for t in s["cache"]:
        t = t.view(torch.uint8) if t.dtype == E4M3 else t
        t[b, :, bo] = t[a, :, ao]
    return tuple(s["cache"])


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for t in s["cache"]:
        t = t.view(torch.uint8) if t.dtype == E4M3 else t
        t[dst] = t[src]
    return tuple(s["cache"])


def _plain_update(s):
    page, refs, table = s["case"]["page"], s["refs"].clone(), s["table"].long()
    (b, cols), pages = table.shape, refs.numel()
    row, col = torch.arange(b, device=DEV), torch.arange(cols, device=DEV)
    parent = row if s["parents"] is None else s["parents"].long()
    lens = s["lens"].long().clamp(0, cols * page)
    refs = torch.cat((refs, refs.new_zeros(cols)))  # what names no page counts behind them

    def count(at, mask, one):
        at = torch.where(mask & (at >= 0), at, pages + col)
        refs.scatter_add_(0, at.view(-1), refs.new_full((1,), one).expand(at.numel()))

    count(table, col < (-(-lens // page))[:, None], -1)
    theirs = table[parent.clamp_min(0)]
    want = s["new"].long().clamp(0, cols * page)
    kept = torch.minimum(want, lens[parent.clamp_min(0)]) * (parent >= 0)
    full, part = kept // page, kept % page > 0
    keep = col < full[:, None]
    count(theirs, keep, 1)
    new = torch.where(keep, theirs, -1)
    # the page a sequence keeps a part of: its own if nobody else holds it, and the first one's that keeps such a part
    at = theirs.gather(1, full.clamp_max(cols - 1)[:, None])[:, 0].clamp_min(0)
    alone = part & (refs[at] == 0)
    first = torch.full((pages,), b, device=DEV).scatter_reduce(0, at, torch.where(alone, row, b), "amin")
    takes = alone & (first[at] == row)
    count(at[:, None].expand(b, cols), (col == 0) & takes[:, None], 1)
    copies = part & ~takes
    new = torch.where((col == full[:, None]) & takes[:, None], at[:, None], new)
    begin = full + takes
    need = (-(-want // page) - begin).clamp_min(0)
    before = need.cumsum(0) - need
    free = refs[:pages] == 0
    order = torch.where(free, free.cumsum(0) - 1, pages)
    listed_ = torch.full((pages + 1,), -1, device=DEV).scatter(0, order, torch.arange(pages, device=DEV))
    asked = (col >= begin[:, None]) & (col < (begin + need)[:, None])
    which = before[:, None] + col - begin[:, None]
    got = torch.where(asked & (which < pages), listed_[which.clamp(0, pages)], -1)
    new = torch.where(asked, got, new)
    count(got, asked, 1)
    missing = torch.where(asked & (got < 0), col, cols).amin(1)
    granted = torch.minimum(want, missing * page)
    dst = torch.where(copies, new.gather(1, full.clamp_max(cols - 1)[:, None])[:, 0], -1)
    return new.int(), granted.int(), torch.where(dst >= 0, at, -1).int(), dst.int(), refs[:pages]


def _plain_lora(s):
    """All adapters at once, each token's own picked out of the products between."""
    n, r, k = s["a"].shape
    mine = (torch.arange(n, device=DEV) == s["who"][:, None]) * s["scales"]
    low = (s["x"].float() @ s["a"].float().view(n * r, k).t()).view(-1, n, r) * mine[..., None]
    up = s["b"].float().transpose(1, 2).reshape(n * r, -1)
    return (s["base"].float() + low.view(-1, n * r) @ up).to(s["base"].dtype)


_PLAIN = {"verify": _plain_verify, "compact": _plain_compact, "copy": _plain_copy, "update": _plain_update, "lora": _plain_lora}


# ------------------------------------------------------------------------------------------------ the framework
def _framework(s):
    import aklr_amd as ops

    op = s["case"]["op"]
    if op == "verify":
        return ops.verify_drafts(s["target"], s["tokens"], s["starts"], s["u"], s["v"], s["most"], draft_probs=s["draft"],
                                 parents=s["parents"])
    if op == "compact":
        return ops.kv_cache_compact_fp8(*s["cache"], s["table"], s["lens"], s["starts"], s["path"], s["counts"])
    if op == "copy":
        return ops.kv_cache_copy_pages_fp8(*s["cache"], s["src"], s["dst"])
    if op == "update":
        refs = s["refs"].clone()
        return ops.kv_cache_update_pages(refs, s["table"], s["lens"], s["new"], s["case"]["page"], s["parents"]) + (refs,)
    return ops.lora_project(s["x"], s["a"], s["b"], s["who"], s["base"], scales=s["scales"], ranks=s["ranks"])


def run(s):
    return _framework(s) if own else _PLAIN[s["case"]["op"]](s)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _proper(x):
    x = x.double().cpu().numpy()
    return np.where(np.isfinite(x) & (x > 0), x, 0.0)


def _exact_verify(s):
    """One sequence after the other, down its tree."""
    b, most, starts = s["case"]["b"], s["most"], s["starts"].tolist()
    out, path, count = np.full((b, most), -1), np.full((b, most), -1), np.zeros(b, dtype=np.int64)
    tokens, u = s["tokens"].tolist(), s["u"].double().tolist()
    for i in range(b):
        lo, t = starts[i], starts[i + 1] - starts[i]
        parent = [-1] + (list(range(t - 1)) if s["parents"] is None else s["parents"][lo + 1:lo + t].tolist())
        node, steps = 0, [0]
        while True:
            p = _proper(s["target"][lo + node])
            q = _proper(s["draft"][lo + node]) if s["draft"] is not None else None
            rest, mass, found = p.copy(), 1.0, None
            for j in range(node + 1, t):
                if parent[j] != node:
                    continue
                x = tokens[lo + j]
                if u[lo + j] * mass * (q[x] if q is not None else 1.0) < rest[x]:
                    found = j
                    break
                if q is not None:
                    rest = np.maximum(rest - mass * q, 0)
                    mass = rest.sum()
                else:
                    mass -= rest[x]
                    rest[x] = 0
            if found is None:
                break
            node = found
            steps.append(node)
        rest = rest if rest.sum() > 0 else p
        level = float(s["v"][i]) * rest.sum()
        ends = np.cumsum(rest)
        last = int(np.argmax(ends > level)) if ends[-1] > level else -1
        count[i] = len(steps)
        path[i, : len(steps)] = steps
        out[i, : len(steps)] = [tokens[lo + j] for j in steps[1:]] + [last]
    return out, path.astype(np.int32), count.astype(np.int32)


def _exact_compact(s):
    page, table, starts = s["case"]["page"], s["table"].cpu().numpy(), s["starts"].cpu().numpy()
    lens, path, counts = (s[x].cpu().numpy() for x in ("lens", "path", "counts"))
    outs = []
    for t in s["cache"]:
        old = t.double().cpu().numpy()
        new = old.copy()
        for i, n in enumerate(counts):
            first = lens[i] - (starts[i + 1] - starts[i])
            a, b = first + path[i, :n], first + np.arange(n)
            new[table[i, b // page], :, b % page] = old[table[i, a // page], :, a % page]
        outs.append(new)
    return tuple(outs)


def _exact_copy(s):
    outs = [t.double().cpu().numpy() for t in s["cache"]]
    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
        for t in outs:
            t[b] = t[a]
    return tuple(outs)


def _exact_update(s):
    """Sequence after sequence: all let go of what they held, take what they keep, then new pages in order."""
    page, refs, old = s["case"]["page"], s["refs"].tolist(), s["table"].tolist()
    lens, wants = s["lens"].tolist(), s["new"].tolist()
    b, cols = len(old), len(old[0])
    parents = list(range(b)) if s["parents"] is None else s["parents"].tolist()
    for i in range(b):
        for p in old[i][: -(-lens[i] // page)]:
            refs[p] -= 1
    new = [[-1] * cols for _ in range(b)]
    keeps = [min(wants[i], cols * page, lens[parents[i]]) if parents[i] >= 0 else 0 for i in range(b)]
    for i in range(b):
        for j in range(keeps[i] // page):
            new[i][j] = old[parents[i]][j]
            refs[new[i][j]] += 1
    src, dst, claimed, copy = [-1] * b, [-1] * b, set(), [False] * b
    for i in range(b):
        if keeps[i] % page:
            p = old[parents[i]][keeps[i] // page]
            if refs[p] == 0:
                claimed.add(p)
                refs[p] = 1
                new[i][keeps[i] // page] = p
            else:
                copy[i] = True
    free, granted = [p for p in range(len(refs)) if refs[p] == 0][::-1], []
    for i in range(b):
        want = min(wants[i], cols * page)
        for j in range(-(-want // page)):
            if new[i][j] >= 0:
                continue
            if not free:
                want = min(want, j * page)
                break
            new[i][j] = free.pop()
            refs[new[i][j]] = 1
            if copy[i] and j == keeps[i] // page:
                src[i], dst[i] = old[parents[i]][j], new[i][j]
        granted.append(want)
    return tuple(np.array(x, dtype=np.int32) for x in (new, granted, src, dst, refs))


def _exact_lora(s):
    out = s["base"].double()
    for j in range(s["a"].shape[0]):
        rows = torch.nonzero(s["who"] == j)[:, 0]
        low = torch.mm(s["x"][rows].double(), s["a"][j].double().t().contiguous())
        out[rows] += s["scales"][j].double() * torch.mm(low, s["b"][j].double().t().contiguous())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"verify": _exact_verify, "compact": _exact_compact, "copy": _exact_copy, "update": _exact_update,
            "lora": _exact_lora}[s["case"]["op"]](s)
