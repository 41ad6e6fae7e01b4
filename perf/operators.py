"""The operators between a served model's projections, as cases that can be timed and compared.

- ``rotary``: rotary positions of queries and keys (``rotary_embedding``);
- ``write``: keys and values quantized to FP8 as they are written into a paged cache (``kv_cache_write_fp8``);
- ``rotary_write``: both in one pass (``rotary_kv_cache_write_fp8``);
- ``read``: a cached prefix read back (``kv_cache_read_fp8``);
- ``attend``: attention of decoded tokens, trees of drafted tokens or chunks of a prompt over that cache
  (``tree_attention_fp8``).

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
TINY, STEP = 1e-10, float(np.float32(1.0 / 448.0))


def listed():
    return [
        # the 64 rotary values of every head of a decode batch, the last of 192 in a query head and of 576 in a latent
        # row: the smallest call there is
        {"name": "rotary_decode", "op": "rotary", "t": 16, "hq": 128, "hk": 1, "d": 64, "rot": 64, "pad_q": 128,
         "pad_k": 512, "inter": True, "far": 32768, "dtype": "bf16"},
        # an odd number of prompt tokens, half of each head rotated, far positions
        {"name": "rotary_prefill", "op": "rotary", "t": 5003, "hq": 32, "hk": 8, "d": 128, "rot": 64, "pad_q": 0,
         "pad_k": 0, "inter": False, "far": 1048576, "dtype": "f16"},
        # one new token of each sequence of a decode batch
        {"name": "write_decode", "op": "write", "t": 64, "hk": 8, "d": 128, "page": 16, "dtype": "bf16"},
        # a ragged batch of prompts with wide heads
        {"name": "write_prefill", "op": "write", "t": 8191, "hk": 8, "d": 256, "page": 64, "dtype": "f16"},
        # a decode step's queries, keys and values
        {"name": "rotary_write_decode", "op": "rotary_write", "t": 8, "hq": 64, "hk": 8, "d": 128, "rot": 128,
         "inter": False, "far": 32768, "page": 16, "dtype": "bf16"},
        # a prompt's
        {"name": "rotary_write_prefill", "op": "rotary_write", "t": 8192, "hq": 32, "hk": 8, "d": 128, "rot": 128,
         "inter": True, "far": 131072, "page": 64, "dtype": "bf16"},
        # the short prefixes of a few sequences, narrow heads
        {"name": "read_short", "op": "read", "b": 3, "ctx": 700, "hk": 2, "d": 64, "page": 16, "dtype": "f16"},
        # the long prefixes of a batch whose prompts go on
        {"name": "read_long", "op": "read", "b": 16, "ctx": 16384, "hk": 8, "d": 128, "page": 64, "dtype": "bf16"},
        # the next token of one sequence: latency alone
        {"name": "attend_one", "op": "attend", "b": 1, "t": 1, "ctx": 2047, "hk": 8, "group": 4, "d": 128, "page": 16,
         "tree": False, "lse": False, "dtype": "bf16"},
        # the next token of every sequence of a batch, ragged contexts: a stream of the cache
        {"name": "attend_batch", "op": "attend", "b": 64, "t": 1, "ctx": 8192, "hk": 8, "group": 8, "d": 128,
         "page": 16, "tree": False, "lse": False, "dtype": "bf16"},
        # trees of up to 33 drafted tokens to verify, long ragged contexts
        {"name": "attend_tree", "op": "attend", "b": 16, "t": 33, "ctx": 16384, "hk": 8, "group": 4, "d": 128,
         "page": 64, "tree": True, "lse": True, "dtype": "bf16"},
        # a chunk of two long prompts after what is cached of them: matrix products
        {"name": "attend_chunk", "op": "attend", "b": 2, "t": 2048, "ctx": 8192, "hk": 8, "group": 4, "d": 128,
         "page": 64, "tree": False, "lse": False, "dtype": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        c = _drawn(rng)
        w = work(c)
        if w["bytes"] < 1.0e9 and w["flops"] < 2.5e11:
            return c


def _drawn(rng):
    op = rng.choice(["rotary", "write", "rotary_write", "read", "attend", "attend"])
    d = rng.choice([64, 128, 256])
    dtype = rng.choice(["bf16", "f16"])
    page = rng.choice([16, 32, 48, 64, 128])
    hk, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    if op == "rotary":
        return {"op": op, "t": _spread(rng, 1, 9000), "hq": hk * group, "hk": hk, "d": d, "rot": d // rng.choice([1, 2, 4]),
                "pad_q": rng.choice([0, 64, 128]), "pad_k": rng.choice([0, 128, 512]), "inter": rng.random() < 0.5,
                "far": _spread(rng, 64, 1 << 20), "dtype": rng.choice(["bf16", "f16", "f32"])}
    if op == "write":
        return {"op": op, "t": _spread(rng, 1, 9000), "hk": hk, "d": d, "page": page, "dtype": dtype}
    if op == "rotary_write":
        return {"op": op, "t": _spread(rng, 1, 9000), "hq": hk * group, "hk": hk, "d": d, "rot": d // rng.choice([1, 2]),
                "inter": rng.random() < 0.5, "far": _spread(rng, 64, 1 << 20), "page": page, "dtype": dtype}
    if op == "read":
        return {"op": op, "b": _spread(rng, 1, 64), "ctx": _spread(rng, 1, 20000), "hk": hk, "d": d, "page": page,
                "dtype": dtype}
    return {"op": op, "b": _spread(rng, 1, 64), "t": _spread(rng, 1, 64), "ctx": _spread(rng, 1, 32768), "hk": hk,
            "group": group, "d": d, "page": page, "tree": rng.random() < 0.6, "lse": rng.random() < 0.5, "dtype": dtype}


def _contexts(b, ctx):
    """Ragged cached lengths, the first the longest."""
    return [max(1, ctx * (64 - 29 * i % 57) // 64) for i in range(b)]


def _drafts(b, t):
    """Ragged numbers of drafted tokens, the first the most; chunks of a prompt and single tokens are alike."""
    return [max(1, t - 5 * i % (t // 2 + 1)) if t <= 64 else t for i in range(b)]


def work(c):
    n = SIZE[c["dtype"]]
    if c["op"] == "rotary":
        values = c["t"] * (c["hq"] + c["hk"]) * c["d"]
        return {"bytes": 2 * n * values + 8 * c["t"], "flops": 3 * c["t"] * (c["hq"] + c["hk"]) * c["rot"]}
    if c["op"] in ("write", "rotary_write"):
        heads = c["t"] * c["hk"]
        bytes_, flops = 2 * heads * (c["d"] * (n + 1) + 4) + 8 * c["t"], 6 * heads * c["d"]
        if c["op"] == "rotary_write":
            bytes_ += 2 * n * c["t"] * c["hq"] * c["d"] + 8 * c["t"]
            flops += 3 * c["t"] * (c["hq"] + c["hk"]) * c["rot"]
        return {"bytes": bytes_, "flops": flops}
    if c["op"] == "read":
        tokens = sum(_contexts(c["b"], c["ctx"]))
        return {"bytes": 2 * tokens * c["hk"] * (c["d"] * (n + 1) + 4), "flops": 2 * tokens * c["hk"] * c["d"]}
    ctx, drafts, hq = _contexts(c["b"], c["ctx"]), _drafts(c["b"], c["t"]), c["hk"] * c["group"]
    kept = sum(drafts) * hq * (2 * n * c["d"] + (4 if c["lse"] else 0))
    if c["tree"]:
        kept += sum(t * t for t in drafts)
    pairs = sum(t * x + (t * (t + 1) // 2 if not c["tree"] else t * t) for x, t in zip(ctx, drafts))
    return {"bytes": 2 * sum(x + t for x, t in zip(ctx, drafts)) * c["hk"] * (c["d"] + 4) + kept,
            "flops": 4 * pairs * hq * c["d"]}


def _normal(shape, dtype, g, outliers=0.0):
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)
    if outliers:
        x = torch.where(torch.rand(shape, generator=g, device=DEV) < outliers, 20 * x, x)
    return x.to(dtype)


def _frequencies(rot):
    """Angles a position turns each pair by, interpolated by parts to eight times the length they were trained on."""
    f = 10000.0 ** -(torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    turns = 4096 * f / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    return (f / 8 * (1 - keep) + f * keep).to(DEV), 0.1 * math.log(8) + 1


def _cache(pages, c):
    shape = (pages, c["hk"], c["page"])
    codes = [torch.zeros(shape + (c["d"],), dtype=E4M3, device=DEV) for _ in "kv"]
    return codes + [torch.zeros(shape, dtype=torch.float32, device=DEV) for _ in "kv"]


def _paged(lens, c, g, spare=3):
    """A cache that holds sequences of these lengths, its pages in any order, and their block table."""
    need = [-(-n // c["page"]) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros((len(lens), max(need)), dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    got = []
    for _ in "kv":
        x = _normal((pages, c["hk"], c["page"], c["d"]), torch.float32, g, 0.002)
        got.append(_quantized(x))
    (kc, ks), (vc, vs) = got
    return [kc, vc, ks, vs], table


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(v):
    return _i32([0] + np.cumsum(v).tolist())


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dtype = TYPE[c["dtype"]]
    s = {"case": c}
    if c["op"] in ("rotary", "rotary_write"):
        pq, pk = c.get("pad_q", 0), c.get("pad_k", 0)
        s["q"] = _normal((c["t"], c["hq"], pq + c["d"]), dtype, g)[..., pq:]
        s["k"] = _normal((c["t"], c["hk"], pk + c["d"]), dtype, g, 0.002)[..., pk:]
        s["positions"] = torch.randint(0, c["far"], (c["t"],), generator=g, device=DEV)
        s["frequencies"], s["magnitude"] = _frequencies(c["rot"])
    if c["op"] in ("write", "rotary_write"):
        if c["op"] == "write":
            s["k"] = _normal((c["t"], c["hk"], c["d"]), dtype, g, 0.002)
        s["v"] = _normal((c["t"], c["hk"], c["d"]), dtype, g, 0.002)
        pages = -(-c["t"] // c["page"]) + 3
        s["cache"] = _cache(pages, c)
        if c["t"] <= 64:  # decode: a place of its own for each sequence's token
            s["slots"] = torch.randperm(pages * c["page"], generator=g, device=DEV)[: c["t"]].contiguous()
        else:  # prompts: whole pages, in any order
            i = torch.arange(c["t"], device=DEV)
            order = torch.randperm(pages, generator=g, device=DEV)
            s["slots"] = order[i // c["page"]] * c["page"] + i % c["page"]
    if c["op"] == "read":
        lens = _contexts(c["b"], c["ctx"])
        s["cache"], s["table"] = _paged(lens, c, g)
        s["starts"], s["total"] = _starts(lens), sum(lens)
    if c["op"] == "attend":
        ctx, drafts = _contexts(c["b"], c["ctx"]), _drafts(c["b"], c["t"])
        s["cache"], s["table"] = _paged([x + t for x, t in zip(ctx, drafts)], c, g)
        s["lens"], s["starts"] = _i32([x + t for x, t in zip(ctx, drafts)]), _starts(drafts)
        s["q"] = _normal((sum(drafts), c["hk"] * c["group"], c["d"]), torch.float32, g).mul(2).to(dtype)
        s["mask"], s["most"], s["longest"] = None, max(drafts), max(x + t for x, t in zip(ctx, drafts))
        if c["tree"]:  # every draft sees itself and the drafts it follows
            pick = np.random.RandomState(int(seed) % (1 << 31))
            rows = []
            for t in drafts:
                m = np.zeros((t, max(drafts)), dtype=bool)
                for i in range(t):
                    if i:
                        parent = pick.randint(-1, i)
                        m[i] = m[parent] if parent >= 0 else False
                    m[i, i] = True
                rows.append(m)
            s["mask"] = torch.from_numpy(np.concatenate(rows)).to(DEV)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _rotated(x, positions, frequencies, magnitude, inter):
    """In 32 bits, the angles in 64."""
    angle = positions[:, None].double() * frequencies
    cos, sin = ((f * magnitude).float()[:, None, :] for f in (angle.cos(), angle.sin()))
    rot = 2 * frequencies.numel()
    x = x.float()
    if inter:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _quantized(x):
    scale = x.abs().amax(-1).clamp_min(TINY) * STEP
    return (x * (1 / scale)[..., None]).clamp(-448, 448).to(E4M3), scale


def _written(cache, slots, page, k, v):
    at, off = slots // page, slots % page
    for codes, scales, x in ((cache[0], cache[2], k), (cache[1], cache[3], v)):
        q, s = _quantized(x.float())
        codes.view(torch.uint8)[at, :, off] = q.view(torch.uint8)
        scales[at, :, off] = s
    return cache


def _plain_attention(s):
    c, (kc, vc, ks, vs) = s["case"], s["cache"]
    b, n, hk, d = c["b"], s["longest"], c["hk"], c["d"]
    k, v = ((codes[s["table"]].float() * scales[s["table"]][..., None]).transpose(1, 2).reshape(b, hk, -1, d)[:, :, :n]
            for codes, scales in ((kc, ks), (vc, vs)))
    rows = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(s["starts"][1:].long(), rows, right=True)
    draft = rows - s["starts"][seq]
    q = torch.zeros((b, s["most"]) + s["q"].shape[1:], device=DEV)
    q[seq, draft] = s["q"].float()
    q = q.view(b, s["most"], hk, c["group"], d).permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)
    first = s["lens"] - (s["starts"][1:] - s["starts"][:-1])
    j = torch.arange(n, device=DEV)[None, :] - first[:, None]  # which draft a position holds; negative: the context
    i = torch.arange(s["most"], device=DEV)
    if s["mask"] is None:
        seen = j[:, None, :] <= i[None, :, None]
    else:
        mask = torch.zeros((b, s["most"], s["most"]), dtype=torch.bool, device=DEV)
        mask[seq, draft] = s["mask"]
        seen = mask.gather(2, j.clamp(0, s["most"] - 1)[:, None, :].expand(b, s["most"], n)) | (j < 0)[:, None, :]
    seen = seen & (torch.arange(n, device=DEV) < s["lens"][:, None])[:, None, :]
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5).view(b, hk, s["most"], c["group"], n)
    score.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-1e30)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(b, hk, -1, n), v).view(b, hk, s["most"], c["group"], d) / total
    out = out.permute(0, 2, 1, 3, 4).reshape(b, s["most"], -1, d)[seq, draft].to(s["q"].dtype)
    if not c["lse"]:
        return out
    return out, (top + total.log()).squeeze(-1).permute(0, 2, 1, 3).reshape(b, s["most"], -1)[seq, draft]


def _plain(s):
    c = s["case"]
    if c["op"] == "rotary":
        return tuple(_rotated(s[x], s["positions"], s["frequencies"], s["magnitude"], c["inter"]).to(s[x].dtype) for x in "qk")
    if c["op"] == "write":
        return tuple(_written(s["cache"], s["slots"], c["page"], s["k"], s["v"]))
    if c["op"] == "rotary_write":
        q, k = (_rotated(s[x], s["positions"], s["frequencies"], s["magnitude"], c["inter"]) for x in "qk")
        return (q.to(s["q"].dtype),) + tuple(_written(s["cache"], s["slots"], c["page"], k, s["v"]))
    if c["op"] == "read":
        rows = torch.arange(s["total"], device=DEV)
        seq = torch.searchsorted(s["starts"][1:].long(), rows, right=True)
        at = rows - s["starts"][seq]
        page, off = s["table"][seq, at // c["page"]], at % c["page"]
        kc, vc, ks, vs = s["cache"]
        return tuple((codes.view(torch.uint8)[page, :, off].view(E4M3).float() * scales[page, :, off][..., None]).to(TYPE[c["dtype"]])
                     for codes, scales in ((kc, ks), (vc, vs)))
    return _plain_attention(s)


# ------------------------------------------------------------------------------------------------ the framework
def _framework(s):
    import aklr_amd as ops

    c = s["case"]
    if c["op"] == "rotary":
        return ops.rotary_embedding(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=c["inter"],
                                    magnitude=s["magnitude"])
    if c["op"] == "write":
        return ops.kv_cache_write_fp8(s["k"], s["v"], *s["cache"], s["slots"])
    if c["op"] == "rotary_write":
        q = ops.rotary_kv_cache_write_fp8(s["q"], s["k"], s["v"], s["positions"], s["frequencies"], *s["cache"],
                                          s["slots"], interleaved=c["inter"], magnitude=s["magnitude"])
        return (q,) + tuple(s["cache"])
    if c["op"] == "read":
        return ops.kv_cache_read_fp8(*s["cache"], s["table"], s["starts"], s["total"], out_dtype=TYPE[c["dtype"]])
    return ops.tree_attention_fp8(s["q"], *s["cache"], s["table"], s["lens"], s["starts"], s["mask"],
                                  return_lse=c["lse"])


def run(s):
    return _framework(s) if own else _plain(s)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _turn64(s, x):
    """Each pair as a complex number, times the unit number of its angle."""
    f = s["frequencies"].cpu().numpy()
    turn = np.exp(1j * np.outer(s["positions"].cpu().numpy().astype(np.float64), f)) * s["magnitude"]
    x = x.double().cpu().numpy().copy()
    r = 2 * len(f)
    lo, hi = (slice(0, r, 2), slice(1, r, 2)) if s["case"]["inter"] else (slice(0, r // 2), slice(r // 2, r))
    z = (x[..., lo] + 1j * x[..., hi]) * turn[:, None, :]
    x[..., lo], x[..., hi] = z.real, z.imag
    return x


def _store64(s, k, v):
    """Codes before their rounding, and scales; what no slot names stays zero."""
    got = []
    at = np.divmod(s["slots"].cpu().numpy(), s["case"]["page"])
    for like, x in ((s["cache"][0], k), (s["cache"][1], v)):
        scale = np.maximum(np.abs(x).max(-1), TINY) / 448
        codes, scales = np.zeros(tuple(like.shape)), np.zeros(tuple(like.shape[:3]))
        codes[at[0], :, at[1]], scales[at[0], :, at[1]] = x / scale[..., None], scale
        got.append((codes, scales))
    return got[0][0], got[1][0], got[0][1], got[1][1]


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "rotary":
        return _turn64(s, s["q"]), _turn64(s, s["k"])
    if c["op"] == "write":
        return _store64(s, s["k"].double().cpu().numpy(), s["v"].double().cpu().numpy())
    if c["op"] == "rotary_write":
        return (_turn64(s, s["q"]),) + _store64(s, _turn64(s, s["k"]), s["v"].double().cpu().numpy())
    kc, vc, ks, vs = s["cache"]
    starts = s["starts"].tolist()
    lens = s["lens"].tolist() if c["op"] == "attend" else np.diff(starts).tolist()
    outs, ends = [], []
    for i, n in enumerate(lens):
        pages = s["table"][i, : -(-n // c["page"])].long()
        k, v = ((codes.view(torch.uint8)[pages].view(E4M3).double() * scales[pages].double().unsqueeze(-1)).permute(0, 2, 1, 3)
                .reshape(-1, c["hk"], c["d"])[:n] for codes, scales in ((kc, ks), (vc, vs)))
        if c["op"] == "read":
            outs.append(k)
            ends.append(v)
            continue
        t = starts[i + 1] - starts[i]
        q = s["q"][starts[i]:starts[i + 1]].double()
        sees = torch.ones((t, n), dtype=torch.bool, device=DEV)
        sees[:, n - t:] = torch.ones((t, t), device=DEV).tril().bool() if s["mask"] is None else s["mask"][starts[i]:starts[i + 1], :t]
        out, end = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float64, device=DEV)
        for h in range(q.shape[1]):
            score = (q[:, h] @ k[:, h // c["group"]].t()) / math.sqrt(c["d"])
            score = torch.where(sees, score, -math.inf)
            end[:, h] = torch.logsumexp(score, -1)
            out[:, h] = torch.exp(score - end[:, h, None]) @ v[:, h // c["group"]]
        outs.append(out)
        ends.append(end)
    first, second = torch.cat(outs), torch.cat(ends)
    return (first, second) if c["op"] == "read" or c["lse"] else first
