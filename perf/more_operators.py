"""Attention of prompts, scores that are capped or lean on distance, and a cache of 4-bit keys and values: what a
decoding program calls, its inputs, one pass of each, and the 64-bit answer.

A case is a dict of plain values. Its "kind" names the operator:

  prompt   prompt_attention: the new tokens of every sequence over its pages, masked by position
  shaped   paged_attention with a cap or slopes: one new token of every sequence
  store    PackedPages.append and .read: keys and values into 4-bit pages, and what these then stand for
  packed   PackedPages.attend: one new token of every sequence over its 4-bit pages

`own` says whose operators run: elementary torch operations in 32 bits (False), or this package's (True).
"""

import math
import random

import torch

own = False

DEV = "cuda"
_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_GROUP = 64  # elements that share a scale and an offset
_MOST = 65504.0  # float16's largest


def listed():
    """The cases that are timed and compared by name."""
    return [
        # a short question of one user: bound by the call
        dict(name="prompt-bf16-short", kind="prompt", dtype="bfloat16", sequences=1, new=77, past=0, kv=8, heads=32,
             dim=128, vdim=128, page=64, window=0, prefix=0, cap=0.0, slopes=False, heads_first=False, ragged=1),
        # one long prompt, all of it new
        dict(name="prompt-bf16-8k", kind="prompt", dtype="bfloat16", sequences=1, new=8_192, past=0, kv=8, heads=32,
             dim=128, vdim=128, page=64, window=0, prefix=0, cap=0.0, slopes=False, heads_first=False, ragged=2),
        # the next 512 tokens of a document behind 65,536 that the cache holds, capped scores
        dict(name="prompt-bf16-chunk", kind="prompt", dtype="bfloat16", sequences=1, new=512, past=65_536, kv=8,
             heads=32, dim=128, vdim=128, page=64, window=0, prefix=0, cap=50.0, slopes=False, heads_first=True,
             ragged=3),
        # prompts of seven users of different lengths in one call, a head for every query head, a bias by distance
        dict(name="prompt-f16-slopes", kind="prompt", dtype="float16", sequences=7, new=2_000, past=300, kv=16,
             heads=16, dim=64, vdim=64, page=16, window=0, prefix=0, cap=0.0, slopes=True, heads_first=False, ragged=4),
        # single precision, odd sizes, a prefix that is read in both directions
        dict(name="prompt-f32-prefix", kind="prompt", dtype="float32", sequences=3, new=1_001, past=0, kv=4, heads=12,
             dim=80, vdim=72, page=24, window=0, prefix=300, cap=0.0, slopes=False, heads_first=False, ragged=5),
        # a server's step with capped scores: 64 sequences of very different lengths
        dict(name="shaped-bf16-cap", kind="shaped", dtype="bfloat16", sequences=64, kv=8, heads=32, dim=128, vdim=128,
             page=64, longest=8_192, window=0, cap=50.0, slopes=False, heads_first=False, ragged=6),
        # a few sequences whose scores lean on distance
        dict(name="shaped-f16-slopes", kind="shaped", dtype="float16", sequences=3, kv=4, heads=32, dim=64, vdim=64,
             page=16, longest=3_001, window=0, cap=0.0, slopes=True, heads_first=False, ragged=7),
        # one decoding step: a token of each of 64 sequences
        dict(name="store-bf16-step", kind="store", dtype="bfloat16", sequences=64, new=1, kv=8, dim=128, vdim=128,
             page=64, longest=1_000, ragged=8),
        # the prompts of seven sequences of different lengths in one call, small pages
        dict(name="store-f16-prompt", kind="store", dtype="float16", sequences=7, new=5_000, kv=8, dim=64, vdim=64,
             page=16, longest=6_000, ragged=9),
        # a short chat of one user: bound by the call
        dict(name="packed-bf16-short", kind="packed", dtype="bfloat16", sequences=1, kv=8, heads=32, dim=128, vdim=128,
             page=64, longest=77, window=0, cap=0.0, slopes=False, ragged=10),
        # a server's step: 64 sequences of very different lengths
        dict(name="packed-bf16-64seq", kind="packed", dtype="bfloat16", sequences=64, kv=8, heads=32, dim=128, vdim=128,
             page=64, longest=8_192, window=0, cap=0.0, slopes=False, ragged=11),
        # one sequence as long as the key cache of the benchmark, single precision queries
        dict(name="packed-f32-131k", kind="packed", dtype="float32", sequences=1, kv=8, heads=32, dim=128, vdim=128,
             page=64, longest=131_072, window=0, cap=0.0, slopes=False, ragged=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    return kv, kv * rng.choice([1, 2, 3, 4, 4, 6, 8, 16])


def _dim(rng):
    return rng.choice([64, 128, 128, 256, rng.randrange(8, 257, 8), rng.randrange(33, 250)])


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    while True:
        kind = rng.choice(["prompt", "prompt", "shaped", "store", "packed", "packed"])
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        kv, heads = _heads(rng)
        dim = _dim(rng)
        vdim = dim if rng.random() < 0.7 else _dim(rng)
        page = rng.choice([16, 32, 64, 64, 128, 8 * rng.randrange(1, 20)])
        case = dict(kind=kind, dtype=dtype, kv=kv, dim=dim, vdim=vdim, page=page, ragged=rng.randrange(1 << 20))
        if kind != "store":
            case.update(heads=heads, window=rng.choice([0, 0, 0, _log(rng, 16, 5_000)]),
                        cap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.3)
        if kind in ("prompt", "shaped"):
            case["heads_first"] = rng.random() < 0.5
        if kind == "shaped" and not case["cap"]:
            case["slopes"] = True
        if kind == "prompt":
            case.update(sequences=_log(rng, 1, 32), new=_log(rng, 1, 8_000), past=rng.choice([0, _log(rng, 1, 60_000)]))
            case["prefix"] = rng.choice([0, 0, _log(rng, 1, case["new"])])
            b, n, most = case["sequences"], case["new"], case["new"] + case["past"]
            fits = b * heads * n * most <= 800_000_000 and b * kv * most * (dim + vdim) <= 300_000_000
        elif kind == "store":
            case.update(sequences=_log(rng, 1, 128), new=rng.choice([1, 1, _log(rng, 1, 4_000)]),
                        longest=_log(rng, 16, 30_000))
            held = case["sequences"] * (case["longest"] + case["new"] + page) * kv * (dim + vdim)
            fits = held <= 200_000_000 and case["sequences"] * case["new"] * kv * (dim + vdim) <= 50_000_000
        else:
            case.update(sequences=_log(rng, 1, 128), longest=_log(rng, 1, 131_072))
            fits = case["sequences"] * case["longest"] * kv * (dim + vdim) <= 300_000_000
        if fits and _most(work(case)):
            return case


def _most(w):
    return w["bytes"] <= 9e8 and w["flops"] <= 3e11


def _lengths(case):
    """Positions of every sequence in the cache: `longest` for the first, log-uniform below it for the
    others, and from four sequences on an empty one. Of the case, not of the seed."""
    rng = random.Random(case["ragged"])
    b, top = case["sequences"], case["longest"]
    lens = [top] + [_log(rng, max(1, top // 8), top) for _ in range(b - 1)]
    if b >= 4:
        lens[b // 2] = 0
    return lens


def _news(case):
    """New tokens of every sequence: one each, or prompts of different lengths up to `new`."""
    rng = random.Random(case["ragged"] + 1)
    return [case["new"]] + [_log(rng, max(1, case["new"] // 4), case["new"]) for _ in range(case["sequences"] - 1)]


def _pasts(case):
    """What every sequence of prompts has in the cache already, and from four sequences on one that has nothing."""
    rng = random.Random(case["ragged"] + 2)
    b, top = case["sequences"], case["past"]
    return [top] + [_log(rng, 1, top) if top and 4 * s != b else 0 for s in range(1, b)]


def _seen(case):
    return [min(n, case["window"]) if case["window"] else n for n in _lengths(case)]


def _pairs(case):
    """Pairs of a query and a position that it sees, over all sequences, and the positions that any query sees."""
    pairs, seen = 0, 0
    for n, past in zip(_news(case), _pasts(case)):
        w, x = case["window"] or 1 << 40, min(case["prefix"], past + n)
        for p in range(past, past + n):
            pairs += max(p + 1, x) - max(0, p + 1 - w)
        seen += past + n - max(0, past + 1 - w)
    return pairs, seen


def _row_bytes(case):
    """Bytes of a packed position of one head: half a byte an element, four a group."""
    return sum((d + 1) // 2 + 4 * -(-d // _GROUP) for d in (case["dim"], case["vdim"]))


def work(case):
    """Bytes and operations that one pass cannot do without."""
    e, kv, width = _TYPES[case["dtype"]].itemsize, case["kv"], case["dim"] + case["vdim"]
    if case["kind"] == "prompt":
        (pairs, seen), t = _pairs(case), sum(_news(case))
        return {"bytes": seen * kv * width * e + t * case["heads"] * width * e, "flops": 2 * pairs * case["heads"] * width}
    if case["kind"] == "store":
        t = sum(_news(case))  # read, packed, the packed read again, and written
        return {"bytes": 2 * t * kv * (width * e + _row_bytes(case)) + 8 * t, "flops": 6 * t * kv * width}
    seen, rows = sum(_seen(case)), case["sequences"] * case["heads"]
    one = width * e if case["kind"] == "shaped" else _row_bytes(case)
    return {"bytes": seen * kv * one + rows * width * e, "flops": 2 * seen * case["heads"] * width}


# ---- inputs ----


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, shape, dtype, loud=0, scale=1.0):
    """Normal values, `loud` channels of them four times as large (as projections' outputs have them)."""
    x = torch.empty(shape, dtype=dtype, device=DEV)
    for part in x.split(max(1, (1 << 28) // max(1, x[0].numel()))) if x.numel() else ():
        y = torch.randn(part.shape, generator=g, device=DEV) * scale
        if loud:
            y[..., :: max(1, shape[-1] // loud)] *= 4.0
        part.copy_(y)
    return x


def _pool(g, pages, case, dim, loud):
    """A pool of pages, (pages, slots, heads, dim) as a view of either order of slots and heads."""
    s, h = case["page"], case["kv"]
    if case.get("heads_first"):
        return _randn(g, (pages, h, s, dim), _TYPES[case["dtype"]], loud).transpose(1, 2)
    return _randn(g, (pages, s, h, dim), _TYPES[case["dtype"]], loud)


def _table(g, lens, page):
    """Page table (sequences, most pages) int32 over a shuffled pool, -1 past a sequence's pages."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(max(1, sum(need)), generator=g, device=DEV).to(torch.int32).tolist()
    rows, at = [], 0
    for n in need:
        rows.append(order[at : at + n] + [-1] * (max(max(need), 1) - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device=DEV), max(1, sum(need))


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _inputs(case, seed):
    g = _gen(seed)
    dtype, b = _TYPES[case["dtype"]], case["sequences"]
    x = {}
    if case.get("slopes"):  # a geometric series, the steepest first
        x["slopes"] = 2.0 ** (-8.0 * torch.arange(1, case["heads"] + 1, device=DEV) / case["heads"])
    # trained queries make scores that a cap has something to do with
    loudness = 4.0 if case.get("cap") else 1.0
    if case["kind"] == "prompt":
        news, pasts = _news(case), _pasts(case)
        lens = [a + n for a, n in zip(pasts, news)]
        x["table"], pages = _table(g, lens, case["page"])
        x["k_pages"], x["v_pages"] = _pool(g, pages, case, case["dim"], 4), _pool(g, pages, case, case["vdim"], 0)
        x["q"] = _randn(g, (sum(news), case["heads"], case["dim"]), dtype, scale=loudness)
        x["lengths"], x["first"] = _ints(lens), _ints([sum(news[:s]) for s in range(b + 1)])
        if case["prefix"]:
            x["prefix"] = _ints([min(case["prefix"], n) for n in lens])
    elif case["kind"] == "shaped":
        lens = _lengths(case)
        x["table"], pages = _table(g, lens, case["page"])
        x["k_pages"], x["v_pages"] = _pool(g, pages, case, case["dim"], 4), _pool(g, pages, case, case["vdim"], 0)
        x["q"] = _randn(g, (b, case["heads"], case["dim"]), dtype, scale=loudness)
        x["lengths"] = _ints(lens)
    elif case["kind"] == "store":
        news, lens = _news(case), _lengths(case)
        x["table"], x["pages"] = _table(g, [a + n for a, n in zip(lens, news)], case["page"])
        x["k"] = _randn(g, (sum(news), case["kv"], case["dim"]), dtype, 4)
        x["v"] = _randn(g, (sum(news), case["kv"], case["vdim"]), dtype)
        x["positions"] = _ints([a + i for a, n in zip(lens, news) for i in range(n)])
        x["sequences"] = _ints([s for s, n in enumerate(news) for _ in range(n)])
    else:
        lens = _lengths(case)
        x["table"], x["pages"] = _table(g, lens, case["page"])
        # what fills the cache: every slot of every page, in the order of the pool
        x["k"] = _randn(g, (x["pages"] * case["page"], case["kv"], case["dim"]), dtype, 4)
        x["v"] = _randn(g, (x["pages"] * case["page"], case["kv"], case["vdim"]), dtype)
        x["q"] = _randn(g, (b, case["heads"], case["dim"]), dtype, scale=loudness)
        x["lengths"] = _ints(lens)
    return x


def _pack(x):
    """Elements (..., dim) as 4-bit codes, two a byte, and a float16 scale and offset for every 64 of them."""
    d = x.shape[-1]
    groups = -(-d // _GROUP)
    f = x.float()
    f = torch.cat([f, f[..., -1:].expand(*f.shape[:-1], groups * _GROUP - d)], -1).unflatten(-1, (groups, _GROUP))
    low = f.amin(-1).clamp(-_MOST, _MOST).half()
    step = ((f.amax(-1) - low.float()) / 15).clamp(0, _MOST).half()
    # 64 bits: which of two codes is nearer is to be the same whatever computes it
    code = ((f.double() - low.double()[..., None]) / step.double()[..., None]).round().clamp(0, 15)
    code = torch.where(step[..., None] > 0, code, 0.0).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, step, low


def _unpack(packed, step, low, dim):
    """The values in 32 bits."""
    code = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).float()
    return (low.float()[..., None] + step.float()[..., None] * code).flatten(-2)[..., :dim]


def prepare(case, seed):
    """Inputs on the GPU, and the cache that a program keeps: 4-bit pages of the package, or codes, scales and offsets."""
    state = dict(case=case, **_inputs(case, seed))
    if case["kind"] == "store":
        if own:
            import libcertex_amd as certex

            state["cache"] = certex.PackedPages(state["pages"], case["page"], case["kv"], case["dim"], case["vdim"])
        else:
            state["cache"] = []
            for d in (case["dim"], case["vdim"]):
                shape = (state["pages"], case["page"], case["kv"], -(-d // _GROUP))
                state["cache"].append([torch.zeros(shape + (_GROUP // 2,), dtype=torch.uint8, device=DEV),
                                       *[torch.zeros(shape, dtype=torch.float16, device=DEV) for _ in range(2)]])
    elif case["kind"] == "packed":
        k, v, page = state.pop("k"), state.pop("v"), case["page"]
        if own:
            import libcertex_amd as certex

            state["cache"] = certex.PackedPages(state["pages"], page, case["kv"], case["dim"], case["vdim"])
            where = torch.arange(state["pages"], dtype=torch.int32, device=DEV)[:, None]
            slots = torch.arange(k.shape[0], dtype=torch.int32, device=DEV)
            state["cache"].append(k, v, where, slots % page, sequences=slots // page)
        else:
            state["cache"] = [[t.unflatten(0, (-1, page)) for t in _pack(x)] for x in (k, v)]
    return state


# ---- one pass ----


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    import libcertex_amd as certex

    case = s["case"]
    if case["kind"] == "store":
        s["cache"].append(s["k"], s["v"], s["table"], s["positions"], sequences=s["sequences"])
        return list(s["cache"].read(s["table"], s["positions"], sequences=s["sequences"], dtype=s["k"].dtype))
    shape = dict(window=case["window"] or None, cap=case["cap"] or None, slopes=s.get("slopes"))
    if case["kind"] == "prompt":
        return [certex.prompt_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["first"],
                                        prefix=s.get("prefix"), **shape)]
    if case["kind"] == "shaped":
        return [certex.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], **shape)]
    return [s["cache"].attend(s["q"], s["table"], s["lengths"], **shape)]


def _plain(s):
    case = s["case"]
    if case["kind"] == "store":
        p, n = s["positions"].long(), s["k"].shape[0]
        page, slot = s["table"][s["sequences"].long(), p // case["page"]].long(), p % case["page"]
        out = []
        for x, cache in zip((s["k"], s["v"]), s["cache"]):
            for held, new in zip(cache, _pack(x)):
                held[page, slot] = new.view(n, case["kv"], *held.shape[3:])
            out.append(_unpack(*[held[page, slot] for held in cache], x.shape[-1]).to(x.dtype))
        return out
    # pages of every sequence, one after the other: (b, positions, kv, dim) in 32 bits
    at = s["table"].long().clamp(min=0)
    if case["kind"] == "packed":
        keys, values = (_unpack(*[t[at].flatten(1, 2) for t in cache], d)
                        for cache, d in zip(s["cache"], (case["dim"], case["vdim"])))
    else:
        keys, values = (s[name][at].flatten(1, 2).float() for name in ("k_pages", "v_pages"))
    b, kv, d = case["sequences"], case["kv"], case["dim"]
    g, length = case["heads"] // kv, s["lengths"].long()
    if case["kind"] == "prompt":
        # the queries of every sequence, padded to the longest
        news = s["first"].long().diff()
        most = case["new"]
        i = torch.arange(most, device=DEV)
        row, real = (s["first"].long()[:-1, None] + i).clamp(max=s["q"].shape[0] - 1), i < news[:, None]
        q, p = s["q"][row], (length - news)[:, None] + i
    else:
        most, q, p = 1, s["q"][:, None], length[:, None] - 1
    # (b, kv, queries x group, d) and (b, kv, d, positions)
    q = q.float().view(b, most, kv, g, d).permute(0, 2, 1, 3, 4).reshape(b, kv, most * g, d)
    scores = (q @ keys.permute(0, 2, 3, 1).contiguous()).view(b, kv, most, g, -1)
    del keys
    scores *= d**-0.5
    if case["cap"]:
        scores = case["cap"] * torch.tanh(scores / case["cap"])
    t, p = torch.arange(scores.shape[-1], device=DEV), p[..., None]
    if case["slopes"]:
        scores -= s["slopes"].view(1, kv, 1, g, 1) * (p - t).abs().float()[:, None, :, None]
    seen = t <= p
    if case.get("prefix"):
        seen |= t < s["prefix"].long()[:, None, None]
    seen &= t < length[:, None, None]
    if case["window"]:
        seen &= t > p - case["window"]
    scores = scores.masked_fill_(~seen[:, None, :, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores -= torch.where(top.isinf(), 0.0, top)
    w = scores.exp_()
    total = w.sum(-1, keepdim=True)
    w /= torch.where(total == 0, 1.0, total)
    out = w.view(b, kv, most * g, -1) @ values.permute(0, 2, 1, 3).contiguous()
    out = out.view(b, kv, most, g, -1).permute(0, 2, 1, 3, 4).reshape(b, most, case["heads"], -1).to(s["q"].dtype)
    return [out[real] if case["kind"] == "prompt" else out[:, 0]]


# ---- the definition in 64 bits ----


def _stored(x):
    """What 4-bit pages hold of x (rows, heads, dim), element for element, in 64 bits."""
    out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    for at in range(0, x.shape[-1], _GROUP):
        part = x[..., at : at + _GROUP].double()
        offset = part.min(-1, keepdim=True).values.clamp(-_MOST, _MOST).to(torch.float16)
        # a scale is the float16 of a float32 quotient: that is the format, not a rounding of this computation
        span = part.max(-1, keepdim=True).values.float() - offset.float()
        scale = (span / 15.0).clamp(0.0, _MOST).to(torch.float16).double()
        offset = offset.double()
        steps = torch.where(scale > 0, (part - offset) / torch.where(scale > 0, scale, 1.0), 0.0)
        out[..., at : at + _GROUP] = offset + scale * torch.clamp(torch.round(steps), 0, 15)
    return out


def _rows_attended(case, x, q, positions, length, prefix, keys, values):
    """Queries (n, heads, dim) at `positions` over keys and values (length, kv, .) of one sequence, in 64 bits."""
    heads, g = case["heads"], case["heads"] // case["kv"]
    out = torch.zeros((q.shape[0], heads, values.shape[-1]), dtype=torch.float64, device=DEV)
    t = torch.arange(length, device=DEV)
    for h in range(heads):
        k, v = keys[:, h // g].double(), values[:, h // g].double()
        for part in torch.arange(q.shape[0], device=DEV).split(max(1, (1 << 26) // max(1, length))):
            p = positions[part][:, None]
            s = q[part, h].double() @ k.T / case["dim"] ** 0.5
            if case["cap"]:
                s = case["cap"] * torch.tanh(s / case["cap"])
            if case["slopes"]:
                s = s - x["slopes"][h].double() * (p - t).abs()
            hidden = (t > p) & (t >= prefix)
            if case["window"]:
                hidden |= p - t >= case["window"]
            s = s.masked_fill(hidden, float("-inf"))
            out[part, h] = torch.nan_to_num(torch.softmax(s, -1)) @ v
    return out


def exact(case, seed):
    """What run returns, from the operators' definitions in 64 bits."""
    x = _inputs(case, seed)
    if case["kind"] == "store":
        return [_stored(x["k"]), _stored(x["v"])]
    if case["kind"] == "packed":
        k_pages, v_pages = (x[name].unflatten(0, (-1, case["page"])) for name in ("k", "v"))
    else:
        k_pages, v_pages = x["k_pages"], x["v_pages"]
    out = []
    for b, n in enumerate(x["lengths"].tolist()):
        if case["kind"] == "prompt":
            lo, hi = x["first"][b : b + 2].tolist()
        else:
            lo, hi = b, b + 1
        if n == 0:
            out.append(torch.zeros((hi - lo, case["heads"], case["vdim"]), dtype=torch.float64, device=DEV))
            continue
        at = torch.arange(n, device=DEV)
        page, slot = x["table"][b].long()[at // case["page"]], at % case["page"]
        keys, values = k_pages[page, slot], v_pages[page, slot]
        if case["kind"] == "packed":
            keys, values = _stored(keys), _stored(values)
        prefix = int(x["prefix"][b]) if "prefix" in x else 0
        out.append(_rows_attended(case, x, x["q"][lo:hi], torch.arange(n - (hi - lo), n, device=DEV), n, prefix, keys,
                                  values))
    return [torch.cat(out)]
