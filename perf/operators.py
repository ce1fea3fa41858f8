"""The attention operators next to the key cache: what a decoding program calls, its inputs, one pass
of each, and the 64-bit answer.

A case is a dict of plain values. Its "kind" names the operator:

  rotate   Rotary: queries or keys rotated by their positions, in training with the gradient
  append   append_pages: new keys and values into a paged cache, the rotation on the way
  attend   paged_attention: one new token of every sequence over its pages
  select   selected_attention: softmax over the top k that a KeyCache returned, and their values

`own` says whose operators run: elementary torch operations in 32 bits (False), or this package's (True).
"""

import math
import random

import torch

own = False

DEV = "cuda"
_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_BASE = 10000.0


def listed():
    """The cases that are timed and compared by name."""
    return [
        # the queries of one decoding step of 64 sequences, at positions up to the cache's length
        dict(name="rotate-bf16-step", kind="rotate", dtype="bfloat16", tokens=64, heads=32, dim=128, rotary=128,
             layout="half", longest=131_072, train=False),
        # all keys of a long cache, before they go to a KeyCache
        dict(name="rotate-bf16-keys", kind="rotate", dtype="bfloat16", tokens=131_072, heads=8, dim=128, rotary=128,
             layout="half", longest=131_072, train=False),
        # a training step of a model that rotates part of each head, an odd number of tokens
        dict(name="rotate-f32-train", kind="rotate", dtype="float32", tokens=4_099, heads=20, dim=80, rotary=32,
             layout="interleaved", longest=4_099, train=True),
        # one decoding step: a token of each of 64 sequences, its queries rotated in the same call
        dict(name="append-bf16-step", kind="append", dtype="bfloat16", sequences=64, new=1, kv=8, heads=32, dim=128,
             vdim=128, rotary=128, layout="half", page=64, longest=1_000, heads_first=False, ragged=1),
        # 256 more keys of one long sequence
        dict(name="append-bf16-grow", kind="append", dtype="bfloat16", sequences=1, new=256, kv=8, heads=0, dim=128,
             vdim=128, rotary=128, layout="half", page=64, longest=131_072, heads_first=True, ragged=2),
        # the prompts of seven sequences of different lengths in one call, small pages
        dict(name="append-f16-prompt", kind="append", dtype="float16", sequences=7, new=5_000, kv=8, heads=32, dim=64,
             vdim=64, rotary=64, layout="interleaved", page=16, longest=6_000, heads_first=False, ragged=3),
        # a short chat of one user: bound by the call
        dict(name="attend-bf16-short", kind="attend", dtype="bfloat16", sequences=1, kv=8, heads=32, dim=128, vdim=128,
             page=64, longest=77, window=0, heads_first=False, ragged=4),
        # a server's step: 64 sequences of very different lengths
        dict(name="attend-bf16-64seq", kind="attend", dtype="bfloat16", sequences=64, kv=8, heads=32, dim=128,
             vdim=128, page=64, longest=8_192, window=0, heads_first=False, ragged=5),
        # one sequence as long as the key cache of the benchmark: split over its length
        dict(name="attend-bf16-131k", kind="attend", dtype="bfloat16", sequences=1, kv=8, heads=32, dim=128, vdim=128,
             page=64, longest=131_072, window=0, heads_first=True, ragged=6),
        # a head for every query head, single precision, dimensions and pages off the usual ones
        dict(name="attend-f32-mha", kind="attend", dtype="float32", sequences=5, kv=16, heads=16, dim=80, vdim=72,
             page=24, longest=5_001, window=0, heads_first=False, ragged=7),
        # sparse attention of one new token: 2,048 keys of each query head's 131,072
        dict(name="select-bf16-1q", kind="select", dtype="bfloat16", kv=8, heads=32, queries=1, k=2_048, n=131_072,
             vdim=128, page=64),
        # the benchmark's key cache: 64 queries a head
        dict(name="select-bf16-64q", kind="select", dtype="bfloat16", kv=8, heads=32, queries=64, k=2_048, n=131_072,
             vdim=128, page=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    return kv, kv * rng.choice([1, 2, 3, 4, 4, 6, 8, 16])


def _dim(rng):
    return rng.choice([64, 128, 128, 256, rng.randrange(8, 257, 8), rng.randrange(34, 250, 2)])


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    while True:
        kind = rng.choice(["rotate", "append", "attend", "attend", "select"])
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        layout = rng.choice(["half", "interleaved"])
        kv, heads = _heads(rng)
        dim = _dim(rng)
        rotary = dim if rng.random() < 0.6 else 2 * rng.randrange(1, dim // 2 + 1)
        vdim = dim if rng.random() < 0.7 else _dim(rng)
        page = rng.choice([16, 32, 64, 64, 128, 8 * rng.randrange(1, 20)])
        if kind == "rotate":
            case = dict(kind=kind, dtype=dtype, tokens=_log(rng, 1, 100_000), heads=heads, dim=dim, rotary=rotary,
                        layout=layout, longest=_log(rng, 1_000, 1_000_000), train=rng.random() < 0.3)
            size = case["tokens"] * heads * dim * (2 if case["train"] else 1)
            fits = size <= 100_000_000
        elif kind == "append":
            case = dict(kind=kind, dtype=dtype, sequences=_log(rng, 1, 128), new=rng.choice([1, 1, _log(rng, 1, 4_000)]),
                        kv=kv, heads=rng.choice([0, heads]), dim=dim, vdim=vdim, rotary=rotary, layout=layout,
                        page=page, longest=_log(rng, 16, 30_000), heads_first=rng.random() < 0.5,
                        ragged=rng.randrange(1 << 20))
            pool = case["sequences"] * (case["longest"] + case["new"] + page) * kv * (dim + vdim)
            fits = pool <= 200_000_000 and case["sequences"] * case["new"] * (kv * (dim + vdim) + heads * dim) <= 50_000_000
        elif kind == "attend":
            case = dict(kind=kind, dtype=dtype, sequences=_log(rng, 1, 128), kv=kv, heads=heads, dim=dim, vdim=vdim,
                        page=page, longest=_log(rng, 1, 131_072),
                        window=rng.choice([0, 0, 0, _log(rng, 16, 5_000)]), heads_first=rng.random() < 0.5,
                        ragged=rng.randrange(1 << 20))
            fits = case["sequences"] * case["longest"] * kv * (dim + vdim) <= 400_000_000
        else:
            n = _log(rng, 64, 131_072)
            case = dict(kind=kind, dtype=dtype, kv=kv, heads=heads, queries=_log(rng, 1, 64),
                        k=min(n, 2_048, _log(rng, 8, 4_000)), n=n, vdim=vdim, page=rng.choice([0, page]))
            rows = heads * case["queries"]
            fits = rows * case["k"] * vdim <= 400_000_000 and rows * n <= 200_000_000 and kv * n * vdim <= 130_000_000
        if fits and _most(work(case)):
            return case


def _most(w):
    return w["bytes"] <= 9e8 and w["flops"] <= 4e9


def _lengths(case, spare=0):
    """Tokens of every sequence in the cache: `longest` for the first, log-uniform below it for the
    others, and from four sequences on an empty one. Of the case, not of the seed."""
    rng = random.Random(case["ragged"])
    b, top = case["sequences"], case["longest"]
    lens = [top] + [_log(rng, max(1, top // 8), top) for _ in range(b - 1)]
    if b >= 4:
        lens[b // 2] = 0
    return [n + spare for n in lens]


def _news(case):
    """New tokens of every sequence: one each, or prompts of different lengths up to `new`."""
    rng = random.Random(case["ragged"] + 1)
    return [case["new"]] + [_log(rng, max(1, case["new"] // 4), case["new"]) for _ in range(case["sequences"] - 1)]


def _seen(case):
    return [min(n, case["window"]) if case["window"] else n for n in _lengths(case)]


def work(case):
    """Bytes and operations that one pass cannot do without."""
    e = _TYPES[case["dtype"]].itemsize
    if case["kind"] == "rotate":
        t, width = case["tokens"], case["heads"] * case["dim"]
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * t * width * e + 8 * t, "flops": passes * 3 * t * case["heads"] * case["rotary"]}
    if case["kind"] == "append":
        t = sum(_news(case))
        width = case["kv"] * (case["dim"] + case["vdim"]) + case["heads"] * case["dim"]
        return {"bytes": 2 * t * width * e + 12 * t, "flops": 3 * t * (case["kv"] + case["heads"]) * case["rotary"]}
    if case["kind"] == "attend":
        seen, b = sum(_seen(case)), case["sequences"]
        width = case["dim"] + case["vdim"]
        return {"bytes": seen * case["kv"] * width * e + b * case["heads"] * width * e,
                "flops": 2 * seen * case["heads"] * width}
    n, rows = case["n"], case["heads"] * case["queries"]
    # rows of values that at least one of a head's queries selects
    touched = n * (1.0 - (1.0 - case["k"] / n) ** (rows // case["kv"]))
    return {"bytes": int(12 * rows * case["k"] + case["kv"] * touched * case["vdim"] * e + rows * case["vdim"] * e),
            "flops": 2 * rows * case["k"] * case["vdim"]}


# ---- inputs ----


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, shape, dtype, loud=0):
    """Normal values, `loud` channels of them four times as large (as projections' outputs have them)."""
    x = torch.empty(shape, dtype=dtype, device=DEV)
    for part in x.split(max(1, (1 << 28) // max(1, x[0].numel()))) if x.numel() else ():
        y = torch.randn(part.shape, generator=g, device=DEV)
        if loud:
            y[..., :: max(1, shape[-1] // loud)] *= 4.0
        part.copy_(y)
    return x


def _pool(g, pages, case, dim, loud):
    """A pool of pages, (pages, slots, heads, dim) as a view of either order of slots and heads."""
    s, h = case["page"], case["kv"]
    if case["heads_first"]:
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


def _inputs(case, seed):
    g = _gen(seed)
    dtype = _TYPES[case["dtype"]]
    if case["kind"] == "rotate":
        t, h, d = case["tokens"], case["heads"], case["dim"]
        x = dict(x=_randn(g, (t, h, d), dtype, 4),
                 positions=torch.randint(0, case["longest"], (t,), generator=g, device=DEV))
        if case["train"]:
            x["dy"] = _randn(g, (t, h, d), dtype)
        return x
    if case["kind"] == "append":
        news = _news(case)
        t = sum(news)
        first = _lengths(case)
        table, pages = _table(g, [a + b for a, b in zip(first, news)], case["page"])
        x = dict(k=_randn(g, (t, case["kv"], case["dim"]), dtype, 4), v=_randn(g, (t, case["kv"], case["vdim"]), dtype),
                 k_pages=_pool(g, pages, case, case["dim"], 4), v_pages=_pool(g, pages, case, case["vdim"], 0),
                 table=table, q=None,
                 positions=torch.tensor([a + i for a, b in zip(first, news) for i in range(b)], dtype=torch.int32,
                                        device=DEV),
                 sequences=torch.tensor([s for s, b in enumerate(news) for _ in range(b)], dtype=torch.int32,
                                        device=DEV))
        if case["heads"]:
            x["q"] = _randn(g, (t, case["heads"], case["dim"]), dtype, 4)
        return x
    if case["kind"] == "attend":
        lens = _lengths(case)
        table, pages = _table(g, lens, case["page"])
        return dict(q=_randn(g, (case["sequences"], case["heads"], case["dim"]), dtype),
                    k_pages=_pool(g, pages, case, case["dim"], 4), v_pages=_pool(g, pages, case, case["vdim"], 0),
                    table=table, lengths=torch.tensor(lens, dtype=torch.int32, device=DEV))
    n, m, k = case["n"], case["queries"], case["k"]
    scores, ids = [], []
    for _ in range(case["heads"]):  # products of N(0, 1) vectors of 128 coordinates, the k best of n
        s, i = torch.topk(torch.randn((m, n), generator=g, device=DEV) * 128**0.5, k, dim=-1)
        scores.append(s)
        ids.append(i)
    x = dict(scores=torch.stack(scores), ids=torch.stack(ids), table=None)
    if case["page"]:
        pages = -(-n // case["page"])
        x["table"] = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        x["values"] = _randn(g, (pages, case["page"], case["kv"], case["vdim"]), dtype)
    else:
        x["values"] = _randn(g, (case["kv"], n, case["vdim"]), dtype)
    return x


def _freqs(case):
    r = case["rotary"]
    return _BASE ** (-torch.arange(0, r, 2, dtype=torch.float64, device=DEV) / r)


def prepare(case, seed):
    """Inputs on the GPU, and the rotation that a program keeps: a Rotary, or tables of cosines and sines."""
    state = dict(case=case, **_inputs(case, seed))
    if "rotary" in case:
        if own:
            import libcertex_amd as certex

            state["rope"] = certex.Rotary(case["dim"], rotary_dim=case["rotary"], base=_BASE, layout=case["layout"])
        else:
            most = int(state["positions"].max()) + 1
            angle = torch.arange(most, dtype=torch.float64, device=DEV)[:, None] * _freqs(case)
            state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    return state


# ---- one pass ----


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    import libcertex_amd as certex

    case = s["case"]
    if case["kind"] == "rotate":
        if not case["train"]:
            return [s["rope"](s["x"], s["positions"])]
        x = s["x"].detach().requires_grad_()
        y = s["rope"](x, s["positions"])
        return [y.detach(), torch.autograd.grad(y, x, s["dy"])[0]]
    if case["kind"] == "append":
        q = certex.append_pages(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["positions"],
                                sequences=s["sequences"], rotary=s["rope"], q=s["q"])
        return [s["k_pages"], s["v_pages"]] + ([] if q is None else [q])
    if case["kind"] == "attend":
        return [certex.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"],
                                       window=case["window"] or None)]
    return [certex.selected_attention(s["scores"], s["ids"], s["values"], 128**-0.5, page_table=s["table"])]


def _turn(x, cos, sin, case):
    """Rotation in 32 bits: cos and sin are (tokens, 1, rotary / 2)."""
    r = case["rotary"]
    f = x[..., :r].float()
    if case["layout"] == "half":
        a, b = f[..., : r // 2], f[..., r // 2 :]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = f[..., 0::2], f[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([y.to(x.dtype), x[..., r:]], -1)


def _plain(s):
    case = s["case"]
    if case["kind"] in ("rotate", "append"):
        p = s["positions"].long()
        cos, sin = s["cos"][p][:, None], s["sin"][p][:, None]
    if case["kind"] == "rotate":
        y = _turn(s["x"], cos, sin, case)
        return [y, _turn(s["dy"], cos, -sin, case)] if case["train"] else [y]
    if case["kind"] == "append":
        page = s["table"][s["sequences"].long(), p // case["page"]].long()
        slot = p % case["page"]
        s["k_pages"][page, slot] = _turn(s["k"], cos, sin, case)
        s["v_pages"][page, slot] = s["v"]
        return [s["k_pages"], s["v_pages"]] + ([] if s["q"] is None else [_turn(s["q"], cos, sin, case)])
    if case["kind"] == "attend":
        q, b, kv = s["q"], case["sequences"], case["kv"]
        g, d, dv = case["heads"] // kv, case["dim"], case["vdim"]
        at = s["table"].long().clamp(min=0)
        keys = s["k_pages"][at].flatten(1, 2).permute(0, 2, 3, 1).float().contiguous()  # (b, kv, d, positions)
        scores = q.float().view(b, kv, g, d) @ keys * d**-0.5
        del keys
        t = torch.arange(scores.shape[-1], device=DEV)
        n = s["lengths"].long()[:, None]
        seen = t < n
        if case["window"]:
            seen &= t >= n - case["window"]
        seen = seen[:, None, None]
        scores = torch.where(seen, scores, float("-inf"))
        top = scores.amax(-1, keepdim=True)
        w = torch.exp(scores - torch.where(top.isinf(), 0.0, top))
        total = w.sum(-1, keepdim=True)
        values = s["v_pages"][at].flatten(1, 2).permute(0, 2, 1, 3).float().contiguous()
        out = w @ values / torch.where(total == 0, 1.0, total)
        return [out.reshape(b, case["heads"], dv).to(q.dtype)]
    values, r = s["values"], case["heads"] // case["kv"]
    if s["table"] is not None:
        values = values[s["table"].long()].flatten(0, 1).transpose(0, 1)
    out = []
    for h in range(case["kv"]):
        mine = s["scores"][h * r : (h + 1) * r]
        w = torch.exp((mine - mine.amax(-1, keepdim=True)) * 128**-0.5)
        rows = values[h][s["ids"][h * r : (h + 1) * r]].float()
        out.append(((w / w.sum(-1, keepdim=True))[..., None, :] @ rows)[..., 0, :])
    return [torch.cat(out).to(values.dtype)]


# ---- the definition in 64 bits ----


def _turned(x, positions, case, sign=1.0):
    """Every pair as a complex number times exp(i angle)."""
    r = case["rotary"]
    z = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                    sign * positions.double()[:, None, None] * _freqs(case))
    out = x.double().clone()
    first, second = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
    y = torch.complex(out[..., first].contiguous(), out[..., second].contiguous()) * z
    out[..., first], out[..., second] = y.real, y.imag
    return out


def exact(case, seed):
    """What run returns, from the operators' definitions in 64 bits."""
    x = _inputs(case, seed)
    if case["kind"] == "rotate":
        out = [_turned(x["x"], x["positions"], case)]
        if case["train"]:
            out.append(_turned(x["dy"], x["positions"], case, -1.0))
        return out
    if case["kind"] == "append":
        pools = [x["k_pages"].double(), x["v_pages"].double()]
        for pool, new in zip(pools, (_turned(x["k"], x["positions"], case), x["v"].double())):
            where = x["positions"].long()
            flat = x["table"].long()[x["sequences"].long(), where.div(case["page"], rounding_mode="floor")]
            pool.index_put_((flat, where.remainder(case["page"])), new)
        return pools + ([] if x["q"] is None else [_turned(x["q"], x["positions"], case)])
    if case["kind"] == "attend":
        g = case["heads"] // case["kv"]
        out = torch.zeros((case["sequences"], case["heads"], case["vdim"]), dtype=torch.float64, device=DEV)
        for b, (n, seen) in enumerate(zip(_lengths(case), _seen(case))):
            if seen == 0:
                continue
            at = torch.arange(n - seen, n, device=DEV)
            page, slot = x["table"][b].long()[at // case["page"]], at % case["page"]
            for h in range(case["kv"]):
                keys = x["k_pages"][page, slot, h].double()
                values = x["v_pages"][page, slot, h].double()
                p = torch.softmax(x["q"][b, h * g : (h + 1) * g].double() @ keys.T / case["dim"] ** 0.5, -1)
                out[b, h * g : (h + 1) * g] = p @ values
        return [out]
    g = case["heads"] // case["kv"]
    out = torch.empty((case["heads"], case["queries"], case["vdim"]), dtype=torch.float64, device=DEV)
    for h in range(case["heads"]):
        p = torch.softmax(x["scores"][h].double() / 128**0.5, -1)
        for j in range(case["queries"]):
            i = x["ids"][h, j]
            if x["table"] is None:
                rows = x["values"][h // g, i]
            else:
                rows = x["values"][x["table"].long()[i // case["page"]], i % case["page"], h // g]
            out[h, j] = p[j] @ rows.double()
    return [out]
