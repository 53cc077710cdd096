"""The operators of a paged key-value cache: appending (with the position rotation), reading back, and the attention of
one new token.  They serve what follows a search: a model answers a query from the passages that the index found, whose
keys and values lie in pages.

`listed` and `draw` give cases, `prepare` their inputs, `run` one pass (plain torch operations in fp32, or the
framework's operators where `own` is true), `exact` the same from the definition in 64 bits, `work` what a pass cannot
do without.
"""
import importlib
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"


def listed():
    return [
        # one decoding step of 32 requests: a token each, its query heads rotated in the same call; latency counts
        dict(name="append step of 32", op="append", dtype="bf16", store="same", seqs=32, fewest=1, most=1, past=4096,
             hq=32, hkv=8, d=128, rot=128, pairs="halves", page=64, pad=1),
        # a prompt chunk of a few requests, every head with its own keys (no sharing), small pages
        dict(name="append prompts", op="append", dtype="f16", store="same", seqs=5, fewest=700, most=4096, past=1000,
             hq=16, hkv=16, d=64, rot=64, pairs="halves", page=16, pad=0),
        # keys and values of passages stored ahead of any query, as int8 codes; no query heads, half of each head rotated
        dict(name="append passages int8", op="append", dtype="bf16", store="int8", seqs=200, fewest=20, most=200, past=1,
             hq=0, hkv=8, d=128, rot=64, pairs="neighbours", page=32, pad=0),
        # one passage read back, as when it moves to another position
        dict(name="read one passage", op="read", dtype="bf16", store="same", seqs=1, fewest=100, most=100, hkv=8, d=128,
             page=64),
        # many requests' int8 rows as floating point, for a dense prefill; a head size that is no power of two
        dict(name="read int8", op="read", dtype="f16", store="int8", seqs=64, fewest=33, most=2048, hkv=4, d=96,
             page=32),
        # the smallest answer: one request over one short passage
        dict(name="attend one passage", op="attend", dtype="bf16", store="same", seqs=1, fewest=100, most=100, found=0,
             hq=32, hkv=8, d=128, page=64),
        # 32 queries, each over the 10 passages that a search returns (some missing: id -1), whose last pages are partly
        # filled, and then its own tokens
        dict(name="attend 10 passages", op="attend", dtype="f16", store="same", seqs=32, fewest=1, most=500, found=10,
             hq=12, hkv=12, d=64, page=16),
        # a serving batch of very different lengths, shared key heads
        dict(name="attend ragged", op="attend", dtype="bf16", store="same", seqs=64, fewest=1, most=8192, found=0,
             hq=32, hkv=8, d=128, page=64),
        # one long document: the work has to be split over its length
        dict(name="attend long", op="attend", dtype="bf16", store="same", seqs=1, fewest=131071, most=131071, found=0,
             hq=32, hkv=8, d=128, page=64),
        # a search batch of 2000 queries over short int8 contexts
        dict(name="attend 2000 short int8", op="attend", dtype="f16", store="int8", seqs=2000, fewest=1, most=200,
             found=0, hq=16, hkv=2, d=128, page=32),
        # the largest: long int8 contexts
        dict(name="attend large int8", op="attend", dtype="bf16", store="int8", seqs=48, fewest=2048, most=16384,
             found=0, hq=64, hkv=8, d=128, page=128),
        # one key head for all query heads, wide heads, a page size that is no power of two
        dict(name="attend one key head", op="attend", dtype="f16", store="same", seqs=16, fewest=500, most=5000, found=0,
             hq=16, hkv=1, d=256, page=48),
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["append", "append", "read", "attend", "attend", "attend", "attend"])
    d = rng.choice([64, 96, 128, 128, 192, 256])
    hkv = rng.choice([1, 2, 3, 4, 8, 8, 12])
    case = dict(op=op, dtype=rng.choice(["bf16", "f16"]), store=rng.choice(["same", "int8"]), hkv=hkv, d=d,
                page=rng.choice([1, 16, 16, 20, 32, 48, 64, 64, 128, 256]))
    if op == "attend":
        seqs = _spread(rng, 1, 2000)
        room = int(3.0e8 / (hkv * d * seqs))  # keys a request: keeps the padded plain form below the largest case's
        most = _spread(rng, 1, max(1, min(131072, room)))
        case.update(seqs=seqs, fewest=_spread(rng, 1, most), most=most, found=rng.choice([0, 0, 10]) if seqs <= 64 else 0,
                    hq=hkv * rng.choice([1, 2, 4, 5, 8, 8, 16]))
        return case
    seqs = _spread(rng, 1, 256)
    room = int(1.6e7 / (hkv * d * seqs))
    most = _spread(rng, 1, max(1, min(4096, room)))
    case.update(seqs=seqs, fewest=_spread(rng, 1, most), most=most)
    if op == "append":
        case.update(past=_spread(rng, 1, 4096), hq=hkv * rng.choice([0, 1, 4, 8]), rot=rng.choice([d, d, d // 2]),
                    pairs=rng.choice(["halves", "neighbours"]), pad=rng.choice([0, 1]))
        if case["hq"] * most * seqs * d > 6e7:
            case["hq"] = hkv
    return case


def _lengths(case):
    """Tokens of each request: from the case alone, spread over their logarithm."""
    rng = random.Random("lengths %(seqs)d %(fewest)d %(most)d %(page)d" % case)
    return [_spread(rng, case["fewest"], case["most"]) for _ in range(case["seqs"])]


def _pasts(case):
    rng = random.Random("pasts %(seqs)d %(past)d %(page)d" % case)
    return [rng.randrange(case["past"]) for _ in range(case["seqs"])]


def _passages(case):
    """Lengths of each request's passages, 0 where the search found none."""
    rng = random.Random("passages %(seqs)d %(found)d %(page)d" % case)
    return [[0 if rng.random() < 0.1 else rng.randint(60, 200) for _ in range(case["found"])]
            for _ in range(case["seqs"])]


def _up(n, m):
    return -(-n // m)


def _layout(case):
    """Rows of (page number or -1, slots filled) of each request in order, and each request's length in slots.

    Page numbers are consecutive here; prepare() shuffles them."""
    page, nxt, rows, lens = case["page"], 0, [], []
    tails = _lengths(case)
    pasts = _pasts(case) if case["op"] == "append" else [0] * case["seqs"]
    found = _passages(case) if case["op"] == "attend" else [[]] * case["seqs"]
    for b in range(case["seqs"]):
        row = []
        for n in found[b]:
            for p in range(max(1, _up(n, page))):
                row.append((nxt if n else -1, min(page, n - p * page) if n else 0))
                nxt += bool(n)
        n = tails[b]
        if case["op"] == "attend" and case["seqs"] >= 16 and b % 16 == 5:
            n = 0  # a request that has ended: its row of the batch is empty
            if not found[b]:
                row = []
        lens.append(len(row) * page + n)
        for p in range(_up(n + pasts[b], page)):
            row.append((nxt, page))
            nxt += 1
        rows.append(row)
    return rows, lens, nxt


def _visible(case):
    """Keys that the new tokens of all requests attend to."""
    rows, lens, _ = _layout(case)
    page = case["page"]
    return sum(max(0, min(fill, n - p * page)) for row, n in zip(rows, lens) for p, (at, fill) in enumerate(row) if at >= 0)


def work(case):
    e = 2
    stored = case["d"] * (1 if case["store"] == "int8" else e) + (4 if case["store"] == "int8" else 0)  # a head's row
    if case["op"] == "attend":
        n, q = _visible(case), case["seqs"] * case["hq"]
        table = sum(len(row) for row in _layout(case)[0])
        return {"bytes": n * 2 * case["hkv"] * stored + q * (2 * case["d"] * e + 4) + 4 * table,
                "flops": 4 * n * case["hq"] * case["d"]}
    n = sum(_lengths(case))
    if case["op"] == "read":
        return {"bytes": n * 2 * case["hkv"] * (stored + case["d"] * e) + 4 * n, "flops": n * 2 * case["hkv"] * case["d"]}
    heads = case["hq"] * 2 * case["d"] * e + 2 * case["hkv"] * (case["d"] * e + stored)
    more = n * 2 * case["hkv"] * (stored + case["d"] * e) if case["store"] == "int8" else 0  # the codes are read back
    return {"bytes": n * (heads + 4 * case["rot"] + 12) + more, "flops": 3 * n * (case["hq"] + case["hkv"]) * case["rot"]}


def _codes(x):
    """int8 codes and fp32 scales of rows, the largest value of a row at 127."""
    top = x.abs().amax(-1, keepdim=True)
    codes = torch.round(x * torch.where(top > 0, 127.0 / top, torch.zeros_like(top)))
    return codes.to(torch.int8), (top / 127.0).squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, page, hkv, d = TYPES[case["dtype"]], case["page"], case["hkv"], case["d"]
    rows, lens, used = _layout(case)
    pages = used + 3
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32).to(DEV)  # noqa: E731
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    wide = max(1, max(len(r) for r in rows))
    table = ints([[at for at, _ in r] + [-1] * (wide - len(r)) for r in rows])
    table = torch.where(table >= 0, order[table.clamp(min=0).long()], table).contiguous()
    s = dict(case=case, table=table, lens=ints(lens), fill=None, k_scale=None, v_scale=None)
    if any(f < page for r in rows for at, f in r if at >= 0):
        filled = [page] * pages
        for r in rows:
            for at, f in r:
                if at >= 0:
                    filled[at] = f
        fill = torch.empty(pages, dtype=torch.int32, device=DEV)
        fill[order.long()] = ints(filled)
        s["fill"] = fill
    # what lies in the cache: pages at a time, so that wide caches need no fp32 copy
    kind = torch.int8 if case["store"] == "int8" else dt
    for name in "kv":
        cache = torch.empty(pages, hkv, page, d, dtype=kind, device=DEV)
        scale = torch.empty(pages, hkv, page, device=DEV) if kind == torch.int8 else None
        step = max(1, (1 << 26) // (hkv * page * d))
        for a in range(0, pages, step):
            x = normal(min(step, pages - a), hkv, page, d)
            if scale is None:
                cache[a:a + step] = x.to(dt)
            else:
                cache[a:a + step], scale[a:a + step] = _codes(x)
        s[name], s[name + "_scale"] = cache, scale
    if case["op"] == "attend":
        # slots that no token can see hold what memory holds: not-a-numbers among it
        t = torch.arange(wide * page, device=DEV)
        at = s["table"].long().repeat_interleave(page, 1)
        seen = torch.zeros(pages, page, dtype=torch.bool, device=DEV)
        mine = (t < s["lens"][:, None]) & (at >= 0)
        seen.index_put_((at[mine], (t % page).expand_as(at)[mine]), torch.tensor(True, device=DEV))
        if s["fill"] is not None:
            seen &= torch.arange(page, device=DEV) < s["fill"][:, None]
        for name in "kv":
            if s[name + "_scale"] is not None:
                s[name + "_scale"].masked_fill_(~seen[:, None], math.nan)
            else:
                s[name].masked_fill_(~seen[:, None, :, None], math.nan)
        s["q"] = (normal(case["seqs"], case["hq"], d) * 1.5).to(dt)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(case["seqs"], case["hq"], device=DEV)
    else:
        n, past = _lengths(case), _pasts(case) if case["op"] == "append" else [0] * case["seqs"]
        s["seq"] = ints([b for b in range(case["seqs"]) for _ in range(n[b])])
        idx = [past[b] + i for b in range(case["seqs"]) for i in range(n[b])]
        if case.get("pad") and len(idx) > 8:
            idx[len(idx) // 2] = -1  # a place of the batch that no request has: nothing is written
        s["idx"] = ints(idx)
        if case["op"] == "append":
            # the projection's output holds the heads of query, key and value side by side
            hq, tokens = case["hq"], len(idx)
            heads = normal(tokens, hq + 2 * hkv, d).to(dt)
            s["q_new"] = heads[:, :hq] if hq else None
            s["k_new"], s["v_new"] = heads[:, hq:hq + hkv], heads[:, hq + hkv:]
            s["q_out"] = torch.empty(tokens, hq, d, dtype=dt, device=DEV) if hq else None
            # positions count on from a chunk's place in its document
            start = random.Random(seed).randrange(256)
            s["pos"] = ints([max(0, i) + start for i in idx])
            top = max(idx) + 257
            freq = 10000.0 ** (-torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float64) / case["rot"])
            angle = torch.arange(top, device=DEV, dtype=torch.float64)[:, None] * freq
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    if own:
        kv = importlib.import_module("fanarvse-paper_b200.kvcache")
        s["cache"] = kv.PagedKV(s["k"], s["v"], k_scale=s["k_scale"], v_scale=s["v_scale"], fill=s["fill"])
    return s


# ------------------------------------------------------------------------------------------------ the plain form

def _rows_of(s, seq, idx):
    """Page, slot and whether there is one, of logical tokens idx of the requests seq."""
    page = s["case"]["page"]
    at = s["table"][seq.long(), idx.clamp(min=0).long() // page].long()
    there = (idx >= 0) & (at >= 0)
    return at.clamp(min=0), idx.clamp(min=0).long() % page, there


def _rotated(x, cos, sin, rot, pairs):
    x = x.float()
    y = x.clone()
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if pairs == "halves" else (x[..., 0:rot:2], x[..., 1:rot:2])
    cos, sin = cos[:, None], sin[:, None]
    left, right = a * cos - b * sin, b * cos + a * sin
    if pairs == "halves":
        y[..., :rot // 2], y[..., rot // 2:rot] = left, right
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = left, right
    return y


def _plain_read(s):
    at, slot, there = _rows_of(s, s["seq"], s["idx"])
    got = []
    for name in "kv":
        x = s[name][at, :, slot].float()
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][at, :, slot][..., None]
        got.append(torch.where(there[:, None, None], x, torch.zeros_like(x)).to(TYPES[s["case"]["dtype"]]))
    return got


def _plain_append(s):
    case = s["case"]
    at, slot, there = _rows_of(s, s["seq"], s["idx"])
    cos, sin = s["cos"][s["pos"].long()], s["sin"][s["pos"].long()]
    if case["hq"]:
        q = _rotated(s["q_new"], cos, sin, case["rot"], case["pairs"])
        s["q_out"].copy_(torch.where(there[:, None, None], q, torch.zeros_like(q)))
    # a token without a place writes what a token with one writes, to the same place
    first = there.int().argmax()
    src = torch.where(there, torch.arange(len(at), device=DEV), first)
    at, slot = at[src], slot[src]
    new = {"k": _rotated(s["k_new"], cos, sin, case["rot"], case["pairs"])[src], "v": s["v_new"].float()[src]}
    for name, x in new.items():
        if case["store"] == "int8":
            codes, scale = _codes(x)
            s[name][at, :, slot] = codes
            s[name + "_scale"][at, :, slot] = scale
        else:
            s[name][at, :, slot] = x.to(s[name].dtype)


def _plain_attend(s):
    case = s["case"]
    hkv, d, page = case["hkv"], case["d"], case["page"]
    seqs, wide = s["table"].shape
    at = s["table"].clamp(min=0).long()
    t = torch.arange(wide * page, device=DEV)
    seen = (t < s["lens"][:, None]) & (s["table"] >= 0).repeat_interleave(page, 1)
    if s["fill"] is not None:
        seen &= t % page < s["fill"][at].repeat_interleave(page, 1)

    def dense(name):
        x = s[name][at].float()
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][at][..., None]
        return x.permute(0, 2, 1, 3, 4).reshape(seqs, hkv, wide * page, d)

    q = s["q"].float().view(seqs, hkv, case["hq"] // hkv, d)
    score = (q @ dense("k").transpose(-1, -2)) * (1.0 / math.sqrt(d))
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    v = dense("v").masked_fill(~seen[:, None, :, None], 0.0)
    out = (p @ v) / torch.where(total > 0, total, torch.ones_like(total))
    return out.reshape(seqs, case["hq"], d).to(s["q"].dtype), (top + torch.log(total)).reshape(seqs, case["hq"])


def run(state):
    s, case, dt = state, state["case"], TYPES[state["case"]["dtype"]]
    if case["op"] == "attend":
        out, lse = s["cache"].attend(s["q"], s["table"], s["lens"], out=s["out"], lse=s["lse"]) if own else _plain_attend(s)
        return {"out": out, "lse": lse}
    if case["op"] == "read":
        k, v = s["cache"].read(s["table"], s["idx"], seq=s["seq"], dtype=dt) if own else _plain_read(s)
        return {"k": k, "v": v}
    if own:
        s["cache"].append(s["k_new"], s["v_new"], s["table"], s["idx"], seq=s["seq"], pos=s["pos"],
                          rope=(s["cos"], s["sin"]), pairs=case["pairs"], q=s["q_new"], q_out=s["q_out"])
    else:
        _plain_append(s)
    got = {"q": s["q_out"]} if case["hq"] else {}
    if case["store"] == "int8":  # codes come back as the values that they stand for
        k, v = s["cache"].read(s["table"], s["idx"], seq=s["seq"], dtype=dt) if own else _plain_read(s)
        return {**got, "k": k, "v": v}
    return {**got, "k": s["k"], "v": s["v"]}


# ------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    page, d, hkv = case["page"], case["d"], case["hkv"]
    table = s["table"].tolist()

    def value(name, at, slot):
        x = s[name][at, :, slot].double()
        return x if s[name + "_scale"] is None else x * s[name + "_scale"][at, :, slot].double()[..., None]

    if case["op"] == "attend":
        out = torch.zeros(case["seqs"], case["hq"], d, dtype=torch.float64, device=DEV)
        lse = torch.full((case["seqs"], case["hq"]), -math.inf, dtype=torch.float64, device=DEV)
        fill = s["fill"].tolist() if s["fill"] is not None else None
        for b, n in enumerate(s["lens"].tolist()):
            at, slot = [], []
            for p in range(_up(n, page)):
                if table[b][p] >= 0:
                    m = min(page, n - p * page, fill[table[b][p]] if fill else page)
                    at += [table[b][p]] * m
                    slot += range(m)
            if not at:
                continue
            at, slot = torch.tensor(at).to(DEV), torch.tensor(slot).to(DEV)
            k, v = value("k", at, slot).transpose(0, 1), value("v", at, slot).transpose(0, 1)
            q = s["q"][b].double().reshape(hkv, -1, d)
            score = torch.einsum("hgd,htd->hgt", q, k) / math.sqrt(d)
            lse[b] = torch.logsumexp(score, -1).reshape(-1)
            out[b] = torch.einsum("hgt,htd->hgd", torch.softmax(score, -1), v).reshape(-1, d)
        return {"out": out, "lse": lse}
    idx = s["idx"].tolist()
    place = [(t, table[b][i // page], i % page) for t, (b, i) in enumerate(zip(s["seq"].tolist(), idx)) if i >= 0]
    token, at, slot = (torch.tensor(x).to(DEV) for x in zip(*place))
    tokens = len(idx)
    if case["op"] == "read":
        got = {}
        for name in "kv":
            got[name] = torch.zeros(tokens, hkv, d, dtype=torch.float64, device=DEV)
            got[name][token] = value(name, at, slot)
        return got
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]

    def turned(x):
        x, rot = x.double(), case["rot"]
        head = x[..., :rot]
        if case["pairs"] == "halves":
            z = torch.complex(head[..., :rot // 2], head[..., rot // 2:]) * turn
            head = torch.cat([z.real, z.imag], -1)
        else:
            head = torch.view_as_real(torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous()) * turn).flatten(-2)
        return torch.cat([head, x[..., rot:]], -1)

    got = {}
    if case["hq"]:
        got["q"] = torch.zeros(tokens, case["hq"], d, dtype=torch.float64, device=DEV)
        got["q"][token] = turned(s["q_new"])[token]
    for name, x in (("k", turned(s["k_new"])), ("v", s["v_new"].double())):
        if case["store"] == "int8":
            step = x.abs().amax(-1, keepdim=True) / 127
            near = torch.where(step > 0, torch.round(x / step.clamp(min=1e-300)), torch.zeros_like(x)) * step
            got[name] = torch.zeros(tokens, hkv, d, dtype=torch.float64, device=DEV)
            got[name][token] = near[token]
        else:
            got[name] = s[name].double()
            got[name][at, :, slot] = x[token]
    return got
