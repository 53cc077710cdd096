"""The operators of answering with drafted tokens over a paged key-value cache: a small model drafts a tree of tokens behind
each sequence, and the target model takes as many of them in one step as its own probabilities allow.  The drafted tokens
are appended (norm of each head and rotation in one pass), attend over the cache and their own ancestors, are verified
against the target's probabilities, and the rows of the ones taken move together behind the sequence.

`listed` and `draw` give cases, `prepare` their inputs, `run` one pass (plain torch operations in fp32, or the
framework's operators where `own` is true), `exact` the same from the definition in 64 bits, `work` what a pass cannot
do without.
"""
import importlib
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEV = "cuda"


def listed():
    return [
        # one decoding step of 32 requests by a model that norms its query and key heads; latency counts
        dict(name="append normed step of 32", op="append", dtype="bf16", store="same", seqs=32, fewest=1, most=1, past=4096,
             hq=32, hkv=8, d=128, rot=128, pairs="halves", page=64, pad=1, weight="bf16"),
        # prompt chunks stored as int8 codes, half of each head rotated, fp32 weights
        dict(name="append normed prompts int8", op="append", dtype="f16", store="int8", seqs=5, fewest=700, most=4096,
             past=1000, hq=16, hkv=4, d=96, rot=48, pairs="neighbours", page=32, pad=0, weight="f32"),
        # the smallest verification step: one request over one short passage, a tree of 8
        dict(name="tree one passage", op="attend", dtype="bf16", store="same", seqs=1, nodes=8, tree="random", fewest=100,
             most=100, found=0, hq=32, hkv=8, d=128, page=64),
        # 32 queries, each over the 10 passages that a search returns (some missing, last pages partly filled) and its own
        # tokens; every head with keys of its own; one tree shape for all
        dict(name="tree 10 passages", op="attend", dtype="f16", store="same", seqs=32, nodes=25, tree="levels", fewest=1,
             most=500, found=10, hq=12, hkv=12, d=64, page=16),
        # a serving batch of very different lengths, shared key heads, some requests with fewer nodes
        dict(name="tree ragged", op="attend", dtype="bf16", store="same", seqs=64, nodes=16, tree="random", fewest=1,
             most=8192, found=0, hq=32, hkv=8, d=128, page=64),
        # one long document and a large tree: the work has to be split over the length
        dict(name="tree long", op="attend", dtype="bf16", store="same", seqs=1, nodes=64, tree="random", fewest=131000,
             most=131000, found=0, hq=32, hkv=8, d=128, page=64),
        # the largest: long int8 contexts
        dict(name="tree large int8", op="attend", dtype="bf16", store="int8", seqs=24, nodes=32, tree="random", fewest=2048,
             most=16384, found=0, hq=64, hkv=8, d=128, page=128),
        # the smallest verification: one request, eight drafted tokens
        dict(name="verify one", op="verify", dtype="f32", seqs=1, nodes=8, tree="random", vocab=32000, draft=1),
        # a serving batch over a large vocabulary
        dict(name="verify batch", op="verify", dtype="f32", seqs=64, nodes=16, tree="levels", vocab=131072, draft=1),
        # drafts without probabilities of their own (found in the passages, say), an odd vocabulary
        dict(name="verify plain drafts", op="verify", dtype="bf16", seqs=200, nodes=5, tree="chain", vocab=50021, draft=0),
        # after a step of 32 requests: the rows of the tokens taken, behind the sequence
        dict(name="compact step of 32", op="compact", dtype="bf16", store="same", seqs=32, nodes=16, past=4096, hkv=8, d=128,
             page=64),
        # large trees of many requests, int8 rows read back
        dict(name="compact many int8", op="compact", dtype="f16", store="int8", seqs=200, nodes=64, past=500, hkv=12, d=64,
             page=16),
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "attend", "verify", "verify", "compact"])
    if op == "verify":
        seqs = _spread(rng, 1, 256)
        nodes = _spread(rng, 1, max(1, min(64, 140000 // seqs)))
        vocab = _spread(rng, 1000, max(1000, min(200000, int(1.3e8 / (seqs * (nodes + 1))))))
        return dict(op=op, dtype=rng.choice(["f32", "f32", "bf16", "f16"]), seqs=seqs, nodes=nodes,
                    tree=rng.choice(["random", "levels", "chain"]), vocab=vocab, draft=rng.choice([0, 1, 1]))
    d = rng.choice([64, 96, 128, 128, 192, 256])
    hkv = rng.choice([1, 2, 3, 4, 8, 8, 12])
    case = dict(op=op, dtype=rng.choice(["bf16", "f16"]), store=rng.choice(["same", "int8"]), hkv=hkv, d=d,
                page=rng.choice([1, 16, 16, 20, 32, 48, 64, 64, 128, 256]))
    if op == "attend":
        group = rng.choice([1, 2, 4, 5, 8, 8, 16])
        nodes = _spread(rng, 1, max(1, min(256, 4096 // group)))
        seqs = _spread(rng, 1, 128)
        # keys a request: the padded plain form and the products stay below the largest case's
        room = int(min(1.5e8 / (hkv * d * seqs), 3.5e10 / (nodes * hkv * group * d * seqs)))
        most = _spread(rng, 1, max(1, min(131072, room)))
        short = seqs * nodes * hkv * group * d * (most + 1500) <= 3.5e10
        case.update(seqs=seqs, nodes=nodes, tree=rng.choice(["random", "levels", "chain"]), fewest=_spread(rng, 1, most),
                    most=most, found=rng.choice([0, 0, 10]) if short and seqs <= 32 else 0, hq=hkv * group)
        return case
    seqs = _spread(rng, 1, 256)
    if op == "compact":
        nodes = _spread(rng, 1, max(1, min(256, 12800 // seqs)))
        room = int(6e7 / (hkv * d * seqs))
        case.update(seqs=seqs, nodes=nodes, past=_spread(rng, 1, max(1, min(4096, room))))
        return case
    room = int(1.6e7 / (hkv * d * seqs))
    most = _spread(rng, 1, max(1, min(4096, room)))
    case.update(seqs=seqs, fewest=_spread(rng, 1, most), most=most, past=_spread(rng, 1, 4096),
                hq=hkv * rng.choice([1, 1, 4, 8]), rot=rng.choice([d, d, d // 2]), pairs=rng.choice(["halves", "neighbours"]),
                pad=rng.choice([0, 1]), weight=rng.choice([case["dtype"], "f32"]))
    if case["hq"] * most * seqs * d > 2e7:
        case["hq"] = hkv
    return case


# ------------------------------------------------------------------------------------------------ what a case consists of

def _lengths(case):
    """Tokens of each request before the drafted ones (append: new tokens), spread over their logarithm."""
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


def _trees(case):
    """Parents of each request's nodes (-1: behind the sequence) and how many nodes it has.

    "levels": one shape for all, whose levels narrow from left to right; "random": each request a shape and, for every
    fourth, a size of its own; "chain": each node behind the one before."""
    nodes, rng = case["nodes"], random.Random("tree %(seqs)d %(nodes)d" % case)
    if case["tree"] == "chain":
        return [list(range(-1, nodes - 1))] * case["seqs"], [nodes] * case["seqs"]
    if case["tree"] == "levels":
        parents, above, at = [], [-1], 0
        while at < nodes:
            new = []
            for rank, p in enumerate(above):
                for _ in range(max(1 if rank == 0 else 0, (4 if p < 0 else 3) - rank)):
                    if at < nodes:
                        parents.append(p)
                        new.append(at)
                        at += 1
            above = new
        return [parents] * case["seqs"], [nodes] * case["seqs"]
    parents = [[max(-1, i - 1 - int(rng.expovariate(0.4))) for i in range(nodes)] for _ in range(case["seqs"])]
    counts = [rng.randint(0 if case["op"] == "attend" else 1, nodes) if b % 4 == 3 else nodes for b in range(case["seqs"])]
    return parents, counts


def _ancestors(parents):
    """For each node the nodes that it sees, itself among them."""
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else []) + [i])
    return seen


def _up(n, m):
    return -(-n // m)


def _layout(case):
    """Rows of (page number or -1, slots filled) of each request in order, and each request's length in slots before the
    drafted nodes (append: new tokens).  Page numbers are consecutive here; prepare() shuffles them."""
    page, nxt, rows, lens = case["page"], 0, [], []
    tails = _lengths(case) if case["op"] != "compact" else [p + 1 for p in _pasts(case)]
    pasts = _pasts(case) if case["op"] == "append" else [0] * case["seqs"]
    found = _passages(case) if case["op"] == "attend" else [[]] * case["seqs"]
    more = 0 if case["op"] == "append" else case["nodes"]
    for b in range(case["seqs"]):
        row = []
        for n in found[b]:
            for p in range(max(1, _up(n, page))):
                row.append((nxt if n else -1, min(page, n - p * page) if n else 0))
                nxt += bool(n)
        n = tails[b]
        if case["op"] == "attend" and case["seqs"] >= 16 and b % 16 == 5:
            n = 0  # a request that begins: its tree has nothing before it but what was found
        lens.append(len(row) * page + n)
        for p in range(_up(n + pasts[b] + more, page)):
            row.append((nxt, page))
            nxt += 1
        rows.append(row)
    return rows, lens, nxt


def _visible(case):
    """Keys that any node sees, and pairs of a node and a key that it sees, of all requests."""
    rows, lens, _ = _layout(case)
    parents, counts = _trees(case)
    page, keys, pairs = case["page"], 0, 0
    for row, n, up, count in zip(rows, lens, parents, counts):
        if count:
            before = sum(max(0, min(fill, n - p * page)) for p, (at, fill) in enumerate(row) if at >= 0)
            keys += before + count
            pairs += before * count + sum(len(a) for a in _ancestors(up[:count]))
    return keys, pairs


def _paths(case):
    """The nodes that verification took: some from the start on, then later ones.  No row that moves is another's place,
    so that a second pass over the same cache finds the same rows."""
    rng, nodes, paths = random.Random("path %(seqs)d %(nodes)d" % case), case["nodes"], []
    for _ in range(case["seqs"]):
        kept = rng.randint(0, nodes)
        first = rng.randint(max(0, 2 * kept - nodes), kept)
        paths.append(list(range(first)) + sorted(rng.sample(range(kept, nodes), kept - first)))
    return paths


def work(case):
    if case["op"] == "verify":
        e, seqs, nodes = TYPES[case["dtype"]].itemsize, case["seqs"], case["nodes"]
        # the distribution of the last node taken, and the draft's where its probabilities count
        return {"bytes": seqs * (case["vocab"] * e * (1 + case["draft"]) + 16 * nodes), "flops": 3 * seqs * case["vocab"]}
    e = 2
    stored = case["d"] * (1 if case["store"] == "int8" else e) + (4 if case["store"] == "int8" else 0)  # a head's row
    if case["op"] == "attend":
        keys, pairs = _visible(case)
        q = sum(_trees(case)[1]) * case["hq"]
        table = sum(len(row) for row in _layout(case)[0])
        return {"bytes": keys * 2 * case["hkv"] * stored + q * (2 * case["d"] * e + 4) + 4 * table,
                "flops": 4 * pairs * case["hq"] * case["d"]}
    if case["op"] == "compact":
        paths = _paths(case)
        n, moved = sum(len(p) for p in paths), sum(i != x for p in paths for i, x in enumerate(p))
        back = n * 2 * case["hkv"] * (stored + case["d"] * e) if case["store"] == "int8" else 0  # the codes are read back
        return {"bytes": moved * 4 * case["hkv"] * stored + 4 * case["nodes"] * case["seqs"] + back, "flops": 0}
    n = sum(_lengths(case))
    heads = case["hq"] * 2 * case["d"] * e + 2 * case["hkv"] * (case["d"] * e + stored)
    more = n * 2 * case["hkv"] * (stored + case["d"] * e) if case["store"] == "int8" else 0  # the codes are read back
    return {"bytes": n * (heads + 4 * case["rot"] + 12) + more,
            "flops": n * (case["hq"] + case["hkv"]) * (3 * case["rot"] + 4 * case["d"])}


# ------------------------------------------------------------------------------------------------ inputs

def _codes(x):
    """int8 codes and fp32 scales of rows, the largest value of a row at 127."""
    top = x.abs().amax(-1, keepdim=True)
    codes = torch.round(x * torch.where(top > 0, 127.0 / top, torch.zeros_like(top)))
    return codes.to(torch.int8), (top / 127.0).squeeze(-1)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32).to(DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "verify":
        return _prepare_verify(case, g)
    dt, page, hkv, d = TYPES[case["dtype"]], case["page"], case["hkv"], case["d"]
    rows, lens, used = _layout(case)
    pages = used + 3
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)  # noqa: E731
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    wide = max(1, max(len(r) for r in rows))
    table = _ints([[at for at, _ in r] + [-1] * (wide - len(r)) for r in rows])
    table = torch.where(table >= 0, order[table.clamp(min=0).long()], table).contiguous()
    s = dict(case=case, table=table, lens=_ints(lens), fill=None, k_scale=None, v_scale=None)
    if any(f < page for r in rows for at, f in r if at >= 0):
        filled = [page] * pages
        for r in rows:
            for at, f in r:
                if at >= 0:
                    filled[at] = f
        fill = torch.empty(pages, dtype=torch.int32, device=DEV)
        fill[order.long()] = _ints(filled)
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
        _prepare_attend(s, normal, wide, pages)
    elif case["op"] == "compact":
        paths = _paths(case)
        s["path"] = _ints([p + [-1] * (case["nodes"] - len(p)) for p in paths])
        s["seq"] = _ints([b for b, p in enumerate(paths) for _ in p])
        s["idx"] = _ints([lens[b] + i for b, p in enumerate(paths) for i in range(len(p))])
    else:
        _prepare_append(s, normal, seed)
    if own:
        kv = importlib.import_module("fanarvse-paper_b200.kvcache")
        s["cache"] = kv.PagedKV(s["k"], s["v"], k_scale=s["k_scale"], v_scale=s["v_scale"], fill=s["fill"])
    return s


def _prepare_attend(s, normal, wide, pages):
    case, page = s["case"], s["case"]["page"]
    parents, counts = _trees(case)
    s["counts"] = _ints(counts) if case["tree"] == "random" else None
    s["parents"] = _ints(parents[0] if case["tree"] == "levels" else parents)
    # slots that no token can see hold what memory holds: not-a-numbers among it
    t = torch.arange(wide * page, device=DEV)
    at = s["table"].long().repeat_interleave(page, 1)
    seen = torch.zeros(pages, page, dtype=torch.bool, device=DEV)
    mine = (t < (s["lens"] + _ints(counts))[:, None]) & (at >= 0)
    seen.index_put_((at[mine], (t % page).expand_as(at)[mine]), torch.tensor(True, device=DEV))
    if s["fill"] is not None:
        seen &= torch.arange(page, device=DEV) < s["fill"][:, None]
    for name in "kv":
        if s[name + "_scale"] is not None:
            s[name + "_scale"].masked_fill_(~seen[:, None], math.nan)
        else:
            s[name].masked_fill_(~seen[:, None, :, None], math.nan)
    s["q"] = (normal(case["seqs"], case["nodes"], case["hq"], case["d"]) * 1.5).to(TYPES[case["dtype"]])
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty(case["seqs"], case["nodes"], case["hq"], device=DEV)


def _prepare_append(s, normal, seed):
    case, dt = s["case"], TYPES[s["case"]["dtype"]]
    n, past = _lengths(case), _pasts(case)
    s["seq"] = _ints([b for b in range(case["seqs"]) for _ in range(n[b])])
    idx = [past[b] + i for b in range(case["seqs"]) for i in range(n[b])]
    if case["pad"] and len(idx) > 8:
        idx[len(idx) // 2] = -1  # a place of the batch that no request has: nothing is written
    s["idx"] = _ints(idx)
    # the projection's output holds the heads of query, key and value side by side
    hq, hkv, d, tokens = case["hq"], case["hkv"], case["d"], len(idx)
    heads = (normal(tokens, hq + 2 * hkv, d) * torch.exp(0.5 * normal(tokens, 1, 1))).to(dt)
    s["q_new"], s["k_new"], s["v_new"] = heads[:, :hq], heads[:, hq:hq + hkv], heads[:, hq + hkv:]
    s["q_out"] = torch.empty(tokens, hq, d, dtype=dt, device=DEV)
    s["q_weight"], s["k_weight"] = ((1.0 + 0.2 * normal(d)).to(TYPES[case["weight"]]) for _ in range(2))
    s["eps"] = 1e-6
    # positions count on from a chunk's place in its document
    start = random.Random(seed).randrange(256)
    s["pos"] = _ints([max(0, i) + start for i in idx])
    top = max(idx) + 257
    freq = 10000.0 ** (-torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float64) / case["rot"])
    angle = torch.arange(top, device=DEV, dtype=torch.float64)[:, None] * freq
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()


def _prepare_verify(case, g):
    """The target's probabilities from logits that spread as a model's do, the draft's from the same with an error, and
    each node drawn from the draft's probabilities behind its parent."""
    seqs, nodes, vocab, dt = case["seqs"], case["nodes"], case["vocab"], TYPES[case["dtype"]]
    parents, counts = _trees(case)
    s = dict(case=case, parents=_ints(parents[0] if case["tree"] == "levels" else parents),
             counts=_ints(counts) if case["tree"] == "random" else None)
    s["target"] = torch.empty(seqs, nodes + 1, vocab, dtype=dt, device=DEV)
    s["draft"] = torch.empty_like(s["target"]) if case["draft"] else None
    s["tokens"] = torch.empty(seqs, nodes, dtype=torch.int32, device=DEV)
    behind = _ints(parents).long() + 1
    for b in range(seqs):
        logits = torch.randn(nodes + 1, vocab, generator=g, device=DEV) * 2.5
        s["target"][b] = torch.softmax(logits, -1).to(dt)
        logits += torch.randn(nodes + 1, vocab, generator=g, device=DEV) * 0.7
        q = torch.softmax(logits, -1)
        if s["draft"] is not None:
            s["draft"][b] = q.to(dt)
            q = s["draft"][b].float()
        total = q.double().cumsum(-1)
        at = torch.rand(nodes, 1, generator=g, device=DEV, dtype=torch.float64) * total[behind[b], -1:]
        s["tokens"][b] = torch.searchsorted(total[behind[b]], at, right=True)[:, 0].clamp(max=vocab - 1)
    s["u"] = torch.rand(seqs, nodes + 1, generator=g, device=DEV)
    if own:
        s["verify"] = importlib.import_module("fanarvse-paper_b200.drafts").verify
    return s


# ------------------------------------------------------------------------------------------------ the plain form

def _rows_of(s, seq, idx):
    """Page, slot and whether there is one, of logical tokens idx of the requests seq."""
    page = s["case"]["page"]
    at = s["table"][seq.long(), idx.clamp(min=0).long() // page].long()
    there = (idx >= 0) & (at >= 0)
    return at.clamp(min=0), idx.clamp(min=0).long() % page, there


def _rotated(x, cos, sin, rot, pairs):
    y = x.clone()
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if pairs == "halves" else (x[..., 0:rot:2], x[..., 1:rot:2])
    cos, sin = cos[:, None], sin[:, None]
    left, right = a * cos - b * sin, b * cos + a * sin
    if pairs == "halves":
        y[..., :rot // 2], y[..., rot // 2:rot] = left, right
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = left, right
    return y


def _normed(x, weight, eps):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float()


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
    q = _rotated(_normed(s["q_new"], s["q_weight"], s["eps"]), cos, sin, case["rot"], case["pairs"])
    s["q_out"].copy_(torch.where(there[:, None, None], q, torch.zeros_like(q)))
    # a token without a place writes what a token with one writes, to the same place
    first = there.int().argmax()
    src = torch.where(there, torch.arange(len(at), device=DEV), first)
    at, slot = at[src], slot[src]
    k = _rotated(_normed(s["k_new"], s["k_weight"], s["eps"]), cos, sin, case["rot"], case["pairs"])
    for name, x in (("k", k[src]), ("v", s["v_new"].float()[src])):
        if case["store"] == "int8":
            codes, scale = _codes(x)
            s[name][at, :, slot] = codes
            s[name + "_scale"][at, :, slot] = scale
        else:
            s[name][at, :, slot] = x.to(s[name].dtype)


def _plain_attend(s):
    case = s["case"]
    hkv, d, page, nodes, seqs = case["hkv"], case["d"], case["page"], case["nodes"], case["seqs"]
    wide = s["table"].shape[1]
    at = s["table"].clamp(min=0).long()
    t = torch.arange(wide * page, device=DEV)
    there = (s["table"] >= 0).repeat_interleave(page, 1)
    if s["fill"] is not None:
        there &= t % page < s["fill"][at].repeat_interleave(page, 1)
    # which nodes each node sees: its parent's and itself
    parents = s["parents"].expand(seqs, nodes).long()
    own_bit = torch.eye(nodes, dtype=torch.bool, device=DEV)
    sees = own_bit.expand(seqs, nodes, nodes).clone()
    for i in range(1, nodes):
        up = parents[:, i]
        above = sees.gather(1, up.clamp(min=0)[:, None, None].expand(seqs, 1, nodes))[:, 0]
        sees[:, i] |= above & (up >= 0)[:, None]
    counts = s["counts"] if s["counts"] is not None else torch.full((seqs,), nodes, device=DEV)
    real = torch.arange(nodes, device=DEV) < counts[:, None]
    node = (t - s["lens"][:, None]).long()  # the node that a place holds
    tree = sees.gather(2, node.clamp(0, nodes - 1)[:, None].expand(seqs, nodes, wide * page))
    seen = torch.where((node < 0)[:, None], torch.ones_like(tree), tree & ((node >= 0) & (node < nodes))[:, None])
    seen = seen & there[:, None] & real[:, :, None]  # [sequences, nodes, keys]

    def dense(name):
        x = s[name][at].float()
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][at][..., None]
        return x.permute(0, 2, 1, 3, 4).reshape(seqs, hkv, wide * page, d)

    q = s["q"].float().view(seqs, nodes, hkv, -1, d).permute(0, 2, 1, 3, 4).reshape(seqs, hkv, -1, d)
    score = (q @ dense("k").transpose(-1, -2)) * (1.0 / math.sqrt(d))
    score = score.view(seqs, hkv, nodes, -1, wide * page).masked_fill(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    v = dense("v").masked_fill(~seen.any(1)[:, None, :, None], 0.0)
    out = (p.view(seqs, hkv, -1, wide * page) @ v).view(seqs, hkv, nodes, -1, d)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    back = lambda x: x.permute(0, 2, 1, 3, 4).reshape(seqs, nodes, case["hq"], -1)  # noqa: E731
    return back(out).to(s["q"].dtype), back(top + torch.log(total))[..., 0]


def _plain_verify(s):
    """All requests side by side, node after node: children come after their parent and are tried in order."""
    case, target, draft = s["case"], s["target"], s["draft"]
    seqs, nodes, vocab = case["seqs"], case["nodes"], case["vocab"]
    row = torch.arange(seqs, device=DEV)
    parents, tokens = s["parents"].expand(seqs, nodes).long(), s["tokens"].long()
    u = s["u"].double()
    last = torch.full((seqs,), -1, dtype=torch.long, device=DEV)
    kept = torch.zeros(seqs, dtype=torch.long, device=DEV)
    path = torch.full((seqs, nodes), -1, dtype=torch.int32, device=DEV)
    left = target[:, 0].double()
    weight = torch.ones(seqs, dtype=torch.float64, device=DEV)
    for i in range(nodes):
        mine = parents[:, i] == last
        if s["counts"] is not None:
            mine &= i < s["counts"]
        x = tokens[:, i]
        if draft is not None:
            q = draft[row, last + 1].double()
            qx = q[row, x]
        else:
            q = torch.zeros_like(left)
            q[row, x] = 1.0
            qx = torch.ones_like(weight)
        taken = mine & (u[:, i] * weight * qx < left[row, x])
        turned = mine & ~taken
        rest = (left - weight[:, None] * q).clamp(min=0.0) if draft is not None else left * (1.0 - q)
        total = rest.sum(-1)
        turned = turned & (total > 0)
        left = torch.where(turned[:, None], rest, left)
        weight = torch.where(turned, total, weight)
        left = torch.where(taken[:, None], target[:, i + 1].double(), left)
        weight = torch.where(taken, torch.ones_like(weight), weight)
        last = torch.where(taken, torch.full_like(last, i), last)
        path[row, kept.clamp(max=nodes - 1)] = torch.where(taken, torch.full_like(last, i).int(), path[row, kept.clamp(max=nodes - 1)])
        kept = kept + taken
    total = left.cumsum(-1)
    token = torch.searchsorted(total, u[:, nodes:] * total[:, -1:], right=True)[:, 0]
    final = vocab - 1 - (left > 0).flip(-1).int().argmax(-1)
    return path, kept.int(), torch.minimum(token, final).int()


def _plain_compact(s):
    case = s["case"]
    moves = s["path"] >= 0
    to = s["lens"][:, None] + torch.arange(case["nodes"], device=DEV)
    start = s["lens"][:, None] + s["path"]
    seq = torch.arange(case["seqs"], device=DEV)[:, None].expand_as(to)
    # a node that was not taken stays where it is, unless its place was needed
    kept = moves.sum(1, keepdim=True)
    start = torch.where(moves, start, to)
    live = (torch.arange(case["nodes"], device=DEV) < kept)
    at, slot, _ = _rows_of(s, seq.reshape(-1), torch.where(live, start, to).reshape(-1))
    at2, slot2, _ = _rows_of(s, seq.reshape(-1), to.reshape(-1))
    for name in ("k", "v", "k_scale", "v_scale"):
        if s[name] is not None:
            s[name][at2, :, slot2] = s[name][at, :, slot]


def run(state):
    s, case = state, state["case"]
    if case["op"] == "attend":
        if own:
            out, lse = s["cache"].attend_tree(s["q"], s["table"], s["lens"], s["parents"], counts=s["counts"],
                                              out=s["out"], lse=s["lse"])
        else:
            out, lse = _plain_attend(s)
        return {"out": out, "lse": lse}
    if case["op"] == "verify":
        if own:
            path, kept, token = s["verify"](s["target"], s["parents"], s["tokens"], s["u"], draft=s["draft"],
                                            counts=s["counts"])
        else:
            path, kept, token = _plain_verify(s)
        return {"path": path, "kept": kept, "token": token}
    if case["op"] == "compact":
        if own:
            s["cache"].compact(s["table"], s["lens"], s["path"])
        else:
            _plain_compact(s)
        got = {}
    else:
        if own:
            s["cache"].append(s["k_new"], s["v_new"], s["table"], s["idx"], seq=s["seq"], pos=s["pos"],
                              rope=(s["cos"], s["sin"]), pairs=case["pairs"], q=s["q_new"], q_out=s["q_out"],
                              norm=(s["q_weight"], s["k_weight"]), eps=s["eps"])
        else:
            _plain_append(s)
        got = {"q": s["q_out"]}
    if case["store"] == "int8":  # codes come back as the values that they stand for
        if not len(s["idx"]):
            return got
        dt = TYPES[case["dtype"]]
        k, v = s["cache"].read(s["table"], s["idx"], seq=s["seq"], dtype=dt) if own else _plain_read(s)
        return {**got, "k": k, "v": v}
    return {**got, "k": s["k"], "v": s["v"]}


# ------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "verify":
        return _exact_verify(s)
    page, d, hkv = case["page"], case["d"], case["hkv"]
    table = s["table"].tolist()

    def value(name, at, slot):
        x = s[name][at, :, slot].double()
        return x if s[name + "_scale"] is None else x * s[name + "_scale"][at, :, slot].double()[..., None]

    if case["op"] == "attend":
        nodes, hq = case["nodes"], case["hq"]
        parents, counts = _trees(case)
        out = torch.zeros(case["seqs"], nodes, hq, d, dtype=torch.float64, device=DEV)
        lse = torch.full((case["seqs"], nodes, hq), -math.inf, dtype=torch.float64, device=DEV)
        fill = s["fill"].tolist() if s["fill"] is not None else None
        for b, n in enumerate(s["lens"].tolist()):
            count = counts[b]
            if not count:
                continue
            at, slot, first = [], [], 0
            for p in range(_up(n + count, page)):
                if table[b][p] >= 0:
                    m = min(page, n + count - p * page, fill[table[b][p]] if fill else page)
                    at += [table[b][p]] * m
                    slot += range(m)
            first = len(at) - count  # the nodes' own rows are the last ones
            at, slot = torch.tensor(at).to(DEV), torch.tensor(slot).to(DEV)
            k, v = value("k", at, slot).transpose(0, 1), value("v", at, slot).transpose(0, 1)
            hidden = torch.zeros(count, len(at), dtype=torch.bool)
            hidden[:, first:] = True
            for i, seen in enumerate(_ancestors(parents[b][:count])):
                hidden[i, [first + j for j in seen]] = False
            hidden = hidden.to(DEV)
            q = s["q"][b, :count].double().reshape(count, hkv, -1, d)
            score = torch.einsum("chgd,htd->hgct", q, k) / math.sqrt(d)
            score.masked_fill_(hidden, -math.inf)
            lse[b, :count] = torch.logsumexp(score, -1).permute(2, 0, 1).reshape(count, hq)
            out[b, :count] = torch.einsum("hgct,htd->chgd", torch.softmax(score, -1), v).reshape(count, hq, d)
        return {"out": out, "lse": lse}
    if case["op"] == "compact":
        got = {name: s[name].clone() for name in ("k", "v", "k_scale", "v_scale") if s[name] is not None}
        lens = s["lens"].tolist()
        pairs = [(b, lens[b] + x, lens[b] + i) for b, p in enumerate(_paths(case)) for i, x in enumerate(p)]
        if pairs:
            here, there = ([(table[b][t // page], t % page) for b, t in ends] for ends in
                           ([(b, x) for b, x, _ in pairs], [(b, y) for b, _, y in pairs]))
            (a1, s1), (a2, s2) = (torch.tensor(x).to(DEV).T for x in (here, there))
            for name, x in got.items():
                x[a2, :, s2] = s[name][a1, :, s1]
        if case["store"] != "int8":
            return {"k": got["k"], "v": got["v"]}
        if not pairs:
            return {}
        return {name: got[name][a2, :, s2].double() * got[name + "_scale"][a2, :, s2].double()[..., None] for name in "kv"}
    idx = s["idx"].tolist()
    place = [(t, table[b][i // page], i % page) for t, (b, i) in enumerate(zip(s["seq"].tolist(), idx)) if i >= 0]
    token, at, slot = (torch.tensor(x).to(DEV) for x in zip(*place))
    tokens = len(idx)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]

    def turned(x, weight):
        x, rot = x.double(), case["rot"]
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / d + s["eps"]) * weight.double()
        head = x[..., :rot]
        if case["pairs"] == "halves":
            z = torch.complex(head[..., :rot // 2], head[..., rot // 2:]) * turn
            head = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous()) * turn
            head = torch.view_as_real(z).flatten(-2)
        return torch.cat([head, x[..., rot:]], -1)

    got = {"q": torch.zeros(tokens, case["hq"], d, dtype=torch.float64, device=DEV)}
    got["q"][token] = turned(s["q_new"], s["q_weight"])[token]
    for name, x in (("k", turned(s["k_new"], s["k_weight"])), ("v", s["v_new"].double())):
        if case["store"] == "int8":
            step = x.abs().amax(-1, keepdim=True) / 127
            near = torch.where(step > 0, torch.round(x / step.clamp(min=1e-300)), torch.zeros_like(x)) * step
            got[name] = torch.zeros(tokens, hkv, d, dtype=torch.float64, device=DEV)
            got[name][token] = near[token]
        else:
            got[name] = s[name].double()
            got[name][at, :, slot] = x[token]
    return got


def _exact_verify(s):
    """One request after the other, walking down from the sequence's end."""
    case, nodes = s["case"], s["case"]["nodes"]
    parents, counts = _trees(case)
    tokens, u = s["tokens"].tolist(), s["u"].double().tolist()
    path = torch.full((case["seqs"], nodes), -1, dtype=torch.int32)
    kept, picked = [], []
    for b in range(case["seqs"]):
        children = {}
        for i in range(counts[b]):
            children.setdefault(parents[b][i], []).append(i)
        at, taken = -1, []
        while True:
            p, mass, step = s["target"][b, at + 1].double(), 1.0, None
            for i in children.get(at, []):
                x = tokens[b][i]
                qx = float(s["draft"][b, at + 1, x].double()) if case["draft"] else 1.0
                if u[b][i] * mass * qx < float(p[x]):
                    step = i
                    break
                if case["draft"]:
                    rest = torch.clamp(p - mass * s["draft"][b, at + 1].double(), min=0)
                else:
                    rest = p.clone()
                    rest[x] = 0.0
                total = float(rest.sum())
                if total > 0:
                    p, mass = rest, total
            if step is None:
                break
            taken.append(step)
            at = step
        path[b, :len(taken)] = torch.tensor(taken, dtype=torch.int32)
        kept.append(len(taken))
        upto = torch.cumsum(p, 0)
        over = torch.nonzero(upto > u[b][nodes] * float(upto[-1]))
        picked.append(int(over[0]) if len(over) else int(torch.nonzero(p)[-1]))
    return {"path": path.to(DEV), "kept": _ints(kept), "token": _ints(picked)}
