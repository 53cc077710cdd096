"""Answering from found passages: an index search, its passages' cached keys and values, and a decoding loop over them.

    python examples/answer_from_passages.py

Ahead of any query, the keys and values of every passage are stored in pages of one cache as int8 codes (`append`, with the
passage's own positions).  A query's search returns passage ids, which become the first part of a page table
(`passage_table`); the model's new tokens go to pages of the sequence's own behind them.  Each step of the loop appends
one token per sequence (its query and key rotated on the way) and attends over everything before it.  The model here is
one attention layer of random weights behind a norm; a real one does the same in each layer, with a cache for each."""
import importlib
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def pkg(name):
    return importlib.import_module("fanarvse-paper_b200." + name)


def main(steps=8, found=4, device="cuda"):
    from __graft_entry__ import _tiny_index
    g = torch.Generator().manual_seed(0)
    ds, _, _, _, index = _tiny_index(device)
    engine = pkg("engine").EngineB200I8(index)
    kv = pkg("kvcache")
    rand = lambda *s: torch.randn(*s, generator=g).to(device, torch.bfloat16)

    # a layer: hidden size, heads, key heads, head dim
    hidden, hq, heads, dim, page = 256, 8, 2, 64, 16
    wqkv, wo = rand(hidden, (hq + 2 * heads) * dim) / math.sqrt(hidden), rand(hq * dim, hidden) / math.sqrt(hq * dim)
    angle = torch.arange(512)[:, None] * 10000.0 ** (-torch.arange(0, dim, 2) / dim)
    rope = (angle.cos().to(device), angle.sin().to(device))

    # the passages that the queries find, in pages: passage i has length[i] tokens
    B = 6
    ids, _, _ = engine.search(ds["queries"][:B].contiguous(), 40, 1.25, 12, found)
    stored = torch.unique(ids[ids >= 0])
    length = torch.randint(5, 40, (len(stored),), generator=g)
    need = (length + page - 1) // page
    first = torch.cumsum(need, 0) - need
    own_pages = -(-steps // page)
    pages = int(need.sum()) + B * own_pages
    fill = torch.full((pages,), page, dtype=torch.int32)
    pages_of = torch.full((index.N, int(need.max())), -1, dtype=torch.int32)
    for i, p in enumerate(stored.tolist()):
        pages_of[p, :need[i]] = torch.arange(first[i], first[i] + need[i], dtype=torch.int32)
        fill[first[i] + need[i] - 1] = length[i] - (need[i] - 1) * page
    pages_of = pages_of.to(device)
    cache = kv.PagedKV.empty(pages, heads, page, dim, dtype=torch.int8, device=device, fill=fill.to(device))

    tokens = int(length.sum())
    x = rand(tokens, hidden)
    qkv = (x @ wqkv).view(tokens, hq + 2 * heads, dim)
    seq = torch.repeat_interleave(torch.arange(len(stored)), length).to(device, torch.int32)
    idx = torch.cat([torch.arange(n) for n in length]).to(device, torch.int32)
    cache.append(qkv[:, hq:hq + heads], qkv[:, hq + heads:], pages_of[stored].contiguous(), idx, seq=seq, rope=rope)

    # the decoding loop
    own = torch.arange(pages - B * own_pages, pages, dtype=torch.int32, device=device).view(B, own_pages)
    table = kv.passage_table(ids, pages_of, own)
    at = torch.full((B,), found * pages_of.shape[1] * page, dtype=torch.int32, device=device)   # behind the passages
    pos = torch.full((B,), 64, dtype=torch.int32, device=device)
    lens = at + 1
    h = rand(B, hidden)
    for _ in range(steps):
        x = (h.float() * h.float().square().mean(1, keepdim=True).rsqrt()).to(h.dtype)
        qkv = (x @ wqkv).view(B, hq + 2 * heads, dim)
        q = cache.append(qkv[:, hq:hq + heads], qkv[:, hq + heads:], table, at, pos=pos, rope=rope, q=qkv[:, :hq])
        out, lse = cache.attend(q, table, lens)
        h = h + out.reshape(B, -1) @ wo
        for n in (at, pos, lens):
            n.add_(1)
    cache.check_status()

    # the last step again from the cache's values as plain products
    lens = lens - 1
    worst = 0.0
    for b in range(B):
        t = torch.arange(int(lens[b]), dtype=torch.int32, device=device)
        p = table[b, (t // page).long()]
        seen = (p >= 0) & (t % page < cache.fill[p.clamp(min=0).long()])
        k, v = cache.read(table[b:b + 1], t[seen].contiguous(), seq=torch.zeros(int(seen.sum()), dtype=torch.int32, device=device))
        k, v = (z.repeat_interleave(hq // heads, 1) for z in (k, v))
        w = torch.softmax(torch.einsum("hd,thd->ht", q[b].float(), k) / math.sqrt(dim), 1)
        plain = torch.einsum("ht,thd->hd", w, v)
        worst = max(worst, float((plain - out[b].float()).abs().max() / plain.abs().max()))
    print(f"{len(stored)} passages of {tokens} tokens in {pages} pages; {steps} steps of {B} sequences; largest difference "
          f"from plain products {worst:.5f} of the largest output")
    return worst


if __name__ == "__main__":
    sys.exit(0 if main() < 2 ** -7 else 1)
