"""Answering from found passages with drafted tokens: each step takes as many of a small model's tokens as the target model's
own probabilities allow.

    python examples/answer_with_drafts.py

Behind the passages that a search found (see answer_from_passages.py) each sequence has one pending token, drawn but not yet
in the cache.  A step drafts a tree behind it, appends the pending token and the tree's nodes (their heads normed and
rotated in the same pass, at the positions that their depth gives), attends over the cache and each node's ancestors
(`attend_tree`), takes nodes by the target's probabilities (`drafts.verify`) and moves the rows of the taken ones together
(`compact`).  The pending token is node 0 of the attention's tree and always taken, so the rows of its outputs are those that
`verify` looks at: row 0 behind the pending token, row i + 1 behind draft i.  The target here is one attention layer of random
weights, the draft model a table of next tokens; a real target does the same in each layer, with a cache for each."""
import importlib
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def pkg(name):
    return importlib.import_module("fanarvse-paper_b200." + name)


def main(steps=6, found=3, device="cuda"):
    from __graft_entry__ import _tiny_index
    g = torch.Generator().manual_seed(0)
    ds, _, _, _, index = _tiny_index(device)
    engine = pkg("engine").EngineB200I8(index)
    kv, drafts = pkg("kvcache"), pkg("drafts")
    rand = lambda *s: torch.randn(*s, generator=g).to(device, torch.bfloat16)
    ints = lambda x: torch.as_tensor(x, dtype=torch.int32).to(device)

    # the target: hidden size, heads, key heads, head dim, vocabulary; the draft model: next-token logits
    hidden, hq, heads, dim, page, vocab = 256, 8, 2, 64, 16, 50
    embed, wqkv = rand(vocab, hidden), rand(hidden, (hq + 2 * heads) * dim) / math.sqrt(hidden)
    wo, norm = rand(hq * dim, hidden) / math.sqrt(hq * dim), (1 + 0.1 * rand(dim), 1 + 0.1 * rand(dim))
    angle = torch.arange(512)[:, None] * 10000.0 ** (-torch.arange(0, dim, 2) / dim)
    rope = (angle.cos().to(device), angle.sin().to(device))
    guess = torch.softmax((embed.float() @ embed.float().T) / 16 + torch.randn(vocab, vocab, generator=g).to(device), -1)

    # the passages that the queries find: one page each, their keys and values stored ahead of any query
    B = 6
    ids, _, _ = engine.search(ds["queries"][:B].contiguous(), 40, 1.25, 12, found)
    length = torch.arange(index.N) % page + 1
    own_pages = -(-steps * 8 // page)
    fill = ints(torch.cat([length, torch.full((B * own_pages,), page)]))
    cache = kv.PagedKV.empty(index.N + B * own_pages, heads, page, dim, device=device, fill=fill)
    pages_of = ints(torch.arange(index.N)).view(-1, 1)
    idx = torch.cat([torch.arange(n) for n in length.tolist()])
    k, v = (rand(len(idx), heads, dim) for _ in range(2))
    cache.append(k, v, pages_of, ints(idx), seq=ints(torch.repeat_interleave(torch.arange(index.N), length)), rope=rope,
                 norm=(None, norm[1]))
    own = ints(torch.arange(index.N, index.N + B * own_pages)).view(B, own_pages)
    table = kv.passage_table(ids, pages_of, own)

    # a tree of drafts behind the pending token, and the attention's tree: the pending token before it
    shape = [-1, -1, 0, 0, 2]
    parents, nodes = ints(shape), len(shape)
    tree = ints([-1] + [p + 1 for p in shape])
    depth = [0]
    for p in shape:
        depth.append(depth[p + 1] + 1)
    depth = ints(depth)
    lens = torch.full((B,), found * page, dtype=torch.int32, device=device)
    pos = torch.full((B,), page, dtype=torch.int32, device=device)
    pending = ints(torch.randint(0, vocab, (B,), generator=g))
    row = torch.arange(B, device=device)
    answer, worst = [], 0.0
    for step in range(steps):
        # draft: each node's token from the draft model's distribution behind its parent
        tokens = torch.empty(B, nodes + 1, dtype=torch.int32, device=device)
        tokens[:, 0] = pending
        for i, p in enumerate(shape):
            draw = torch.rand(B, 1, generator=g).to(device)
            tokens[:, i + 1] = torch.searchsorted(guess[tokens[:, p + 1].long()].cumsum(-1), draw)[:, 0].clamp(max=vocab - 1)
        # the target: one call of each kind for all nodes
        x = embed[tokens.long()].view(B * (nodes + 1), hidden)
        qkv = (x @ wqkv).view(-1, hq + 2 * heads, dim)
        at = (lens[:, None] + torch.arange(nodes + 1, device=device, dtype=torch.int32)).view(-1)
        q = cache.append(qkv[:, hq:hq + heads], qkv[:, hq + heads:], table, at,
                         seq=torch.repeat_interleave(row, nodes + 1).int(), pos=(pos[:, None] + depth).view(-1), rope=rope,
                         q=qkv[:, :hq], norm=norm)
        out, _ = cache.attend_tree(q.view(B, nodes + 1, hq, dim), table, lens, tree)
        if step == steps - 1:
            worst = against_plain(cache, q.view(B, nodes + 1, hq, dim), out, table, lens, tree)
        h = x + out.reshape(B * (nodes + 1), -1) @ wo
        target = torch.softmax((h @ embed.T).float() / 16, -1).view(B, nodes + 1, vocab)
        u = torch.rand(B, nodes + 1, generator=g).to(device)
        path, kept, token = drafts.verify(target, parents, tokens[:, 1:].contiguous(), u, draft=guess[tokens.long()])
        # the pending token and the taken nodes stay, one behind the other; the drawn token is pending now
        taken = torch.cat([torch.zeros_like(path[:, :1]), torch.where(path >= 0, path + 1, path)], 1)
        cache.compact(table, lens, taken)
        answer.append((tokens, taken, kept))
        lens, pos, pending = lens + kept + 1, pos + kept + 1, token
    cache.check_status()
    taken = sum(int(kept.sum()) for *_, kept in answer)
    print(f"{steps} steps of {B} sequences: {taken} of {steps * B * nodes} drafted tokens taken, {steps * B} drawn by the target; "
          f"largest difference of the last step's attention from plain products {worst:.5f} of the largest output")
    return worst, taken


def against_plain(cache, q, out, table, lens, tree):
    """Each node's attention as plain products over the rows that it sees."""
    B, nodes, hq, dim = q.shape
    sees = []
    for i, p in enumerate(tree.tolist()):
        sees.append((sees[p] if p >= 0 else []) + [i])
    worst = 0.0
    for b in range(B):
        n = int(lens[b])
        t = torch.arange(n + nodes, dtype=torch.int32, device=q.device)
        p = table[b, (t // cache.page).long()]
        there = (p >= 0) & (t % cache.page < cache.fill[p.clamp(min=0).long()])
        k, v = cache.read(table[b:b + 1], t, seq=torch.zeros_like(t), dtype=torch.float32)
        k, v = (x.repeat_interleave(hq // cache.heads, 1) for x in (k, v))
        for i in range(nodes):
            seen = there.clone()
            seen[n:] &= torch.tensor([j in sees[i] for j in range(nodes)], device=q.device)
            w = torch.softmax(torch.einsum("hd,thd->ht", q[b, i].float(), k[seen]) / math.sqrt(dim), 1)
            plain = torch.einsum("ht,thd->hd", w, v[seen])
            worst = max(worst, float((plain - out[b, i].float()).abs().max() / plain.abs().max()))
    return worst


if __name__ == "__main__":
    sys.exit(0 if main()[0] < 2 ** -7 else 1)
