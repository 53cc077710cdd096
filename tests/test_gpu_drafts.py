"""Drafted tokens: appending with norms, verification, and moving the rows that were taken, against the 64-bit oracle.

Bounds, from the arithmetic alone (u: unit roundoff of the output type):
* append with norm: the sum of dim squares in fp32 passes at most dim / 8 + 4 roundings for any element, the square root
  halves their effect, then one root, two products and three operations of the rotation: within (dim / 16 + 8) 2^-24 of sum
  |terms|, then one rounding to the stored type; an int8 code is within half a step of the value.
* verification: whole numbers, equal to the oracle's (both decide in 64 bits).
* compaction: the same bytes at other places.
"""
import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import drafts_oracle as O
from oracle import kv_oracle as K
from test_gpu_kv import BF16, DEV, F16, I8, U, c, full_table, kv, make_cache, rope, values  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def drafts():
    pkg("build").build()
    return pkg("drafts")


def ints(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to(DEV)


def some_trees(B, nodes, rng):
    return np.stack([[rng.integers(-1, i) if i else -1 for i in range(nodes)] for _ in range(B)]).reshape(B, nodes)


# ------------------------------------------------------------------------------------------------ append with norm

@pytest.mark.parametrize("dim,rot", [(64, 64), (64, 0), (96, 96), (96, 48), (128, 128), (128, 16), (192, 192), (256, 128)])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("dtype,store,wtype", [(BF16, BF16, BF16), (F16, F16, torch.float32), (BF16, I8, torch.float32), (F16, I8, F16)])
def test_append_norm(kv, dim, rot, pairs, dtype, store, wtype):  # noqa: F811
    g = torch.Generator().manual_seed(dim + rot)
    heads, hq, page, n, eps = 3, 5, 20, 37, 1e-5
    table, pages = full_table([60, 45, 0], page, g)
    cache = make_cache(kv, pages, heads, page, dim, store, g)
    fused = torch.randn(n, hq + 2 * heads, dim, generator=g) * torch.exp(2 * torch.randn(n, 1, 1, generator=g))
    fused[3] = 0
    fused[4] *= 1e-4                                       # eps counts
    fused = fused.to(DEV, dtype)
    q, k, v = fused[:, :hq], fused[:, hq:hq + heads], fused[:, hq + heads:]
    place = torch.randperm(105, generator=g)[:n]
    seq, idx = (place >= 60).int(), torch.where(place >= 60, place - 60, place).int()
    idx[5] = -1
    pos = torch.randint(0, 50, (n,), generator=g, dtype=torch.int32)
    table, seq, idx, pos = (x.to(DEV) for x in (table, seq, idx, pos))
    wq, wk = ((1 + 0.5 * torch.randn(dim, generator=g)).to(DEV, wtype) for _ in range(2))
    cs = rope(50, rot, g) if rot else None
    got = cache.append(k, v, table, idx, seq=seq, pos=pos, rope=cs, pairs=pairs, q=q, norm=(wq, wk), eps=eps)
    torch.cuda.synchronize()
    cache.check_status()
    cos, sin = (c(x)[c(pos)] for x in cs) if rot else (None, None)
    eq, mq = K.rotate(O.norm(c(q), c(wq), eps), cos, sin, rot, pairs)
    ek, mk = K.rotate(O.norm(c(k), c(wk), eps), cos, sin, rot, pairs)
    ev, mv = c(v), np.zeros_like(c(v))
    at = K.rows_of(c(table), page, c(seq), c(idx), pages)
    there = np.array([a is not None for a in at])
    u, es = U[dtype], (dim / 16 + 8) * 2.0 ** -24
    got = c(got)
    assert (got[~there] == 0).all() and there.sum() == n - 1
    tiny = 2.0 ** -25 if F16 in (dtype,) else 0.0
    assert (np.abs(got - eq) <= u * np.abs(eq) * (1 + 2 ** -8) + es * mq + tiny)[there].all()
    kk, vv = values(cache)
    for t, a in enumerate(at):
        if a is None:
            continue
        for have, want, mag in ((kk, ek, mk), (vv, ev, mv)):
            row, e = have[a[0], :, a[1]], want[t]
            if store == I8:
                step = np.abs(e).max(-1, keepdims=True) / 127
                bound = 0.5 * step + 2.0 ** -20 * 127 * step + es * (mag[t] + mag[t].max(-1, keepdims=True))
            else:
                bound = u * np.abs(e) * (1 + 2 ** -8) + es * mag[t] + tiny
            assert (np.abs(row - e) <= bound).all(), t


def test_append_norm_of_one_kind_of_heads(kv):  # noqa: F811
    """Only keys or only queries normed; without weights and rotation as the plain call; q in place; no query heads."""
    g = torch.Generator().manual_seed(3)
    table, pages = full_table([40, 40, 40], 8, g)
    table, idx = table.to(DEV), ints([7, 20, 39])
    x = [torch.randn(3, h, 64, generator=g).to(DEV, F16) for h in (4, 2, 2)]
    w = (1 + 0.5 * torch.randn(64, generator=g)).to(DEV, F16)
    cs = rope(64, 64, g)
    fresh = lambda: make_cache(kv, pages, 2, 8, 64, F16, torch.Generator().manual_seed(1))  # noqa: E731
    plain, both, only_k, only_q, none = (fresh() for _ in range(5))
    q0 = plain.append(x[1], x[2], table, idx, rope=cs, q=x[0])
    q1 = both.append(x[1], x[2], table, idx, rope=cs, q=x[0], norm=(w, w))
    q2 = only_k.append(x[1], x[2], table, idx, rope=cs, q=x[0], norm=(None, w))
    mine = x[0].clone()
    q3 = only_q.append(x[1], x[2], table, idx, rope=cs, q=mine, q_out=mine, norm=(w, None))
    q4 = none.append(x[1], x[2], table, idx, rope=cs, q=x[0], norm=(None, None))
    assert torch.equal(q0, q2) and torch.equal(q1, q3) and torch.equal(q0, q4) and not torch.equal(q0, q1)
    assert torch.equal(only_k.k, both.k) and torch.equal(only_q.k, plain.k) and torch.equal(none.k, plain.k)
    assert all(torch.equal(o.v, plain.v) for o in (both, only_k, only_q, none))
    keys = fresh()
    assert keys.append(x[1], x[2], table, idx, rope=cs, norm=(None, w)) is None
    assert torch.equal(keys.k, both.k)


def test_append_norm_refusals(kv):  # noqa: F811
    g = torch.Generator().manual_seed(4)
    cache = make_cache(kv, 4, 2, 16, 64, F16, g)
    t, n, k = ints(np.zeros((3, 2))), ints(np.zeros(3)), torch.zeros(3, 2, 64, dtype=F16, device=DEV)
    w = torch.ones(64, dtype=F16, device=DEV)
    learned = torch.ones(64, dtype=F16, device=DEV, requires_grad=True)
    wide = torch.ones(128, dtype=F16, device=DEV)
    for norm, q in (((w, w), None), ((w.to(BF16), None), k), ((w, w.float()), k), ((None, w[:32]), k), ((None, wide[::2]), k),
                    ((None, wide[4:68]), k), ((None, w.cpu()), k), ((None, learned), k), ((w.view(1, 64), None), k)):
        with pytest.raises(ValueError):
            cache.append(k, k, t, n, q=q, norm=norm)
    for eps in (0.0, -1.0, float("nan")):
        with pytest.raises(pkg("_lib").FvsError):
            cache.append(k, k, t, n, norm=(None, w), eps=eps)
    assert cache.launches == 0


# ------------------------------------------------------------------------------------------------ verification

def check_verify(drafts, target, parents, tokens, u, draft=None, counts=None):
    path, kept, token = drafts.verify(target, parents, tokens, u, draft=draft, counts=counts)
    torch.cuda.synchronize()
    B, nodes = tokens.shape
    up = np.broadcast_to(c(parents), (B, nodes))
    ep, ek, et = O.verify(c(target), up, c(tokens), c(u), None if draft is None else c(draft), None if counts is None else c(counts))
    np.testing.assert_array_equal(c(kept), ek)
    np.testing.assert_array_equal(c(path), ep)
    np.testing.assert_array_equal(c(token), et)
    return ek


def make_probabilities(B, nodes, vocab, dtype, g, spread=1.5, error=0.8):
    logits = torch.randn(B, nodes + 1, vocab, generator=g) * spread
    target = torch.softmax(logits, -1).to(DEV, dtype)
    draft = torch.softmax(logits + error * torch.randn(B, nodes + 1, vocab, generator=g), -1).to(DEV, dtype)
    return target, draft


def drawn(draft, parents, g):
    B, nodes = parents.shape
    rows = draft.float().cpu()[torch.arange(B)[:, None], torch.as_tensor(parents).long() + 1]
    if nodes == 0:
        return torch.zeros(B, 0, dtype=torch.int32, device=DEV)
    return torch.multinomial(rows.reshape(B * nodes, -1) + 1e-30, 1, generator=g).view(B, nodes).to(DEV, torch.int32)


@pytest.mark.parametrize("dtype", [torch.float32, F16, BF16])
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("B,nodes,vocab", [(70, 12, 31), (9, 40, 7), (5, 256, 11), (3, 6, 4099), (1, 7, 70001), (2, 3, 33333), (40, 0, 501),
                                           (33, 1, 1), (300, 4, 9001)])
def test_verify(drafts, dtype, with_draft, B, nodes, vocab):
    rng, g = np.random.default_rng(B), torch.Generator().manual_seed(vocab)
    parents = some_trees(B, nodes, rng)
    target, draft = make_probabilities(B, nodes, vocab, dtype, g)
    tokens = drawn(draft, parents, g)
    u = torch.rand(B, nodes + 1, generator=g).to(DEV)
    counts = ints(rng.integers(0, nodes + 2, B))
    kept = check_verify(drafts, target, ints(parents), tokens, u, draft if with_draft else None, counts)
    if B == 70:  # a small vocabulary: some paths are long, some empty
        assert kept.max() >= 2 and kept.min() == 0
    check_verify(drafts, target, ints(np.arange(nodes) - 1), tokens, u, draft if with_draft else None)


@pytest.mark.parametrize("with_draft", [True, False])
def test_verify_many_siblings(drafts, with_draft):
    """Residual after residual: wide levels whose tokens are refused one after the other, the same token more than once."""
    g = torch.Generator().manual_seed(5)
    B, nodes, vocab = 64, 30, 13
    parents = np.full((B, nodes), -1)
    parents[:, 20:] = 7
    target, draft = make_probabilities(B, nodes, vocab, torch.float32, g, error=2.0)
    tokens = drawn(draft, parents, g)
    u = 1 - torch.rand(B, nodes + 1, generator=g).to(DEV) ** 6 * 0.999 - 1e-6
    check_verify(drafts, target, ints(parents), tokens, u, draft if with_draft else None)


def test_verify_borders(drafts):
    """p = q is never refused, a token without probability never taken, u of 0 and near 1, sure rows, empty rows, padding."""
    vocab, near = 50, float(np.nextafter(np.float32(1), np.float32(0)))
    g = torch.Generator().manual_seed(6)
    target, draft = make_probabilities(6, 3, vocab, torch.float32, g)
    tokens = torch.randint(0, vocab, (6, 3), generator=g, dtype=torch.int32).to(DEV)
    chain = ints([-1, 0, 1])
    u = torch.full((6, 4), near, device=DEV)
    assert (check_verify(drafts, target, chain, tokens, u, target) == 3).all()
    u[:] = 0
    target[0, 0, int(tokens[0, 0])] = 0
    target[1, 1] = 0
    target[1, 1, int(tokens[1, 1])] = 1
    kept = check_verify(drafts, target, chain, tokens, u, draft)
    assert kept[0] == 0 and (kept[1:] == 3).all()
    target[2] = 0                                           # no probability anywhere
    target[3, 0, 5], target[3, 0, 6], target[3, 0, 7] = float("nan"), -1.0, float("inf")
    u[:] = near
    tokens[4, 0], tokens[5, 0] = -1, vocab
    for d in (draft, None):
        check_verify(drafts, target, chain, tokens, u, d)
    bad = ints([[0, 0, 1], [-1, 1, 0], [-2, -1, 0], [-1, 5, -1], [2, -1, 1], [-1, -1, -1]])
    check_verify(drafts, target, bad, tokens, u, draft)
    assert int(drafts.verify(target, chain, tokens, u)[2][2]) == -1
    u[:] = 1.0                                              # outside [0, 1): still a token
    check_verify(drafts, target, chain, tokens, u, draft)


def test_verify_rows_that_are_not_needed(drafts):
    """Rows behind nodes without children, and the draft's, hold anything; strided rows; shared and odd addresses."""
    g = torch.Generator().manual_seed(7)
    B, nodes, vocab = 8, 6, 1001
    parents = np.array([-1, -1, 0, 0, 1, 1])
    target, draft = make_probabilities(B, nodes, vocab, F16, g)
    tokens = drawn(draft, np.tile(parents, (B, 1)), g)
    u = torch.rand(B, nodes + 1, generator=g).to(DEV)
    draft[:, 3:] = float("nan")
    want = drafts.verify(target, ints(parents), tokens, u, draft=draft)
    check_verify(drafts, target, ints(parents), tokens, u, draft)
    room = torch.full((nodes + 1, B, vocab + 7), float("nan"), dtype=F16, device=DEV)
    view = room[:, :, 3:3 + vocab].transpose(0, 1)
    view.copy_(target)
    for a, b in zip(drafts.verify(view, ints(parents), tokens, u, draft=draft), want):
        assert torch.equal(a, b)
    one = target[:1].expand(B, nodes + 1, vocab)
    for a, b in zip(drafts.verify(one, ints(parents), tokens, u), drafts.verify(one.contiguous(), ints(parents), tokens, u)):
        assert torch.equal(a, b)


def test_verify_offsets_past_32_bits(drafts):
    g = torch.Generator().manual_seed(8)
    nodes, vocab = 2, 200003
    target = torch.zeros(3600, nodes + 1, vocab, dtype=F16, device=DEV)  # 2.2e9 elements
    small, draft = make_probabilities(1, nodes, vocab, F16, g)
    target[-1] = small[0]
    parents, u = ints([-1, 0]), torch.rand(3600, nodes + 1, generator=g).to(DEV)
    tokens = drawn(draft, np.array([[-1, 0]]), g).expand(3600, nodes).contiguous()
    path, kept, token = drafts.verify(target, parents, tokens, u)
    ep, ek, et = O.verify(c(small), [[-1, 0]], c(tokens[-1:]), c(u[-1:]))
    assert (c(token)[:-1] == -1).all() and (c(kept)[:-1] == 0).all()
    assert c(token)[-1] == et[0] and c(kept)[-1] == ek[0] and (c(path)[-1] == ep[0]).all()


def test_verify_graph_and_streams(drafts):
    g = torch.Generator().manual_seed(9)
    B, nodes, vocab = 12, 9, 5003
    parents = some_trees(B, nodes, np.random.default_rng(9))
    target, draft = make_probabilities(B, nodes, vocab, torch.float32, g)
    tokens, u = drawn(draft, parents, g), torch.rand(B, nodes + 1, generator=g).to(DEV)
    up = ints(parents)
    want = [x.clone() for x in drafts.verify(target, up, tokens, u, draft=draft)]
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        got = drafts.verify(target, up, tokens, u, draft=draft)
    u2 = torch.rand(B, nodes + 1, generator=g).to(DEV)
    torch.cuda.synchronize()
    for _ in range(3):
        graph.replay()
        with torch.cuda.stream(other):
            beside = drafts.verify(target, up, tokens, u2, draft=draft)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    check_verify(drafts, target, up, tokens, u2, draft)
    u.copy_(u2)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, beside))


def test_verify_refusals(drafts):
    f = lambda *s: torch.rand(*s, device=DEV)  # noqa: E731
    t, p, k, u = f(2, 4, 10), ints([-1, 0, 1]), ints(np.zeros((2, 3))), f(2, 4)
    learned = f(2, 4, 10).requires_grad_()
    for args, more in (((t.double(), p, k, u), {}), ((t[0], p, k, u), {}), ((t.cpu(), p, k, u), {}),
                       ((f(2, 4, 20)[..., ::2], p, k, u), {}), ((t, p[:2], k, u), {}), ((t, p.long(), k, u), {}),
                       ((t, p, k[:1], u), {}), ((t, p, k.long(), u), {}), ((t, p, k, u[:, :3]), {}), ((t, p, k, u.double()), {}),
                       ((t, p, k, u), dict(draft=t.half())), ((t, p, k, u), dict(draft=t[:, :3])), ((learned, p, k, u), {}),
                       ((t, p, k, u), dict(counts=ints([1]))), ((f(1, 258, 4), ints(np.arange(257) - 1), ints(np.zeros((1, 257))), f(1, 258)), {}),
                       ((f(2, 0, 10), ints(np.zeros(0)), ints(np.zeros((2, 0))), f(2, 0)), {})):
        with pytest.raises(ValueError):
            drafts.verify(*args, **more)
    empty = drafts.verify(f(0, 4, 10), p, ints(np.zeros((0, 3))), f(0, 4))
    assert [tuple(x.shape) for x in empty] == [(0, 3), (0,), (0,)]


# ------------------------------------------------------------------------------------------------ compaction

def rising(rng, nodes, kept):
    return np.concatenate([np.sort(rng.choice(nodes, kept, replace=False)), np.full(nodes - kept, -1)]).astype(np.int32)


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("store", [BF16, F16, I8])
@pytest.mark.parametrize("page,nodes", [(16, 9), (1, 5), (7, 70), (64, 256)])
def test_compact(kv, dim, store, page, nodes):  # noqa: F811
    rng, g = np.random.default_rng(dim + page), torch.Generator().manual_seed(nodes)
    B, heads = 6, 3
    lens = rng.integers(0, 90, B)
    table, pages = full_table([int(n) + nodes for n in lens], page, g)
    cache = make_cache(kv, pages, heads, page, dim, store, g, token_major=page == 16)
    path = np.stack([rising(rng, nodes, k) for k in (nodes, nodes - 1, nodes // 2, 1, 0, min(nodes, 33))])
    names = ["k", "v"] + (["k_scale", "v_scale"] if store == I8 else [])
    want = [O.compact(c(getattr(cache, n)), c(table), lens, path, page) for n in names]
    cache.compact(table.to(DEV), ints(lens), ints(path))
    torch.cuda.synchronize()
    for n, w in zip(names, want):
        np.testing.assert_array_equal(c(getattr(cache, n)), w)
    cache.check_status()


def test_compact_overlapping_moves_many_times(kv):  # noqa: F811
    """Shifts by one, whose every place is the next row's source."""
    g = torch.Generator().manual_seed(10)
    B, nodes, page = 80, 256, 32
    table, pages = full_table([nodes + 40] * B, page, g)
    cache = make_cache(kv, pages, 2, page, 64, F16, g)
    path = np.tile(np.append(np.arange(1, nodes), -1), (B, 1))
    k, v = c(cache.k), c(cache.v)
    for _ in range(3):
        cache.compact(table.to(DEV), ints([40] * B), ints(path))
        k, v = (O.compact(x, c(table), [40] * B, path, page) for x in (k, v))
    torch.cuda.synchronize()
    np.testing.assert_array_equal(c(cache.k), k)
    np.testing.assert_array_equal(c(cache.v), v)


def test_compact_holes_and_bad_paths(kv):  # noqa: F811
    FvsError = pkg("_lib").FvsError
    g = torch.Generator().manual_seed(11)
    page, nodes = 4, 8
    table, pages = full_table([16] * 3, page, g)
    cache = make_cache(kv, pages, 2, page, 64, F16, g)
    holes = c(table).copy()
    holes[0, 3], holes[1, 2] = -1, -1
    path = np.tile(np.array([1, 3, 4, 7, -1, -1, -1, -1]), (3, 1))
    want = O.compact(c(cache.k), holes, [7, 8, 5], path, page)
    cache.compact(ints(holes), ints([7, 8, 5]), ints(path))
    np.testing.assert_array_equal(c(cache.k), want)
    cache.check_status()
    # an entry that does not rise, one past the nodes, a length that is none, one past the table, a page past the cache
    worse = c(table).copy()
    worse[0, 1] = pages + 3
    for bad, lens, tab, upto in (([1, 3, 3, 7], 5, table, 2), ([2, 1, 5, 6], 5, table, 1), ([1, 8, 9, 10], 5, table, 1),
                                 ([0, 2, 4, 5], -1, table, 0), ([1, 2, 4, 5], 14, table, 1), ([1, 2, 4, 5], 2 ** 31 - 2, table, 0)):
        row = np.tile(np.array(bad + [-1] * 4), (3, 1))
        good = row.copy()
        good[:, upto:] = -1
        want = O.compact(c(cache.k), c(tab), [max(0, lens) if upto else 0] * 3, good, page)
        cache.compact(ints(c(tab)), ints([lens] * 3), ints(row))
        with pytest.raises(FvsError):
            cache.check_status()
        np.testing.assert_array_equal(c(cache.k), want)
    cache.compact(ints(worse), ints([4] * 3), ints(np.tile([1, 2, -1, -1, -1, -1, -1, -1], (3, 1))))
    with pytest.raises(FvsError):
        cache.check_status()


def test_compact_refusals_and_empty_calls(kv):  # noqa: F811
    g = torch.Generator().manual_seed(12)
    cache = make_cache(kv, 4, 2, 16, 64, F16, g)
    t, n, p = ints(np.zeros((3, 2))), ints(np.zeros(3)), ints(np.zeros((3, 5)))
    for args in ((t.long(), n, p), (t, n[:2], p), (t, n.long(), p), (t, n, p[:2]), (t, n, p.long()), (t, n, p[0]),
                 (t, n, ints(np.zeros((3, 10)))[:, ::2]), (t, n, p.cpu())):
        with pytest.raises(ValueError):
            cache.compact(*args)
    assert cache.launches == 0
    k0 = cache.k.clone()
    cache.compact(t, n, ints(np.zeros((3, 0))))
    cache.compact(t[:0], n[:0], p[:0])
    assert torch.equal(cache.k, k0)


# ------------------------------------------------------------------------------------------------ together

def test_a_step_as_it_is_used(kv, drafts):  # noqa: F811
    """Two steps of append with norm, tree attention, verification and compaction, eagerly and in one captured graph, against the
    oracles one after the other."""
    g, rng = torch.Generator().manual_seed(20), np.random.default_rng(20)
    B, heads, group, dim, page, nodes, vocab = 5, 2, 4, 128, 16, 9, 301
    hq = heads * group
    shape = [int(rng.integers(-1, i)) if i else -1 for i in range(nodes)]
    lens0 = [30, 0, 77, 16, 5]
    table, pages = full_table([n + 3 * nodes for n in lens0], page, g)
    start = make_cache(kv, pages, heads, page, dim, BF16, g)
    norm = tuple((1 + 0.2 * torch.randn(dim, generator=g)).to(DEV, BF16) for _ in range(2))
    cs = rope(200, dim, g)
    parents, depth = ints(shape), [0] * nodes
    for i, p in enumerate(shape):
        depth[i] = depth[p] + 1 if p >= 0 else 0
    table, depth, seq = table.to(DEV), ints(depth), ints(np.repeat(np.arange(B), nodes))
    fused = [(torch.randn(B * nodes, hq + 2 * heads, dim, generator=g)).to(DEV, BF16) for _ in range(2)]
    logits = torch.randn(B, nodes + 1, vocab, generator=g).to(DEV)
    draft = torch.softmax(logits + 0.5 * torch.randn(B, nodes + 1, vocab, generator=g).to(DEV), -1)
    tokens = [drawn(draft, np.tile(shape, (B, 1)), g) for _ in range(2)]
    u = [torch.rand(B, nodes + 1, generator=g).to(DEV) for _ in range(2)]
    mix = torch.randn(hq * dim, vocab, generator=g).to(DEV) / 8

    def step(cache, lens, i):
        x = fused[i]
        at = (lens[:, None] + torch.arange(nodes, dtype=torch.int32, device=DEV)).view(-1)
        q = cache.append(x[:, hq:hq + heads], x[:, hq + heads:], table, at, seq=seq, pos=(lens[:, None] + depth).view(-1), rope=cs,
                         q=x[:, :hq], norm=norm)
        out, lse = cache.attend_tree(q.view(B, nodes, hq, dim), table, lens, parents)
        behind = torch.cat([logits[:, :1], logits[:, 1:] + out.reshape(B, nodes, -1).float() @ mix], 1)
        target = torch.softmax(behind, -1)
        path, kept, token = drafts.verify(target, parents, tokens[i], u[i], draft=draft)
        before = cache.k.clone(), cache.v.clone()
        cache.compact(table, lens, path)
        return dict(q=q, out=out, lse=lse, target=target, path=path, kept=kept, token=token, k=before[0], v=before[1], lens=lens + kept)

    fresh = lambda: kv.PagedKV(start.k.clone(), start.v.clone())  # noqa: E731
    eager, captured = fresh(), fresh()
    lens, got = ints(lens0), []
    for i in range(2):
        got.append(step(eager, lens, i))
        lens = got[-1]["lens"]
    torch.cuda.synchronize()
    first = ints(lens0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one = step(captured, first, 0)
        two = step(captured, one["lens"], 1)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, (one, two)):
        assert all(torch.equal(a[name], b[name]) for name in a)
    assert torch.equal(eager.k, captured.k) and torch.equal(eager.v, captured.v)
    eager.check_status()
    lens = np.array(lens0)
    for i, s in enumerate(got):
        k, v = c(s["k"]), c(s["v"])
        eo, el, pv, _ = O.attend_tree(c(s["q"]).reshape(B, nodes, hq, dim), k, v, c(table), lens, np.tile(shape, (B, 1)), None, dim ** -0.5)
        assert np.abs(c(s["out"]) - eo).max() <= 2.0 ** -8 * np.abs(eo).max() + 2.0 ** -14 * pv.max()
        ep, ek, et = O.verify(c(s["target"]), np.tile(shape, (B, 1)), c(tokens[i]), c(u[i]), c(draft))
        np.testing.assert_array_equal(c(s["path"]), ep)
        np.testing.assert_array_equal(c(s["token"]), et)
        want = O.compact(k, c(table), lens, ep, page)
        after = c(got[i + 1]["k"]) if i == 0 else c(eager.k)
        stay = np.ones(k.shape, bool)
        if i == 0:                                          # the next step has appended behind its own start
            for b in range(B):
                for t in range(int(lens[b] + ek[b]), int(lens[b] + ek[b] + nodes)):
                    stay[c(table)[b][t // page], :, t % page] = False
        np.testing.assert_array_equal(after[stay], want[stay])
        lens = lens + ek


def test_example_answers_with_drafts():
    import importlib.util
    import os

    from conftest import REPO
    spec = importlib.util.spec_from_file_location("answer_with_drafts", os.path.join(REPO, "examples", "answer_with_drafts.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    worst, taken = m.main(steps=4)
    assert worst < 2 ** -7 and taken > 0
