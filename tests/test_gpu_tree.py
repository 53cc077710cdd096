"""Attention of trees of drafted tokens over a paged cache, against the 64-bit oracle.

Bounds, from the arithmetic alone (u: unit roundoff of the output type):
* a score is off by es <= (dim + 4) 2^-23 scale sum |q k| (fp32 sums; the tensor cores may cut instead of round), which
  changes its weight by a factor e^(es);
* a weight enters the second product as two parts of the 16-bit type: 2^-17 of it with bf16, 2^-21 with fp16, where weights
  below 2^-25 of the largest lose more (2^-36 of the largest, absolute); the exponential is within 2^-21;
* sums over L keys in fp32, cut or rounded: (L + 64) 2^-22 of sum p |v|; one rounding of the output.
"""
import threading
import weakref

import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import drafts_oracle as O
from test_gpu_drafts import ints, some_trees
from test_gpu_kv import BF16, DEV, F16, I8, U, c, full_table, kv, make_cache, values  # noqa: F401

pytestmark = pytest.mark.gpu


def check_tree(cache, q, table, lens, parents, counts=None, scale=None, got=None):
    out, lse = got or cache.attend_tree(q, table, lens, parents, counts=counts, scale=scale)
    torch.cuda.synchronize()
    d = cache.dim
    scale = 1 / np.sqrt(d) if scale is None else scale
    k, v = values(cache)
    up = np.broadcast_to(c(parents), q.shape[:2])
    eo, el, pv, mag = O.attend_tree(c(q), k, v, c(table), c(lens), up, None if counts is None else c(counts), scale,
                                    None if cache.fill is None else c(cache.fill))
    out, lse = c(out), c(lse)
    L = int(max(1, c(lens).max() + q.shape[1]))
    es = (d + 4) * 2.0 ** -23 * mag
    part = 2.0 ** -17 if BF16 in (q.dtype,) or cache.dtype == I8 else 2.0 ** -21
    u = U[q.dtype]
    tiny = 2.0 ** -25 if q.dtype == F16 else 0.0
    tol = u * np.abs(eo) + (part + 2 * es[..., None] + 2.0 ** -20 + (L + 64) * 2.0 ** -22) * pv * 1.01 + tiny + 2.0 ** -36 * np.abs(np.nan_to_num(v)).max()
    empty = np.isinf(el)
    assert (out[empty] == 0).all() and np.array_equal(np.isneginf(lse), empty)
    assert np.isfinite(out).all()
    worst = (np.abs(out - eo) / tol).max()
    assert worst <= 1, f"out is {worst:.2f} of its bound"
    tol = 2 * es + (L + 64) * 2.0 ** -22 + 2.0 ** -20 * (1 + np.abs(np.where(empty, 0, el)))
    worst = (np.abs(lse[~empty] - el[~empty]) / tol[~empty]).max(initial=0)
    assert worst <= 1, f"lse is {worst:.2f} of its bound"
    cache.check_status()


def setup(kv, lens, nodes, heads, group, page, dim, dtype, store, g, **more):  # noqa: F811
    table, pages = full_table([n + nodes for n in lens], page, g)
    cache = make_cache(kv, pages, heads, page, dim, store, g, **more)
    q = (torch.randn(len(lens), nodes, heads * group, dim, generator=g) * 1.5).to(DEV, dtype)
    return cache, q, table.to(DEV), ints(lens)


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype,store", [(BF16, BF16), (F16, F16), (BF16, I8), (F16, I8)])
@pytest.mark.parametrize("heads,group,nodes", [(2, 1, 5), (1, 7, 20), (2, 4, 64)])
def test_tree_types_and_dims(kv, dim, dtype, store, heads, group, nodes):  # noqa: F811
    g, rng = torch.Generator().manual_seed(dim + heads), np.random.default_rng(dim)
    lens = [0, 1, 17, 63, 64, 127, 128, 200, 391]
    cache, q, table, n = setup(kv, lens, nodes, heads, group, 16, dim, dtype, store, g)
    check_tree(cache, q, table, n, ints(some_trees(len(lens), nodes, rng)))


@pytest.mark.parametrize("nodes,group", [(1, 1), (1, 16), (2, 3), (31, 1), (33, 2), (128, 1), (129, 1), (43, 3), (32, 8), (64, 16),
                                         (256, 1), (256, 3), (255, 5), (100, 71)])
@pytest.mark.parametrize("store", [BF16, I8])
def test_tree_rows(kv, nodes, group, store):  # noqa: F811
    """Fewer rows than a warp, one more than a tile, several tiles; one tree for all and a chain."""
    g, rng = torch.Generator().manual_seed(nodes + group), np.random.default_rng(nodes)
    lens = [300, 45, 0]
    cache, q, table, n = setup(kv, lens, nodes, 2, group, 32, 64, BF16, store, g)
    check_tree(cache, q, table, n, ints(some_trees(1, nodes, rng)[0]))
    check_tree(cache, q, table, n, ints(np.arange(nodes) - 1))
    check_tree(cache, q, table, n, ints(np.full(nodes, -1)), counts=ints([nodes // 2, 0, max(0, nodes - 1)]))


@pytest.mark.parametrize("page", [1, 3, 7, 16, 20, 48, 100, 256])
@pytest.mark.parametrize("store", [F16, I8])
def test_tree_page_sizes(kv, page, store):  # noqa: F811
    g, rng = torch.Generator().manual_seed(page), np.random.default_rng(page)
    lens = [page - 1, page, page + 1, 5 * page, 333, 0, 1000]
    cache, q, table, n = setup(kv, lens, 12, 2, 3, page, 128, F16, store, g, token_major=page == 16)
    check_tree(cache, q, table, n, ints(some_trees(len(lens), 12, rng)), counts=ints([12, 3, 0, 1, 12, 12, 7]))


@pytest.mark.parametrize("store", [BF16, I8])
@pytest.mark.parametrize("page", [5, 16, 64])
@pytest.mark.parametrize("dim", [64, 192])
def test_tree_holes_fill_and_what_memory_holds(kv, page, store, dim):  # noqa: F811
    g, rng = torch.Generator().manual_seed(page), np.random.default_rng(page)
    B, nodes, w = 7, 9, 12
    own = -(-nodes // page) + 1
    pages = B * (w + own) + 2
    perm = torch.randperm(pages - 2, generator=g).view(B, w + own).int()
    table = perm.clone()
    table[:, :w][torch.rand(B, w, generator=g) < 0.3] = -1
    table[2, :w] = -1
    fill = torch.randint(0, page + 1, (pages,), generator=g, dtype=torch.int32)
    fill[perm[:, w:].reshape(-1).long()] = page
    lens = torch.full((B,), w * page, dtype=torch.int32)
    lens[3] += 1
    cache = make_cache(kv, pages, 2, page, dim, store, g, fill=fill.to(DEV))
    # every slot that nothing sees holds not-a-numbers
    seen = torch.zeros(pages, page, dtype=torch.bool)
    for b in range(B):
        for t in range(int(lens[b]) + nodes):
            p = int(table[b, t // page])
            if p >= 0 and t % page < int(fill[p]):
                seen[p, t % page] = True
    seen = seen.to(DEV)
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        (x if s is None else s).masked_fill_(~seen[:, None, :, None] if s is None else ~seen[:, None], float("nan"))
    q = torch.randn(B, nodes, 6, dim, generator=g).to(DEV, BF16)
    check_tree(cache, q, table.to(DEV), lens.to(DEV), ints(some_trees(B, nodes, rng)))


@pytest.mark.parametrize("dtype,store", [(F16, F16), (BF16, BF16), (BF16, I8)])
@pytest.mark.parametrize("B,heads,group,dim,nodes,longest", [(1, 1, 1, 64, 1, 20000), (1, 8, 4, 128, 8, 9000), (1, 2, 4, 128, 64, 5000),
                                                             (3, 2, 16, 96, 5, 4099), (2, 1, 4, 256, 30, 3001), (5, 3, 2, 192, 65, 700)])
def test_tree_splits_over_the_length(kv, dtype, store, B, heads, group, dim, nodes, longest):  # noqa: F811
    g, rng = torch.Generator().manual_seed(dim), np.random.default_rng(dim)
    lens = [longest - i * (longest // 3) for i in range(B)] if B <= 3 else [longest] * B
    cache, q, table, n = setup(kv, lens, nodes, heads, group, 64, dim, dtype, store, g)
    check_tree(cache, q, table, n, ints(some_trees(B, nodes, rng)))


@pytest.mark.parametrize("dtype,store,group,dim,nodes", [(BF16, BF16, 2, 64, 3), (F16, I8, 1, 128, 40), (F16, F16, 8, 64, 33)])
def test_tree_one_item_over_every_sm(kv, dtype, store, group, dim, nodes):  # noqa: F811
    """One key head of a long context: as many shares as the GPU has places, some of them behind a page that is not there."""
    g, rng = torch.Generator().manual_seed(11), np.random.default_rng(11)
    cache, q, table, n = setup(kv, [90001], nodes, 1, group, 64, dim, dtype, store, g)
    table[0, 200:900] = -1
    check_tree(cache, q, table, n, ints(some_trees(1, nodes, rng)))


@pytest.mark.parametrize("B,lens", [(300, (0, 300)), (900, (0, 40)), (1500, (0, 3)), (129, (0, 2000))])
def test_tree_many_sequences(kv, B, lens):  # noqa: F811
    g, rng = torch.Generator().manual_seed(B), np.random.default_rng(B)
    n = list(rng.integers(*lens, B))
    cache, q, table, n = setup(kv, n, 4, 1, 2, 16, 64, F16, F16, g)
    check_tree(cache, q, table, n, ints(some_trees(B, 4, rng)), counts=ints(rng.integers(0, 5, B)))


def test_tree_batches_of_changing_size(kv):  # noqa: F811
    """Calls on one stream share a workspace."""
    g, rng = torch.Generator().manual_seed(3), np.random.default_rng(3)
    for B, nodes, longest in ((1, 64, 4000), (9, 5, 700), (1, 8, 6000), (40, 3, 100), (2, 200, 1000)):
        cache, q, table, n = setup(kv, list(rng.integers(1, longest, B)), nodes, 2, 4, 16, 128, BF16, BF16, g)
        check_tree(cache, q, table, n, ints(some_trees(B, nodes, rng)))


@pytest.mark.parametrize("dtype,store", [(F16, F16), (BF16, BF16), (F16, I8)])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 5.0])
def test_tree_scores_far_apart(kv, dtype, store, scale):  # noqa: F811
    """Scores that rise and fall by hundreds, a scale of its own, below zero or zero."""
    g, rng = torch.Generator().manual_seed(4), np.random.default_rng(4)
    cache, q, table, n = setup(kv, [900, 130], 10, 2, 2, 16, 64, dtype, store, g)
    ramp = torch.linspace(-3, 3, cache.page * cache.pages, device=DEV)[torch.randperm(cache.page * cache.pages, generator=g).to(DEV)]
    ramp = ramp.view(cache.pages, 1, cache.page)
    if store == I8:
        cache.k_scale *= ramp.abs() + 0.1
    else:
        cache.k *= ramp[..., None].to(dtype)
    check_tree(cache, q, table, n, ints(some_trees(2, 10, rng)), scale=scale)


@pytest.mark.parametrize("dtype,store", [(F16, F16), (BF16, BF16), (BF16, I8)])
def test_tree_scores_that_keep_rising(kv, dtype, store):  # noqa: F811
    """Each tile's scores a little above those before, around the step at which outputs are scaled again."""
    g = torch.Generator().manual_seed(5)
    n, nodes, dim = 3000, 4, 64
    table, pages = full_table([n + nodes], 16, g)
    cache = make_cache(kv, pages, 1, 16, dim, F16 if store == F16 else BF16, g)
    t = torch.arange(n + nodes).float() * (40.0 / n)
    k = torch.zeros(pages, 1, 16, dim)
    order = table[0].long().repeat_interleave(16)[:n + nodes]
    k[order, 0, torch.arange(n + nodes) % 16, 0] = t
    if store == I8:
        scale = k.abs().amax(-1) / 127 + 1e-9
        codes = (k / scale[..., None]).round().to(I8)
        vs = c(cache.v)
        vscale = torch.tensor(np.abs(vs).max(-1) / 127, dtype=torch.float32, device=DEV)
        cache = kv.PagedKV(codes.to(DEV), (cache.v.float() / vscale[..., None]).round().to(I8), scale.to(DEV), vscale)
    else:
        cache.k.copy_(k)
    q = torch.zeros(1, nodes, 2, dim)
    q[..., 0] = torch.linspace(0.2, 8, 2 * nodes).view(1, nodes, 2)
    check_tree(cache, q.to(DEV, dtype), table.to(DEV), ints([n]), ints([-1, 0, 0, 1]), scale=1.0)


@pytest.mark.parametrize("dtype,store", [(F16, F16), (BF16, BF16)])
def test_tree_weights_are_not_cut(kv, dtype, store):  # noqa: F811
    """Equal scores over values that all but cancel: one part of a weight would be off by its own rounding."""
    g = torch.Generator().manual_seed(6)
    cache, q, table, n = setup(kv, [4000], 3, 1, 2, 16, 128, dtype, store, g)
    check_tree(cache, q * 0.1, table, n, ints([-1, 0, 1]))


def test_tree_non_finite_inputs(kv):  # noqa: F811
    """A node's not-a-numbers stay in its own outputs; an infinite score is not-a-number as in the formula; rows whose
    scores are all -infinity have no weight."""
    g = torch.Generator().manual_seed(7)
    cache, q, table, n = setup(kv, [40, 40], 4, 1, 2, 16, 64, F16, F16, g)
    parents = ints([-1, 0, 0, -1])
    want, _ = cache.attend_tree(q, table, n, parents)
    q2 = q.clone()
    q2[0, 1] = float("nan")
    out, lse = cache.attend_tree(q2, table, n, parents)
    assert torch.isnan(out[0, 1]).all() and torch.isnan(lse[0, 1]).all()
    out[0, 1] = want[0, 1]
    assert torch.equal(out, want)
    cache.k[:] = 1.0
    cache.k[..., 0] = float("-inf")
    q[:] = 1.0
    out, lse = cache.attend_tree(q, table, n, parents)
    assert (out == 0).all() and torch.isneginf(lse).all()
    cache.k[table[0, 0].item(), 0, 3, 0] = float("inf")
    out, lse = cache.attend_tree(q, table, n, parents)
    assert torch.isnan(out[0]).all() and (out[1] == 0).all()


def test_tree_strides_streams_and_graphs(kv):  # noqa: F811
    g, rng = torch.Generator().manual_seed(8), np.random.default_rng(8)
    B, nodes = 3, 12
    cache, q, table, n = setup(kv, [700, 90, 2500], nodes, 2, 4, 16, 128, BF16, BF16, g)
    parents = ints(some_trees(B, nodes, rng))
    want, wlse = cache.attend_tree(q, table, n, parents)
    check_tree(cache, q, table, n, parents, got=(want, wlse))
    room = torch.full((B, 8, nodes, 256), float("nan"), dtype=BF16, device=DEV)
    view = room[..., 64:192].transpose(1, 2)
    view.copy_(q)
    out, lse = cache.attend_tree(view, table, n, parents)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    wide = torch.full((B, table.shape[1] + 5), 10 ** 6, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    out, lse = cache.attend_tree(q, wide[:, :table.shape[1]], n, parents)
    assert torch.equal(out, want)
    one = q[:1].expand(B, nodes, 8, 128)
    a, b = cache.attend_tree(one, table, n, parents), cache.attend_tree(one.contiguous(), table, n, parents)
    assert torch.equal(a[0], b[0])
    # two captured calls, replayed beside eager ones on another stream, and with new lengths and trees
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        got = cache.attend_tree(q, table, n, parents)
    with torch.cuda.graph(second, stream=side):
        got2 = cache.attend_tree(q, table, n, parents)
    torch.cuda.synchronize()
    for _ in range(4):
        with torch.cuda.stream(side):
            graph.replay()
        with torch.cuda.stream(other):
            second.replay()
            beside = cache.attend_tree(q, table, n, parents)
        torch.cuda.synchronize()
        for x in (got, got2, beside):
            assert torch.equal(x[0], want) and torch.equal(x[1], wlse)
    n.copy_(ints([20, 90, 1234]))
    parents.copy_(ints(some_trees(B, nodes, rng)))
    graph.replay()
    torch.cuda.synchronize()
    check_tree(cache, q, table, n, parents, got=got)


def test_tree_offsets_past_32_bits(kv):  # noqa: F811
    g = torch.Generator().manual_seed(9)
    pages, page, heads, dim = 9000, 64, 32, 128                   # 2.36e9 elements each of k and v
    k, v = (torch.zeros(pages, heads, page, dim, dtype=F16, device=DEV) for _ in range(2))
    cache = kv.PagedKV(k, v)
    used = torch.tensor([pages - 1, pages - 3, 1, pages - 2])
    for x in (k, v):
        x[used.to(DEV)] = torch.randn(4, heads, page, dim, generator=g).to(DEV, F16)
    q = torch.randn(1, 5, 32, dim, generator=g).to(DEV, F16)
    out, lse = cache.attend_tree(q, ints(used[None]), ints([200]), ints([-1, 0, 0, 1, 2]))
    small = kv.PagedKV(k[used.to(DEV)].contiguous(), v[used.to(DEV)].contiguous())
    check_tree(small, q, ints([[0, 1, 2, 3]]), ints([200]), ints([-1, 0, 0, 1, 2]), got=(out, lse))


def test_tree_of_one_node_is_attend(kv):  # noqa: F811
    g = torch.Generator().manual_seed(10)
    cache, q, table, n = setup(kv, [0, 5, 700, 64], 1, 2, 4, 16, 128, F16, F16, g)
    out, lse = cache.attend_tree(q, table, n, ints([-1]))
    one, olse = cache.attend(q[:, 0], table, n + 1)
    assert (out[:, 0].float() - one.float()).abs().max() <= 2.0 ** -10 * one.float().abs().max()
    assert (lse[:, 0] - olse).abs().max() <= 1e-5 * olse.abs().max()


def test_tree_bad_indices_are_reported(kv):  # noqa: F811
    """Lengths and nodes past the table, pages past the cache: cut or skipped, and reported; wrong parents are none."""
    FvsError = pkg("_lib").FvsError
    g = torch.Generator().manual_seed(11)
    cache, q, table, n = setup(kv, [40, 40], 8, 1, 2, 16, 64, F16, F16, g)
    parents = ints([-1, 0, 0, 1, 1, 2, 3, 3])
    k, v = values(cache)

    def reported(tab, lens, up=parents):
        out, lse = cache.attend_tree(q, tab, lens, up)
        with pytest.raises(FvsError):
            cache.check_status()
        room = tab.shape[1] * 16
        eo, el, *_ = O.attend_tree(c(q), k, v, c(tab), np.clip(c(lens), 0, room), np.broadcast_to(c(up), (2, 8)), None, 0.125)
        assert np.abs(c(out) - eo).max() < 2e-3 and np.array_equal(np.isinf(c(lse)), np.isinf(el))

    reported(table, ints([44, 40]))
    reported(table, ints([1000, 2 ** 31 - 1]))
    bad = table.clone()
    bad[0, 1] = cache.pages
    reported(bad, n)
    check_tree(cache, q, table, ints([-5, 40]), parents)
    for wrong in ([0, 0, 5, 1, 4, -7, 3, 2 ** 31 - 1], [-(2 ** 31)] * 8, [7] * 8):
        check_tree(cache, q, table, n, ints(wrong))


def test_tree_refusals(kv):  # noqa: F811
    g = torch.Generator().manual_seed(12)
    z = lambda *s, dtype=F16: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    cache = make_cache(kv, 4, 2, 16, 64, F16, g)
    t, n, p, q = ints(np.zeros((3, 2))), ints(np.zeros(3)), ints([-1, 0]), z(3, 2, 4, 64)
    learned = z(3, 2, 4, 64).requires_grad_()
    for args, more in (((q.float(), t, n, p), {}), ((q.to(BF16), t, n, p), {}), ((z(3, 2, 5, 64), t, n, p), {}), ((z(3, 2, 4, 96), t, n, p), {}),
                       ((z(3, 4, 64), t, n, p), {}), ((q, t.long(), n, p), {}), ((q, t[:2], n, p), {}), ((q, t, n.long(), p), {}),
                       ((q, t, n, p[:1]), {}), ((q, t, n, p.long()), {}), ((q, t, n, ints(np.zeros((2, 2)))), {}), ((q.cpu(), t, n, p), {}),
                       ((z(3, 2, 64, 4).transpose(2, 3), t, n, p), {}), ((learned, t, n, p), {}), ((z(3, 2, 4, 68)[..., :64], t, n, p), {}),
                       ((z(3, 257, 2, 64), t, n, ints(np.arange(257) - 1)), {}), ((q, t, n, p), dict(counts=n[:2])),
                       ((q, t, n, p), dict(out=q.float())), ((q, t, n, p), dict(lse=z(3, 2, 4))), ((q, t, n, p), dict(lse=z(3, 2, 2, dtype=torch.float32)))):
        with pytest.raises(ValueError):
            cache.attend_tree(*args, **more)
    assert cache.launches == 0
    out, lse = cache.attend_tree(z(0, 2, 4, 64), t[:0], n[:0], p)
    assert out.shape == (0, 2, 4, 64) and lse.shape == (0, 2, 4)
    out, lse = cache.attend_tree(z(3, 0, 4, 64), t, n, p[:0])
    assert out.shape == (3, 0, 4, 64) and lse.shape == (3, 0, 4)


def test_tree_waits_that_run_out(kv):  # noqa: F811
    """With no polls allowed every wait inside the kernel gives up: the call reports it, and the next one works."""
    L = pkg("_lib")
    g = torch.Generator().manual_seed(13)
    cache, q, table, n = setup(kv, [700, 90], 6, 2, 4, 16, 128, BF16, BF16, g)
    parents = ints([-1, 0, 1, 2, 3, 4])
    old = L.lib().fvs_set_wait_limit(0)
    try:
        cache.attend_tree(q, table, n, parents)
        with pytest.raises(L.FvsError, match="ran out"):
            cache.check_status()
    finally:
        L.lib().fvs_set_wait_limit(old)
    check_tree(cache, q, table, n, parents)


def test_tree_two_streams_at_once(kv):  # noqa: F811
    """Calls of different shapes side by side, and workspaces given back between calls."""
    g, rng = torch.Generator().manual_seed(14), np.random.default_rng(14)
    sides = []
    for B, nodes, group, longest in ((1, 64, 4, 9000), (7, 6, 2, 900)):
        cache, q, table, n = setup(kv, list(rng.integers(1, longest, B)), nodes, 2, group, 16, 128, BF16, BF16, g)
        sides.append((cache, q, table, n, ints(some_trees(B, nodes, rng)), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for i in range(10):
        for cache, q, table, n, parents, stream in sides:
            with torch.cuda.stream(stream):
                got.append(cache.attend_tree(q, table, n, parents))
        if i == 5:
            kv.release_workspaces()
    torch.cuda.synchronize()
    for i, (cache, q, table, n, parents, _) in enumerate(sides):
        check_tree(cache, q, table, n, parents, got=got[i])
        assert all(torch.equal(x[0], got[i][0]) and torch.equal(x[1], got[i][1]) for x in got[i::2])


@pytest.mark.parametrize("page", [8, 24, 64, 192])
@pytest.mark.parametrize("dim", [64, 96, 192])
def test_tree_boxes_of_a_page(kv, page, dim):  # noqa: F811
    """Tensor copies of 8 to 64 keys, token-major memory, pages behind one another in a larger tensor, a hole in each box's place."""
    g, rng = torch.Generator().manual_seed(page), np.random.default_rng(page)
    lens, nodes = [200, 63, 65, 1, 511], 7
    cache, q, table, n = setup(kv, lens, nodes, 2, 3, page, dim, BF16, BF16, g, token_major=True)
    room = torch.full((cache.pages, 5, page + 3, dim + 8), float("nan"), dtype=BF16, device=DEV)
    wide = []
    for x in (cache.k, cache.v):
        view = room.clone()[:, 1:3, 2:2 + page, 8:]
        view.copy_(x)
        wide.append(view)
    holes = table.clone()
    holes[0, ::3] = -1
    holes[0, 200 // page:] = table[0, 200 // page:]
    parents = ints(some_trees(len(lens), nodes, rng))
    check_tree(cache, q, holes, n, parents)
    a = cache.attend_tree(q, holes, n, parents)
    b = kv.PagedKV(*wide).attend_tree(q, holes, n, parents)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype,store,dim,group,nodes", [(BF16, BF16, 64, 2, 8), (BF16, BF16, 128, 4, 32), (F16, F16, 96, 1, 100),
                                                         (BF16, I8, 128, 8, 32), (F16, I8, 64, 4, 64), (BF16, I8, 96, 2, 40),
                                                         (BF16, BF16, 128, 4, 64), (BF16, BF16, 192, 2, 16)])
@pytest.mark.parametrize("rise", [4, 8, 10])
def test_tree_references_that_rise_in_every_half(kv, dtype, store, dim, group, nodes, rise):  # noqa: F811
    """Every 32 keys weigh 2^rise times those before them, so that a row's reference rises twice in a tile of 64, the first and
    the later ones, and what was stored for its first half is read again at once.  Keys before a rise keep 2^-rise of the
    output, which is far above its bound."""
    g, rng = torch.Generator().manual_seed(rise), np.random.default_rng(rise)
    lens, heads, page = [160, 225, 31, 64, 97, 128] * 4, 2, 32
    cache, q, table, n = setup(kv, lens, nodes, heads, group, page, dim, dtype, store, g)
    q *= 0.1
    q[..., 0] = 1.0
    step = torch.zeros(cache.pages, device=DEV)  # a page is one step
    for b, m in enumerate(lens):
        row = table[b][table[b] >= 0].long()
        step[row] = torch.arange(len(row), device=DEV).float()
    if store == I8:
        cache.k_scale.copy_((0.01 * (1 + step))[:, None, None].expand_as(cache.k_scale))
        cache.k[..., 0] = 127
        scale = rise * np.log(2) / 1.27  # 0.01 * 127 * scale a step, beside what the other elements add
    else:
        cache.k[..., 0] = step[:, None, None].to(store)
        scale = rise * np.log(2)
    cache.k[..., 1:] = 0
    check_tree(cache, q, table, n, ints(some_trees(len(lens), nodes, rng)), scale=float(scale))


def test_tree_two_threads_on_one_stream(kv):  # noqa: F811
    """Threads share torch's default stream and its workspace: a call's two launches stay together."""
    g, rng = torch.Generator().manual_seed(15), np.random.default_rng(15)
    calls, want = [], []
    for B, nodes, group, longest in ((1, 64, 4, 9000), (20, 6, 2, 900)):
        cache, q, table, n = setup(kv, list(rng.integers(longest // 2, longest, B)), nodes, 2, group, 16, 128, BF16, BF16, g)
        calls.append((cache, q, table, n, ints(some_trees(B, nodes, rng))))
        want.append(calls[-1][0].attend_tree(*calls[-1][1:]))
        check_tree(*calls[-1], got=want[-1])
    start, got = threading.Barrier(4), [[] for _ in range(4)]

    def work(i):
        cache, *args = calls[i % 2]
        start.wait()
        for _ in range(100):
            got[i].append(cache.attend_tree(*args))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        assert len(outs) == 100
        assert all(torch.equal(x[0], want[i % 2][0]) and torch.equal(x[1], want[i % 2][1]) for x in outs)


def check_special(cache, q, table, lens, parents, counts=None, scale=None, got=None):
    """check_tree for values that are not finite: a column is what the formula makes of its infinities and not-a-numbers, and
    the others lie within their bound."""
    out, lse = got or cache.attend_tree(q, table, lens, parents, counts=counts, scale=scale)
    torch.cuda.synchronize()
    d = cache.dim
    scale = 1 / np.sqrt(d) if scale is None else scale
    k, v = values(cache)
    with np.errstate(invalid="ignore", over="ignore"):
        eo, el, pv, mag = O.attend_tree(c(q), k, v, c(table), c(lens), np.broadcast_to(c(parents), q.shape[:2]),
                                        None if counts is None else c(counts), scale, None if cache.fill is None else c(cache.fill))
    out, lse = c(out), c(lse)
    assert np.array_equal(np.isnan(out), np.isnan(eo))
    inf = np.isinf(eo)
    assert np.array_equal(np.isinf(out), inf) and np.array_equal(out[inf], eo[inf])
    fine = np.isfinite(eo)
    L = int(max(1, c(lens).max() + q.shape[1]))
    es = (d + 4) * 2.0 ** -23 * np.broadcast_to(mag[..., None], eo.shape)
    part = 2.0 ** -17 if q.dtype == BF16 or cache.dtype == I8 else 2.0 ** -21
    tol = U[q.dtype] * np.abs(eo[fine]) + (part + 2 * es[fine] + 2.0 ** -20 + (L + 64) * 2.0 ** -22) * pv[fine] * 1.01 + (2.0 ** -25 if q.dtype == F16 else 0.0)
    tol += 2.0 ** -36 * np.abs(v[np.isfinite(v)]).max()
    worst = (np.abs(out[fine] - eo[fine]) / tol).max(initial=0)
    assert worst <= 1, f"out is {worst:.2f} of its bound"
    empty = np.isneginf(el)
    assert np.array_equal(np.isneginf(lse), empty) and (out[empty] == 0).all()
    assert np.array_equal(np.isnan(lse), np.isnan(el))
    fine = np.isfinite(el)
    tol = 2 * (d + 4) * 2.0 ** -23 * mag[fine] + (L + 64) * 2.0 ** -22 + 2.0 ** -20 * (1 + np.abs(el[fine]))
    worst = (np.abs(lse[fine] - el[fine]) / tol).max(initial=0)
    assert worst <= 1, f"lse is {worst:.2f} of its bound"
    cache.check_status()


def put(cache, table, b, t, h, col, x):
    """Value `x` in column `col` of token t of sequence b (codes: a scale makes it of the row)."""
    page, slot = int(table[b, t // cache.page]), t % cache.page
    if cache.v_scale is None:
        cache.v[page, h, slot, col] = x
    else:
        cache.v[page, h, slot] = 1
        cache.v[page, h, slot, col] = 1 if x > 0 else -1 if x < 0 else 0
        cache.v_scale[page, h, slot] = abs(x)


KINDS = [(BF16, BF16, 64, 2, 9), (BF16, BF16, 128, 4, 20), (F16, F16, 96, 8, 25), (BF16, I8, 128, 8, 32), (F16, I8, 64, 2, 10), (BF16, BF16, 192, 2, 70),
         (F16, F16, 128, 5, 1)]


@pytest.mark.parametrize("dtype,store,dim,group,nodes", KINDS)
@pytest.mark.parametrize("lens,page", [([300, 40, 129, 0, 70], 16), ([20000, 3], 64), ([100] * 90, 20)])
def test_tree_visible_values_that_are_not_finite(kv, dtype, store, dim, group, nodes, lens, page):  # noqa: F811
    """An infinity is the column's output, two against each other and not-a-numbers are not-a-number, as in `attend`; items of
    one CTA and cut ones, copies of boxes and of rows, in the sequence and in its nodes."""
    g, rng = torch.Generator().manual_seed(16), np.random.default_rng(16)
    heads = 2
    cache, q, table, n = setup(kv, lens, nodes, heads, group, page, dim, dtype, store, g)
    tab, inf, nan = table.cpu(), float("inf"), float("nan")
    put(cache, tab, 0, 7, 0, 5, inf)
    put(cache, tab, 0, lens[0] - 1, 1, dim - 1, -inf)
    put(cache, tab, 0, 3, 1, dim - 1, inf)               # not-a-number in that column
    put(cache, tab, 1, 2, 0, 33, -inf)
    put(cache, tab, 1, 1, 1, 40, nan)
    last = len(lens) - 1
    put(cache, tab, last, lens[last] + nodes - 1, 0, 8, inf)   # a node: its own rows and those of its descendants
    put(cache, tab, last, lens[last], 1, 9, -inf)
    put(cache, tab, last, lens[last] + nodes // 2, 1, 9, inf)
    q *= 0.3                                                # no weight is 0 in 64 bits
    parents = ints(some_trees(len(lens), nodes, rng))
    check_special(cache, q, table, n, parents)
    counts = ints(rng.integers(0, nodes + 1, len(lens)))
    check_special(cache, q, table, n, parents, counts=counts)


@pytest.mark.parametrize("dtype,store,dim,group,nodes", KINDS)
@pytest.mark.parametrize("lens,page", [([300, 40, 129, 0, 70], 16), ([20000, 3], 64), ([100] * 90, 20)])
def test_tree_values_near_the_ends_of_their_range(kv, dtype, store, dim, group, nodes, lens, page):  # noqa: F811
    """Large finite values, whose products with weights that are not normed pass fp32's range: outputs are their means."""
    if dtype == F16 and store == F16:
        big = 6e4
    else:
        big = 3e38 if dtype == BF16 else 1e4
    g, rng = torch.Generator().manual_seed(17), np.random.default_rng(17)
    cache, q, table, n = setup(kv, lens, nodes, 2, group, page, dim, dtype, store, g)
    if store == I8:
        cache.v_scale.fill_(big / 127)
        cache.v[:, :, :, ::2] = torch.randint(90, 128, cache.v[:, :, :, ::2].shape, generator=g).to(DEV, I8)
    else:
        cache.v.copy_((torch.rand(cache.v.shape, generator=g) * 2 - 1).to(DEV) * big)
        cache.v[:, :, :, ::2] = (big * (0.9 + 0.1 * torch.rand(cache.v[:, :, :, ::2].shape, generator=g).to(DEV))).to(store)
    check_special(cache, q, table, n, ints(some_trees(len(lens), nodes, rng)))


def test_tree_not_finite_rows_and_values_together(kv):  # noqa: F811
    """A query of not-a-numbers beside infinite values: its row is not-a-number in every column; without a place for the sums'
    logarithms as well."""
    L = pkg("_lib")
    g = torch.Generator().manual_seed(18)
    cache, q, table, n = setup(kv, [9000, 100, 40], 6, 2, 2, 16, 64, BF16, BF16, g)
    q[0, 2, 1] = float("nan")
    q[1, 3] = float("nan")
    tab = table.cpu()
    for b in range(3):
        put(cache, tab, b, 5, b % 2, 7, float("inf"))
    parents = ints([-1, 0, 1, 0, -1, 4])
    check_special(cache, q, table, n, parents)
    want, _ = cache.attend_tree(q, table, n, parents)
    out = torch.full_like(want, float("nan"))
    work = torch.empty(L.lib().fvs_kv_attend_tree_work(64, 12), dtype=torch.uint8, device=DEV)
    rc = L.lib().fvs_kv_attend_tree(torch.cuda.current_stream().cuda_stream, cache._ref, L.BF16, q.data_ptr(), *q.stride()[:3], 4,
                                    table.data_ptr(), 3, table.shape[1], table.stride(0), n.data_ptr(), parents.data_ptr(), 0, None, 6,
                                    0.125, out.data_ptr(), None, work.data_ptr())
    torch.cuda.synchronize()
    assert rc == 0 and torch.equal(out.view(torch.int16) & 0x7fff, want.view(torch.int16) & 0x7fff)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_tree_infinite_key_scales(kv, dtype):  # noqa: F811
    """Codes of both signs times an infinite scale: a score of not-a-number, whatever the sign of the codes' own product."""
    g = torch.Generator().manual_seed(20)
    cache, q, table, n = setup(kv, [90, 300], 5, 2, 2, 16, 64, dtype, I8, g)
    cache.k_scale[int(table[1, 4]), 1, 3] = float("inf")
    check_special(cache, q, table, n, ints([-1, 0, 1, 1, -1]))


@pytest.mark.parametrize("dtype,store,dim,group,nodes", KINDS[:6])
@pytest.mark.parametrize("lens,page", [([300, 0, 129], 16), ([15000, 3, 1], 64), ([70] * 80, 20)])
@pytest.mark.parametrize("x", [float("nan"), float("inf")])
def test_tree_nodes_that_are_not_finite(kv, dtype, store, dim, group, nodes, lens, page, x):  # noqa: F811
    """A draft's key or value of not-a-numbers or infinities is seen by itself and its descendants alone."""
    g, rng = torch.Generator().manual_seed(19), np.random.default_rng(19)
    cache, q, table, n = setup(kv, lens, nodes, 2, group, page, dim, dtype, store, g)
    tab, parents = table.cpu(), some_trees(len(lens), nodes, rng)
    for b in range(min(3, len(lens))):
        for t, rows, scale in ((lens[b] + 1, cache.k, cache.k_scale), (lens[b] + nodes - 1, cache.v, cache.v_scale), (lens[b] + 2, cache.v, cache.v_scale)):
            at = int(tab[b, t // page]), b % 2, t % page
            if scale is None:
                rows[at] = x
            else:
                scale[at] = x
    q *= 0.3
    sees = [O.sees(p) for p in parents[:3]]
    assert any(not m[:, 1].all() and m[:, 1].sum() > 1 for m in sees)
    check_special(cache, q, table, n, ints(parents))
    out, lse = cache.attend_tree(q, table, n, ints(parents))
    for b, m in enumerate(sees[:len(lens)]):
        fine = torch.isfinite(out[b]).all(-1).all(-1).cpu().numpy()
        clean = ~(m[:, 1] | m[:, 2] | m[:, nodes - 1])
        assert fine[clean].all() and clean.any()


def test_tree_status_names_all_that_was_met(kv):  # noqa: F811
    """A wait that ran out hides no index outside its table."""
    FvsError = pkg("_lib").FvsError
    cache = make_cache(kv, 4, 1, 16, 64, F16, torch.Generator().manual_seed(21))
    for status, words in ((1, ["index"]), (2, ["ran out"]), (3, ["index", "ran out"])):
        cache.status.fill_(status)
        with pytest.raises(FvsError) as e:
            cache.check_status()
        assert [w for w in ("index", "ran out") if w in str(e.value)] == words
        cache.check_status()


@pytest.mark.parametrize("dtype,dim,group,nodes", [(BF16, 128, 8, 32), (F16, 64, 2, 10), (F16, 96, 4, 40), (BF16, 192, 1, 3)])
@pytest.mark.parametrize("kind", ["wide", "rising", "falling", "zeros", "signs"])
def test_tree_value_scales_far_apart(kv, dtype, dim, group, nodes, kind):  # noqa: F811
    """int8 values whose scales differ by 2^60 from key to key, rise or fall along the sequence, are 0 beside the largest weights,
    or negative.  Weights times scales enter the product as fp16 numbers of 22 bits, of 2^-25 beside 2^9 for the largest met so
    far: off by 2^-34 of it a key.  A scale of 0 counts as 2^-80 there: where such a key weighs most, 2^-25 beside 2^(9 + 80) for
    its weight, which is at most the sum, times a code of 127 is 2^-107 a key."""
    g, rng = torch.Generator().manual_seed(22), np.random.default_rng(22)
    lens, page, heads = [300, 40, 1000], 16, 2
    cache, q, table, n = setup(kv, lens, nodes, heads, group, page, dim, dtype, I8, g)
    q *= 0.5
    tab = table.cpu().long()
    order = torch.zeros(cache.pages * page)
    for b, m in enumerate(lens):
        t = torch.arange(m + nodes)
        order[tab[b, t // page] * page + t % page] = t.float()
    order = order.view(cache.pages, 1, page).to(DEV)
    far = torch.rand(cache.v_scale.shape, generator=g).to(DEV)
    if kind == "wide":
        cache.v_scale *= 2.0 ** (60 * far - 30).round()
    elif kind in ("rising", "falling"):
        cache.v_scale *= 2.0 ** ((order if kind == "rising" else 1000 - order) / 10 - 50).round()
    elif kind == "zeros":
        top = far < 0.3                                       # these keys weigh most, and have no value
        cache.k_scale[top] *= 30
        cache.v_scale[top] = 0
    else:
        cache.v_scale[far < 0.5] *= -1
    parents = ints(some_trees(len(lens), nodes, rng))
    out, lse = cache.attend_tree(q, table, n, parents)
    torch.cuda.synchronize()
    k, v = values(cache)
    scale = dim ** -0.5
    eo, el, pv, mag = O.attend_tree(c(q), k, v, c(table), c(n), c(parents), None, scale)
    L = max(lens) + nodes
    es = (dim + 4) * 2.0 ** -23 * mag[..., None]
    bound = U[dtype] * np.abs(eo) + (2.0 ** -21 + 2 * es + 2.0 ** -20 + (L + 64) * 2.0 ** -22) * pv + L * (2.0 ** -34 * pv.max(-1, keepdims=True) + 2.0 ** -107) + (2.0 ** -25 if dtype == F16 else 0)
    out = c(out).astype(np.float64)
    over = np.abs(eo) >= 65504 * (1 - 2.0 ** -12) if dtype == F16 else np.zeros(eo.shape, bool)   # outputs past fp16's range
    assert np.isfinite(out[~over]).all() and (np.abs(out[over]) >= 65504 * (1 - 2.0 ** -10)).all()
    with np.errstate(invalid="ignore"):
        worst = (np.abs(out - eo) / bound)[~over].max(initial=0)
    assert worst <= 1, f"out is {worst:.2f} of its bound"
    tol = 2 * es[..., 0] + (L + 64) * 2.0 ** -22 + 2.0 ** -20 * (1 + np.abs(el))
    assert (np.abs(c(lse) - el) <= tol).all()
    cache.check_status()


@pytest.mark.parametrize("dtype,store,part", [(BF16, BF16, 2.0 ** -17), (F16, F16, 2.0 ** -21), (BF16, I8, 2.0 ** -21), (F16, I8, 2.0 ** -21)])
@pytest.mark.parametrize("dim,group", [(64, 2), (128, 40), (192, 1)])
def test_tree_weights_keep_their_second_part(kv, dtype, store, part, dim, group):  # noqa: F811
    """Two keys whose weighted values all but cancel: what is left shows a weight's own rounding, which with one 16-bit part
    misses the bound by far.  Scores are single exact products, so that no sum adds to the bound; an exponential is within
    2^-21, a sum of two and the quotient within 2^-23 together."""
    g = torch.Generator().manual_seed(23)
    B, nodes = 24, 5
    cache, q, table, n = setup(kv, [2] * B, nodes, 1, group, 16, dim, dtype, store, g)
    at = table[:, 0].long()
    first = torch.rand(B, generator=g) * 1.4 + 0.1             # scores' difference
    q.zero_()
    q[..., 0] = 1.0
    cache.k[at] = 0
    if store == I8:
        cache.k[at, :, 0, 0] = 64
        cache.k_scale[at] = (first / 64).to(DEV)[:, None, None]
        cache.v_scale[at] = 1 / 64
    else:
        cache.k[at, :, 0, 0] = first.to(DEV, store)[:, None]
    k, _ = values(cache)
    d = torch.tensor(k[c(at), 0, 0, 0])                       # 64 bits
    ratio = torch.exp(d)                                       # of the two weights
    if store == I8:                                            # w0 a - w1 b, of codes near a / b = w1 / w0
        b = torch.arange(dim) % 60 + 60
        a = (b[None] / ratio[:, None]).round()
        cache.v[at, 0, 0], cache.v[at, 0, 1] = a.to(DEV, I8), -b.expand(B, dim).to(DEV, I8)
    else:
        b = 1 + torch.arange(dim) / 256
        cache.v[at, 0, 0], cache.v[at, 0, 1] = (b[None] / ratio[:, None]).to(DEV, store), -b.expand(B, dim).to(DEV, store)
    # each node sees the two keys and itself: its own key weighs nothing beside them
    own = at
    for i in range(nodes):
        cache.k[own, 0, 2 + i] = 0
        if store == I8:
            cache.k[own, 0, 2 + i, 0], cache.k_scale[own, 0, 2 + i] = -127, 1.0
        else:
            cache.k[own, 0, 2 + i, 0] = -100.0
    parents = ints(np.full(nodes, -1))
    out, lse = cache.attend_tree(q, table, n, parents, scale=1.0)
    k, v = values(cache)
    eo, el, pv, _ = O.attend_tree(c(q), k, v, c(table), c(n), np.broadcast_to(c(parents), (B, nodes)), None, 1.0)
    bound = U[dtype] * np.abs(eo) + (part + 2.0 ** -21 + 2.0 ** -23 + 2.0 ** -22) * pv + 2.0 ** -34 * np.abs(v[c(at)]).max() + (2.0 ** -25 if dtype == F16 else 0)
    worst = (np.abs(c(out) - eo) / bound).max()
    assert worst <= 1, f"out is {worst:.2f} of its bound"
    # the same with weights rounded to one part
    w = np.stack([np.ones(B), np.exp(-c(d))], 1)
    one = torch.tensor(w * (512 if store != BF16 else 1)).to(F16 if store != BF16 else BF16).double().numpy()
    vv = v[c(at), 0, :2]
    cut = (one[..., None] * vv).sum(1) / (w.sum(1) * (512 if store != BF16 else 1))[:, None]
    assert (np.abs(cut - eo[:, 0, 0]) / bound[:, 0, 0]).max() > 20


@pytest.mark.parametrize("dtype,store,group,dim,nodes", [(BF16, BF16, 2, 64, 3), (F16, I8, 1, 128, 40), (F16, F16, 8, 64, 33), (BF16, BF16, 4, 192, 5)])
def test_tree_no_share_is_lost(kv, dtype, store, group, dim, nodes):  # noqa: F811
    """One long context whose every run of keys has a column of its own: an output without one CTA's share (a 296th of the keys or
    more) would be far off its bound in that run's column, and so would its lse's tighter one."""
    g, rng = torch.Generator().manual_seed(24), np.random.default_rng(24)
    L = 60000
    cache, q, table, n = setup(kv, [L], nodes, 1, group, 64, dim, dtype, store, g)
    q *= 0.1
    run = torch.zeros(cache.pages, 64, dtype=torch.long)
    t = torch.arange(L + nodes)
    run[table.cpu()[0, t // 64].long(), t % 64] = t * dim // (L + nodes)
    one = torch.nn.functional.one_hot(run, dim)[:, None].to(DEV)
    if store == I8:
        cache.v.copy_(one)
        cache.v_scale.fill_(1.0)
    else:
        cache.v.copy_(one)
    parents = ints(some_trees(1, nodes, rng))
    check_tree(cache, q, table, n, parents)
    # the same bounds for an output without 200 keys of a run (a share has 202 or more)
    k, v = values(cache)
    eo, el, pv, mag = O.attend_tree(c(q), k, v, c(table), c(n), c(parents), None, dim ** -0.5)
    bound = U[dtype] * np.abs(eo) + (2.0 ** -17 + 2.0 ** -20 + (L + nodes + 64) * 2.0 ** -22) * pv * 1.01
    assert (eo[..., :dim - 1] * 200 / ((L + nodes) / dim) / 2 > 2 * bound[..., :dim - 1]).all()


@pytest.mark.parametrize("dtype,store,dim", [(BF16, BF16, 128), (F16, F16, 64), (BF16, I8, 64)])
@pytest.mark.parametrize("n", [200, 30000])
def test_tree_infinite_value_of_a_small_weight(kv, dtype, store, dim, n):  # noqa: F811
    """A weight that fp32 does not hold is above zero all the same: in its own tile, and as a share of its own."""
    g = torch.Generator().manual_seed(25)
    cache, q, table, lens = setup(kv, [n], 6, 1, 4, 16, dim, dtype, store, g)
    tab = table.cpu()
    q *= 0.1
    q[..., 0] = 20.0
    row = table[0, :3 if n < 1000 else 64].long()           # the first keys (more than a share): 400 nats below the others
    if store == I8:
        cache.k_scale.fill_(0.01)
        cache.k[..., 0] = 0
        cache.k[row, :, :, 0], cache.k_scale[row] = -127, 20 / 127
    else:
        cache.k[..., 0] = 0
        cache.k[row, :, :, 0] = -20.0
    put(cache, tab, 0, 5, 0, 7, float("inf"))
    put(cache, tab, 0, 40, 0, 9, float("-inf"))
    check_special(cache, q, table, lens, ints([-1, 0, 0, 1, 2, -1]), scale=1.0)


def test_tree_long_run_of_values_of_zero(kv):  # noqa: F811
    """Every key but a few has a value scale of 0 and all of the weight: the sum of their weights, 2^89 each, stays finite."""
    g = torch.Generator().manual_seed(26)
    n = 400000
    cache, q, table, lens = setup(kv, [n], 2, 1, 2, 64, 64, BF16, I8, g)
    cache.v_scale[:] = 0
    cache.k[:] = 0
    cache.v_scale[table[0, -1].long(), :, :(n + 2) % 64] = 1.0
    out, lse = cache.attend_tree(q, table, lens, ints([-1, 0]))
    k, v = values(cache)
    eo, el, pv, _ = O.attend_tree(c(q), k, v, c(table), c(lens), np.array([[-1, 0]]), None, 0.125)
    assert (np.abs(c(lse) - el) <= 2.0 ** -20 * np.abs(el) + (n + 64) * 2.0 ** -22).all() and np.isfinite(c(lse)).all()
    assert (np.abs(c(out) - eo) <= 2.0 ** -8 * np.abs(eo) + (n + 64) * 2.0 ** -22 * pv).all()


def test_tree_not_finite_in_graphs_and_on_streams(kv):  # noqa: F811
    """Rows that are computed again: captured, replayed after the values changed, and beside another stream's calls."""
    g, rng = torch.Generator().manual_seed(27), np.random.default_rng(27)
    cache, q, table, n = setup(kv, [5000, 90, 300], 12, 2, 4, 16, 128, BF16, BF16, g)
    q *= 0.3
    tab, parents = table.cpu(), ints(some_trees(3, 12, rng))
    put(cache, tab, 0, 77, 0, 3, float("inf"))
    put(cache, tab, 2, 301, 1, 100, float("nan"))
    other, q2, table2, n2 = setup(kv, [4000], 64, 2, 4, 16, 128, BF16, BF16, g)
    put(other, table2.cpu(), 0, 4001, 1, 5, float("-inf"))
    parents2 = ints(some_trees(1, 64, rng))
    want, want2 = cache.attend_tree(q, table, n, parents), other.attend_tree(q2, table2, n2, parents2)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        got = cache.attend_tree(q, table, n, parents)
    same = lambda a, b: all(torch.equal(x.view(torch.int16 if x.element_size() == 2 else torch.int32), y.view(torch.int16 if y.element_size() == 2 else torch.int32)) for x, y in zip(a, b))  # noqa: E731
    for _ in range(5):
        with torch.cuda.stream(side):
            graph.replay()
        beside = other.attend_tree(q2, table2, n2, parents2)
        torch.cuda.synchronize()
        assert same(got, want) and same(beside, want2)
    check_special(cache, q, table, n, parents, got=got)
    put(cache, tab, 0, 77, 0, 3, 1.0)
    put(cache, tab, 1, 3, 1, 60, float("-inf"))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph.replay()
    torch.cuda.synchronize()
    check_special(cache, q, table, n, parents, got=got)


def test_tree_workspace_is_held_for_the_launches(kv, monkeypatch):  # noqa: F811
    """Another thread may give the stream's workspace back, or put a larger one in its place, while a call is made: its memory is
    nobody else's before the launches are on the stream."""
    g = torch.Generator().manual_seed(28)
    cache, q, table, n = setup(kv, [70], 3, 1, 2, 16, 64, BF16, BF16, g)
    held = []
    find, launch = cache._tree_workspace, cache._attend_tree

    def found(*args):
        work = find(*args)
        held.append(weakref.ref(work))
        kv.release_workspaces()
        return work

    def launched(*args):
        assert held[-1]() is not None and args[-1] == held[-1]().data_ptr()
        return launch(*args)

    monkeypatch.setattr(cache, "_tree_workspace", found)
    monkeypatch.setattr(cache, "_attend_tree", launched)
    check_tree(cache, q, table, n, ints([-1, 0, 0]))
    assert len(held) == 1 and held[0]() is None


@pytest.mark.parametrize("dtype,store,part,parts_of_attend", [(BF16, BF16, 2.0 ** -17, 2.0 ** -24), (BF16, I8, 2.0 ** -21, 2.0 ** -21), (F16, I8, 2.0 ** -21, 2.0 ** -21)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_tree_of_one_node_is_attend_in_every_type(kv, dtype, store, part, parts_of_attend, dim):  # noqa: F811
    """The two calls' outputs are apart by no more than both bounds together, and by one number of the type at most in nearly all."""
    g = torch.Generator().manual_seed(29)
    lens = [0, 5, 700, 64, 3000] * 3
    cache, q, table, n = setup(kv, lens, 1, 2, 4, 16, dim, dtype, store, g)
    out, lse = cache.attend_tree(q, table, n, ints([-1]))
    one, olse = cache.attend(q[:, 0].contiguous(), table, n + 1)
    k, v = values(cache)
    eo, el, pv, mag = O.attend_tree(c(q), k, v, c(table), c(n), np.full((len(lens), 1), -1), None, dim ** -0.5)
    es = (dim + 4) * 2.0 ** -23 * mag[:, 0, :, None]
    L = max(lens) + 1
    each = U[dtype] * np.abs(eo[:, 0]) + (2 * es + 2.0 ** -20 + (L + 64) * 2.0 ** -22) * pv[:, 0] + (2.0 ** -25 if dtype == F16 else 0)
    a, b = c(out)[:, 0].astype(np.float64), c(one).astype(np.float64)
    assert (np.abs(a - b) <= 2 * each + (part + parts_of_attend) * pv[:, 0]).all()
    assert (np.abs(a - b) <= 4 * U[dtype] * np.abs(eo[:, 0])).mean() > 0.99
    assert (np.abs(c(lse)[:, 0] - c(olse)) <= 2 * (2 * es[..., 0] + (L + 64) * 2.0 ** -22 + 2.0 ** -20 * (1 + np.abs(el[:, 0])))).all()
