"""Paged key-value cache (append, read, attend) against the 64-bit oracle.

Bounds, from the arithmetic alone (u: unit roundoff of the output type, 2^-11 fp16 and 2^-8 bf16):
* append: the rotation is three fp32 operations, each within 2^-24 of sum |terms|, then one rounding to the stored type;
  an int8 code is within half a step of the value.
* read: the fp32 product of code and scale, rounded once: equal to numpy's.
* attend: a score is off by es <= (dim + 4) 2^-23 scale sum |q k| (fp32 sums; the tensor cores may cut instead of round),
  which changes its weight by a factor e^(es); weights enter the second product rounded to the 16-bit type (u of sum
  p |v|, and half the smallest fp16 step, 2^-25, for tiny ones); fp32 sums over L keys; one rounding of the output.
"""
import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import kv_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16, BF16, I8 = torch.float16, torch.bfloat16, torch.int8


def c(x):
    return x.detach().double().cpu().numpy() if x.is_floating_point() else x.detach().cpu().numpy()


@pytest.fixture(scope="module")
def kv():
    pkg("build").build()
    return pkg("kvcache")


def make_cache(kv, pages, heads, page, dim, dtype, g, fill=None, token_major=False):
    """A cache of normal values; token_major: a view of [pages, page, heads, dim] memory."""
    def rows():
        x = torch.randn(pages, page, heads, dim, generator=g).to(DEV)
        return x if token_major else x.transpose(1, 2).contiguous()
    k, v = rows(), rows()
    scales = [None, None]
    if dtype == I8:
        scales = [x.abs().amax(-1) / 127 for x in (k, v)]
        k, v = ((x / s[..., None]).round().to(I8) for x, s in zip((k, v), scales))
    else:
        k, v = k.to(dtype), v.to(dtype)
    if token_major:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
        scales = [None if s is None else s.transpose(1, 2) for s in scales]
    return kv.PagedKV(k, v, *scales, fill=fill)


def values(cache):
    """What the cache's rows stand for, in 64 bits."""
    k, v = c(cache.k).astype(np.float64), c(cache.v).astype(np.float64)
    if cache.k_scale is not None:
        with np.errstate(invalid="ignore"):        # hidden rows may hold anything
            k, v = k * c(cache.k_scale)[..., None], v * c(cache.v_scale)[..., None]
    return k, v


def check_attend(cache, q, table, lens, scale=None, got=None):
    out, lse = got or cache.attend(q, table, lens, scale=scale)
    torch.cuda.synchronize()
    d = cache.dim
    scale = 1 / np.sqrt(d) if scale is None else scale
    k, v = values(cache)
    fill = None if cache.fill is None else c(cache.fill)
    eo, el, pv, av, mag = O.attend(c(q), k, v, c(table), c(lens), scale, fill)
    out, lse = c(out), c(lse)
    u, L = U[q.dtype], int(max(1, c(lens).max()))
    es = (d + 4) * 2.0 ** -23 * mag
    tol = u * np.abs(eo) + (u + 2 * es[..., None] + (L + 64) * 2.0 ** -22) * pv * 1.01 + 2.0 ** -25 * (1 + 2 * av)
    empty = np.isinf(el)
    assert (out[empty] == 0).all() and np.array_equal(np.isneginf(lse), empty)
    worst = (np.abs(out - eo) / tol).max()
    assert worst <= 1, f"out is {worst:.2f} of its bound"
    tol = 2 * es + (L + 64) * 2.0 ** -22 + 2.0 ** -21 * (1 + np.abs(np.where(empty, 0, el)))
    worst = (np.abs(lse[~empty] - el[~empty]) / tol[~empty]).max(initial=0)
    assert worst <= 1, f"lse is {worst:.2f} of its bound"


def full_table(lens, page, g, spare=3, wide=None):
    """Pages in random order for sequences of the given lengths; -1 after each one's last."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=g)
    t, at = torch.full((len(lens), wide or max(1, max(need))), -1), 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t.to(torch.int32), sum(need) + spare


# ------------------------------------------------------------------------------------------------ attend

@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype,store", [(BF16, BF16), (F16, F16), (BF16, I8), (F16, I8)])
@pytest.mark.parametrize("heads,group", [(2, 1), (1, 7)])
def test_attend_types_and_dims(kv, dim, dtype, store, heads, group):
    g = torch.Generator().manual_seed(dim + heads)
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 200]
    table, pages = full_table(lens, 16, g)
    cache = make_cache(kv, pages, heads, 16, dim, store, g)
    q = (torch.randn(len(lens), heads * group, dim, generator=g) * 1.5).to(DEV, dtype)
    check_attend(cache, q, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))
    cache.check_status()


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 9, 12, 16, 17, 24, 32, 33, 40, 71])
@pytest.mark.parametrize("store", [BF16, I8])
def test_attend_head_groups(kv, group, store):
    g = torch.Generator().manual_seed(group)
    lens = [333, 40, 1]
    table, pages = full_table(lens, 32, g)
    cache = make_cache(kv, pages, 3, 32, 64, store, g)
    q = torch.randn(3, 3 * group, 64, generator=g).to(DEV, BF16)
    check_attend(cache, q, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("page", [1, 2, 3, 7, 16, 20, 48, 100, 256])
@pytest.mark.parametrize("store", [F16, I8])
def test_attend_page_sizes(kv, page, store):
    g = torch.Generator().manual_seed(page)
    lens = [1, page, page + 1, 2 * page - 1, 130, 5]
    table, pages = full_table(lens, page, g)
    cache = make_cache(kv, pages, 2, page, 128, store, g)
    q = torch.randn(len(lens), 8, 128, generator=g).to(DEV, F16)
    check_attend(cache, q, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("store", [BF16, I8])
@pytest.mark.parametrize("page", [5, 16, 64])
def test_attend_holes_fill_and_what_memory_holds(kv, page, store):
    """Holes, partly filled pages, sequences with nothing visible; hidden slots hold not-a-numbers and infinities."""
    g = torch.Generator().manual_seed(3 * page)
    B, wide = 6, 9
    pages = B * wide + 2
    table = torch.randperm(pages, generator=g)[:B * wide].reshape(B, wide).to(torch.int32)
    table[torch.rand(B, wide, generator=g) < 0.3] = -1
    table[2] = -1                                    # all holes
    table[3, :-1] = -1                               # only the last page
    fill = torch.randint(0, page + 1, (pages,), generator=g, dtype=torch.int32)
    fill[table[4].clamp(min=0).long()] = 0           # pages without any token
    fill[table[3, -1].long()] = 1
    table[3, -1] = table[3, -1].clamp(min=0)
    lens = torch.tensor([wide * page, wide * page - page // 2 - 1, wide * page, wide * page, wide * page, 0], dtype=torch.int32)
    cache = make_cache(kv, pages, 2, page, 64, store, g, fill=fill.to(DEV))
    seen = torch.zeros(pages, page, dtype=torch.bool)
    for b in range(B):
        for t in range(int(lens[b])):
            p = int(table[b, t // page])
            if p >= 0 and t % page < fill[p]:
                seen[p, t % page] = True
    hid = ~seen.to(DEV)
    for x, odd in ((cache.k_scale if store == I8 else cache.k, np.nan), (cache.v_scale if store == I8 else cache.v, np.inf)):
        x.masked_fill_(hid[:, None] if store == I8 else hid[:, None, :, None], odd)
    q = torch.randn(B, 6, 64, generator=g).to(DEV, BF16)
    check_attend(cache, q, table.to(DEV), lens.to(DEV))
    cache.check_status()


@pytest.mark.parametrize("store", [F16, I8])
@pytest.mark.parametrize("B,heads,group,dim,longest", [(1, 1, 1, 64, 20000), (1, 8, 4, 128, 9000), (3, 2, 16, 96, 4099),
                                                       (40, 3, 5, 64, 700), (700, 2, 1, 64, 90)])
def test_attend_splits_over_the_length(kv, B, heads, group, dim, longest, store):
    """Few rows over a long axis, and many short ones: parts of one sequence are joined; the same call twice gives the
    same bits."""
    g = torch.Generator().manual_seed(B + longest)
    lens = torch.randint(0, longest + 1, (B,), generator=g, dtype=torch.int32)
    lens[0] = longest
    table, pages = full_table(lens.tolist(), 64, g)
    cache = make_cache(kv, pages, heads, 64, dim, store, g)
    q = (torch.randn(B, heads * group, dim, generator=g) * 2).to(DEV, F16)
    table, lens = table.to(DEV), lens.to(DEV)
    a = cache.attend(q, table, lens)
    check_attend(cache, q, table, lens, got=a)
    for _ in range(3):
        b = cache.attend(q, table, lens)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    perm = torch.arange(B - 1, -1, -1, device=DEV)                 # another batch order: the same rows within the bounds
    check_attend(cache, q[perm].contiguous(), table[perm].contiguous(), lens[perm].contiguous())


def test_attend_batches_of_changing_size(kv):
    """Calls of different batch and head counts share a stream's workspace; every one is split over its length."""
    g = torch.Generator().manual_seed(77)
    lens = torch.tensor([3000, 2500, 2700, 100, 2900], dtype=torch.int32)
    table, pages = full_table(lens.tolist(), 32, g)
    cache = make_cache(kv, pages, 2, 32, 64, BF16, g)
    table, lens = table.to(DEV), lens.to(DEV)
    for n, hq in ((2, 4), (5, 16), (1, 2), (5, 16), (3, 40), (2, 4), (5, 16), (3, 40)):
        q = torch.randn(n, hq, 64, generator=g).to(DEV, BF16)
        check_attend(cache, q, table[:n], lens[:n])


@pytest.mark.parametrize("store", [F16, I8])
@pytest.mark.parametrize("B,lens", [(300, (1, 300)), (900, (1, 40)), (3000, (0, 3)), (2500, (100, 130)), (129, (0, 2000))])
def test_attend_many_short_and_a_few_long(kv, store, B, lens):
    """Ranges of work that begin and end inside items, at their ends and over sequences without tokens."""
    g = torch.Generator().manual_seed(B)
    n = torch.randint(lens[0], lens[1] + 1, (B,), generator=g)
    n[torch.rand(B, generator=g) < 0.2] = 0
    n[B // 3] = 1500
    n[B // 3 + 1:B // 3 + 40] = 0
    n[0] = n[-1] = 0
    table, pages = full_table(n.tolist(), 16, g)
    cache = make_cache(kv, pages, 1, 16, 64, store, g)
    q = torch.randn(B, 2, 64, generator=g).to(DEV, F16)
    check_attend(cache, q, table.to(DEV), n.to(DEV, torch.int32))
    cache.check_status()


@pytest.mark.parametrize("store", [BF16, I8])
def test_attend_scores_far_apart(kv, store):
    """A running maximum that keeps rising, one that falls, one key that takes all the weight."""
    g = torch.Generator().manual_seed(9)
    lens = [700, 700, 700]
    table, pages = full_table(lens, 64, g)
    cache = make_cache(kv, pages, 1, 64, 64, store, g)
    t = torch.arange(700)
    size = torch.stack([t * 0.05, 35 - t * 0.05, (t == 350) * 60.0])            # <q, k> along the sequence
    for b in range(3):
        p, s = table[b][t // 64].long(), t % 64
        if store == I8:
            cache.k[p, 0, s] = 64
            cache.k_scale[p, 0, s] = (size[b] / 64).to(DEV)
        else:
            cache.k[p, 0, s] = size[b][:, None].to(DEV, BF16)
    q = torch.ones(3, 1, 64, device=DEV, dtype=BF16)
    check_attend(cache, q, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("store", [F16, I8])
def test_attend_large_and_small_values(kv, store):
    """Value rows of very different scale (int8 scales from 2^-40 to 2^6, a row of zeros), queries near the type's ends."""
    g = torch.Generator().manual_seed(5)
    table, pages = full_table([150, 90], 16, g)
    cache = make_cache(kv, pages, 2, 16, 64, store, g)
    if store == I8:
        cache.v_scale.copy_(2.0 ** torch.randint(-40, 7, cache.v_scale.shape, generator=g))
        cache.v_scale[table[0, 0].long(), :, :3] = 0
        cache.k_scale[table[0, 0].long(), :, 3] = 0
    q = torch.randn(2, 4, 64, generator=g)
    q[0, 0] *= 1e-4
    q[0, 1] = 0
    lens = torch.tensor([150, 90], dtype=torch.int32, device=DEV)
    check_attend(cache, q.to(DEV, F16), table.to(DEV), lens)
    if store == I8:     # bf16 queries beyond fp16's range over int8 codes
        q[1, 0] *= 2.0 ** 40
        q[1, 1] *= 2.0 ** -60
        cache.k_scale.mul_(2.0 ** -40)
        check_attend(cache, q.to(DEV, BF16), table.to(DEV), lens)


def test_attend_non_finite_inputs(kv):
    """Visible infinities and not-a-numbers do what the formula does; a score of -infinity weighs nothing, also where
    a whole tile has no other."""
    g = torch.Generator().manual_seed(6)
    lens = torch.tensor([300, 300, 300, 300], dtype=torch.int32)
    table, pages = full_table(lens.tolist(), 64, g)
    cache = make_cache(kv, pages, 1, 64, 64, BF16, g)
    q = torch.randn(4, 2, 64, generator=g).abs().to(DEV, BF16) + 0.1
    p = table.long()
    cache.k[p[0, 1], 0, 5, 7] = float("nan")
    cache.k[p[1, :3], 0, :, 3] = float("-inf")              # tokens 0 .. 191 have no weight
    cache.k[p[2], 0, :, 3] = float("-inf")                  # none has
    cache.v[p[3, 0], 0, 2, 9] = float("inf")
    out, lse = cache.attend(q, table.to(DEV), lens.to(DEV))
    k, v = values(cache)
    eo, el, *_ = O.attend(c(q), k, v, c(table), c(lens), 1 / 8)
    out, lse = c(out), c(lse)
    assert np.isnan(out[0]).all() and np.isnan(lse[0]).all()
    np.testing.assert_allclose(out[1], eo[1], atol=0.03)
    np.testing.assert_allclose(lse[1], el[1], rtol=1e-5)
    assert (out[2] == 0).all() and np.isneginf(lse[2]).all()
    assert (out[3][:, 9] == np.inf).all() and np.isfinite(np.delete(out[3], 9, 1)).all()


def test_attend_strides_streams_and_graphs(kv):
    """Token-major cache memory, queries inside a fused projection, a slice of a wider table, another stream, a replayed
    graph with new lengths."""
    g = torch.Generator().manual_seed(8)
    lens = [100, 37, 260]
    table, pages = full_table(lens, 16, g, wide=30)
    cache = make_cache(kv, pages, 2, 16, 128, F16, g, token_major=True)
    fused = torch.randn(3, 12, 128, generator=g).to(DEV, F16)
    q = fused[:, 2:10]
    wide = torch.cat([torch.full((3, 4), 10 ** 6, dtype=torch.int32), table], 1).to(DEV)
    t, n = wide[:, 4:], torch.tensor(lens, dtype=torch.int32, device=DEV)
    check_attend(cache, q, t, n)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = cache.attend(q, t, n)
    torch.cuda.current_stream().wait_stream(s)
    mine = cache.attend(q, t, n)
    torch.cuda.synchronize()
    assert torch.equal(other[0], mine[0]) and torch.equal(other[1], mine[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cache.attend(q, t, n)
        again = cache.attend(q, t, n)
    for new in (lens, [0, 1, 400], [480, 480, 480]):
        n.copy_(torch.tensor(new, dtype=torch.int32))
        table_now = torch.where(t < 0, torch.zeros_like(t), t)
        t.copy_(table_now)
        graph.replay()
        check_attend(cache, q, t, n, got=got)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_attend_offsets_past_32_bits(kv):
    """The last pages of a cache of more than 2^31 elements (and 2^32 bytes) per tensor."""
    heads, page, dim = 8, 64, 256
    pages = 2 ** 31 // (heads * page * dim) + 40
    k, v = (torch.empty(pages, heads, page, dim, dtype=F16, device=DEV) for _ in range(2))
    g = torch.Generator().manual_seed(1)
    last = torch.arange(pages - 6, pages)
    for x in (k, v):
        x[-6:] = torch.randn(6, heads, page, dim, generator=g).to(DEV, F16)
    cache = kv.PagedKV(k, v)
    small = kv.PagedKV(k[-6:].clone(), v[-6:].clone())
    q = torch.randn(2, 8, dim, generator=g).to(DEV, F16)
    lens = torch.tensor([190, 100], dtype=torch.int32, device=DEV)
    high = last.reshape(2, 3).to(DEV, torch.int32)
    a, b = cache.attend(q, high, lens), small.attend(q, high - (pages - 6), lens)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    idx = torch.tensor([189, 5], dtype=torch.int32, device=DEV)
    x = torch.randn(2, heads, dim, generator=g).to(DEV, F16)
    cache.append(x, x, high, idx)
    got = cache.read(high, idx)
    assert torch.equal(got[0], x) and torch.equal(got[1], x)
    cache.check_status()


def test_attend_joins_by_lse(kv):
    """Two caches attended apart and joined by lse give the attention over both."""
    g = torch.Generator().manual_seed(2)
    table, pages = full_table([96], 16, g, spare=0)
    cache = make_cache(kv, pages, 2, 16, 64, F16, g)
    q = torch.randn(1, 4, 64, generator=g).to(DEV, F16)
    n = lambda x: torch.tensor([x], dtype=torch.int32, device=DEV)
    table = table.to(DEV)
    o1, l1 = cache.attend(q, table[:, :2].contiguous(), n(32))
    o2, l2 = cache.attend(q, table[:, 2:].contiguous(), n(64))
    o, l = cache.attend(q, table, n(96))
    m = torch.maximum(l1, l2)
    w1, w2 = (l1 - m).exp()[..., None], (l2 - m).exp()[..., None]
    joined = (o1.float() * w1 + o2.float() * w2) / (w1 + w2)
    assert (joined - o.float()).abs().max() <= 4 * U[F16] * max(1.0, float(cache.v.abs().max()))
    assert (torch.logaddexp(l1, l2) - l).abs().max() < 1e-5


def test_attend_bad_indices_are_reported(kv):
    g = torch.Generator().manual_seed(4)
    table, pages = full_table([64, 64], 16, g)
    cache = make_cache(kv, pages, 1, 16, 64, F16, g)
    q = torch.randn(2, 1, 64, generator=g).to(DEV, F16)
    ok = table.to(DEV)
    bad = ok.clone()
    bad[0, 1] = pages                                   # a page that there is not: as a hole
    hole = ok.clone()
    hole[0, 1] = -1
    n = torch.tensor([64, 64], dtype=torch.int32, device=DEV)
    a = cache.attend(q, bad, n)
    with pytest.raises(pkg("_lib").FvsError):
        cache.check_status()
    b = cache.attend(q, hole, n)
    cache.check_status()
    assert torch.equal(a[0], b[0])
    a = cache.attend(q, ok, torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device=DEV))     # cut to the table; none
    with pytest.raises(pkg("_lib").FvsError):
        cache.check_status()
    b = cache.attend(q, ok, torch.tensor([64, 0], dtype=torch.int32, device=DEV))
    cache.check_status()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------------------------------------ append and read

def rope(positions, rot, g):
    angle = torch.rand(positions, rot // 2, generator=g) * 6.3
    return angle.cos().to(DEV), angle.sin().to(DEV)


@pytest.mark.parametrize("dim,rot", [(64, 64), (64, 32), (96, 96), (96, 48), (128, 128), (128, 16), (192, 192), (192, 0),
                                     (256, 256), (256, 128)])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("dtype,store", [(BF16, BF16), (F16, F16), (BF16, I8), (F16, I8)])
def test_append(kv, dim, rot, pairs, dtype, store):
    g = torch.Generator().manual_seed(dim + rot)
    heads, hq, page, n = 3, 5, 20, 37
    table, pages = full_table([60, 45, 0], page, g)
    cache = make_cache(kv, pages, heads, page, dim, store, g)
    before = [x.clone() for x in (cache.k, cache.v)]
    fused = torch.randn(n, hq + 2 * heads, dim, generator=g).to(DEV, dtype)
    fused[3] = 0
    q, k, v = fused[:, :hq], fused[:, hq:hq + heads], fused[:, hq + heads:]
    place = torch.randperm(105, generator=g)[:n]
    seq, idx = (place >= 60).int(), torch.where(place >= 60, place - 60, place).int()
    idx[5] = -1
    seq[6], idx[6] = 2, 0                                  # a hole
    pos = torch.randint(0, 50, (n,), generator=g, dtype=torch.int32)
    table, seq, idx, pos = (x.to(DEV) for x in (table, seq, idx, pos))
    cs = rope(50, rot, g) if rot else None
    got = cache.append(k, v, table, idx, seq=seq, pos=pos, rope=cs, pairs=pairs, q=q)
    torch.cuda.synchronize()
    cache.check_status()
    cos, sin = (c(x)[c(pos)] for x in cs) if rot else (None, None)
    eq, mq = O.rotate(c(q), cos, sin, rot, pairs)
    ek, mk = O.rotate(c(k), cos, sin, rot, pairs)
    ev, mv = c(v), np.zeros_like(c(v))
    at = O.rows_of(c(table), page, c(seq), c(idx), pages)
    there = np.array([a is not None for a in at])
    assert not there[5] and not there[6] and there.sum() == n - 2
    u = U[dtype]
    got = c(got)
    assert (got[~there] == 0).all()
    assert (np.abs(got - eq) <= u * np.abs(eq) * (1 + 2 ** -8) + 3 * 2.0 ** -24 * mq + 2.0 ** -25)[there].all()
    kk, vv = values(cache)
    touched = np.zeros((pages, page), bool)
    for t, a in enumerate(at):
        if a is None:
            continue
        touched[a] = True
        for have, want, mag in ((kk, ek, mk), (vv, ev, mv)):
            row, e = have[a[0], :, a[1]], want[t]
            if store == I8:
                step = np.abs(e).max(-1, keepdims=True) / 127
                bound = 0.5 * step + 2.0 ** -20 * 127 * step + 3 * 2.0 ** -24 * mag[t]
            else:
                bound = u * np.abs(e) * (1 + 2 ** -8) + 3 * 2.0 ** -24 * mag[t] + 2.0 ** -25
            assert (np.abs(row - e) <= bound).all(), t
    keep = torch.from_numpy(~touched).to(DEV)
    for x, old in zip((cache.k, cache.v), before):
        assert torch.equal(x.transpose(1, 2)[keep], old.transpose(1, 2)[keep])


def test_append_defaults_in_place_and_single_tokens(kv):
    """seq and pos by default, q rotated in place, one token, none."""
    g = torch.Generator().manual_seed(12)
    table, pages = full_table([40, 40, 40], 8, g)
    table = table.to(DEV)
    cs = rope(64, 64, g)
    for n in (3, 1, 0):
        idx = torch.tensor([7, 20, 39], dtype=torch.int32, device=DEV)[:n]
        x = [torch.randn(n, h, 64, generator=g).to(DEV, F16) for h in (4, 2, 2)]
        one, two = (make_cache(kv, pages, 2, 8, 64, F16, torch.Generator().manual_seed(1)) for _ in range(2))
        a = one.append(x[1], x[2], table, idx, rope=cs, q=x[0])
        q = x[0].clone()
        b = two.append(x[1], x[2], table, idx, seq=torch.arange(n, dtype=torch.int32, device=DEV), pos=idx, rope=cs,
                       q=q, q_out=q)
        assert torch.equal(a, b) and b is q
        assert torch.equal(one.k, two.k) and torch.equal(one.v, two.v)
        assert one.append(x[1], x[2], table, idx, rope=cs) is None


@pytest.mark.parametrize("value,code", [(float("nan"), None), (float("inf"), None), (1e-40, 0), (3e38, 127)])
def test_append_int8_odd_rows(kv, value, code):
    """Rows that no code can hold read back as not-a-numbers; rows at the type's ends stay finite."""
    cache = kv.PagedKV.empty(1, 1, 4, 64, dtype=I8)
    x = torch.zeros(1, 1, 64, device=DEV, dtype=BF16)
    x[0, 0, 5] = value
    table, idx = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([2], dtype=torch.int32, device=DEV)
    cache.append(x, x, table, idx)
    k, v = cache.read(table, idx)
    if code is None:
        assert torch.isnan(k).all() and torch.isnan(v).all()
    else:
        assert torch.isfinite(k).all() and int(cache.k[0, 0, 2].max()) == code
        if code:
            assert abs(float(k[0, 0, 5]) / float(x[0, 0, 5]) - 1) < 1e-5


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("store", [F16, BF16, I8])
@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
def test_read(kv, dim, store, dtype):
    g = torch.Generator().manual_seed(dim)
    table, pages = full_table([50, 31], 7, g)
    cache = make_cache(kv, pages, 3, 7, dim, store, g, token_major=dim == 96)
    seq = torch.tensor([0] * 50 + [1] * 31 + [0, 1], dtype=torch.int32)
    idx = torch.tensor([*range(50), *range(31), -1, 49], dtype=torch.int32)        # no token; a hole of sequence 1
    got = cache.read(table.to(DEV), idx.to(DEV), seq=seq.to(DEV), dtype=dtype)
    cache.check_status()
    at = O.rows_of(table.numpy(), 7, seq.numpy(), idx.numpy(), pages)
    assert at[-1] is None and at[-2] is None
    for x, y, s in zip(got, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        assert x.dtype == dtype and x.shape == (83, 3, dim)
        want = torch.zeros(83, 3, dim)
        for t, a in enumerate(at):
            if a is not None:
                row = y[a[0], :, a[1]].float()
                want[t] = (row if s is None else row * s[a[0], :, a[1]][:, None]).cpu()
        assert torch.equal(x.cpu(), want.to(dtype))


def test_append_and_read_bad_indices_are_reported(kv):
    FvsError = pkg("_lib").FvsError
    g = torch.Generator().manual_seed(14)
    table, pages = full_table([32, 32], 16, g)
    cache = make_cache(kv, pages, 1, 16, 64, F16, g)
    k0, v0 = cache.k.clone(), cache.v.clone()
    x = torch.randn(1, 1, 64, generator=g).to(DEV, F16)
    i = lambda n: torch.tensor([n], dtype=torch.int32, device=DEV)
    ok = table.to(DEV)
    worse = ok.clone()
    worse[0, 0] = pages + 7
    cs = rope(8, 64, g)
    for t, seq, idx, pos in ((ok, 2, 0, 0), (ok, -1, 0, 0), (ok, 0, 32, 0), (ok, 0, 2 ** 31 - 1, 0), (worse, 0, 3, 0),
                             (ok, 0, 0, 8), (ok, 0, 0, -1)):
        q = cache.append(x, x, t, i(idx), seq=i(seq), pos=i(pos), rope=cs, q=x)
        assert (q == 0).all()
        with pytest.raises(FvsError):
            cache.check_status()
        if 0 <= pos < 8:
            k, v = cache.read(t, i(idx), seq=i(seq))
            assert (k == 0).all() and (v == 0).all()
            with pytest.raises(FvsError):
                cache.check_status()
    cache.check_status()
    assert torch.equal(cache.k, k0) and torch.equal(cache.v, v0)


# ------------------------------------------------------------------------------------------------ refusals, together

def test_refusals(kv):
    g = torch.Generator().manual_seed(15)
    z = lambda *s, dtype=F16: torch.zeros(*s, dtype=dtype, device=DEV)
    for args in ((z(2, 1, 4, 80), z(2, 1, 4, 80)),                                        # head dim
                 (z(2, 1, 4, 64), z(2, 1, 4, 64, dtype=BF16)), (z(2, 1, 4, 64), z(2, 1, 5, 64)),
                 (z(2, 1, 4, 64, dtype=torch.float32), z(2, 1, 4, 64, dtype=torch.float32)),
                 (z(2, 1, 4, 64, dtype=I8), z(2, 1, 4, 64, dtype=I8)),                    # codes without scales
                 (z(2, 1, 4, 64), z(2, 1, 4, 64), z(2, 1, 4, dtype=torch.float32), z(2, 1, 4, dtype=torch.float32)),
                 (z(2, 1, 4, 68)[..., :64], z(2, 1, 4, 68)[..., :64]),                    # rows not 16-byte aligned
                 (z(2, 1, 4, 128)[..., ::2], z(2, 1, 4, 128)[..., ::2]),
                 (torch.zeros(2, 1, 4, 64), torch.zeros(2, 1, 4, 64)),                    # host memory
                 (z(2, 1, 4, 64), z(2, 1, 4, 64), None, None, z(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            kv.PagedKV(*args)
    cache = make_cache(kv, 4, 2, 16, 64, F16, g)
    t, n = z(3, 2, dtype=torch.int32), z(3, dtype=torch.int32)
    q = z(3, 4, 64)
    for args, more in (((q.float(), t, n), {}), ((q.to(BF16), t, n), {}), ((z(3, 5, 64), t, n), {}),
                       ((z(3, 4, 96), t, n), {}), ((q, t.long(), n), {}), ((q, t[:2], n), {}), ((q, t, n.long()), {}),
                       ((q, t, n[:2]), {}), ((q.cpu(), t, n), {}), ((z(3, 64, 4).transpose(1, 2), t, n), {}),
                       ((z(3 * 4 * 64 + 4)[4:].view(3, 4, 64), t, n), {}),
                       ((q, t, n), dict(out=q.float())), ((q, t, n), dict(lse=z(3, 4)))):
        with pytest.raises(ValueError):
            cache.attend(*args, **more)
    k = z(3, 2, 64)
    cs = rope(8, 64, g)
    for args, more in (((k.to(BF16), k, t, n), {}), ((z(3, 3, 64), k, t, n), {}), ((k, k, t, n.long()), {}),
                       ((k, k, t[:2], n), {}), ((k, k, t, n), dict(rope=(cs[0].half(), cs[1].half()))),
                       ((k, k, t, n), dict(rope=rope(8, 24, g))), ((k, k, t, n), dict(rope=rope(8, 80, g))),
                       ((k, k, t, n), dict(rope=cs, pairs="thirds")), ((k, k, t, n), dict(pos=n.long())),
                       ((k, k, t, n), dict(q=q, q_out=z(3, 4, 128)[..., :64]))):
        with pytest.raises(ValueError):
            cache.append(*args, **more)
    with pytest.raises(ValueError):
        cache.read(t, n, dtype=torch.float64)
    assert cache.launches == 0


def test_search_then_answer(kv):
    """The ids of a search become a page table; a decoding loop appends its own tokens and attends over both."""
    eng = pkg("engine")
    import __graft_entry__ as ge
    ds, s1, i8, code, ix = ge._tiny_index(DEV)
    E = eng.EngineB200I8(ix)
    I, _, _ = E.search(ds["queries"], 40, 1.25, 12, 4)
    I = I[:6].clone()
    I[0, 2] = -1                                                       # a search that found fewer
    g = torch.Generator().manual_seed(16)
    N, page, heads, hq, dim, B = ix.N, 16, 2, 8, 64, 6
    found = torch.unique(I[I >= 0])
    length = torch.randint(1, 33, (len(found),), generator=g)
    pages_of = torch.full((N, 2), -1, dtype=torch.int32, device=DEV)
    need = (length + page - 1) // page
    first = torch.cumsum(need, 0) - need
    total = int(need.sum()) + B * 2
    fill = torch.full((total,), page, dtype=torch.int32)
    for i, (f, n) in enumerate(zip(first.tolist(), length.tolist())):
        for p in range(int(need[i])):
            pages_of[found[i], p] = f + p
            fill[f + p] = min(page, n - p * page)
    own = torch.arange(total - 2 * B, total, dtype=torch.int32, device=DEV).view(B, 2)
    cache = make_cache(kv, total, heads, page, dim, BF16, g, fill=fill.to(DEV))
    table = kv.passage_table(I, pages_of, own)
    assert table.shape == (B, 4 * 2 + 2)
    base = 4 * 2 * page
    cs = rope(64, dim, g)
    for step in range(18):
        idx = torch.full((B,), base + step, dtype=torch.int32, device=DEV)
        pos = torch.full((B,), step, dtype=torch.int32, device=DEV)
        qkv = torch.randn(B, hq + 2 * heads, dim, generator=g).to(DEV, BF16)
        q = cache.append(qkv[:, hq:hq + heads], qkv[:, hq + heads:], table, idx, pos=pos, rope=cs, q=qkv[:, :hq])
        got = cache.attend(q, table, idx + 1)
        if step in (0, 15, 17):
            check_attend(cache, q, table, idx + 1, got=got)
    cache.check_status()


def test_example_answers_from_passages():
    """examples/answer_from_passages.py: the attention of its last step against plain products of what the cache holds:
    within the rounding of bf16 outputs (2^-8) and as much again."""
    import importlib.util
    import os
    from conftest import REPO
    pkg("build").build()
    spec = importlib.util.spec_from_file_location("answer", os.path.join(REPO, "examples", "answer_from_passages.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main(steps=20) < 2 ** -7


def test_attend_one_table_for_all_and_long_rows(kv):
    """A page table whose rows are one row (stride 0), and more sequences than a grid axis holds."""
    g = torch.Generator().manual_seed(21)
    table, pages = full_table([70], 16, g)
    cache = make_cache(kv, pages, 1, 16, 64, F16, g)
    n = 70000
    q = torch.randn(3, 2, 64, generator=g).to(DEV, F16)
    shared = table.to(DEV).expand(n, -1)
    lens = (torch.arange(n, device=DEV) % 71).int()
    many = q[torch.arange(n, device=DEV) % 3]
    out, lse = cache.attend(many, shared, lens)
    some = torch.arange(0, n, 997, device=DEV)
    a, b = out[some].contiguous(), lse[some].contiguous()
    check_attend(cache, many[some].contiguous(), shared[some].contiguous(), lens[some].contiguous(), got=(a, b))


def test_attend_two_streams_at_once(kv):
    """Calls in flight on two streams have workspaces of their own."""
    g = torch.Generator().manual_seed(22)
    table, pages = full_table([9000, 8000], 64, g)
    cache = make_cache(kv, pages, 4, 64, 128, BF16, g)
    lens = torch.tensor([9000, 8000], dtype=torch.int32, device=DEV)
    q = [torch.randn(2, 8, 128, generator=g).to(DEV, BF16) for _ in range(2)]
    table = table.to(DEV)
    want = [cache.attend(x, table, lens) for x in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(cache.attend(q[k], table, lens))
    torch.cuda.synchronize()
    for k in range(2):
        for o, l in got[k]:
            assert torch.equal(o, want[k][0]) and torch.equal(l, want[k][1])


def test_attend_graph_of_several_caches(kv):
    """Layers captured together (their workspaces follow one another in the graph's memory), replayed beside eager calls on
    another stream."""
    g = torch.Generator().manual_seed(23)
    table, pages = full_table([5000, 4000, 10], 32, g)
    caches = [make_cache(kv, pages, 2, 32, d, BF16, g) for d in (64, 128, 64)]
    lens = torch.tensor([5000, 4000, 10], dtype=torch.int32, device=DEV)
    table = table.to(DEV)
    q = [torch.randn(3, 8, c.dim, generator=g).to(DEV, BF16) for c in caches]
    want = [c.attend(x, table, lens) for c, x in zip(caches, q)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [c.attend(x, table, lens) for c, x in zip(caches, q)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for o, l in got:
            o.zero_()
        graph.replay()
        with torch.cuda.stream(side):
            beside = [c.attend(x, table, lens) for c, x in zip(caches, q)]
        torch.cuda.synchronize()
        for a in (got, beside):
            for (o, l), (wo, wl) in zip(a, want):
                assert torch.equal(o, wo) and torch.equal(l, wl)
