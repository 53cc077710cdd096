"""The paged cache where its arithmetic could lose something: attention weights far below the largest, value scales and keys
of very different size, rows that hold infinities, codes of very small rows; and calls large enough to take the attention
kernel's other ways of dividing the work.

Bounds, from the arithmetic alone, with u the unit roundoff of the output type and n the keys of a sequence:
* a score is a sum of exact products (codes, 16-bit numbers), 16 to an instruction, in D / 16 instructions, each of which may
  cut up to 2^-23 of the largest term or partial sum, plus 20 such steps for the ends (scale, factors of the heads, the
  difference to the running maximum): es = (D / 16 + 20) 2^-23 scale sum |q k|, which changes a weight by a factor e^(es);
* a weight enters the second product with 21 bits or more: ep = 2^-20 of sum p |v|; over fp16 values and codes its parts end
  at 2^-36 of the largest weight (of the largest weight times value scale over codes), so a key that is smaller still may be off
  by 2^-35 of that;
* sums of fp32 over at most n / 16 + 64 steps, each cutting 2^-23: (n / 16 + 64) 2^-23 of sum p |v|;
* one rounding of the output, u of it (2^-25 where fp16 has no more bits, 2^-134 where bf16 has none).
"""
import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import kv_oracle as O
from test_gpu_kv import BF16, DEV, F16, I8, U, c, full_table, make_cache, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    pkg("build").build()
    return pkg("kvcache")


def close(cache, q, table, lens, got=None):
    """attend against the oracle within the bounds above."""
    out, lse = got or cache.attend(q, table, lens)
    torch.cuda.synchronize()
    d, scale = cache.dim, 1 / np.sqrt(cache.dim)
    k, v = values(cache)
    fill = None if cache.fill is None else c(cache.fill)
    eo, el, pv, av, mag = O.attend(c(q), k, v, c(table), c(lens), scale, fill)
    out, lse = c(out), c(lse)
    assert np.isfinite(out).all() and np.isfinite(lse[np.isfinite(el)]).all()
    es = (d / 16 + 20) * 2.0 ** -23 * mag
    sums = (c(lens) / 16 + 64)[:, None] * 2.0 ** -23
    least = 2.0 ** -35 * av                              # av: sum |v| over the sum of the weights
    if cache.dtype == I8:                                # in units of the largest weighted scale
        top = np.zeros_like(el)
        n = np.zeros_like(el)
        for b in range(len(top)):
            t = np.arange(int(lens[b]))
            p, s = c(table)[b][t // cache.page], t % cache.page
            g = q.shape[1] // cache.heads
            for h in range(q.shape[1]):
                w = np.exp(k[p, h // g, s] @ c(q)[b, h] * scale - el[b, h])
                top[b, h], n[b, h] = (w * np.abs(c(cache.v_scale)[p, h // g, s])).max(initial=0), len(t)
        least = (2.0 ** -35 * 127 * n * top)[..., None]
    tol = U[q.dtype] * np.abs(eo) + (2 * es[..., None] + 2.0 ** -20 + sums[..., None]) * pv * 1.01 + least
    tol += 2.0 ** -25 if q.dtype == F16 else 2.0 ** -134
    worst = (np.abs(out - eo) / np.maximum(tol, 1e-300)).max()
    assert worst <= 1, f"out is {worst:.2f} of its bound"
    tol = es + sums + 2.0 ** -22 * (1 + np.abs(np.where(np.isfinite(el), el, 0)))
    seen = np.isfinite(el)
    worst = (np.abs(lse[seen] - el[seen]) / tol[seen]).max(initial=0)
    assert worst <= 1, f"lse is {worst:.2f} of its bound"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------------------ weights

@pytest.mark.parametrize("dtype,store", [(F16, F16), (BF16, BF16), (F16, I8), (BF16, I8)])
@pytest.mark.parametrize("bits", [12, 17, 22, 25.2, 29])
def test_weights_far_below_the_largest(kv, dtype, store, bits):
    """Keys without a value take nearly all of the weight; the others, 2^-bits of one of them, make the output."""
    g = torch.Generator().manual_seed(int(bits))
    n, page, dim = 4000, 16, 64
    table, pages = full_table([n], page, g)
    first = torch.zeros(pages * page, dtype=torch.bool)
    t = torch.arange(n)
    place = table[0].long()[t // page] * page + t % page
    first[place[t % 32 == 3]] = True                                # in every unit of work
    first = first.view(pages, 1, page, 1).to(DEV)
    score = np.log(2) * bits                                        # <q, k> / 8 = 8 k for q = 1
    k = torch.where(first, score / 8, 0.0) * torch.ones(pages, 1, page, dim, device=DEV)
    v = (torch.rand(pages, 1, page, dim, generator=g).to(DEV) + 0.5) * 1000
    if store == I8:
        one = torch.ones(pages, 1, page, device=DEV)
        cache = kv.PagedKV((first * 64 * torch.ones_like(k)).to(I8), torch.where(first, 0.0, v / 12).round().to(I8),
                           one * float(score) / 8 / 64, one * 12)
    else:
        cache = kv.PagedKV(k.to(store), torch.where(first, 0.0, v).to(store))
    close(cache, torch.ones(1, 2, dim, dtype=dtype, device=DEV), table.to(DEV), ints([n]))


@pytest.mark.parametrize("dtype,store", [(F16, F16), (F16, I8), (BF16, I8), (BF16, BF16)])
def test_weights_are_not_cut(kv, dtype, store):
    """Two keys whose values nearly cancel show how many bits of their weights reach the output."""
    g = torch.Generator().manual_seed(31)
    B, dim, page = 256, 64, 16
    table = torch.arange(B, dtype=torch.int32).view(B, 1)
    size = torch.rand(B, 1, page, generator=g) * 0.25
    v = torch.ones(B, 1, page, dim) * 96
    v[:, :, 1] = -v[:, :, 0] * torch.exp(8 * (size[:, :, 0] - size[:, :, 1]))[..., None]
    size, v = size.to(DEV), v.to(DEV)
    if store == I8:
        cache = kv.PagedKV(torch.full((B, 1, page, dim), 64, dtype=I8, device=DEV), (v / 8).round().to(I8), size / 64,
                           torch.full_like(size, 8))
    else:
        cache = kv.PagedKV((size[..., None] * torch.ones(dim, device=DEV)).to(store), v.to(store))
    close(cache, torch.ones(B, 1, dim, dtype=dtype, device=DEV), table.to(DEV), ints([2] * B))


@pytest.mark.parametrize("dtype,store", [(F16, F16), (BF16, BF16), (F16, I8), (BF16, I8)])
def test_outputs_are_the_nearest_numbers(kv, dtype, store):
    """Errors of 2^-19 of an output, some ulps of fp32, put it on a neighbouring number of its type only where the 64-bit value
    lies that near to the middle of two, and these are u to 2 u of it apart: 2 * 2^-19 / u of the outputs."""
    g = torch.Generator().manual_seed(40)
    lens = torch.randint(500, 2500, (24,), generator=g).tolist()
    table, pages = full_table(lens, 32, g)
    cache = make_cache(kv, pages, 2, 32, 128, store, g)
    q = (torch.randn(24, 16, 128, generator=g) * 1.5).to(DEV, dtype)
    out, _ = cache.attend(q, table.to(DEV), ints(lens))
    eo, *_ = O.attend(c(q), *values(cache), table.numpy(), np.array(lens), 1 / np.sqrt(128))
    nearest = torch.from_numpy(eo).to(dtype)        # by way of fp32, whose rounding is of no account here
    apart = float((out.cpu() != nearest).double().mean())
    assert apart <= 2.0 ** -18 / U[dtype], apart


@pytest.mark.parametrize("dtype,store", [(F16, F16), (BF16, I8)])
def test_scores_that_keep_rising(kv, dtype, store):
    """Every unit of work passes the running maximum, by steps small and large."""
    g = torch.Generator().manual_seed(32)
    n, page, dim = 1500, 32, 64
    table, pages = full_table([n] * 3, page, g)
    cache = make_cache(kv, pages, 1, page, dim, store, g)
    for b, step in enumerate((0.001, 0.02, 0.4)):
        t = torch.arange(n)
        p, s = table[b].long()[t // page], t % page
        if store == I8:
            cache.k[p, 0, s] = 32
            cache.k_scale[p, 0, s] = (t * step / 8 / 32).to(DEV)
        else:
            cache.k[p, 0, s] = (t * step / 8)[:, None].to(DEV, store)
    close(cache, torch.ones(3, 2, dim, dtype=dtype, device=DEV), table.to(DEV), ints([n] * 3))


# ------------------------------------------------------------------------------------------------ value scales of codes

@pytest.mark.parametrize("ratio", [2.0 ** 12, 2.0 ** 16, 2.0 ** 20, 2.0 ** 24, 2.0 ** 40])
@pytest.mark.parametrize("below", [60, 100])
def test_large_value_scales_that_weigh_nothing(kv, ratio, below):
    """Rows of a scale far above the others', at 2^-below of their weight, leave the others' bits alone."""
    g = torch.Generator().manual_seed(33)
    n, page, dim = 1000, 16, 64
    table, pages = full_table([n, n], page, g)
    cache = make_cache(kv, pages, 1, page, dim, I8, g)
    cache.k.fill_(64)
    cache.k_scale.fill_(0)
    cache.v_scale.fill_(1 / 64)
    t = torch.arange(7, n, 32)                                      # one in every unit of work, in one sequence at the end
    for b, t in ((0, t), (1, torch.tensor([n - 1]))):
        p, s = table[b].long()[t // page], t % page
        cache.k_scale[p, 0, s] = -below * float(np.log(2)) / 8 / 64
        cache.v_scale[p, 0, s] = ratio / 64
    close(cache, torch.ones(2, 2, dim, dtype=BF16, device=DEV), table.to(DEV), ints([n, n]))


def test_heads_that_weigh_rows_of_different_scale(kv):
    """Query heads that share codes and prefer rows of different scale each keep their bits."""
    g = torch.Generator().manual_seed(34)
    n, page, dim, hq = 600, 16, 64, 8
    table, pages = full_table([n], page, g)
    cache = make_cache(kv, pages, 1, page, dim, I8, g)
    t = torch.arange(n)
    p, s = table[0].long()[t // page], t % page
    cache.k[p, 0, s] = 0
    cache.k[p, 0, s, t % hq] = 64                                   # head h prefers the tokens t = h mod 8
    cache.k_scale.fill_(1 / 64)
    cache.v_scale[p, 0, s] = (2.0 ** (-6.0 * (t % hq)) / 64).to(DEV)
    q = torch.zeros(1, hq, dim)
    q[0, torch.arange(hq), torch.arange(hq)] = 8 * 40               # scores of 40 and 0: 2^-57
    close(cache, q.to(DEV, BF16), table.to(DEV), ints([n]))


@pytest.mark.parametrize("log", [-126, -110, -60, 0, 60, 100, 103, 110])
def test_value_scales_near_the_ends_of_fp32(kv, log):
    g = torch.Generator().manual_seed(35)
    table, pages = full_table([300, 1], 16, g)
    cache = make_cache(kv, pages, 2, 16, 64, I8, g)
    cache.v_scale.mul_(2.0 ** 5).mul_(2.0 ** log)                   # about 2^log of a code
    q = torch.randn(2, 4, 64, generator=g).to(DEV, BF16)
    close(cache, q, table.to(DEV), ints([300, 1]))


# ------------------------------------------------------------------------------------------------ scores over codes

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_scores_of_rows_with_one_large_element(kv, dtype, dim):
    """One element takes a row's scale, and no query has it; a sequence of one key has its score as lse."""
    g = torch.Generator().manual_seed(dim)
    B, page = 64, 16
    x = torch.rand(B, 1, page, dim, generator=g) + 0.5
    x[..., 5] = 127
    cache = kv.PagedKV(x.round().to(DEV, I8), x.round().to(DEV, I8), *(torch.ones(B, 1, page, device=DEV) for _ in range(2)))
    q = torch.rand(B, 8, dim, generator=g) + 0.5
    q[..., 5] = 0
    close(cache, q.to(DEV, dtype), torch.arange(B).view(B, 1).to(DEV, torch.int32), ints([1] * B))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_queries_with_one_large_element(kv, dtype):
    """Elements far below the head's largest keep their bits."""
    g = torch.Generator().manual_seed(36)
    B, page, dim = 64, 16, 64
    cache = make_cache(kv, B, 1, page, dim, I8, g)
    cache.k[..., 9] = 0
    q = torch.randn(B, 8, dim, generator=g) * 2.0 ** -6
    q[..., 9] = 2.0 ** 15
    close(cache, q.to(DEV, dtype), torch.arange(B).view(B, 1).to(DEV, torch.int32), ints([1] * B))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("odd", [float("inf"), float("nan")])
def test_key_rows_of_codes_that_are_not_finite(kv, dtype, odd):
    """A key row stored with an infinity or a not-a-number makes every head that sees it not-a-number, and nothing else."""
    g = torch.Generator().manual_seed(37)
    B, hq, page, dim = 16, 64, 16, 128
    lens = [40 + b for b in range(B)]
    table, pages = full_table(lens, page, g)
    cache = make_cache(kv, pages, 1, page, dim, I8, g)
    table = table.to(DEV)
    k = torch.randn(B // 2, 1, dim, generator=g)
    k[:, 0, 3] = odd
    v = torch.randn(B // 2, 1, dim, generator=g).to(DEV, dtype)
    cache.append(k.to(DEV, dtype), v, table, ints([b * 5 for b in range(B // 2)]))
    q = torch.randn(B, hq, dim, generator=g).to(DEV, dtype)
    out, lse = cache.attend(q, table, ints(lens))
    assert torch.isnan(lse[:B // 2]).all() and torch.isnan(out[:B // 2]).all()
    assert torch.isfinite(lse[B // 2:]).all() and torch.isfinite(out[B // 2:]).all()


def test_value_rows_of_codes_that_are_not_finite(kv):
    g = torch.Generator().manual_seed(38)
    table, pages = full_table([200, 200], 16, g)
    cache = make_cache(kv, pages, 1, 16, 64, I8, g)
    table = table.to(DEV)
    x = torch.randn(1, 1, 64, generator=g).to(DEV, F16)
    odd = x.clone()
    odd[0, 0, 7] = float("-inf")
    cache.append(x, odd, table, ints([123]))
    out, lse = cache.attend(torch.randn(2, 2, 64, generator=g).to(DEV, F16), table, ints([200, 200]))
    assert torch.isnan(out[0]).all() and torch.isfinite(lse).all() and torch.isfinite(out[1]).all()


def test_infinite_fp16_values(kv):
    """A visible infinite value whose weight has no lower half gives an infinity, not a not-a-number."""
    g = torch.Generator().manual_seed(39)
    table, pages = full_table([50], 16, g)
    cache = make_cache(kv, pages, 1, 16, 64, F16, g)
    cache.k.zero_()                                                 # all weights are the same power of two before the end
    p = table[0].long()
    cache.v[p[1], 0, 4, 9] = float("inf")
    cache.v[p[2], 0, 1, 3] = float("-inf")
    out, _ = cache.attend(torch.ones(1, 2, 64, dtype=F16, device=DEV), table.to(DEV), ints([50]))
    assert (out[0, :, 9] == float("inf")).all() and (out[0, :, 3] == float("-inf")).all()
    assert torch.isfinite(out[0]).sum() == 2 * 62


# ------------------------------------------------------------------------------------------------ large calls, wide heads

@pytest.mark.parametrize("dtype,store,dim,group", [(BF16, I8, 128, 8), (F16, F16, 64, 4), (F16, I8, 64, 12)])
def test_large_calls(kv, dtype, store, dim, group):
    """Calls whose pieces are taken as blocks finish, with items cut at uneven places; then a small call on the same stream.
    The sequences share the pages of one pool, each in an order of its own."""
    g = torch.Generator().manual_seed(dim + group)
    heads, page, pool, B = 8, 64, 256, 160
    cache = make_cache(kv, pool, heads, page, dim, store, g)
    table = torch.stack([torch.randperm(pool, generator=g) for _ in range(B)]).to(DEV, torch.int32)
    lens = torch.randint(2000, pool * page + 1, (B,), generator=g, dtype=torch.int32)
    lens[3], lens[40], lens[41], lens[B - 1] = 0, 1, 100, pool * page
    units = int((lens.long() // (32 if store == I8 or dim == 64 else 16) + 3).sum()) * heads * -(-group // 16)
    assert units >= 512 * 444, "too small a call to be divided that way"
    q = torch.randn(B, heads * group, dim, generator=g).to(DEV, dtype)
    lens = lens.to(DEV)
    first = cache.attend(q, table, lens)
    for _ in range(2):
        again = cache.attend(q, table, lens)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    small = cache.attend(q[40:42].contiguous(), table[40:42].contiguous(), lens[40:42].contiguous())
    some = torch.tensor([3, 40, 41, 7, 90, B - 1], device=DEV)
    heads_seen = [0, heads * group // 2 + 1, heads * group - 1]
    # the oracle takes the sampled heads one at a time, each over its own key head
    for h in heads_seen:
        kh = h // group
        scales = [None if s is None else s[:, kh:kh + 1] for s in (cache.k_scale, cache.v_scale)]
        part = kv.PagedKV(cache.k[:, kh:kh + 1], cache.v[:, kh:kh + 1], *scales)
        pick = lambda x: x[some][:, h:h + 1].contiguous()  # noqa: E731
        close(part, pick(q), table[some], lens[some], got=(pick(first[0]), pick(first[1])))
    close(cache, q[40:42].contiguous(), table[40:42], lens[40:42], got=small)


@pytest.mark.parametrize("dtype,store", [(F16, F16), (BF16, BF16), (BF16, I8)])
@pytest.mark.parametrize("dim,group", [(192, 4), (256, 16), (256, 5)])
def test_wide_heads_over_long_sequences(kv, dtype, store, dim, group):
    g = torch.Generator().manual_seed(dim + group)
    lens = [5000, 3000, 1, 0, 4099]
    table, pages = full_table(lens, 48, g)
    cache = make_cache(kv, pages, 1, 48, dim, store, g)
    q = torch.randn(len(lens), group, dim, generator=g).to(DEV, dtype)
    close(cache, q, table.to(DEV), ints(lens))


# ------------------------------------------------------------------------------------------------ append of codes

@pytest.mark.parametrize("top", [2.0 ** -126, 1.3e-38, 1e-37, 3e-37, 3.7e-37, 1e-36, 2.0 ** -100, 7.8e-31, 1e-30])
@pytest.mark.parametrize("dim", [64, 96])
def test_append_of_small_rows(kv, top, dim):
    """Rows of a small largest magnitude: each code within half a step (and 2^-20 of 127 steps of fp32 rounding), the scale
    within half of fp32's smallest number."""
    g = torch.Generator().manual_seed(41)
    cache = kv.PagedKV.empty(2, 2, 16, dim, dtype=I8)
    x = ((torch.rand(20, 2, dim, generator=g) * 2 - 1) * top).to(DEV, BF16)
    x[:, :, 5] = top
    table, idx = torch.tensor([[1, 0]] * 20, dtype=torch.int32, device=DEV), torch.arange(20, dtype=torch.int32, device=DEV)
    cache.append(x, x, table, idx)
    want = c(x)
    step = np.abs(want).max(-1, keepdims=True) / 127
    bound = 0.5 * step + 2.0 ** -20 * 127 * step + 127 * 2.0 ** -149
    for got in cache.read(table, idx):
        assert (np.abs(c(got) - want) <= bound).all()


def test_append_of_subnormal_rows_stores_zeros(kv):
    cache = kv.PagedKV.empty(1, 1, 16, 64, dtype=I8)
    x = torch.full((1, 1, 64), 2.0 ** -127, device=DEV, dtype=BF16)
    table, idx = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([2], dtype=torch.int32, device=DEV)
    cache.append(x, x, table, idx)
    assert not cache.k.any() and not cache.k_scale.any() and not cache.v.any() and not cache.v_scale.any()
