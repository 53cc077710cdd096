"""Paged key-value cache on the host: the C entry points refuse wrong arguments before any device work, the Python layer
refuses host memory, and the 64-bit oracle agrees with torch's own formulas."""
import ctypes as C

import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import kv_oracle as O


@pytest.fixture(scope="module")
def L():
    pkg("build").build()
    return pkg("_lib")


def cache(L, **change):
    """A cache descriptor of addresses that are never followed."""
    c = L.KvCache(4096, 8192, None, None, None, 64, 2 * 16 * 64, 16 * 64, 64, 0, 0, 0, 4, 2, 16, 64, L.F16)
    for k, v in change.items():
        setattr(c, k, v)
    return C.byref(c)


BAD_CACHES = [dict(k=None), dict(v=4100), dict(status=None), dict(pages=0), dict(heads=0), dict(page=0), dict(type=7),
              dict(slot_stride=63), dict(slot_stride=32), dict(page_stride=4), dict(head_stride=-8), dict(type=2)]


def append(L, c, **change):
    a = dict(type=L.F16, k=4096, kt=128, kh=64, v=4096, vt=128, vh=64, q=4096, qt=256, qh=64, hq=4, q_out=4096, table=64,
             seqs=4, wide=2, stride=2, seq=64, idx=64, pos=64, tokens=3, cos=64, sin=64, positions=9, rot=64, pairs=0)
    a.update(change)
    return L.lib().fvs_kv_append(None, c, *a.values())


def read(L, c, **change):
    a = dict(type=L.F16, k=4096, v=4096, table=64, seqs=4, wide=2, stride=2, seq=64, idx=64, tokens=3)
    a.update(change)
    return L.lib().fvs_kv_read(None, c, *a.values())


def attend(L, c, **change):
    a = dict(type=L.F16, q=4096, qs=256, qh=64, hq=4, table=64, seqs=4, wide=2, stride=2, lens=64, scale=0.1, out=4096,
             lse=64, work=64, arrived=64)
    a.update(change)
    return L.lib().fvs_kv_attend(None, c, *a.values())


@pytest.mark.parametrize("change", BAD_CACHES)
def test_bad_caches(L, change):
    for call in (append, read, attend):
        assert call(L, cache(L, **change)) == -1


def test_unsupported_head_dim(L):
    for call in (append, read, attend):
        assert call(L, cache(L, dim=80, slot_stride=80)) == -2


@pytest.mark.parametrize("change", [dict(type=2), dict(type=1), dict(tokens=-1), dict(hq=-1), dict(rot=24), dict(rot=128),
                                    dict(cos=None), dict(sin=68), dict(positions=0), dict(pairs=2), dict(k=4100),
                                    dict(kt=4), dict(vh=32), dict(q=None), dict(q_out=None), dict(q_out=4104),
                                    dict(table=None), dict(seqs=0), dict(wide=0), dict(idx=None),
                                    dict(seq=None, tokens=5)])
def test_append_refuses(L, change):
    assert append(L, cache(L), **change) == -1


@pytest.mark.parametrize("change", [dict(type=2), dict(tokens=-1), dict(k=None), dict(v=4100), dict(table=None),
                                    dict(idx=None), dict(seq=None, tokens=5), dict(wide=0)])
def test_read_refuses(L, change):
    assert read(L, cache(L), **change) == -1


@pytest.mark.parametrize("change", [dict(type=3), dict(type=1), dict(q=None), dict(q=4104), dict(qs=4), dict(qh=-8),
                                    dict(hq=0), dict(hq=5), dict(table=None), dict(seqs=-1), dict(wide=0), dict(lens=None),
                                    dict(out=None), dict(work=None), dict(work=8),
                                    dict(arrived=None), dict(arrived=68)])
def test_attend_refuses(L, change):
    assert attend(L, cache(L), **change) == -1


def test_empty_calls_do_nothing(L):
    assert append(L, cache(L), tokens=0) == 0
    assert read(L, cache(L), tokens=0) == 0
    assert attend(L, cache(L), seqs=0) == 0


def test_workspace_size(L):
    f = L.lib().fvs_kv_attend_work
    assert f(0) == -1 and f(512) == -2
    assert f(64) > 0 and f(64) % 16 == 0


def test_host_memory_is_refused():
    k = torch.zeros(2, 1, 4, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        pkg("kvcache").PagedKV(k, k.clone())


def test_passage_table():
    f = pkg("kvcache").passage_table
    pages_of = torch.tensor([[0, 1], [2, -1], [3, 4]], dtype=torch.int32)
    own = torch.tensor([[7], [8]], dtype=torch.int32)
    got = f(torch.tensor([[2, -1], [1, 0]]), pages_of, own)
    assert got.dtype == torch.int32
    assert got.tolist() == [[3, 4, -1, -1, 7], [2, -1, 0, 1, 8]]
    assert f(torch.tensor([[1]]), pages_of).tolist() == [[2, -1]]
    with pytest.raises(ValueError):
        f(torch.tensor([[1]]), pages_of.long())


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_passage_table_ids_without_a_row(dtype):
    """Ids outside pages_of are holes (nothing is indexed with them), whatever the batch or the number of passages."""
    f = pkg("kvcache").passage_table
    pages_of = torch.tensor([[0, 1], [2, -1]], dtype=torch.int32)
    own = torch.tensor([[7], [8]], dtype=torch.int32)
    ids = torch.tensor([[2, 1, -7], [0, 2 ** 31 - 1, -1]], dtype=dtype)
    assert f(ids, pages_of, own).tolist() == [[-1, -1, 2, -1, -1, -1, 7], [0, 1, -1, -1, -1, -1, 8]]
    for b, k, n, m, w in ((0, 3, 2, 2, 1), (2, 0, 2, 2, 1), (2, 3, 0, 2, 1), (2, 3, 2, 0, 1), (0, 0, 0, 0, 0)):
        got = f(torch.zeros(b, k, dtype=dtype), torch.zeros(n, m, dtype=torch.int32), torch.zeros(b, w, dtype=torch.int32))
        assert got.shape == (b, k * m + w) and got.dtype == torch.int32
        if n == 0:
            assert (got[:, :k * m] == -1).all()


def test_passage_table_refusals():
    f = pkg("kvcache").passage_table
    ids, pages_of, own = torch.zeros(2, 1, dtype=torch.int64), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32)
    for args in ((ids, pages_of, own.long()), (ids, pages_of, own[:1]), (ids, pages_of, own[0]), (ids.float(), pages_of),
                 (ids[0], pages_of), (ids, pages_of[0])):
        with pytest.raises(ValueError):
            f(*args)


def test_oracle_attention_against_torch():
    g = torch.Generator().manual_seed(0)
    q = torch.randn(2, 4, 64, generator=g, dtype=torch.float64)
    k, v = (torch.randn(6, 2, 8, 64, generator=g, dtype=torch.float64) for _ in range(2))
    table = np.array([[4, 1, -1, 0], [2, 5, 3, -1]], np.int32)
    lens, fill = np.array([32, 20], np.int32), np.array([8, 3, 8, 8, 0, 8], np.int32)
    out, lse, *_ = O.attend(q.numpy(), k.numpy(), v.numpy(), table, lens, 0.125, fill)
    for b in range(2):
        at = [(p, s) for i, p in enumerate(table[b]) for s in range(8)
              if p >= 0 and i * 8 + s < lens[b] and s < fill[p]]
        p, s = torch.tensor(at).T
        kk, vv = k[p, :, s].repeat_interleave(2, 1), v[p, :, s].repeat_interleave(2, 1)       # [t, 4, 64]
        score = torch.einsum("hd,thd->ht", q[b], kk) * 0.125
        np.testing.assert_allclose(lse[b], torch.logsumexp(score, 1).numpy(), rtol=1e-12)
        np.testing.assert_allclose(out[b], torch.einsum("ht,thd->hd", score.softmax(1), vv).numpy(), rtol=1e-10)


def test_oracle_rotation_against_complex_product():
    rng = np.random.default_rng(0)
    x, ang = rng.standard_normal((5, 2, 64)), rng.random((5, 16)) * 6
    for pairs in ("halves", "neighbours"):
        y, _ = O.rotate(x, np.cos(ang), np.sin(ang), 32, pairs)
        a, b = (x[..., :16], x[..., 16:32]) if pairs == "halves" else (x[..., 0:32:2], x[..., 1:32:2])
        z = (a + 1j * b) * np.exp(1j * ang)[:, None]
        c, d = (y[..., :16], y[..., 16:32]) if pairs == "halves" else (y[..., 0:32:2], y[..., 1:32:2])
        np.testing.assert_allclose(c, z.real, atol=1e-12)
        np.testing.assert_allclose(d, z.imag, atol=1e-12)
        np.testing.assert_array_equal(y[..., 32:], x[..., 32:])
