"""Drafted tokens on the host: the C entry points refuse wrong arguments before any device work, the Python layer refuses
host memory, and the 64-bit oracles agree with the definitions written another way."""
import ctypes as C

import numpy as np
import pytest
import torch

from conftest import pkg
from oracle import drafts_oracle as O
from test_kv_args import BAD_CACHES, cache


@pytest.fixture(scope="module")
def L():
    pkg("build").build()
    return pkg("_lib")


def append_norm(L, c, **change):
    a = dict(type=L.F16, k=4096, kt=128, kh=64, v=4096, vt=128, vh=64, q=4096, qt=256, qh=64, hq=4, q_out=4096, table=64,
             seqs=4, wide=2, stride=2, seq=64, idx=64, pos=64, tokens=3, cos=64, sin=64, positions=9, rot=64, pairs=0,
             q_weight=64, k_weight=64, weight_type=L.F16, eps=1e-6)
    a.update(change)
    return L.lib().fvs_kv_append_norm(None, c, *a.values())


def compact(L, c, **change):
    a = dict(table=64, seqs=4, wide=2, stride=2, lens=64, path=64, nodes=5)
    a.update(change)
    return L.lib().fvs_kv_compact(None, c, *a.values())


def attend_tree(L, c, **change):
    a = dict(type=L.F16, q=4096, qs=5 * 256, qn=256, qh=64, hq=4, table=64, seqs=4, wide=2, stride=2, lens=64, parents=64, ps=5,
             counts=None, nodes=5, scale=0.1, out=4096, lse=64, work=64)
    a.update(change)
    return L.lib().fvs_kv_attend_tree(None, c, *a.values())


def verify(L, **change):
    a = dict(type=L.F32T, target=64, ts=6 * 100, tr=100, draft=64, ds=6 * 100, dr=100, parents=64, ps=5, tokens=64,
             counts=None, u=64, seqs=2, nodes=5, vocab=100, path=64, kept=64, token=64)
    a.update(change)
    return L.lib().fvs_verify(None, *a.values())


@pytest.mark.parametrize("change", BAD_CACHES)
def test_bad_caches(L, change):
    for call in (append_norm, compact, attend_tree):
        assert call(L, cache(L, **change)) == -1


def test_unsupported_head_dim(L):
    for call in (append_norm, compact, attend_tree):
        assert call(L, cache(L, dim=80, slot_stride=80)) == -2


@pytest.mark.parametrize("change,rc", [(dict(type=3), -1), (dict(type=1), -1), (dict(q=None), -1), (dict(q=4104), -1), (dict(qs=4), -1),
                                       (dict(qn=-8), -1), (dict(qh=12), -1), (dict(hq=0), -1), (dict(hq=5), -1), (dict(table=None), -1),
                                       (dict(seqs=-1), -1), (dict(wide=0), -1), (dict(lens=None), -1), (dict(parents=None), -1),
                                       (dict(ps=-1), -1), (dict(nodes=-1), -1), (dict(out=None), -1), (dict(out=4104), -1),
                                       (dict(work=None), -1), (dict(work=8), -1), (dict(nodes=257), -2), (dict(wide=2 ** 27 + 1), -2)])
def test_attend_tree_refuses(L, change, rc):
    assert attend_tree(L, cache(L), **change) == rc


def test_attend_tree_spans(L):
    """What 32 bits of 16 bytes cannot address is refused before any launch."""
    far = dict(pages=2 ** 31 - 1, page_stride=2 * 16 * 64)
    assert attend_tree(L, cache(L, type=L.I8, k_scale=64, v_scale=64, scale_page_stride=32, scale_head_stride=16, scale_slot_stride=1, **far)) == -2
    assert attend_tree(L, cache(L, page=7, **far)) == -2
    assert attend_tree(L, cache(L), qs=2 ** 36) == -2


def test_tree_workspace_size(L):
    f = L.lib().fvs_kv_attend_tree_work
    assert f(0, 4) == -1 and f(64, -1) == -1 and f(512, 4) == -2
    assert f(64, 1) > 0 and f(64, 1) % 16 == 0 and f(64, 129) >= f(64, 1) and f(256, 4096) >= f(256, 1) > f(192, 1)


@pytest.mark.parametrize("change", [dict(q_weight=68), dict(k_weight=8), dict(weight_type=1), dict(weight_type=2),
                                    dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
                                    dict(type=2), dict(rot=24), dict(q=None), dict(k=None), dict(table=None)])
def test_append_norm_refuses(L, change):
    assert append_norm(L, cache(L), **change) == -1


@pytest.mark.parametrize("change", [dict(table=None), dict(seqs=-1), dict(wide=0), dict(lens=None), dict(path=None),
                                    dict(nodes=-1)])
def test_compact_refuses(L, change):
    assert compact(L, cache(L), **change) == -1


@pytest.mark.parametrize("change,rc", [(dict(type=2), -1), (dict(target=None), -1), (dict(target=66), -1), (dict(draft=65), -1),
                                       (dict(parents=None), -1), (dict(tokens=None), -1), (dict(u=None), -1),
                                       (dict(path=None), -1), (dict(kept=None), -1), (dict(token=None), -1),
                                       (dict(nodes=-1), -1), (dict(vocab=0), -1), (dict(seqs=-1), -1), (dict(ts=-1), -1),
                                       (dict(ps=-1), -1), (dict(nodes=257), -2)])
def test_verify_refuses(L, change, rc):
    assert verify(L, **change) == rc


def test_empty_calls_do_nothing(L):
    assert append_norm(L, cache(L), tokens=0) == 0
    assert compact(L, cache(L), seqs=0) == 0 and compact(L, cache(L), nodes=0) == 0
    assert verify(L, seqs=0) == 0
    assert attend_tree(L, cache(L), seqs=0) == 0 and attend_tree(L, cache(L), nodes=0) == 0


def test_host_memory_is_refused():
    z = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="GPU"):
        pkg("drafts").verify(torch.zeros(1, 3, 8), z(2), z(1, 2), torch.zeros(1, 3))


def test_oracle_norm_against_torch():
    x = torch.randn(5, 3, 64, generator=torch.Generator().manual_seed(0), dtype=torch.float64)
    w = torch.linspace(0.5, 2, 64, dtype=torch.float64)
    want = torch.nn.functional.rms_norm(x, (64,), w, 1e-5)
    np.testing.assert_allclose(O.norm(x.numpy(), w.numpy(), 1e-5), want.numpy(), rtol=1e-12)


def test_oracle_tree_attention_against_one_sequence_per_node():
    """Each node as the last token of a plain sequence of its own."""
    from oracle import kv_oracle as K
    rng = np.random.default_rng(1)
    parents = np.array([-1, 0, 0, -1, 2])
    chains = [[0], [0, 1], [0, 2], [3], [0, 2, 4]]
    assert [list(np.flatnonzero(r)) for r in O.sees(parents)] == chains
    q, k, v = rng.standard_normal((1, 5, 4, 8)), rng.standard_normal((12, 2, 1, 8)), rng.standard_normal((12, 2, 1, 8))
    table = np.array([[7, 3, -1, 9, 0, 1, 2, 4, 5]])        # lens 4, a hole at 2; the nodes lie in pages 0, 1, 2, 4, 5
    out, lse, *_ = O.attend_tree(q, k, v, table, [4], parents[None], None, 0.3)
    for i, chain in enumerate(chains):
        row = [[7, 3, -1, 9] + [int(table[0][4 + j]) for j in chain]]
        eo, el, *_ = K.attend(q[:, i], k, v, row, [len(row[0])], 0.3)
        np.testing.assert_allclose(out[:, i], eo, rtol=1e-12)
        np.testing.assert_allclose(lse[:, i], el, rtol=1e-12)


@pytest.mark.parametrize("with_draft", [True, False])
def test_oracle_verification_keeps_the_target_distribution(with_draft):
    """The first token of the answer is distributed as the target's row: by exact enumeration over the drafted tokens and a
    fine grid of the random numbers (midpoints: an error of at most the grid's step for each number)."""
    rng = np.random.default_rng(2)
    vocab, grid = 3, 24
    p = np.array([0.5, 0.3, 0.2])
    q = np.array([0.2, 0.2, 0.6])
    mid = (np.arange(grid) + 0.5) / grid
    got = np.zeros(vocab)
    drafts = [(x, y, q[x] * q[y]) for x in range(vocab) for y in range(vocab)] if with_draft else [(0, 2, 1.0)]
    u = np.stack(np.meshgrid(mid, mid, mid, indexing="ij"), -1).reshape(-1, 3)
    rows = rng.random((1, 3, vocab))
    rows[0, 0] = p
    n = len(u)
    for x, y, weight in drafts:
        path, kept, token = O.verify(np.repeat(rows, n, 0), np.tile([[-1, -1]], (n, 1)), np.tile([[x, y]], (n, 1)), u,
                                     np.tile(q, (n, 3, 1)) if with_draft else None)
        first = np.where(kept > 0, np.array([x, y])[np.maximum(path[:, 0], 0)], token)
        got += weight * np.bincount(first, minlength=vocab) / n
    np.testing.assert_allclose(got, p, atol=3 / grid)
