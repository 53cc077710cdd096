"""The paged cache's Python layer on the GPU: streams, refusals and memory."""
import pytest
import torch

from conftest import pkg
from test_gpu_kv import BF16, DEV, F16, full_table, make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    pkg("build").build()
    return pkg("kvcache")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_check_status_sees_calls_of_other_streams(kv):
    """A bad index that another stream's call meets while the check is made is reported once."""
    cache = kv.PagedKV.empty(2, 1, 16, 64, dtype=F16)
    table, idx = ints([[0]]), ints([2])
    bad = ints([[9]])
    cache.read(table, idx)                                  # the kernel is loaded by its first call, which waits
    torch.cuda._sleep(1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(50_000_000)                       # some 30 ms
        cache.read(bad, idx)
    with pytest.raises(pkg("_lib").FvsError):
        cache.check_status()
    cache.read(table, idx)
    cache.check_status()


def test_inputs_that_require_gradients_are_refused(kv):
    """Where gradients are recorded; under no_grad the same calls run."""
    g = torch.Generator().manual_seed(1)
    table, pages = full_table([20, 30], 16, g)
    cache = make_cache(kv, pages, 1, 16, 64, F16, g)
    table, n = table.to(DEV), ints([20, 30])
    plain = torch.randn(2, 1, 64, generator=g).to(DEV, F16)
    x = plain.clone().requires_grad_()
    cs = torch.ones(40, 32, device=DEV), torch.zeros(40, 32, device=DEV)
    learnt = cs[0].clone().requires_grad_()
    calls = [lambda: cache.attend(x, table, n), lambda: cache.append(x, plain, table, n - 1),
             lambda: cache.append(plain, x * 2, table, n - 1), lambda: cache.append(plain, plain, table, n - 1, q=x),
             lambda: cache.append(plain, plain, table, n - 1, rope=(learnt, cs[1])),
             lambda: kv.PagedKV(cache.k.clone().requires_grad_(), cache.v)]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
    with torch.no_grad():
        for call in calls:
            call()
        out, _ = cache.attend(x, table, n)
    assert torch.equal(out, cache.attend(plain, table, n)[0]) and not out.requires_grad


def test_release_workspaces(kv):
    """Memory held for streams comes back, calls in flight finish, and the next call works as before."""
    g = torch.Generator().manual_seed(2)
    table, pages = full_table([9000, 7000], 64, g)
    cache = make_cache(kv, pages, 2, 64, 128, BF16, g)
    table, n = table.to(DEV), ints([9000, 7000])
    q = torch.randn(2, 8, 128, generator=g).to(DEV, BF16)
    want = cache.attend(q, table, n)
    kv.release_workspaces()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out, lse = torch.empty_like(want[0]), torch.empty_like(want[1])
    for stream in (torch.cuda.current_stream(), s):
        with torch.cuda.stream(stream):
            for _ in range(20):
                cache.attend(q, table, n, out=out, lse=lse)
        held = torch.cuda.memory_allocated()
        assert held > before + 2 ** 23
        kv.release_workspaces()
        assert torch.cuda.memory_allocated() <= held - 2 ** 23
        with torch.cuda.stream(stream):
            torch.full((2 ** 23,), 255, dtype=torch.uint8, device=DEV)          # in the memory that was given back
            got = cache.attend(q, table, n)
        stream.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        kv.release_workspaces()
