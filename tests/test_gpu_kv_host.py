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
