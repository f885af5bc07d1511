"""Calls of the paged cache and of Rotary next to other streams and to automatic differentiation."""
import pytest
import torch

from test_gpu_paged import ints, make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture()
def gen(gpu_lib):
    return torch.Generator(device="cuda").manual_seed(47)


def test_check_waits_for_every_stream(gen):
    """A report of a call that another stream has not reached yet."""
    cache, _ = make_cache(gen, 4, 2, 64, 4, 4, 16)
    k = torch.zeros(1, 2, 64, device="cuda")
    bad, start, good = ints(9).view(1, 1), ints(0), ints(1).view(1, 1)
    cache.append(k, k, bad, start)
    with pytest.raises(RuntimeError, match="outside the pool"):
        cache.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)   # a tenth of a second
        cache.append(k, k, bad, start)
    with pytest.raises(RuntimeError, match="outside the pool"):
        cache.check()
    cache.append(k, k, good, start)
    cache.check()


def test_status_is_taken_in_one_step(gen, gpu_lib):
    """adaptq_paged_take_status: the word as it was, and zero in its place."""
    cache, _ = make_cache(gen, 4, 2, 64, 4, 4, 16)
    taken = ints(77)
    for word in (0, 1, 2, 3):
        cache._status.fill_(word)
        assert gpu_lib.adaptq_paged_take_status(cache._ref, taken.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        assert int(taken) == word and int(cache._status) == 0
    assert gpu_lib.adaptq_paged_take_status(cache._ref, None, None) == -1 and b"null" in gpu_lib.adaptq_last_error()
    assert gpu_lib.adaptq_paged_take_status(None, taken.data_ptr(), None) == -1 and b"null" in gpu_lib.adaptq_last_error()
