"""pytest plugin (-p paged_checked_plugin): after every test, no index check of the checked build may have failed in a
PagedKVCache of that test, or in a rotation."""
import ctypes as C

import pytest

FAILED = 256
made = []   # of the running test: (descriptor, status word) of its caches, whose pools may be gone by its end


def pytest_configure(config):
    from adaptq_b200.paged import PagedKVCache
    plain = PagedKVCache._set

    def remember(self, *args):
        plain(self, *args)
        made.append((self._desc, self._status))

    PagedKVCache._set = remember


@pytest.hookimpl(hookwrapper=True)
def pytest_runtest_call(item):
    made.clear()
    outcome = yield
    if outcome.excinfo is None:
        import torch
        from adaptq_b200 import PagedKVCache
        own = PagedKVCache(1, 1, 64, page_size=16)   # takes what rotations report
        torch.cuda.synchronize()
        taken = torch.empty(1, dtype=torch.int32, device="cuda")
        for desc, _ in made:
            if own._L.adaptq_paged_take_status(C.addressof(desc), taken.data_ptr(), torch.cuda.current_stream().cuda_stream):
                outcome.force_exception(AssertionError("adaptq_paged_take_status failed"))
            elif int(taken) & FAILED:
                outcome.force_exception(AssertionError("a device-side index check failed"))
    made.clear()
