"""What the paged cache and the rotation keep of their inputs' precision: sums over long runs, tokens far below one,
parts of 16-bit operands, phases, ties."""
import math

import numpy as np
import pytest
import torch

import paged_reference as ref
from test_gpu_paged import BF16, F16, F32, attend_close, ints, make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture()
def gen(gpu_lib):
    return torch.Generator(device="cuda").manual_seed(31)


@pytest.mark.parametrize("dtype,kb,vb,dim", [(F32, 4, 4, 128), (F32, 4, 2, 64), (F32, 3, 3, 256), (F16, 4, 4, 128), (BF16, 4, 2, 128)])
def test_sums_over_long_runs(gen, dtype, kb, vb, dim):
    """As many sequences as there are warps, each of 32768 tokens whose values point the same way, so that every warp
    sums hundreds of units into one item and errors of one sign would add up.  All sequences read the same pages."""
    seqs, n, page = 148 * 16, 32768, 256
    cache, signs = make_cache(gen, n // page, 1, dim, kb, vb, page)
    ref.random_pool(cache, gen)
    cache.v_pages[:] = cache.v_pages[0, 0, 0]
    cache.v_scales.fill_(1.375)
    table = torch.randperm(n // page, generator=gen, device="cuda").int()[None].expand(seqs, -1)
    q = torch.randn(1, 1, dim, generator=gen, device="cuda").to(dtype)
    want = ref.attend(cache, signs, q, table[:1], ints(n))
    got = cache.attend(q.expand(seqs, -1, -1), table, torch.full((seqs,), n, dtype=torch.int32, device="cuda"))
    cache.check()
    attend_close(got, want.expand(seqs, -1, -1), dtype)
