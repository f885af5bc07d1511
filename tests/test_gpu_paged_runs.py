"""The paged cache and rotary positions at sizes where the kernels take several steps.  The smaller cases of
test_gpu_paged.py give every warp one.  Tolerances are those derived there."""
import pytest
import torch

import paged_reference as ref
from test_gpu_paged import BF16, E, F16, close, rotary_bound

pytestmark = pytest.mark.gpu


@pytest.fixture()
def gen(gpu_lib):
    return torch.Generator(device="cuda").manual_seed(23)


# ---------------------------------------------------------------------------
# rotary
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("heads,dim,part,interleaved,dtype", [(65535, 65536, 2, False, BF16), (40000, 65535, 64, True, F16), (65535, 40000, 8192, True, BF16)])
def test_rotary_of_more_coordinates_than_32_bits_count(gen, heads, dim, part, interleaved, dtype):
    """One token of more than 2^31 coordinates: every head is rotated and copied."""
    from adaptq_b200 import Rotary
    r = Rotary(part, interleaved=interleaved)
    x = torch.empty(1, heads, dim, dtype=dtype, device="cuda")
    x.view(-1).view(torch.int16).random_(12288, 16384, generator=gen)   # bit patterns of numbers below two
    pos = torch.tensor([12345], device="cuda")
    y = torch.full_like(x, 77.0)
    r(x, pos, out=y)
    for h in range(0, heads, 4096):
        assert torch.equal(y[:, h: h + 4096, part:], x[:, h: h + 4096, part:]), h
    a = x[..., :part].double()
    want = ref.rotate(a, pos, r)
    b, tiny = rotary_bound(a, pos, r, dtype)
    close(y[..., :part], want, b + E[dtype] * want.abs() + tiny)
