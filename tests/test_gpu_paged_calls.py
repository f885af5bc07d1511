"""Calls of the paged cache and of Rotary next to other streams and to automatic differentiation."""
import pytest
import torch

import paged_reference as ref
from test_gpu_paged import BF16, F32, SCALINGS, ints, make_cache

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


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_forward_mode_derivative(gen, dtype):
    """The tangent of a rotation is the rotated tangent."""
    from torch.autograd import forward_ad
    from adaptq_b200 import Rotary
    r = Rotary(24, scaling=SCALINGS[3])
    x, dx = (torch.randn(5, 2, 40, generator=gen, device="cuda").to(dtype) for _ in range(2))
    pos = torch.arange(3, 8, device="cuda")
    with forward_ad.dual_level():
        y = r(forward_ad.make_dual(x, dx), pos)
        primal, tangent = forward_ad.unpack_dual(y)
        assert tangent is not None and torch.equal(tangent, r(dx, pos)) and torch.equal(primal, r(x, pos))
        leaf = x.clone().requires_grad_()   # both directions at once
        y = r(forward_ad.make_dual(leaf, dx), pos)
        assert torch.equal(forward_ad.unpack_dual(y).tangent, r(dx, pos))
        (g,) = torch.autograd.grad(forward_ad.unpack_dual(y).primal.float().sum(), leaf)
        slope = dx.clone().requires_grad_()  # the tangent has a gradient of its own
        y = r(forward_ad.make_dual(x, slope), pos)
        (h,) = torch.autograd.grad(forward_ad.unpack_dual(y).tangent.float().sum(), slope)
        assert torch.equal(g, h)
        with pytest.raises(ValueError):
            r(forward_ad.make_dual(x, dx), pos, out=torch.empty_like(x))
        assert forward_ad.unpack_dual(r(x, pos)).tangent is None


def test_forward_over_reverse(gen):
    """The tangent of a gradient: of (c / 2) (R x)^2 it is R^T (c R dx)."""
    from torch.autograd import forward_ad
    from adaptq_b200 import Rotary
    r, pos = Rotary(24, scaling=SCALINGS[3]), torch.arange(3, 8, device="cuda")
    x, dx, c = (torch.randn(5, 2, 40, generator=gen, device="cuda") for _ in range(3))
    x.requires_grad_()
    with forward_ad.dual_level():
        y = r(forward_ad.make_dual(x, dx), pos)
        (g,) = torch.autograd.grad((y * y * c).sum() / 2, x, create_graph=True)
        tangent = forward_ad.unpack_dual(g).tangent
    want = ref.rotate(c.double() * ref.rotate(dx.double(), pos, r), pos, r, inverse=True)
    assert tangent is not None and float((tangent.detach().double() - want.detach()).abs().max()) <= 1e-5 * float(want.detach().abs().max())


def test_tensors_written_in_place_are_marked(gen):
    """A tensor that a backward pass still needs cannot be overwritten unnoticed."""
    from adaptq_b200 import Rotary
    r, pos = Rotary(64), torch.arange(3, device="cuda")
    cache, _ = make_cache(gen, 4, 2, 64, 4, 4, 16)
    ref.random_pool(cache, gen)
    table, n = ints(0, 1, 2).view(3, 1), ints(5, 6, 7)
    q = torch.randn(3, 2, 64, generator=gen, device="cuda")
    calls = [lambda o: r(q, pos, out=o), lambda o: r(o, pos, out=o), lambda o: cache.attend(q, table, n, out=o),
             lambda o: cache.read(table, ints(0, 0, 0), ints(0, 1, 2, 3), 3, out=(o, torch.empty_like(o))),
             lambda o: cache.read(table, ints(0, 0, 0), ints(0, 1, 2, 3), 3, out=(torch.empty_like(o), o)),
             lambda o: cache.step(q, q, q, table, n, out=o)]
    for call in calls:
        w = torch.ones(3, 2, 64, device="cuda", requires_grad=True)
        saved = torch.randn(3, 2, 64, generator=gen, device="cuda")
        y = (w * saved).sum()
        call(saved)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        with pytest.raises(ValueError, match="gradient"):
            call(torch.zeros(3, 2, 64, device="cuda", requires_grad=True))
        with torch.no_grad():
            call(torch.zeros(3, 2, 64, device="cuda", requires_grad=True))
        with torch.inference_mode():
            call(torch.zeros(3, 2, 64, device="cuda"))


def test_outputs_whose_rows_overlap_are_refused(gen):
    from adaptq_b200 import Rotary
    r, pos = Rotary(64), torch.arange(3, device="cuda")
    cache, _ = make_cache(gen, 4, 2, 64, 4, 4, 16)
    ref.random_pool(cache, gen)
    table, n = ints(0, 1, 2).view(3, 1), ints(5, 6, 7)
    x = torch.randn(3, 2, 64, generator=gen, device="cuda")
    flat = torch.zeros(4096, device="cuda")
    for bad in (flat[:64].expand(3, 2, 64), flat[:128].view(1, 2, 64).expand(3, 2, 64), flat[:192].view(3, 1, 64).expand(3, 2, 64),
                flat.as_strided((3, 2, 64), (128, 63, 1)), flat.as_strided((3, 2, 64), (32, 512, 1))):
        for call in (lambda: r(x, pos, out=bad), lambda: cache.attend(x, table, n, out=bad),
                     lambda: cache.read(table, ints(0, 0, 0), ints(0, 1, 2, 3), 3, out=(bad, x.clone())),
                     lambda: cache.read(table, ints(0, 0, 0), ints(0, 1, 2, 3), 3, out=(x.clone(), bad))):
            with pytest.raises(ValueError, match="overlap"):
                call()
    with pytest.raises(ValueError, match="one twice"):
        cache.read(table, ints(0, 0, 0), ints(0, 1, 2, 3), 3, out=(x, x))
    assert not flat.any()
    want, one = r(x, pos), r(x[:1], pos[:1])
    for good in (flat[:384].view(2, 3, 64).transpose(0, 1), flat.as_strided((3, 2, 64), (200, 1000, 1))):
        assert torch.equal(r(x, pos, out=good), want)
    assert torch.equal(r(x[:1], pos[:1], out=flat.as_strided((1, 2, 64), (0, 64, 1))), one)


def test_refused_steps_store_nothing(gen):
    cache, _ = make_cache(gen, 4, 2, 64, 4, 4, 16)
    ref.random_pool(cache, gen)
    before = [t.clone() for t in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)]
    table, n = ints(0, 1, 2).view(3, 1), ints(5, 6, 7)
    k, q = torch.randn(3, 2, 64, generator=gen, device="cuda"), torch.randn(3, 4, 64, generator=gen, device="cuda")
    for bad in (lambda: cache.step(k, k, q[:, :3], table, n), lambda: cache.step(k, k, q[:2], table, n), lambda: cache.step(k, k, q.double(), table, n),
                lambda: cache.step(k, k, q, table, n, out=q[:, :2]), lambda: cache.step(k, k, q, table, n, scale=0.0),
                lambda: cache.step(k, k, q, table, n, scale=1e60), lambda: cache.step(k, k[:2], q, table, n), lambda: cache.step(k, k, q, table, n, rotary=1)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
        assert all(torch.equal(a, b) for a, b in zip(before, (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)))
    cache.step(k, k, q, table, n)
    assert not torch.equal(before[0], cache.k_pages)
