"""Calls of the paged cache and of Rotary next to other streams, to automatic differentiation and to missing pages."""
import pytest
import torch

import paged_reference as ref
from test_gpu_paged import BF16, E, F16, F32, SCALINGS, attend_close, close, ints, make_cache, rotary_bound

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


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("interleaved,dim,part", [(False, 128, 128), (True, 80, 40), (False, 67, 30)])
def test_rotary_gradient_in_16_bits(gen, dtype, interleaved, dim, part):
    from adaptq_b200 import Rotary
    r = Rotary(part, interleaved=interleaved, scaling=SCALINGS[3])
    x = torch.randn(40, 3, dim, generator=gen, device="cuda").to(dtype).requires_grad_()
    g = torch.randn(40, 3, dim, generator=gen, device="cuda").to(dtype)
    pos = torch.randint(0, 2 ** 20, (40,), generator=gen, device="cuda")
    (dx,) = torch.autograd.grad(r(x, pos), x, g)
    want = ref.rotate(g.double(), pos, r, inverse=True)
    b, tiny = rotary_bound(g.double(), pos, r, dtype)
    assert dx.dtype == dtype
    close(dx, want, b + E[dtype] * want.abs() + tiny)
    # differences of a linear map are its values: <R s, g> = <s, R^T g>, up to the roundings of both to 16 bits
    s = torch.randn(40, 3, dim, generator=gen, device="cuda").to(dtype)
    left, right = (r(s, pos).double() * g.double()), (s.double() * dx.double())
    room = E[dtype] * float(left.abs().sum() + right.abs().sum()) + 2 * 7e-7 * r.factor * 2 * float((s.double().abs() * g.double().abs().amax()).sum())
    assert abs(float(left.sum() - right.sum())) <= room


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (256, 16), (128, 64), (64, 128)])
def test_units_with_missing_pages_are_left_out(gen, dtype, dim, page):
    """A page that does not exist takes the tokens of its unit along (64 of them, 32 above 128 coordinates; at pages
    larger than that its own); what is left attends as if those tokens had not been there."""
    unit = 32 if dim > 128 else 64
    span = max(unit, page)
    cache, signs = make_cache(gen, 5 * span // page + 2, 2, dim, 4, 3, page)
    ref.random_pool(cache, gen)
    n, per = 4 * span + 5, span // page
    table = ref.random_table(cache, [n, 0], gen)
    table[1] = table[0]
    q = torch.randn(2, 6, dim, generator=gen, device="cuda").to(dtype)
    whole = ref.attend(cache, signs, q, table, ints(n, n))
    got = cache.attend(q, table, ints(n, n))
    attend_close(got, whole, dtype)
    cache.check()
    for missing, value in ((1 * per, -1), (2 * per + per - 1, cache.n_pages), (0, 2 ** 31 - 1), (4 * per, -2 ** 31)):
        broken = table.clone()
        broken[0, missing] = value
        got = cache.attend(q, broken, ints(n, n))
        with pytest.raises(RuntimeError, match="outside the pool"):
            cache.check()
        u = missing // per                       # the span that is gone, the last one has five tokens
        left = torch.cat([table[0, : u * per], table[0, (u + 1) * per:]])
        m = n - (span if u < 4 else 5)
        want = torch.cat([ref.attend(cache, signs, q[:1], left[None], ints(m)), whole[1:]])
        attend_close(got, want, dtype, f"page {missing}")
    got = cache.attend(q, torch.full_like(table, -1), ints(n, 0))
    assert not bool(got.any())
    with pytest.raises(RuntimeError, match="outside the pool"):
        cache.check()


def test_lengths_that_change_during_a_call(gen):
    """A caller's mistake, whose outputs nobody can tell, but which must not lead a kernel out of its tensors."""
    cache, signs = make_cache(gen, 400, 8, 128, 4, 2, 16)
    ref.random_pool(cache, gen)
    table = torch.randint(0, 400, (64, 100), generator=gen, device="cuda", dtype=torch.int32)
    n, other = (torch.randint(0, 1601, (64,), generator=gen, device="cuda", dtype=torch.int32) for _ in range(2))
    other[torch.rand(64, generator=gen, device="cuda") < 0.5] = 0
    q = torch.randn(64, 16, 128, generator=gen, device="cuda").to(BF16)
    lengths, side = n.clone(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(100):
        with torch.cuda.stream(side):
            for new in (other, torch.zeros_like(n), n, other.flip(0)):
                lengths.copy_(new)
        for _ in range(4):
            cache.attend(q, table, lengths)
    torch.cuda.synchronize()
    cache.check()
    attend_close(cache.attend(q, table, n), ref.attend(cache, signs, q, table, n), BF16)
