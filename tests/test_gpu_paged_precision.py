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


@pytest.mark.parametrize("dtype,kb,vb,dim,n,cuts", [(F16, 4, 4, 128, 131072, "even"), (F16, 3, 2, 128, 131072, "even"), (F16, 2, 3, 64, 131072, "even"),
                                                    (F16, 4, 2, 256, 65536, "even"), (F16, 4, 4, 128, 131072, "ragged")])
def test_sums_of_16_bit_calls_over_long_runs(gen, dtype, kb, vb, dim, n, cuts):
    """As above, by how far the output is off along its own direction, where errors of one sign show and the output's
    rounding (known from the definition) mostly cancels.  The tensor cores cut 2^-23 off a sum at every product and hand
    it over after 256 of them: 2^-15.  The codebook of 4 bits moves the row of values by 7.8e-5 of itself at random
    (3 sigma over its coordinates: 2.1e-5 at 128), the other two by less.  A shift of up to 5.2e-5 crosses a border of
    the output's rounding, 2^-11 of the value apart at least, for a share of 0.11 of the outputs at random: 3 sigma over
    them are 3 sqrt(0.11 / 128) 2^-11 = 4.3e-5 along it.  1e-4 in all."""
    seqs, page = 148 * 16, 256
    cache, signs = make_cache(gen, n // page, 1, dim, kb, vb, page)
    ref.random_pool(cache, gen)
    cache.v_pages[:] = cache.v_pages[0, 0, 0]
    cache.v_scales.fill_(1.375)
    table = torch.randperm(n // page, generator=gen, device="cuda").int()[None].expand(seqs, -1)
    if cuts == "even":
        lengths = torch.full((seqs,), n, dtype=torch.int32, device="cuda")
    else:   # empty and shorter sequences between the others
        lengths = torch.randint(0, n + 1, (seqs,), generator=gen, device="cuda", dtype=torch.int32)
        lengths[::7] = 0
        lengths[1::7] = n
    q = torch.randn(1, 1, dim, generator=gen, device="cuda").to(dtype)
    want = ref.attend(cache, signs, q, table[:1], ints(n))[0, 0]   # one row, whatever the weights and the length
    got = cache.attend(q.expand(seqs, -1, -1), table, lengths)[:, 0]
    cache.check()
    along = lambda y: (y.double() @ want) / (want @ want)  # noqa: E731
    off = (along(got) - along(want.to(dtype)))[lengths > 0].abs()
    assert float(off.max()) <= 1e-4 * max(1.0, math.sqrt(128 / dim)), float(off.max())
    assert not got[lengths == 0].any()
    # the reference of the exponentials moves while sums lie in the workspace: weights that grow along the sequence
    if cuts == "even":
        cache.v_scales.copy_(1.375 * torch.exp2(24.0 * (torch.arange(n, device="cuda") - n) / n)[torch.argsort(table[0])[:, None] * page + torch.arange(page, device="cuda")][:, None])
        want = ref.attend(cache, signs, q, table[:1], ints(n))[0, 0]
        got = cache.attend(q.expand(seqs, -1, -1), table, lengths)[:, 0]
        off = (along(got) - along(want.to(dtype))).abs()
        assert float(off.max()) <= 1e-4 * max(1.0, math.sqrt(128 / dim)), float(off.max())


def test_phases_are_exact_to_float32():
    """The phase is reduced to an eighth of a turn in integers before it is rounded to 24 bits, so cosine and sine are
    off by 2^-24 of themselves from that rounding and by 2^-23 (one step) each from the functions: below 2^-22 of the
    value wherever it is, next to a zero crossing as well."""
    from adaptq_b200 import Rotary
    r = Rotary(64, 10000.0)
    gen = torch.Generator().manual_seed(3)
    pos = torch.randint(0, 2 ** 40, (4000,), generator=gen)
    pos[0], pos[1] = 0, 1
    x = torch.zeros(4000, 1, 64, device="cuda")
    x[..., :32] = 1.0
    y = r(x, pos.cuda()).double().cpu()[:, 0]
    c = np.empty((4000, 32))
    s = np.empty((4000, 32))
    for j, w in enumerate(int(t) % 2 ** 64 for t in r._turns.cpu().tolist()):
        for i, p in enumerate(pos.tolist()):
            phase = (p * w) % 2 ** 64
            quarter = (phase + 2 ** 61) >> 62
            a = (phase - (quarter << 62)) / 2.0 ** 64 * 2 * math.pi
            c[i, j], s[i, j] = [(math.cos(a), math.sin(a)), (-math.sin(a), math.cos(a)), (-math.cos(a), -math.sin(a)), (math.sin(a), -math.cos(a))][quarter % 4]
    for got, want in ((y[:, :32], c), (y[:, 32:], s)):
        want = torch.from_numpy(want)
        assert float(want.abs().min()) < 1e-4   # zero crossings are among them
        err = ((got - want).abs() - 2.0 ** -22 * want.abs()).max()
        assert float(err) <= 1e-30, float(err)


@pytest.mark.parametrize("bits", [2, 3, 4])
def test_coordinates_at_a_threshold(gen, bits):
    """A code counts the thresholds at or below its coordinate: (a, b, 0, ...) has the coordinates (a +- b) / norm, and
    pairs are searched (float32, rounded operation by operation as the kernel does it) that give a threshold exactly."""
    from adaptq_b200 import PagedKVCache
    f = np.float32
    m = [f(v) for v in ref.MAGNITUDES[bits]]
    level = [-v for v in reversed(m)] + m
    thresholds = [(p + q) * f(0.5) for p, q in zip(level, level[1:])]
    rng = np.random.default_rng(bits)
    rows, want = [], []
    for t in thresholds:
        if abs(t) >= math.sqrt(2):
            continue
        size, sign = abs(t), f(-1 if t < 0 else 1)
        found = 0
        for a in rng.uniform(1, 2, 200).astype(f):
            b = f(a * math.tan(math.asin(float(size) / math.sqrt(2)) - math.pi / 4))
            bb = next((c for c in (f(b + f(k) * np.spacing(b)) for k in range(-3, 4))
                       if f(f(a + c) * (f(1) / np.sqrt(f(f(f(a * a) + f(c * c)) + f(1e-12))))) == size), None)
            if bb is not None and found < 4:
                other = sign * f(f(a - bb) * (f(1) / np.sqrt(f(f(f(a * a) + f(bb * bb)) + f(1e-12)))))
                rows.append((sign * a, sign * bb))
                want.append((sum(x <= t for x in thresholds), sum(x <= other for x in thresholds)))
                found += 1
        assert found == 4
    n = len(rows)
    x = torch.zeros(n, 1, 64)
    x[:, 0, :2] = torch.from_numpy(np.array(rows, np.float32))
    cache = PagedKVCache(1, 1, 64, bits, bits, 64, signs=torch.ones(1, 64))
    cache.append(x.cuda(), x.cuda(), ints(0).view(1, 1), ints(0), ints(0, n))
    for pages in (cache.k_pages, cache.v_pages):
        code = ref.unpack(pages[0, 0, :n], bits).cpu()
        expect = torch.tensor(want)
        assert torch.equal(code[:, ::2], expect[:, :1].expand(n, 32)) and torch.equal(code[:, 1::2], expect[:, 1:].expand(n, 32))


@pytest.mark.parametrize("dtype,power,tolerance", [(F32, 27, 2e-5), (F32, 30, 2e-5), (F16, 24, 3.8e-3), (BF16, 22, 1.06e-2)])
def test_many_tokens_far_below_one_in_a_warp(gen, dtype, power, tolerance):
    """One value 2^power times as long as 131071 others of its sequence under equal weights, thousands of whose units
    one warp holds together with it: without them the output would be off by 131071 / 2^power, which is above what is
    tolerated."""
    seqs, n, page = 148 * 16, 131072, 256
    assert (n - 1) * 2.0 ** -power > 2 * tolerance
    cache, signs = make_cache(gen, n // page, 1, 128, 4, 4, page)
    ref.random_pool(cache, gen)
    cache.k_scales.zero_()                                   # equal logits
    cache.v_pages[:] = cache.v_pages[0, 0, 0]                # one row for all but one
    cache.v_scales.fill_(1.375)
    order = torch.randperm(n // page, generator=gen, device="cuda").int()
    for unit in (0, 300, 511):
        cache.v_pages[:] = cache.v_pages[int(order[100]), 0, 0]
        cache.v_scales.fill_(1.375)
        page_of = int(order[unit])
        cache.v_scales[page_of, 0, 11] = 1.375 * 2.0 ** power
        cache.v_pages[page_of, 0, 11] = cache.v_pages[page_of, 0, 11].flip(0)   # another direction
        q = torch.randn(1, 1, 128, generator=gen, device="cuda").to(dtype)
        want = ref.attend(cache, signs, q, order[None], ints(n))
        got = cache.attend(q.expand(seqs, -1, -1), order[None].expand(seqs, -1), torch.full((seqs,), n, dtype=torch.int32, device="cuda"))
        attend_close(got, want.expand(seqs, -1, -1), dtype, f"page {unit}")


@pytest.mark.parametrize("where", [0, 300, 511])
def test_many_weights_far_below_one_in_a_warp(gen, where):
    """As above in float32 with one weight of 2^27 among equal ones, so that the sum of weights is what would lose
    them.  Their share is 131071 / 2^27 = 9.8e-4.  Logits reach 40 and are off by 2^-20 of one (10 roundings of 2^-23
    each), weights as much of themselves."""
    seqs, n, page, power, dim = 148 * 16, 131072, 256, 27, 128
    cache, signs = make_cache(gen, n // page, 1, dim, 4, 4, page)
    ref.random_pool(cache, gen)
    for t in (cache.k_pages, cache.v_pages):
        t[:] = t[0, 0, 0].clone()
    cache.k_scales.fill_(1.0)
    cache.v_scales.fill_(1.375)
    order = torch.randperm(n // page, generator=gen, device="cuda").int()
    q = torch.randn(1, 1, dim, generator=gen, device="cuda")
    _, level, _ = ref.rows(cache, "k", order[:1].long(), torch.zeros(1, dtype=torch.long, device="cuda"), signs)
    z = (q.double() * signs) @ ref.hadamard(dim).cuda()
    q *= float(10.0 / ((z * level).sum() * dim ** -0.5 / dim))   # a logit of 10 where the norm is one
    cache.k_scales[int(order[where]), 0, 11] = 1.0 + power * math.log(2.0) / 10.0
    cache.v_pages[int(order[where]), 0, 11] = cache.v_pages[int(order[where]), 0, 11].flip(0)   # another direction
    want = ref.attend(cache, signs, q, order[None], ints(n))
    got = cache.attend(q.expand(seqs, -1, -1), order[None].expand(seqs, -1), torch.full((seqs,), n, dtype=torch.int32, device="cuda"))
    share = 131071 / (131071 + 2.0 ** power)
    alone = ref.attend(cache, signs, q, order[None, where: where + 1], ints(12))   # the one and eleven others: without the rest
    assert float((alone - want).norm() / want.norm()) > 20 * 2e-5 and share > 20 * 2e-5
    attend_close(got, want.expand(seqs, -1, -1), F32)


def evaluate(cache, signs, q, table, lengths, queries=lambda z: z, weights=lambda w: w, level=lambda c: c):
    """The attention in 64 bits with roundings planted: of the transformed queries, of weights times norms (relative to the
    largest), of the codebook."""
    p, dim, heads = signs.shape[1], cache.dim, cache.n_kv_heads
    out, group, h = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), q.shape[1] // heads, ref.hadamard(p).cuda()
    for b, n in enumerate(lengths):
        at, off = ref.place(cache, table[b], n)
        _, kl, kn = ref.rows(cache, "k", at, off, signs)
        _, vl, vn = ref.rows(cache, "v", at, off, signs)
        full = torch.zeros(heads, group, p, dtype=torch.float64, device="cuda")
        full[..., :dim] = q[b].double().view(heads, group, dim)
        z = queries((full * signs[:, None]) @ h)
        logit = torch.einsum("hgp,thp->hgt", z, level(kl)) * kn.T[:, None] * dim ** -0.5 / p
        w = torch.softmax(logit, -1)
        out[b] = (torch.einsum("hgt,thp->hgp", weights(w * vn.T[:, None]), level(vl)) @ h * signs[:, None] / p)[..., :dim].reshape(-1, dim)
    return out


LONG, SHORT = [600, 64, 1000, 333, 777, 150], [2 + b % 7 for b in range(24)]


@pytest.mark.parametrize("dtype,kb,vb,lengths", [(F16, 4, 4, LONG), (F16, 3, 2, LONG), (F16, 2, 3, LONG), (F16, 3, 2, SHORT), (F16, 2, 3, SHORT),
                                                 (BF16, 4, 4, LONG), (BF16, 3, 2, LONG)])
def test_precision_of_16_bit_calls(gen, dtype, kb, vb, lengths):
    """Error of float16 and bfloat16 calls against what their arithmetic is said to leave.

    float16: queries and weights have 22 bits; the codebook is off by c = 7.8e-5 (4 bits), 2.7e-6 (3) or 1.7e-8 (2) of a value,
    rms over its use.  Terms add up at random, so logits of spread s move weights by c_k s and values move by c_v, and
    the sums in float32 add 2e-6: eta = sqrt((c_k s)^2 + c_v^2) + 2e-6 of the output.  bfloat16: queries, weights and values
    have 11 bits, 2^-12 rms at most: eta = sqrt(2) 2^-12 sqrt(s^2 + 1).
    Independent of that is rho, the output's own rounding, which the definition tells.  So the norm of the error over all
    outputs is at most sqrt(rho^2 + eta^2), and 5 % for the sample.  A float16 output differs from the rounded definition
    where a border between two roundings, at least 2^-11 |y| apart, lies within the error: a share of at most
    min(1, 2^11 eta Y / |y|), where Y is the rms of its head's outputs.
    The same evaluation with one rounding more, planted in the definition, lies above that."""
    seqs, heads, group, dim = len(lengths), 4, 4, 128
    cache, signs = make_cache(gen, 120, heads, dim, kb, vb, 64)
    ref.random_pool(cache, gen)
    table = ref.random_table(cache, lengths, gen)
    q = (1.5 * torch.randn(seqs, heads * group, dim, generator=gen, device="cuda")).to(dtype)
    want = evaluate(cache, signs, q, table, lengths)
    attend_close(want, ref.attend(cache, signs, q, table, ints(*lengths)), F32)
    error = lambda y: float((y.double() - want).norm() / want.norm())  # noqa: E731
    other = lambda y: float((y != want.to(dtype)).double().mean())  # noqa: E731
    rho, spread = error(want.to(dtype)), 1.5 * 1.1   # norms vary by a third around sqrt(dim), which adds a tenth
    if dtype == F16:
        c = {4: 7.8e-5, 3: 2.7e-6, 2: 1.7e-8}
        eta = math.hypot(c[kb] * spread, c[vb]) + 2e-6
    else:
        eta = math.sqrt(2) * 2.0 ** -12 * math.hypot(spread, 1.0)
    bound = 1.05 * math.hypot(rho, eta)
    share = float((2.0 ** 11 * eta * want.pow(2).mean(-1, keepdim=True).sqrt() / want.abs()).clamp(max=1).mean())
    got = cache.attend(q, table, ints(*lengths))
    assert error(got) <= bound, f"{error(got):.3e} > {bound:.3e} (rounding alone {rho:.3e})"
    if dtype != F16:
        return
    assert other(got) <= share, f"{other(got):.4f} of the outputs are rounded otherwise, {share:.4f} may be"
    # one part of float16 for queries or weights (the largest of them 400, some number that is not a power of two), or the
    # codebook as float16 holds it
    half = lambda x: (x * (400 / x.abs().amax(-1, keepdim=True))).half().double() * (x.abs().amax(-1, keepdim=True) / 400)  # noqa: E731
    planted = evaluate(cache, signs, q, table, lengths, weights=half).to(dtype)
    assert error(planted) > bound or other(planted) > share or kb == vb == 4
    planted = evaluate(cache, signs, q, table, lengths, queries=half).to(dtype)
    assert error(planted) > bound
    planted = evaluate(cache, signs, q, table, lengths, level=lambda x: x.half().double()).to(dtype)
    assert error(planted) > bound
