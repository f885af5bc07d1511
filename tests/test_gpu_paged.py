"""The paged cache and rotary positions on the GPU against their definitions in 64 bits.

Tolerances, with u = 2^-24 (half a step of float32) and e = half a step of the output type:

* rotary: a turn's angle is off by pi * 2^-25 (its rounding to 24 bits of half a turn) and its
  sine and cosine by 2 ulp (2^-23) and the factor's rounding u, 5e-7 together; two products and a
  sum add 2u each -> (|x1| + |x2|) * factor * 7e-7, and e |y|.
* a row read back: log2(P) + 2 roundings on sums of at most P levels -> (log2 P + 2) u sum|c| norm / P, and e |y|.
* a norm: P/32 + 8 roundings on the way of every term -> 20 u, and those of a rotation, 2 * 7e-7.
* a code: the coordinate H(s x) / norm is off by at most (log2 P + 2) u sum|x| / norm <= 10 u sqrt(P), by the
  norm's error 20 u + 1.4e-6 times at most 3 where thresholds are, and by the rotation's 7e-7 * 2 * sqrt(P):
  below 4e-5 for P = 256, so codes may differ where the 64-bit coordinate is that close to a threshold.
* attention in 16 bits: queries, codebook and weights are rounded to float16 once each, 2^-12 rms of a value; a
  logit of P independent terms is then off by sqrt(2) 2^-12 ||z c|| scale norm / P, about 5e-4 for logits of
  spread 1.5, and weights and values add 2^-12 each: 7e-4 of the output's norm, and the output's own rounding
  (bf16 2^-9 rms of the largest step, fp16 2^-12).  Tolerated: 4 x 7e-4 + 2 e of the norm of a head's output.
* attention in float32: the same with u for 2^-12, log2(P) + 8 roundings a logit: 2e-5 of the norm.
"""
import ctypes as C

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

E = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
CODE_SLACK = 4e-5


@pytest.fixture()
def gen(gpu_lib):
    return torch.Generator(device="cuda").manual_seed(11)


def make_cache(gen, n_pages, heads, dim, kb, vb, page):
    from adaptq_b200 import PagedKVCache
    signs = ref.random_signs(heads, ref.padded(dim), gen)
    return PagedKVCache(n_pages, heads, dim, kb, vb, page, signs=signs), signs.double()


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def close(got, want, bound, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst {float((err - bound).max()):.3e} over, err {float(err.max()):.3e}"


def attend_close(got, want, dtype, what=""):
    """Norm of the error over the norm of the output, per head; see the module's text."""
    tol = 2e-5 if dtype == F32 else 4 * 7e-4 + 2 * E[dtype]
    err, size = (got.double() - want).norm(dim=-1), want.norm(dim=-1)
    assert bool((err <= tol * size).all()), f"{what}: {float((err / size.clamp(min=1e-300)).max()):.3e} > {tol:.1e}"


# ---------------------------------------------------------------------------
# rotary
# ---------------------------------------------------------------------------
SCALINGS = [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 2.0},
            {"type": "yarn", "factor": 8.0, "original_max_position": 4096},
            {"type": "llama3", "factor": 8.0, "original_max_position": 8192}]


def rotary_bound(x, positions, rotary, dtype):
    d = rotary.dim
    size = torch.zeros_like(x)
    i = torch.arange(0, d, 2) if rotary.interleaved else torch.arange(d // 2)
    j = i + 1 if rotary.interleaved else i + d // 2
    both = (x[..., i].abs() + x[..., j].abs()) * rotary.factor
    size[..., i], size[..., j] = both, both
    tiny = 2.0 ** -25 if dtype == F16 else 0.0  # half a step of float16's subnormals
    return size * 7e-7, tiny


@pytest.mark.parametrize("tokens,heads,dim,part,interleaved,dtype,scaling", [
    (1, 1, 64, 64, False, BF16, 0), (5, 3, 128, 128, False, F32, 4), (17, 8, 128, 128, True, F16, 3), (33, 2, 80, 40, True, F32, 3),
    (9, 4, 96, 96, False, BF16, 1), (7, 5, 67, 30, False, BF16, 2), (4, 3, 33, 32, True, F16, 0), (3, 1, 256, 2, False, F32, 0),
    (130, 14, 64, 48, False, F16, 4), (2, 40, 128, 64, False, F32, 0), (700, 1, 128, 16, False, BF16, 0)])
def test_rotary_against_64_bits(gen, tokens, heads, dim, part, interleaved, dtype, scaling):
    from adaptq_b200 import Rotary
    r = Rotary(part, 10000.0, interleaved=interleaved, scaling=SCALINGS[scaling])
    x = torch.randn(tokens, heads, dim, generator=gen, device="cuda").to(dtype)
    pos = torch.randint(0, 2 ** 20, (tokens,), generator=gen, device="cuda", dtype=torch.int64)
    pos[0] = 0
    y = r(x, pos)
    assert y.dtype == dtype and y.shape == x.shape
    want = ref.rotate(x.double(), pos, r)
    b, tiny = rotary_bound(x.double(), pos, r, dtype)
    close(y, want, b + E[dtype] * want.abs() + tiny)
    assert torch.equal(y[..., part:], x[..., part:])
    assert torch.equal(r(x, pos.int()), y)
    # far positions keep their phase
    far = pos + 2 ** 40
    turns = r._turns.cpu().tolist()
    y = r(x, far)
    exact = torch.tensor([[((t * int(p)) % 2 ** 64) / 2.0 ** 64 * 2 * torch.pi for t in turns] for p in far.tolist()], dtype=torch.float64)
    c, s = (r.factor * exact.cos()).cuda()[:, None], (r.factor * exact.sin()).cuda()[:, None]
    xd, want = x.double(), x.double().clone()
    i = torch.arange(0, part, 2) if interleaved else torch.arange(part // 2)
    j = i + 1 if interleaved else i + part // 2
    want[..., i], want[..., j] = xd[..., i] * c - xd[..., j] * s, xd[..., j] * c + xd[..., i] * s
    close(y, want, b + E[dtype] * want.abs() + tiny, "far")


def test_rotary_strides_in_place_and_gradient(gen):
    from adaptq_b200 import Rotary
    r = Rotary(32, interleaved=False, scaling=SCALINGS[3])
    wide = torch.randn(6, 12, 100, generator=gen, device="cuda")
    pos = torch.arange(6, device="cuda")
    x = wide[:, 2:7, 3:67]  # unaligned rows
    want = r(x.contiguous(), pos)
    assert torch.equal(r(x, pos), want)
    t = x.transpose(0, 1)   # [5, 6, 64]: another order
    assert torch.equal(r(t, pos[:5]), r(t.contiguous(), pos[:5]))
    s = torch.randn(6, 64, 5, generator=gen, device="cuda").transpose(1, 2)  # rows not contiguous
    assert torch.equal(r(s, pos), r(s.contiguous(), pos))
    inside = wide.clone()
    r(inside[:, 2:7, 3:67], pos, out=inside[:, 2:7, 3:67])
    assert torch.equal(inside[:, 2:7, 3:67], want)
    inside[:, 2:7, 3:67] = wide[:, 2:7, 3:67]
    assert torch.equal(inside, wide)
    # the gradient is the formula's, and that of differences
    x = torch.randn(6, 5, 64, generator=gen, device="cuda", requires_grad=True)
    g = torch.randn(6, 5, 64, generator=gen, device="cuda")
    y = r(x, pos)
    (dx,) = torch.autograd.grad(y, x, g)
    want = ref.rotate(g.double(), pos, r, inverse=True)
    b, _ = rotary_bound(g.double(), pos, r, F32)
    close(dx, want, b + E[F32] * want.abs())
    step = torch.randn(6, 5, 64, generator=gen, device="cuda")
    with torch.no_grad():
        up, down = r(x + step, pos), r(x - step, pos)
    difference = ((up.double() - down.double()) / 2 * g).sum()
    size = float((g.double().abs().sum() * 10))
    assert abs(float(difference - (dx.double() * step).sum())) <= 1e-6 * size
    (dx2,) = torch.autograd.grad(r(x, pos).sum(), x)   # an expanded gradient, stride 0
    close(dx2, ref.rotate(torch.ones_like(g).double(), pos, r, inverse=True), 4 * 7e-7 * r.factor)
    assert r(torch.empty(0, 5, 64, device="cuda"), pos[:0]).shape == (0, 5, 64)


def test_rotary_gradients_of_gradients_and_copies(gen):
    import copy
    import pickle
    from adaptq_b200 import Rotary
    r = Rotary(24, scaling=SCALINGS[3])
    x = torch.randn(5, 2, 40, generator=gen, device="cuda", requires_grad=True)
    pos = torch.arange(3, 8, device="cuda")
    w = torch.randn(5, 2, 40, generator=gen, device="cuda")
    (g,) = torch.autograd.grad((r(x, pos) * x.detach()).pow(2).sum(), x, create_graph=True)
    (h,) = torch.autograd.grad((g * w).sum(), x)   # through both passes: R^T (2 d^2 R w), d = x.detach()
    d = x.detach().double()
    want = ref.rotate(2 * d * d * ref.rotate(w.double(), pos, r), pos, r, inverse=True)
    assert float((h.double() - want).abs().max()) <= 1e-5 * float(want.abs().max())
    y = r(x.detach(), pos)
    for other in (copy.deepcopy(r), pickle.loads(pickle.dumps(r))):
        assert torch.equal(other(x.detach(), pos), y)


def test_rotary_refusals(gpu_lib):
    from adaptq_b200 import Rotary
    r = Rotary(64)
    x, pos = torch.zeros(3, 2, 64, device="cuda"), torch.arange(3, device="cuda")
    for bad in (lambda: Rotary(63), lambda: Rotary(0), lambda: Rotary(64, base=0.0), lambda: Rotary(64, scaling={"type": "other"}),
                lambda: Rotary(64, scaling={"type": "linear"}), lambda: Rotary(64, scaling={"type": "yarn", "factor": 2.0}),
                lambda: Rotary(2, scaling={"type": "ntk", "factor": 2.0}), lambda: Rotary(64, scaling={"type": "linear", "factor": 2.0, "x": 1}),
                lambda: Rotary(64, device="cpu"), lambda: r(x[..., :32], pos), lambda: r(x, pos[:2]), lambda: r(x, pos.float()),
                lambda: r(x.double(), pos), lambda: r(x.cpu(), pos), lambda: r(x, pos.cpu()), lambda: r(x[0], pos),
                lambda: r(x, pos, out=torch.zeros(3, 2, 65, device="cuda")), lambda: r(x.requires_grad_(), pos, out=torch.zeros(3, 2, 64, device="cuda"))):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------
def check_rows(cache, signs, table_row, first, k, v, rotary):
    """The tokens first.. of one sequence hold these rows."""
    n = k.shape[0]
    at, off = ref.place(cache, table_row, n, first)
    for side, bits, x in (("k", cache.k_bits, k), ("v", cache.v_bits, v)):
        x = x.double()
        if side == "k" and rotary is not None:
            x = ref.rotate(x, torch.arange(first, first + n, device="cuda"), rotary)
        u, norm = ref.coordinates(x, signs)
        lv = ref.levels(bits).cuda()
        border = (lv[1:] + lv[:-1]) / 2
        want = torch.bucketize(u, border, right=True)
        store = (cache.k_pages if side == "k" else cache.v_pages)[at, :, off]
        got = ref.unpack(store, bits)
        wrong = got != want
        if wrong.any():
            assert bool(((got - want).abs()[wrong] == 1).all()), f"{side}: codes are off by more than one"
            gap = (u[..., None] - border).abs().amin(-1)[wrong]
            assert float(gap.max()) <= CODE_SLACK, f"{side}: {int(wrong.sum())} codes differ, one at {float(gap.max()):.2e} from a threshold"
        assert int(wrong.sum()) <= 1 + wrong.numel() // 1000
        norms = (cache.k_scales if side == "k" else cache.v_scales)[at, :, off]
        close(norms, norm, norm * (20 * E[F32] + 1.4e-6), f"{side} norms")


@pytest.mark.parametrize("heads,dim,kb,vb,page,dtype,style,part,lengths,past", [
    (1, 64, 4, 2, 16, BF16, "half", 64, [1], [0]),
    (8, 128, 4, 2, 64, BF16, "half", 128, [1, 1, 1, 1, 1], [0, 63, 64, 65, 200]),
    (3, 128, 3, 3, 32, F32, "interleaved", 64, [37, 0, 1, 70], [0, 5, 31, 40]),
    (2, 96, 2, 4, 16, F16, "half", 96, [5, 16, 17], [0, 16, 3]),
    (5, 80, 4, 3, 128, F32, "half", 40, [129, 3], [1, 0]),
    (1, 256, 4, 4, 256, BF16, "half", 256, [300], [10]),
    (2, 200, 3, 2, 64, F16, "interleaved", 200, [9, 2], [60, 0]),
    (4, 67, 2, 2, 16, BF16, "half", 34, [20, 1], [0, 15]),
    (2, 33, 4, 4, 16, F32, "none", 0, [3, 18], [0, 1]),
    (16, 256, 2, 3, 32, F32, "half", 128, [7, 1, 40], [0, 0, 32]),
    (14, 64, 3, 3, 16, F32, "interleaved", 32, [517], [0])])
def test_append_and_read_against_64_bits(gen, heads, dim, kb, vb, page, dtype, style, part, lengths, past):
    from adaptq_b200 import Rotary
    cache, signs = make_cache(gen, 40, heads, dim, kb, vb, page)
    rotary = None if style == "none" else Rotary(part, interleaved=style == "interleaved", scaling=SCALINGS[3])
    total = [a + b for a, b in zip(lengths, past)]
    table = ref.random_table(cache, total, gen)
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    T = cu[-1]
    k = torch.randn(T + 3, heads, dim, generator=gen, device="cuda").to(dtype)   # three rows of padding behind
    v = (3 * torch.randn(T + 3, heads, dim, generator=gen, device="cuda")).to(dtype)
    cache.k_pages.fill_(7); cache.v_pages.fill_(9)
    before = [t.clone() for t in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)]
    cache.append(k, v, table, ints(*past), ints(*cu), rotary=rotary)
    cache.check()
    touched = torch.zeros(cache.n_pages, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        check_rows(cache, signs, table[b], past[b], k[cu[b]: cu[b + 1]], v[cu[b]: cu[b + 1]], rotary)
        at, off = ref.place(cache, table[b], n, past[b])
        touched[at, off] = True
    for t, old in zip((cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales), before):  # nothing else changed
        same = (t == old).flatten(3).all(-1) if t.dim() == 4 else t == old
        assert bool((same | touched[:, None]).all())
    # one row per sequence needs no offsets
    if all(n == 1 for n in lengths):
        again, _ = make_cache(gen, 40, heads, dim, kb, vb, page)
        again._signs.copy_(cache._signs)
        again.append(k[:T], v[:T], table, ints(*past), rotary=rotary)
        for b in range(len(lengths)):
            at, off = ref.place(cache, table[b], 1, past[b])
            assert torch.equal(again.k_pages[at, :, off], cache.k_pages[at, :, off])
    # read back the new rows, in every type, rows behind left alone
    for out_type in (F32, F16, BF16):
        out = tuple(torch.full((T + 2, heads, dim), 77.0, dtype=out_type, device="cuda") for _ in range(2))
        got = cache.read(table, ints(*past), ints(*cu), T + 2, out=out)
        assert got[0] is out[0] and bool((out[0][T:] == 77).all()) and bool((out[1][T:] == 77).all())
        for b, n in enumerate(lengths):
            at, off = ref.place(cache, table[b], n, past[b])
            for side, o in zip("kv", out):
                want, level, norm = ref.rows(cache, side, at, off, signs)
                p = signs.shape[1]
                bound = 10 * E[F32] * level.abs().sum(-1, keepdim=True) * norm[..., None] / p + E[out_type] * want.abs() + (2.0 ** -25 if out_type == F16 else 0)
                close(o[cu[b]: cu[b + 1]], want, bound, f"{side} {out_type}")
    k2, v2 = cache.read(table, ints(*past), ints(*cu), T)
    assert k2.dtype == BF16 and torch.equal(k2, out[0][:T]) and torch.equal(v2, out[1][:T])
    cache.check()


def test_append_matches_the_ring_cache(gen):
    """The same FP32 rows in a ring (MHAContext) and in pages, same seed: norms to the last bits, codes alike."""
    from adaptq_b200 import MHAContext, PagedKVCache
    heads, dim, n = 4, 96, 50
    k, v = (torch.randn(n, heads, dim, generator=gen, device="cuda") for _ in range(2))
    ring = MHAContext(heads, dim, 4, 3, 64, seed=5, v_mass=0.0, hybrid_thresh=0)
    ring.append_all(k, v)
    cache = PagedKVCache(4, heads, dim, 4, 3, 16, seed=5)
    table = ints(2, 0, 3, 1).view(1, 4)
    cache.append(k, v, table, ints(0), ints(0, n))
    at, off = ref.place(cache, table[0], n)
    for h in range(heads):
        e = ring.export_head(h)
        for side, bits, pages, scales in (("k", 4, cache.k_pages, cache.k_scales), ("v", 3, cache.v_pages, cache.v_scales)):
            close(scales[at, h, off].cpu(), torch.from_numpy(e[f"{side}_scale"][:n]).double(), torch.from_numpy(e[f"{side}_scale"][:n]).double() * 2.0 ** -19)
            a = ref.unpack(pages[at, h, off].cpu(), bits)
            b = ref.unpack(torch.from_numpy(e[f"{side}_rows"][:n]), bits)
            assert int((a != b).sum()) <= 1 and int((a - b).abs().max()) <= 1
    # and the attention over both
    q = torch.randn(1, heads, dim, generator=gen, device="cuda")
    got = cache.attend(q, table, ints(n))
    want = ring.compute_all(q[0])
    assert float((got[0] - want).abs().max()) <= 1e-4 + 1e-4 * float(want.abs().max())


def test_special_rows(gen):
    """Zeros, tiny, huge and non-finite rows: no row spoils another."""
    cache, signs = make_cache(gen, 4, 2, 128, 4, 2, 16)
    k = torch.randn(8, 2, 128, generator=gen, device="cuda")
    v = torch.randn(8, 2, 128, generator=gen, device="cuda")
    plain = k.clone(), v.clone()
    for x in (k, v):
        x[1] = 0.0
        x[2] *= 1e-20
        x[3] *= 1e18
        x[4, 0, 5] = float("nan")
        x[5, 1, 7] = float("inf")
        x[6] = 0.0
        x[6, 0, 3] = 1e-30
    table = ints(1, 2).view(1, 2)
    cache.append(k, v, table, ints(0), ints(0, 8))
    kk, vv = cache.read(table, ints(0), ints(0, 8), 8, dtype=F32)
    for got, x, scales, bits in ((kk, k, cache.k_scales, 4), (vv, v, cache.v_scales, 2)):
        assert bool((scales[1, :, 1] == 1e-6).all()) or float((scales[1, :, 1] - 1e-6).abs().max()) < 1e-12
        for i in (0, 3, 7):
            want, level, norm = ref.rows(cache, "k" if bits == 4 else "v", table[0, :1].long(), torch.tensor([i], device="cuda"), signs)
            close(got[i: i + 1], want, 1e-5 * norm[..., None])
            rel = (got[i] - x[i]).norm() / x[i].norm()
            assert float(rel) < (0.15 if bits == 4 else 0.5)
        assert not bool(got[4, 0].isfinite().all()) and not bool(got[5, 1].isfinite().all())
        assert bool(got[4, 1].isfinite().all()) and bool(got[5, 0].isfinite().all())
    cache.check()


def test_bad_pages_and_positions_are_skipped_and_reported(gen):
    cache, signs = make_cache(gen, 4, 2, 64, 4, 4, 16)
    ref.random_pool(cache, gen)
    before = [t.clone() for t in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)]
    k = torch.randn(3, 2, 64, generator=gen, device="cuda")
    q = torch.randn(3, 2, 64, generator=gen, device="cuda")
    same = lambda: all(torch.equal(a, b) for a, b in zip(before, (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)))  # noqa: E731
    table = ints(-1, 4, 2 ** 31 - 1).view(3, 1)
    cache.append(k, k, table, ints(0, 3, 15))
    with pytest.raises(RuntimeError, match="outside the pool"):
        cache.check()
    cache.check()  # reported once
    assert same()
    out = torch.full((3, 2, 64), 5.0, device="cuda")
    cache.read(table, ints(0, 3, 15), ints(0, 1, 2, 3), 3, out=(out, out.clone()))
    assert bool((out == 5).all())
    with pytest.raises(RuntimeError, match="outside the pool"):
        cache.check()
    got = cache.attend(q, table, ints(4, 16, 0))
    with pytest.raises(RuntimeError, match="outside the pool"):
        cache.check()
    assert bool((got[2] == 0).all())
    good = ints(0, 1, 2).view(3, 1)
    cache.append(k, k, good, ints(16, -3, 2 ** 31 - 1))
    with pytest.raises(RuntimeError, match="no room"):
        cache.check()
    assert same()
    got = cache.attend(q, good, ints(17, -5, 2 ** 31 - 1))   # more than the table holds: its 16 tokens
    with pytest.raises(RuntimeError, match="no room"):
        cache.check()
    want = ref.attend(cache, signs, q, good, ints(16, 0, 16))
    attend_close(got, want, F32)
    assert bool((got[1] == 0).all())
    # offsets that run backwards or past the rows touch nothing they should not
    cache.append(k, k, good, ints(0, 0, 0), ints(3, 1, 9, 2))
    cache.read(good, ints(0, 0, 0), ints(3, 1, 9, 2), 3, out=(out, out.clone()))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("heads,group,dim,kb,vb,page,dtype,style,lengths", [
    (1, 1, 64, 4, 4, 16, F32, "none", [1]),
    (1, 1, 64, 2, 2, 16, BF16, "half", [2, 0, 1]),
    (8, 4, 128, 4, 2, 64, BF16, "half", [1000]),
    (8, 4, 128, 4, 2, 64, F32, "half", [1, 63, 64, 65, 128, 129, 700]),
    (2, 8, 128, 4, 4, 32, F16, "interleaved", [31, 32, 33, 500, 0, 2]),
    (14, 1, 64, 3, 2, 16, F16, "interleaved", [301, 17, 15, 16, 0]),
    (6, 3, 96, 4, 3, 32, F32, "none", [409, 1, 100]),
    (1, 12, 128, 2, 3, 128, BF16, "half", [257, 1024]),
    (2, 5, 80, 3, 4, 256, F16, "half", [256, 255, 600]),
    (3, 2, 256, 4, 4, 64, BF16, "half", [130, 1, 64]),
    (2, 9, 256, 2, 2, 16, F32, "half", [45, 200]),
    (4, 1, 67, 2, 4, 16, BF16, "none", [90, 16, 31]),
    (1, 16, 200, 3, 3, 64, F32, "interleaved", [300]),
    (1, 1, 128, 3, 4, 64, F16, "none", [5000]),
    (2, 4, 64, 2, 4, 64, F32, "half", [3000, 10])])
def test_attend_against_64_bits(gen, heads, group, dim, kb, vb, page, dtype, style, lengths):
    from adaptq_b200 import Rotary
    need = sum(-(-n // page) for n in lengths)
    cache, signs = make_cache(gen, need + 3, heads, dim, kb, vb, page)
    ref.random_pool(cache, gen)
    table = ref.random_table(cache, lengths, gen)
    rotary = None if style == "none" else Rotary(dim // 2 * 2, interleaved=style == "interleaved")
    q = (1.5 * torch.randn(len(lengths), heads * group, dim, generator=gen, device="cuda")).to(dtype)
    n = ints(*lengths)
    got = cache.attend(q, table, n, rotary=rotary)
    cache.check()
    assert got.dtype == dtype and got.shape == q.shape
    attend_close(got, ref.attend(cache, signs, q, table, n, rotary), dtype)
    # the same bits every time, another scale, given outputs, strided inputs
    assert torch.equal(cache.attend(q, table, n, rotary=rotary), got)
    attend_close(cache.attend(q, table, n, rotary=rotary, scale=0.02), ref.attend(cache, signs, q, table, n, rotary, scale=0.02), dtype, "scale")
    wide = torch.full((len(lengths), heads * group + 2, dim + 3), 9.0, dtype=dtype, device="cuda")
    wide[:, 1:-1, 1:-2] = q
    out = torch.full_like(wide, 9.0)
    res = cache.attend(wide[:, 1:-1, 1:-2], table, n, rotary=rotary, out=out[:, 1:-1, 1:-2])
    assert torch.equal(res, got)
    out[:, 1:-1, 1:-2] = 9.0
    assert bool((out == 9).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attend_extremes(gen, dtype):
    """Large logits, norms over many orders of magnitude, zero rows and queries, non-finite rows elsewhere."""
    cache, signs = make_cache(gen, 40, 2, 128, 4, 2, 16)
    ref.random_pool(cache, gen)
    lengths = [100, 37, 64, 5]
    table = ref.random_table(cache, lengths, gen)
    n = ints(*lengths)
    q = torch.randn(4, 8, 128, generator=gen, device="cuda").to(dtype)
    q[1] = 0.0                       # equal weights
    at, off = ref.place(cache, table[0], 100)
    cache.v_scales[at[:50], :, off[:50]] *= 1e6
    cache.v_scales[at[50:], :, off[50:]] *= 1e-6
    cache.k_scales[at[3], :, off[3]] *= 30.0       # one token far above the others
    at, off = ref.place(cache, table[2], 64)
    cache.v_scales[at[:63], :, off[:63]] = 0.0
    at, off = ref.place(cache, table[3], 5)
    cache.v_scales[at, :, off] = 1e-30
    # what lies behind a sequence's end in its last page counts for nothing
    for b, m in enumerate(lengths):
        if m % 16:
            page = int(table[b, m // 16])
            cache.k_scales[page, :, m % 16:] = float("nan")
            cache.v_scales[page, :, m % 16:] = float("inf")
    got = cache.attend(q, table, n)
    want = ref.attend(cache, signs, q, table, n)
    keep = [0, 1, 2] if dtype != F32 else [0, 1, 2, 3]
    tol = 1e-3 if dtype == F32 else 0.05   # logits reach hundreds here: their own rounding moves weights
    err, size = (got.double() - want).norm(dim=-1), want.norm(dim=-1)
    assert bool((err[keep] <= tol * size[keep] + 1e-37).all()), (err / size)
    assert bool((got[3].double().abs() <= 1e-29).all())
    cache.k_scales[table[1, 0].long(), :, 4] = float("nan")
    bad = cache.attend(q, table, n)
    assert bool(bad[1].isnan().all()) and torch.equal(bad[[0, 2, 3]], got[[0, 2, 3]])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("power", [10, 20, 27])
def test_many_tokens_far_below_one(gen, dtype, power):
    """One value 2^power times as long as 30000 equal ones under equal weights: their sum still counts."""
    cache, signs = make_cache(gen, 118, 1, 128, 4, 4, 256)
    ref.random_pool(cache, gen)
    cache.k_scales.zero_()                                   # equal logits
    cache.v_pages[:] = cache.v_pages[0, 0, 0]                # one row for all
    cache.v_scales.fill_(1.0)
    table = ref.random_table(cache, [30000], gen)
    page = int(table[0, 7])
    cache.v_scales[page, 0, 11] = 2.0 ** power
    cache.v_pages[page, 0, 11] = cache.v_pages[page, 0, 11].flip(0)   # another direction
    q = torch.randn(1, 1, 128, generator=gen, device="cuda").to(dtype)
    got, want = cache.attend(q, table, ints(30000)), ref.attend(cache, signs, q, table, ints(30000))
    attend_close(got, want, dtype)


def test_shared_pages_and_views(gen):
    """Sequences that share their first pages; tables, lengths and queries that are views; the output in the queries' place."""
    cache, signs = make_cache(gen, 20, 2, 64, 4, 2, 16)
    ref.random_pool(cache, gen)
    wide = torch.full((6, 9), -1, dtype=torch.int32, device="cuda")
    wide[::2, 2:8] = torch.tensor([[3, 4, 5, 6, 7, 8], [3, 4, 9, 10, 11, 12], [3, 4, 5, 6, 13, 13]], dtype=torch.int32, device="cuda")
    table, n = wide[::2, 2:], ints(90, 0, 40, 0, 96, 0)[::2]
    q = torch.randn(3, 2, 5, 64, generator=gen, device="cuda").to(BF16).transpose(1, 2).reshape(3, 10, 64)
    want = ref.attend(cache, signs, q, table, n)
    attend_close(cache.attend(q, table, n), want, BF16)
    assert torch.equal(cache.attend(q, table, n, out=q), q)
    attend_close(q, want, BF16)
    cache.check()


def test_refusals(gpu_lib):
    from adaptq_b200 import PagedKVCache, Rotary
    for bad in (dict(dim=32), dict(dim=257), dict(k_bits=5), dict(v_bits=16), dict(page_size=48), dict(n_pages=0), dict(n_kv_heads=0), dict(device="cpu"),
                dict(signs=torch.zeros(2, 64)), dict(signs=torch.ones(2, 32))):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(n_pages=4, n_kv_heads=2, dim=64, page_size=16), **bad})
    c = PagedKVCache(4, 2, 64, page_size=16)
    k, q, table, n = torch.zeros(2, 2, 64, device="cuda"), torch.zeros(2, 4, 64, device="cuda"), ints(0, 1).view(2, 1), ints(1, 1)
    wide = Rotary(128)
    for bad in (lambda: c.append(k[:, :1], k[:, :1], table, n), lambda: c.append(k, k.half(), table, n), lambda: c.append(k, k[:1], table, n),
                lambda: c.append(k.double(), k.double(), table, n), lambda: c.append(k.cpu(), k.cpu(), table, n), lambda: c.append(k, k, table.long(), n),
                lambda: c.append(k, k, table, n.long()), lambda: c.append(k, k, table, n[:1]), lambda: c.append(k, k, table[:1], n[:1]),
                lambda: c.append(k, k, table, n, n), lambda: c.append(k, k, table, n, rotary=wide), lambda: c.attend(q[:, :3], table, n),
                lambda: c.attend(q[:1], table, n), lambda: c.attend(q, table, n[:1]), lambda: c.attend(q, table, n, rotary="x"),
                lambda: c.attend(q, table[:, :0], n), lambda: c.append(k, k, table[:, :0], n), lambda: c.attend(q, table, n, out=q[:, :2]), lambda: c.attend(q[..., :32], table, n), lambda: c.attend(q.cpu(), table, n),
                lambda: c.read(table, n, n, 2), lambda: c.read(table, n, ints(0, 1, 2), 2, dtype=torch.int8),
                lambda: c.read(table, n, ints(0, 1, 2), 2, out=(k[:1], k[:1]))):
        with pytest.raises(ValueError):
            bad()
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="scale"):
            c.attend(q, table, n, scale=scale)
    with pytest.raises(ValueError):
        PagedKVCache.over(c.k_pages, c.v_pages[:2], c.k_scales, c.v_scales, 64, 4, 4)
    with pytest.raises(ValueError):
        PagedKVCache.over(c.k_pages.cpu(), c.v_pages.cpu(), c.k_scales.cpu(), c.v_scales.cpu(), 64, 4, 4)
    assert c.attend(q[:0], table[:0], n[:0]).shape == (0, 4, 64)
    c.append(k[:0], k[:0], table, n, ints(0, 0, 0))
    c.check()


# ---------------------------------------------------------------------------
# the operators together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_prompts_steps_and_history(gen, dtype):
    """A continuous batch: prompts of different lengths, decode steps with sequences that come and go, a prompt that
    continues in pieces -- every step against the definitions over what the cache holds."""
    from adaptq_b200 import Rotary
    heads, group, dim, page = 2, 4, 128, 16
    cache, signs = make_cache(gen, 64, heads, dim, 4, 2, page)
    rotary = Rotary(dim, scaling=SCALINGS[4])
    lengths = [40, 3, 0, 17]
    table = ref.random_table(cache, [80, 60, 60, 60], gen, extra=0)
    mk = lambda n, h: torch.randn(n, h, dim, generator=gen, device="cuda").to(dtype)  # noqa: E731
    cu = [0, 40, 43, 43, 60]
    k, v = mk(60, heads), mk(60, heads)
    cache.append(k, v, table, ints(0, 0, 0, 0), ints(*cu), rotary=rotary)
    for b in range(4):
        check_rows(cache, signs, table[b], 0, k[cu[b]: cu[b + 1]], v[cu[b]: cu[b + 1]], rotary)
    for step in range(6):
        active = [1, 1, 1 if step >= 2 else 0, 1 if step < 4 else 0]
        now = [n + 1 if a else 0 for n, a in zip(lengths, active)]
        k, v, q = mk(4, heads), mk(4, heads), mk(4, heads * group)
        got = cache.step(k, v, q, table, ints(*now), rotary=rotary)
        cache.check()
        for b in range(4):
            if active[b]:
                check_rows(cache, signs, table[b], lengths[b], k[b: b + 1], v[b: b + 1], rotary)
                lengths[b] += 1
        attend_close(got, ref.attend(cache, signs, q, table, ints(*now), rotary), dtype, f"step {step}")
        assert all(bool((got[b] == 0).all()) for b in range(4) if not active[b])
    # sequence 0 goes on with ten tokens at once and reads its history back
    k, v = mk(10, heads), mk(10, heads)
    cache.append(k, v, table[:1], ints(lengths[0]), ints(0, 10), rotary=rotary)
    n = lengths[0] + 10
    hk, hv = cache.read(table[:1], ints(0), ints(0, n), n, dtype=F32)
    at, off = ref.place(cache, table[0], n)
    want, level, norm = ref.rows(cache, "k", at, off, signs)
    close(hk, want, 10 * E[F32] * level.abs().sum(-1, keepdim=True) * norm[..., None] / 128 + E[F32] * want.abs())
    kr = ref.rotate(k.double(), torch.arange(lengths[0], n, device="cuda"), rotary)
    assert float((hk[-10:].double() - kr).norm() / kr.norm()) < 0.15 and float((hv[-10:].double() - v.double()).norm() / v.double().norm()) < 0.5


def test_streams_and_graphs(gen):
    """A captured decode step replays on new inputs; two graphs and eager calls share a cache and no workspace."""
    from adaptq_b200 import Rotary
    cache, signs = make_cache(gen, 64, 2, 128, 4, 2, 16)
    ref.random_pool(cache, gen)
    rotary = Rotary(128)
    table = ref.random_table(cache, [300, 200, 100], gen)
    mk = lambda h: torch.randn(3, h, 128, generator=gen, device="cuda").to(BF16)  # noqa: E731
    k, v, q, n = mk(2), mk(2), mk(8), ints(250, 130, 99)
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.step(k, v, q, table, n, rotary=rotary)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cache.step(k, v, q, table, n, rotary=rotary))
        graphs.append(g)
    for trial in range(3):
        for t, h in ((k, 2), (v, 2), (q, 8)):
            t.copy_(mk(h))
        n.copy_(ints(251 + trial, 131 + trial, 0 if trial == 1 else 100))
        for g, o in zip(graphs, outs):
            o.fill_(3.0)
            g.replay()
        want = ref.attend(cache, signs, q, table, n, rotary)
        attend_close(outs[0], want, BF16, f"replay {trial}")
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], cache.attend(q, table, n, rotary=rotary))
    # two streams at once over the same pages
    big = torch.randn(3, 8, 128, generator=gen, device="cuda").to(BF16)
    alone = cache.attend(big, table, n, rotary=rotary)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([cache.attend(big, table, n, rotary=rotary) for _ in range(20)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, alone) for per in got for o in per)
    cache.check()


def test_offsets_beyond_32_bits(gen):
    """A pool of more than 4 GiB a side, pages from its end; rows further than 2^31 elements apart."""
    from adaptq_b200 import PagedKVCache, Rotary
    heads, dim = 8, 256
    signs = ref.random_signs(heads, 256, gen)
    cache = PagedKVCache(18000, heads, dim, 4, 4, 256, signs=signs)   # 4.7e9 bytes of keys
    assert cache.k_pages.numel() > 2 ** 32
    table = ints(17999, 9001, 17000, 5).view(2, 2)
    k, v = (torch.randn(600, heads, dim, generator=gen, device="cuda") for _ in range(2))
    rotary = Rotary(dim)
    cache.append(k, v, table, ints(0, 0), ints(0, 400, 600), rotary=rotary)
    cache.check()
    for b, (lo, hi) in enumerate(((0, 400), (400, 600))):
        check_rows(cache, signs.double(), table[b], 0, k[lo:hi], v[lo:hi], rotary)
    q = torch.randn(2, heads, dim, generator=gen, device="cuda")
    attend_close(cache.attend(q, table, ints(400, 200), rotary=rotary), ref.attend(cache, signs.double(), q, table, ints(400, 200), rotary), F32)
    got, _ = cache.read(table, ints(0, 0), ints(0, 400, 600), 600, dtype=F32)
    at, off = ref.place(cache, table[0], 400)
    want, level, norm = ref.rows(cache, "k", at, off, signs.double())
    close(got[:400], want, 10 * E[F32] * level.abs().sum(-1, keepdim=True) * norm[..., None] / 256 + E[F32] * want.abs())
    del cache
    far = torch.zeros(2 ** 31 + 4096, dtype=BF16, device="cuda")
    x = far.as_strided((2, 2, 64), (2 ** 31, 64, 1))
    x.copy_(torch.randn(2, 2, 64, generator=gen, device="cuda").to(BF16))
    r, pos = Rotary(64), torch.tensor([7, 9], device="cuda")
    assert torch.equal(r(x, pos), r(x.contiguous(), pos))


def test_launch_failures_are_errors(gen, gpu_lib):
    cache, _ = make_cache(gen, 4, 2, 64, 4, 4, 16)
    k, q, table = torch.zeros(1, 2, 64, device="cuda"), torch.zeros(1, 2, 64, device="cuda"), ints(0).view(1, 1)
    for call in (lambda: cache.append(k, k, table, ints(0)), lambda: cache.attend(q, table, ints(1)), lambda: cache.read(table, ints(0), ints(0, 1), 1)):
        gpu_lib.adaptq_inject_failure(3, 1)
        try:
            with pytest.raises(RuntimeError, match="CUDA error"):
                call()
        finally:
            gpu_lib.adaptq_inject_failure(3, 0)
        call()
    torch.cuda.synchronize()
