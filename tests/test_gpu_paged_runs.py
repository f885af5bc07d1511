"""The paged cache and rotary positions at sizes where the kernels take several steps: warps that walk over many
units, sequences, heads and passes; warps and blocks with several tokens or tiles.  The smaller cases of
test_gpu_paged.py give every warp one of them.  Tolerances are those derived there."""
import pytest
import torch

import paged_reference as ref
from test_gpu_paged import BF16, CODE_SLACK, E, F16, F32, SCALINGS, attend_close, close, ints, make_cache, rotary_bound

pytestmark = pytest.mark.gpu

SMS = 148


@pytest.fixture()
def gen(gpu_lib):
    return torch.Generator(device="cuda").manual_seed(23)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("seqs,heads,group,dim,kb,vb,page,dtype,longest", [
    (64, 8, 4, 128, 4, 2, 64, BF16, 2400),
    (64, 8, 1, 128, 3, 4, 16, BF16, 2400),
    (60, 4, 12, 96, 4, 4, 32, BF16, 2400),     # two passes
    (64, 8, 3, 128, 4, 3, 64, F16, 2400),
    (50, 4, 9, 112, 2, 2, 16, F16, 2400),      # three passes
    (64, 8, 2, 128, 4, 4, 128, F32, 2400),
    (60, 4, 6, 128, 2, 3, 16, F32, 2400),      # two passes
    (70, 14, 1, 64, 3, 2, 16, F16, 1500),
    (70, 14, 4, 64, 2, 4, 64, BF16, 1500),
    (70, 14, 1, 64, 4, 3, 32, F32, 1500),
    (40, 4, 8, 256, 4, 2, 64, BF16, 1600),
    (50, 4, 4, 200, 3, 3, 16, F16, 1600),
    (40, 4, 1, 256, 4, 4, 256, F32, 1600)])
def test_attend_walks_over_many_units(gen, seqs, heads, group, dim, kb, vb, page, dtype, longest):
    """At least three units a warp, so that both stages of its ring are in use, runs start and end anywhere, and the walk
    goes on to the next pass, head and sequence (past empty ones); values grow along a sequence, so that the
    reference of the exponentials has to move inside a run."""
    lengths = torch.randint(0, longest + 1, (seqs,), generator=torch.Generator().manual_seed(seqs + dim)).tolist()
    lengths[0] = lengths[seqs // 2] = lengths[seqs // 2 + 1] = lengths[-1] = 0
    lengths[3], lengths[4] = 1, longest
    unit, cols, warps = (32 if dim > 128 else 64), (8 if dtype == BF16 else 4), (8 if dim > 128 else 16)
    units = sum(-(-n // unit) for n in lengths) * heads * -(-group // cols)
    assert units >= 3 * SMS * warps
    cache, signs = make_cache(gen, sum(-(-n // page) for n in lengths) + 3, heads, dim, kb, vb, page)
    ref.random_pool(cache, gen)
    table = ref.random_table(cache, lengths, gen)
    for b, n in enumerate(lengths):
        if n:
            at, off = ref.place(cache, table[b], n)
            t = torch.arange(n, device="cuda")
            cache.v_scales[at, :, off] *= torch.exp2((t - longest) / 120.0)[:, None]
            cache.k_scales[at, :, off] *= (1 + t / (2.0 * longest))[:, None]
    q = torch.randn(seqs, heads * group, dim, generator=gen, device="cuda").to(dtype)
    got = cache.attend(q, table, ints(*lengths))
    cache.check()
    want = ref.attend(cache, signs, q, table, ints(*lengths))
    if dtype == F16:   # short sequences are small: outputs below 2^-14 are half a step of 2^-24 off, sqrt(dim) of them in the norm
        over = (got.double() - want).norm(dim=-1) - (4 * 7e-4 + 2 * E[F16]) * want.norm(dim=-1)
        assert float(over.max()) <= 2.0 ** -25 * dim ** 0.5
    else:
        attend_close(got, want, dtype)
    assert torch.equal(cache.attend(q, table, ints(*lengths)), got)


# ---------------------------------------------------------------------------
# append and read-back
# ---------------------------------------------------------------------------
def ragged(gen, total, longest):
    """Lengths of sequences that bring `total` tokens: many short or empty ones."""
    n = torch.randint(0, longest + 1, (2 * total // longest + 8,), generator=gen, device="cuda")
    n[n % 5 == 0] = 0
    end = n.cumsum(0)
    n = torch.where(end <= total, n, (n - (end - total)).clamp(min=0))
    n[-1] += total - n.sum()
    return n


@pytest.mark.parametrize("tokens,heads,dim,kb,vb,page,dtype,style,part,longest", [
    (12000, 8, 128, 4, 2, 64, BF16, "half", 128, 700),
    (12000, 1, 64, 4, 4, 16, F16, "interleaved", 64, 3),
    (12001, 3, 96, 3, 2, 32, F32, "half", 48, 40),
    (40000, 1, 128, 2, 3, 128, BF16, "half", 128, 5),
    (40003, 3, 64, 2, 4, 16, BF16, "half", 32, 200),
    (40000, 8, 80, 4, 3, 64, F16, "none", 0, 3000),
    (20000, 2, 256, 3, 4, 16, BF16, "half", 256, 11),
    (200001, 1, 33, 4, 2, 256, F16, "half", 32, 64)])
def test_append_and_read_many_tokens(gen, tokens, heads, dim, kb, vb, page, dtype, style, part, longest):
    """Several tokens a warp of the append and up to four tiles a block of the read-back, which find the sequences of
    their tokens across many short and empty ones."""
    from adaptq_b200 import Rotary
    new = ragged(gen, tokens, longest)
    assert int(new.sum()) == tokens and int((new == 0).sum()) > 1
    past = torch.randint(0, 2 * page, new.shape, generator=gen, device="cuda")
    need = -(-(past + new) // page)
    cache, signs = make_cache(gen, int(need.sum()) + 2, heads, dim, kb, vb, page)
    table = torch.full((len(new), int(need.max())), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(table.shape[1], device="cuda")[None] < need[:, None]
    table[at] = torch.randperm(cache.n_pages, generator=gen, device="cuda")[: int(need.sum())].int()
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)]).int()
    rotary = None if style == "none" else Rotary(part, interleaved=style == "interleaved", scaling=SCALINGS[3])
    k = torch.randn(tokens + 5, heads, dim, generator=gen, device="cuda").to(dtype)
    v = (3 * torch.randn(tokens + 5, heads, dim, generator=gen, device="cuda")).to(dtype)
    cache.append(k, v, table, past.int(), cu, rotary=rotary)
    cache.check()
    owner = torch.repeat_interleave(torch.arange(len(new), device="cuda"), new)
    pos = past[owner] + torch.arange(tokens, device="cuda") - cu[owner].long()
    pages, off = table[owner, pos // page].long(), pos % page
    for side, bits, x in (("k", kb, k), ("v", vb, v)):
        x = x[:tokens].double()
        if side == "k" and rotary is not None:
            x = ref.rotate(x, pos, rotary)
        u, norm = ref.coordinates(x, signs)
        lv = ref.levels(bits).cuda()
        border = (lv[1:] + lv[:-1]) / 2
        want = torch.bucketize(u, border, right=True)
        got = ref.unpack((cache.k_pages if side == "k" else cache.v_pages)[pages, :, off], bits)
        wrong = got != want
        if wrong.any():
            assert int((got - want).abs().max()) == 1
            assert float((u[wrong][:, None] - border).abs().amin(-1).max()) <= CODE_SLACK
        assert int(wrong.sum()) <= 1 + wrong.numel() // 1000
        norms = (cache.k_scales if side == "k" else cache.v_scales)[pages, :, off]
        close(norms, norm, norm * (20 * E[F32] + 1.4e-6), f"{side} norms")
        del u, want, got, wrong
    for out_type in (F32, dtype):
        out = tuple(torch.full((tokens + 3, heads, dim), 77.0, dtype=out_type, device="cuda") for _ in range(2))
        cache.read(table, past.int(), cu, tokens + 3, out=out)
        for side, o in zip("kv", out):
            assert bool((o[tokens:] == 77).all())
            want, level, norm = ref.rows(cache, side, pages, off, signs)
            bound = 10 * E[F32] * level.abs().sum(-1, keepdim=True) * norm[..., None] / signs.shape[1] + E[out_type] * want.abs()
            close(o[:tokens], want, bound + (2.0 ** -25 if out_type == F16 else 0), f"{side} {out_type}")
    cache.check()


# ---------------------------------------------------------------------------
# rotary
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("tokens,heads,dim,part,interleaved,dtype", [
    (2401, 2, 128, 128, False, BF16), (2403, 3, 64, 64, True, F32), (5003, 4, 128, 64, False, F16), (5001, 1, 67, 30, False, BF16),
    (4738, 14, 80, 40, True, F32), (9999, 2, 64, 64, False, F32)])
def test_rotary_several_tokens_a_block(gen, tokens, heads, dim, part, interleaved, dtype):
    from adaptq_b200 import Rotary
    r = Rotary(part, interleaved=interleaved, scaling=SCALINGS[4])
    x = torch.randn(tokens, heads, dim, generator=gen, device="cuda").to(dtype)
    pos = torch.randint(0, 2 ** 20, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    y = r(x, pos)
    want = ref.rotate(x.double(), pos, r)
    b, tiny = rotary_bound(x.double(), pos, r, dtype)
    close(y, want, b + E[dtype] * want.abs() + tiny)
    assert torch.equal(y[..., part:], x[..., part:])


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
