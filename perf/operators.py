"""What is measured of the paged quantised cache: rotary positions, rows that enter the pages, attention of
one new token over the pages, and rows read back from them.

A page holds `page` tokens of every KV head: packed codes of the rows in the rotated domain (2, 3 or 4 bits a
coordinate, most significant first) and one float32 norm per row, for keys and for values.  A sequence is a
list of pages (a row of the block table) and a length.
"""
from __future__ import annotations

import math

import torch

own = False

CODEBOOK = {
    2: [0.4528, 1.5104],
    3: [0.2451, 0.7560, 1.3439, 2.1529],
    4: [0.1258, 0.3795, 0.6402, 0.9138, 1.2016, 1.5105, 1.8944, 2.4008],
}
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One user, a short conversation: the smallest decode call, four queries per KV head.
        {"name": "attend_1x8_g4_len1000", "kind": "attend", "seqs": 1, "kv_heads": 8, "group": 4, "dim": 128, "k_bits": 4,
         "v_bits": 2, "page": 64, "longest": 1000, "spread": 0.0, "dtype": "bf16", "rotary": "half", "rotary_dim": 128,
         "scaling": "none"},
        # One user, one very long document (the benchmark's longest context).
        {"name": "attend_1x8_g4_len131072", "kind": "attend", "seqs": 1, "kv_heads": 8, "group": 4, "dim": 128, "k_bits": 4,
         "v_bits": 4, "page": 128, "longest": 131072, "spread": 0.0, "dtype": "bf16", "rotary": "half", "rotary_dim": 128,
         "scaling": "yarn"},
        # A continuous batch at the benchmark's context: 64 sequences of 820 to 8192 tokens.
        {"name": "attend_64x8_g4_len8192", "kind": "attend", "seqs": 64, "kv_heads": 8, "group": 4, "dim": 128, "k_bits": 4,
         "v_bits": 2, "page": 64, "longest": 8192, "spread": 0.9, "dtype": "bf16", "rotary": "half", "rotary_dim": 128,
         "scaling": "none"},
        # A small model without grouped queries, short odd sequences, one of them empty, small pages.
        {"name": "attend_33x14_g1_d64_len3001", "kind": "attend", "seqs": 33, "kv_heads": 14, "group": 1, "dim": 64, "k_bits": 3,
         "v_bits": 2, "page": 16, "longest": 3001, "spread": 1.0, "dtype": "fp16", "rotary": "interleaved", "rotary_dim": 64,
         "scaling": "none"},
        # FP32 in and out, a head dimension that is padded, three queries per KV head, no positions.
        {"name": "attend_20x6_g3_d96_fp32", "kind": "attend", "seqs": 20, "kv_heads": 6, "group": 3, "dim": 96, "k_bits": 4,
         "v_bits": 3, "page": 32, "longest": 4099, "spread": 0.7, "dtype": "fp32", "rotary": "none", "rotary_dim": 0,
         "scaling": "none"},
        # The append of a decode step: one token of each of 256 sequences, and the rows as the cache now holds them.
        {"name": "append_256_tokens", "kind": "append", "seqs": 256, "new": 1, "past": 4096, "kv_heads": 8, "dim": 128, "k_bits": 4,
         "v_bits": 2, "page": 64, "spread": 0.9, "dtype": "bf16", "rotary": "half", "rotary_dim": 128, "scaling": "none",
         "history": False},
        # Prompts of different lengths enter together, and are read back for their own attention.
        {"name": "append_prompts_4x8192", "kind": "append", "seqs": 4, "new": 8192, "past": 0, "kv_heads": 8, "dim": 128, "k_bits": 4,
         "v_bits": 2, "page": 64, "spread": 0.6, "dtype": "bf16", "rotary": "half", "rotary_dim": 128, "scaling": "llama3",
         "history": True},
        # A small model's prompts in FP32, interleaved positions on part of the head; read back in 16 bits.
        {"name": "append_7x517_14_d64_fp32", "kind": "append", "seqs": 7, "new": 517, "past": 0, "kv_heads": 14, "dim": 64, "k_bits": 3,
         "v_bits": 3, "page": 16, "spread": 1.0, "dtype": "fp32", "rotary": "interleaved", "rotary_dim": 32, "scaling": "linear",
         "history": True},
        # A long prompt arrives in pieces: 512 tokens more, and the whole history read back for them.
        {"name": "continue_512_after_30000", "kind": "append", "seqs": 1, "new": 512, "past": 30000, "kv_heads": 8, "dim": 128,
         "k_bits": 4, "v_bits": 4, "page": 128, "spread": 0.0, "dtype": "fp16", "rotary": "half", "rotary_dim": 128, "scaling": "ntk",
         "history": True},
        # The queries of a prompt, rotated for its own attention.
        {"name": "rotary_16384x32", "kind": "rotary", "tokens": 16384, "heads": 32, "dim": 128, "dtype": "bf16", "rotary": "half",
         "rotary_dim": 128, "scaling": "llama3", "gradient": False},
        # Rotation with its gradient: part of an odd head dimension, scaled for long contexts.
        {"name": "rotary_gradient_3001x14_d80", "kind": "rotary", "tokens": 3001, "heads": 14, "dim": 80, "dtype": "fp32",
         "rotary": "interleaved", "rotary_dim": 40, "scaling": "yarn", "gradient": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "append", "rotary"])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256, rng.randint(40, 256)])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    style = rng.choice(["half", "half", "interleaved", "none"])
    part = rng.choice([1.0, 1.0, 0.5, rng.random()])
    rotary_dim = 0 if style == "none" else max(4, int(dim * part) // 2 * 2)
    c = {"kind": kind, "dim": dim, "dtype": dtype, "rotary": style, "rotary_dim": rotary_dim,
         "scaling": rng.choice(["none", "linear", "ntk", "yarn", "llama3"])}
    if kind == "rotary":
        if style == "none":
            c["rotary"], c["rotary_dim"] = "half", dim // 2 * 2
        heads = rng.randint(1, 40)
        gradient = rng.random() < 0.5
        room = 60_000_000 // (heads * dim * (2 if dtype == "fp32" else 1) * (2 if gradient else 1))
        c.update(heads=heads, tokens=_log(rng, 1, min(16384, room)), gradient=gradient)
        return c
    heads = rng.choice([1, 2, 4, 8, 8, rng.randint(1, 16)])
    c.update(kv_heads=heads, k_bits=rng.choice([2, 3, 4, 4]), v_bits=rng.choice([2, 2, 3, 4]), page=rng.choice([16, 32, 64, 64, 128, 256]),
             seqs=_log(rng, 1, 256), spread=rng.choice([0.0, 0.5, 0.9, 1.0]))
    if kind == "attend":
        room = 134_000_000 // (c["seqs"] * heads * _padded(dim))
        c.update(group=rng.choice([1, 1, 2, 4, 4, 5, 8, 12]), longest=_log(rng, 16, max(17, min(131072, room))))
    else:
        one = c["seqs"] * heads * _padded(dim)
        past = rng.choice([0, 0, _log(rng, 1, max(1, min(8192, 64_000_000 // one)))])
        c.update(new=_log(rng, 1, max(2, min(8192, 16_000_000 // one))), past=past, history=one * past < 16_000_000 and rng.random() < 0.5)
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _read_dtype(case):
    """History is read back in 16 bits, whatever the model's own type."""
    return torch.float16 if case["dtype"] == "fp16" else torch.bfloat16


def _padded(dim):
    return 1 << (dim - 1).bit_length()


def _sizes(n, longest, spread):
    """n lengths from `longest` down to (1 - spread) * longest; the full spread ends with an empty sequence."""
    low = 0 if spread == 1.0 and n > 1 else 1
    return [max(low, round(longest * (1 - spread * i / max(1, n - 1)))) for i in range(n)]


def _lengths(case, longest, gen):
    """The same lengths for every seed, in another order."""
    order = torch.randperm(case["seqs"], generator=gen, device="cuda")
    return torch.tensor(_sizes(case["seqs"], longest, case["spread"]), device="cuda")[order]


def _pack(code, bits):
    """[..., P] codes -> [..., P * bits / 8] bytes, most significant bits first."""
    code = code.to(torch.int32)
    if bits == 3:
        c = code.view(*code.shape[:-1], -1, 8)
        word = sum(c[..., i] << (21 - 3 * i) for i in range(8))
        return torch.stack([word >> 16, (word >> 8) & 255, word & 255], -1).flatten(-2).to(torch.uint8)
    per = 8 // bits
    c = code.view(*code.shape[:-1], -1, per)
    return sum(c[..., i] << (8 - bits * (i + 1)) for i in range(per)).to(torch.uint8)


def _frequencies(case):
    """(inverse frequencies in float64, factor of cos and sin) of the case's positions."""
    d, base = case["rotary_dim"], 10000.0
    i = torch.arange(0, d, 2, dtype=torch.float64) / d
    kind = case["scaling"]
    if kind == "ntk":
        base = base * 4.0 ** (d / (d - 2))
    w, f = base ** -i, 1.0
    if kind == "linear":
        w = w / 4.0
    elif kind == "llama3":
        wave = 2 * math.pi / w
        s = (8192.0 / wave - 1.0) / (4.0 - 1.0)
        mid = (1 - s) * w / 8.0 + s * w
        w = torch.where(wave > 8192.0, w / 8.0, torch.where(wave < 8192.0 / 4.0, w, mid))
    elif kind == "yarn":
        at = lambda turns: d * math.log(4096.0 / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(0, math.floor(at(32.0))), min(d - 1, math.ceil(at(1.0)))
        ramp = ((torch.arange(d // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        w, f = w / 8.0 * ramp + w * (1 - ramp), 0.1 * math.log(8.0) + 1.0
    return w, f


def _scaling(case):
    """The same choice as the framework names it."""
    return {"none": None, "linear": {"type": "linear", "factor": 4.0}, "ntk": {"type": "ntk", "factor": 4.0},
            "yarn": {"type": "yarn", "factor": 8.0, "original_max_position": 4096},
            "llama3": {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                       "original_max_position": 8192}}[case["scaling"]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    dtype, dim = DTYPE[case["dtype"]], case["dim"]
    s = {"case": dict(case)}
    if case["rotary"] != "none":
        w, f = _frequencies(case)
        s["inv_freq"], s["factor"] = w.cuda(), f
        if own:
            from adaptq_b200 import Rotary
            s["rotary"] = Rotary(case["rotary_dim"], 10000.0, interleaved=case["rotary"] == "interleaved", scaling=_scaling(case),
                                 device="cuda")
    elif own:
        s["rotary"] = None
    if case["kind"] == "rotary":
        s["x"] = normal(case["tokens"], case["heads"], dim).to(dtype)
        # a prompt's positions, from wherever it stands in its conversation
        first = int(torch.randint(0, 100_000, (1,), generator=gen, device="cuda"))
        s["positions"] = torch.arange(first, first + case["tokens"], device="cuda", dtype=torch.int32)
        if case["gradient"]:
            s["x"].requires_grad_(True)
            s["grad"] = normal(case["tokens"], case["heads"], dim).to(dtype)
        return s

    heads, page, p, n = case["kv_heads"], case["page"], _padded(dim), case["seqs"]
    if case["kind"] == "attend":
        held = _lengths(case, case["longest"], gen)
        total = held
    else:
        held = _lengths(case, case["past"], gen) if case["past"] else torch.zeros(n, dtype=torch.int64, device="cuda")
        new = _lengths(case, case["new"], gen) if case["new"] > 1 else held * 0 + 1
        total = held + new
    pages = (total + page - 1) // page
    most, used = int(pages.max()), int(pages.sum())
    n_pages = used + 7
    # the pages of a server that has run for a while: in no order, the table's unused entries point nowhere
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((n, max(most, 1)), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(table.shape[1], device="cuda")[None, :] < pages[:, None]
    table[at] = order[:used]
    s["table"] = table
    # pages as a run of appends leaves them: codes of normally distributed coordinates, norms around sqrt(dim),
    # a first token whose norms stand out
    for side, bits, spread in (("k", case["k_bits"], 0.25), ("v", case["v_bits"], 0.4)):
        c = torch.tensor(CODEBOOK[bits], device="cuda")
        c = torch.cat([-c.flip(0), c])
        border = (c[1:] + c[:-1]) / 2
        code = torch.bucketize(normal(n_pages, heads, page, p), border, out_int32=True, right=True)
        s[side + "_pages"] = _pack(code, bits)
        del code
        s[side + "_scales"] = math.sqrt(dim) * torch.exp(spread * normal(n_pages, heads, page))
    firsts = table[pages > 0, 0].long()
    s["k_scales"][firsts, :, 0] *= 2.0
    s["v_scales"][firsts, :, 0] *= 0.1
    s["signs"] = (torch.randint(0, 2, (heads, p), generator=gen, device="cuda") * 2 - 1).to(torch.int8)
    if case["kind"] == "attend":
        s["lengths"] = held.to(torch.int32)
        s["q"] = (1.5 * normal(n, heads * case["group"], dim)).to(dtype)
    else:
        zero = torch.zeros(1, dtype=torch.int64, device="cuda")
        s["starts"] = held.to(torch.int32)
        s["cu"] = torch.cat([zero, new.cumsum(0)]).to(torch.int32)
        count = int(new.sum())
        # keys with a few strong channels, as models have them
        strong = torch.ones(heads, dim, device="cuda")
        strong.scatter_(1, torch.randint(0, dim, (heads, 3), generator=gen, device="cuda"), 6.0)
        s["k"] = (normal(count, heads, dim) * strong).to(dtype)
        s["v"] = normal(count, heads, dim).to(dtype)
        if case["history"]:
            s["from"] = torch.zeros(n, dtype=torch.int32, device="cuda")
            s["cu_out"] = torch.cat([zero, total.cumsum(0)]).to(torch.int32)
            s["count_out"] = int(total.sum())
        else:
            s["from"], s["cu_out"], s["count_out"] = s["starts"], s["cu"], count
    if own:
        from adaptq_b200 import PagedKVCache
        s["cache"] = PagedKVCache.over(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], dim, case["k_bits"], case["v_bits"],
                                       signs=s["signs"])
    return s


# ---------------------------------------------------------------------------
# the operators in plain form
# ---------------------------------------------------------------------------
def _hadamard(p, dtype):
    """Entry (i, j) is -1 to the number of bits that i and j share."""
    i = torch.arange(p, device="cuda")
    both = i[:, None] & i[None, :]
    ones = sum((both >> b) & 1 for b in range(p.bit_length()))
    return (1 - 2 * (ones & 1)).to(dtype)


def _rotate(x, positions, s, sign=1.0):
    """x [tokens, heads, dim] in 32 bits, rotated by its positions (by their negatives for the gradient)."""
    case = s["case"]
    d = case["rotary_dim"]
    angle = positions.to(torch.float64)[:, None] * s["inv_freq"]
    c = (s["factor"] * torch.cos(angle)).to(torch.float32)[:, None, :]
    t = (s["factor"] * sign * torch.sin(angle)).to(torch.float32)[:, None, :]
    y = x.clone()
    if case["rotary"] == "half":
        a, b = x[..., : d // 2], x[..., d // 2: d]
        y[..., : d // 2], y[..., d // 2: d] = a * c - b * t, b * c + a * t
    else:
        a, b = x[..., 0:d:2], x[..., 1:d:2]
        y[..., 0:d:2], y[..., 1:d:2] = a * c - b * t, b * c + a * t
    return y


def _unpack(rows, bits):
    """[..., bytes] -> [..., P] codes"""
    if bits == 3:
        b = rows.view(*rows.shape[:-1], -1, 3).to(torch.int32)
        word = (b[..., 0] << 16) | (b[..., 1] << 8) | b[..., 2]
        return ((word[..., None] >> torch.arange(21, -1, -3, device="cuda", dtype=torch.int32)) & 7).flatten(-2)
    shift = torch.arange(8 - bits, -1, -bits, device="cuda", dtype=torch.int32)
    return ((rows[..., None].to(torch.int32) >> shift) & (2 ** bits - 1)).flatten(-2)


def _levels(bits):
    c = torch.tensor(CODEBOOK[bits], device="cuda", dtype=torch.float64)
    return torch.cat([-c.flip(0), c])


def _where(positions, owner, s):
    """Page and place in it of tokens at `positions` of the sequences `owner`."""
    page = s["case"]["page"]
    return s["table"][owner, positions // page].long(), positions % page


def _tokens(starts, cu, count):
    """Sequence and position of each of `count` tokens."""
    i = torch.arange(count, device="cuda")
    owner = torch.searchsorted(cu[1:].long(), i, right=True)
    return owner, starts[owner].long() + i - cu[owner].long()


def _append(s):
    case = s["case"]
    dim, p, count = case["dim"], _padded(case["dim"]), s["k"].shape[0]
    owner, pos = _tokens(s["starts"], s["cu"], count)
    at, place = _where(pos, owner, s)
    for side, bits in (("k", case["k_bits"]), ("v", case["v_bits"])):
        x = s[side].float()
        if side == "k" and case["rotary"] != "none":
            x = _rotate(x, pos, s)
        # 64 bits from here: the codes are decided by values next to a border
        x = x.double()
        norm = torch.sqrt(x.square().sum(-1) + 1e-12)
        full = torch.zeros(*x.shape[:-1], p, dtype=torch.float64, device="cuda")
        full[..., :dim] = x
        # sums first: sums of 16-bit values that are zero stay zero, which is a border
        u = ((full * s["signs"]) @ _hadamard(p, torch.float64)) / norm[..., None]
        level = _levels(bits)
        code = torch.bucketize(u, (level[1:] + level[:-1]) / 2, right=True, out_int32=True)
        s[side + "_pages"][at, :, place] = _pack(code, bits)
        s[side + "_scales"][at, :, place] = norm.float()


def _read(s):
    case = s["case"]
    dim, p = case["dim"], _padded(case["dim"])
    owner, pos = _tokens(s["from"], s["cu_out"], s["count_out"])
    at, place = _where(pos, owner, s)
    out = []
    for side, bits in (("k", case["k_bits"]), ("v", case["v_bits"])):
        c = _levels(bits).float()[_unpack(s[side + "_pages"][at, :, place], bits)]
        y = (c @ _hadamard(p, torch.float32)) * s["signs"] * (s[side + "_scales"][at, :, place][..., None] / p)
        out.append(y[..., :dim].to(_read_dtype(case)))
    return out


def _attend(s):
    case = s["case"]
    dim, p, heads, group, page = case["dim"], _padded(case["dim"]), case["kv_heads"], case["group"], case["page"]
    q, n = s["q"].float(), s["q"].shape[0]
    lengths = s["lengths"].long()
    if case["rotary"] != "none":
        q = _rotate(q, (lengths - 1).clamp(min=0), s)
    h = _hadamard(p, torch.float32)
    full = torch.zeros(n, heads, group, p, device="cuda")
    full[..., :dim] = q.view(n, heads, group, dim)
    z = (full * s["signs"][None, :, None, :]) @ h
    pages = s["table"].clamp(min=0).long()
    rows = lambda t: t[pages].transpose(2, 3).reshape(n, pages.shape[1] * page, heads, -1)  # noqa: E731
    level = lambda bits: _levels(bits).float()  # noqa: E731
    inside = torch.arange(pages.shape[1] * page, device="cuda")[None, :] < lengths[:, None]
    k = level(case["k_bits"])[_unpack(rows(s["k_pages"]), case["k_bits"])]
    score = torch.einsum("nhgp,nthp->nhgt", z, k) * (rows(s["k_scales"][..., None])[..., 0].transpose(1, 2) / (p * math.sqrt(dim)))[:, :, None]
    del k
    score = score.masked_fill(~inside[:, None, None, :], -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    weight = e / e.sum(-1, keepdim=True).clamp(min=1e-38)
    v = level(case["v_bits"])[_unpack(rows(s["v_pages"]), case["v_bits"])]
    vs = rows(s["v_scales"][..., None])[..., 0].transpose(1, 2)[:, :, None]
    acc = torch.einsum("nhgt,nthp->nhgp", weight * vs, v)
    out = (acc @ h) * s["signs"][None, :, None, :] / p
    return out[..., :dim].reshape(n, heads * group, dim).to(DTYPE[case["dtype"]])


def run(s):
    kind = s["case"]["kind"]
    if own:
        if kind == "rotary":
            y = s["rotary"](s["x"], s["positions"])
            return (y.detach(), torch.autograd.grad(y, s["x"], s["grad"])[0]) if s["case"]["gradient"] else y
        if kind == "attend":
            return s["cache"].attend(s["q"], s["table"], s["lengths"], rotary=s["rotary"])
        s["cache"].append(s["k"], s["v"], s["table"], s["starts"], s["cu"], rotary=s["rotary"])
        return s["cache"].read(s["table"], s["from"], s["cu_out"], s["count_out"], dtype=_read_dtype(s["case"]))
    with torch.no_grad():
        if kind == "rotary":
            y = _rotate(s["x"].float(), s["positions"], s).to(s["x"].dtype)
            return (y, _rotate(s["grad"].float(), s["positions"], s, -1.0).to(s["x"].dtype)) if s["case"]["gradient"] else y
        if kind == "attend":
            return _attend(s)
        _append(s)
        return _read(s)


# ---------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    dim, p = case["dim"], _padded(case["dim"])
    if case["kind"] == "rotary":
        one = case["tokens"] * case["heads"] * dim
        passes = 2 if case["gradient"] else 1
        return {"bytes": passes * (2 * one * size + 4 * case["tokens"]), "flops": passes * 3 * case["tokens"] * case["heads"] * case["rotary_dim"]}
    row = p * (case["k_bits"] + case["v_bits"]) // 8 + 8
    heads, n = case["kv_heads"], case["seqs"]
    stages = p.bit_length() - 1
    if case["kind"] == "attend":
        tokens = sum(_sizes(n, case["longest"], case["spread"]))
        queries = n * heads * case["group"]
        return {"bytes": tokens * heads * row + 2 * queries * dim * size + 4 * tokens / case["page"],
                "flops": tokens * heads * case["group"] * 4 * p + queries * 2 * stages * p}
    new = sum(_sizes(n, case["new"], case["spread"])) if case["new"] > 1 else n
    out = new + sum(_sizes(n, case["past"], case["spread"])) if case["history"] and case["past"] else new
    return {"bytes": new * heads * (2 * dim * size + row) + out * heads * (2 * dim * 2 + row),
            "flops": (new + out) * heads * 2 * p * (stages + 3)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _transform64(x):
    """Walsh-Hadamard transform of the last axis, by butterflies."""
    p, step = x.shape[-1], 1
    while step < p:
        x = x.unflatten(-1, (-1, 2, step))
        a, b = x[..., 0, :], x[..., 1, :]
        x = torch.stack([a + b, a - b], -2).flatten(-3)
        step *= 2
    return x


def _turn64(x, positions, s, back=False):
    """The rotation as a product of complex numbers."""
    d, half = s["case"]["rotary_dim"], s["case"]["rotary"] == "half"
    x = x.double()
    phase = torch.outer(positions.double(), s["inv_freq"])
    turn = torch.polar(torch.full_like(phase, s["factor"]), -phase if back else phase)[:, None]
    part = x[..., :d]
    pairs = part.unflatten(-1, (2, d // 2)).transpose(-1, -2) if half else part.unflatten(-1, (d // 2, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z.transpose(-1, -2).flatten(-2) if half else z.flatten(-2)
    return torch.cat([z, x[..., d:]], -1)


def _rows64(s, side, bits, seq, count, first=0):
    """[count, heads, P] levels and [count, heads] norms of one sequence's tokens from `first` on."""
    page = s["case"]["page"]
    t = torch.arange(first, first + count, device="cuda")
    at, place = s["table"][seq].long()[t // page], t % page
    rows = s[side + "_pages"][at, :, place].long()
    p = _padded(s["case"]["dim"])
    bit = torch.arange(p, device="cuda")[:, None] * bits + torch.arange(bits, device="cuda")
    ones = (rows[..., (bit // 8).flatten()] >> (7 - bit % 8).flatten()) & 1
    code = (ones.unflatten(-1, (p, bits)) << torch.arange(bits - 1, -1, -1, device="cuda")).sum(-1)
    magnitude = torch.tensor(CODEBOOK[bits], dtype=torch.float64, device="cuda")
    top = 2 ** (bits - 1)
    level = torch.where(code >= top, magnitude[(code - top).clamp(min=0)], -magnitude[(top - 1 - code).clamp(min=0)])
    return level, s[side + "_scales"][at, :, place].double()


def exact(case, seed):
    s = prepare(case, seed)
    dim, kind = case["dim"], case["kind"]
    if kind == "rotary":
        x = s["x"].detach()
        y = _turn64(x, s["positions"], s)
        return (y, _turn64(s["grad"], s["positions"], s, back=True)) if case["gradient"] else y
    p, heads, n = _padded(dim), case["kv_heads"], case["seqs"]
    sign = s["signs"].double()
    if kind == "attend":
        out = torch.zeros(n, heads, case["group"], dim, dtype=torch.float64, device="cuda")
        lengths = s["lengths"].tolist()
        for b, length in enumerate(lengths):
            if length == 0:
                continue
            q = s["q"][b: b + 1].double()
            if case["rotary"] != "none":
                q = _turn64(q, s["lengths"][b: b + 1] - 1, s)
            z = torch.nn.functional.pad(q.view(heads, case["group"], dim), (0, p - dim)) * sign[:, None]
            z = _transform64(z) / (p * math.sqrt(dim))
            top = torch.full((heads, case["group"], 1), -math.inf, dtype=torch.float64, device="cuda")
            mass, acc = torch.zeros_like(top), torch.zeros(heads, case["group"], p, dtype=torch.float64, device="cuda")
            for first in range(0, length, 16384):
                count = min(16384, length - first)
                k, ks = _rows64(s, "k", case["k_bits"], b, count, first)
                logit = (z @ k.permute(1, 2, 0)) * ks.T[:, None]
                above = torch.maximum(top, logit.amax(-1, keepdim=True))
                w, old = torch.exp(logit - above), torch.exp(top - above)
                v, vs = _rows64(s, "v", case["v_bits"], b, count, first)
                mass, acc, top = mass * old + w.sum(-1, keepdim=True), acc * old + (w * vs.T[:, None]) @ v.transpose(0, 1), above
            out[b] = (_transform64(acc / mass) * sign[:, None] / p)[..., :dim]
        return out.view(n, -1, dim)
    # append, then the rows that are read back
    found = {"k": [], "v": []}
    cu, starts, cu_out, first = (s[x].tolist() for x in ("cu", "starts", "cu_out", "from"))
    for b in range(n):
        new, many = cu[b + 1] - cu[b], cu_out[b + 1] - cu_out[b]
        for side, bits in (("k", case["k_bits"]), ("v", case["v_bits"])):
            x = s[side][cu[b]: cu[b + 1]].double()
            if side == "k" and case["rotary"] != "none":
                x = _turn64(x, torch.arange(starts[b], starts[b] + new, device="cuda"), s)
            norm = (x * x).sum(-1).add(1e-12).sqrt()
            u = _transform64(torch.nn.functional.pad(x, (0, p - dim)) * sign) / norm[..., None]
            magnitude = torch.tensor(CODEBOOK[bits], dtype=torch.float64, device="cuda")
            size = magnitude[sum((u.abs() > (a + c) / 2).long() for a, c in zip(CODEBOOK[bits], CODEBOOK[bits][1:]))]
            level = torch.where(u >= 0, size, -size)
            if many > new:
                old, held = _rows64(s, side, bits, b, many - new, first[b])
                level, norm = torch.cat([old, level]), torch.cat([held, norm])
            found[side].append((_transform64(level) * sign * (norm[..., None] / p))[..., :dim])
    return [torch.cat(found["k"]), torch.cat(found["v"])]
