"""The paged cache's operators in 64 bits, written from their definitions (torch, on whatever device the
inputs are on), and inputs for their tests."""
from __future__ import annotations

import math

import torch

MAGNITUDES = {2: [0.4528, 1.5104], 3: [0.2451, 0.7560, 1.3439, 2.1529],
              4: [0.1258, 0.3795, 0.6402, 0.9138, 1.2016, 1.5105, 1.8944, 2.4008]}


def padded(dim):
    p = 64
    while p < dim:
        p *= 2
    return p


def levels(bits):
    m = torch.tensor(MAGNITUDES[bits], dtype=torch.float64)
    return torch.cat([-m.flip(0), m])


def hadamard(p):
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < p:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)])
    return h


def unpack(rows, bits):
    """[..., bytes] -> [..., P] codes; the row read as one long number, most significant bit first."""
    bit = (rows[..., None].long() >> torch.arange(7, -1, -1, device=rows.device)) & 1
    bit = bit.flatten(-2).unflatten(-1, (-1, bits))
    return (bit << torch.arange(bits - 1, -1, -1, device=rows.device)).sum(-1)


def pack(code, bits):
    bit = (code[..., None].long() >> torch.arange(bits - 1, -1, -1, device=code.device)) & 1
    byte = bit.flatten(-2).unflatten(-1, (-1, 8)) << torch.arange(7, -1, -1, device=code.device)
    return byte.sum(-1).to(torch.uint8)


def rotate(x, positions, rotary, inverse=False):
    """x [T, H, D] float64"""
    d = rotary.dim
    w = rotary.inv_freq.to(x.device)
    a = positions.double()[:, None] * w
    c, s = (rotary.factor * a.cos())[:, None], (rotary.factor * a.sin())[:, None]
    if inverse:
        s = -s
    y = x.clone()
    i = torch.arange(0, d, 2) if rotary.interleaved else torch.arange(d // 2)
    j = i + 1 if rotary.interleaved else i + d // 2
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    return y


def coordinates(x, signs):
    """[..., H, dim] rows -> (H(sign * x) / norm, norm)"""
    p = signs.shape[1]
    full = torch.zeros(*x.shape[:-1], p, dtype=torch.float64, device=x.device)
    full[..., : x.shape[-1]] = x
    norm = (x * x).sum(-1).add(1e-12).sqrt()
    return (full * signs) @ hadamard(p).to(x.device) / norm[..., None], norm


def rows(cache, side, page_ids, places, signs):
    """Stored rows [T, H, dim] as the cache stands for them, and (codes' levels, norms)."""
    bits = cache.k_bits if side == "k" else cache.v_bits
    store = (cache.k_pages if side == "k" else cache.v_pages)[page_ids, :, places]
    norm = (cache.k_scales if side == "k" else cache.v_scales)[page_ids, :, places].double()
    level = levels(bits).to(store.device)[unpack(store, bits)]
    p = signs.shape[1]
    return (level @ hadamard(p).to(store.device) * signs * norm[..., None] / p)[..., : cache.dim], level, norm


def place(cache, table_row, n, first=0):
    t = torch.arange(first, first + n, device=table_row.device)
    return table_row[t // cache.page_size].long(), t % cache.page_size


def attend(cache, signs, q, table, lengths, rotary=None, scale=None):
    """[B, Hq, dim] float64; also how large logits and values are: (max |z.c| sums, sum w vs)."""
    p, dim = signs.shape[1], cache.dim
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    group = q.shape[1] // cache.n_kv_heads
    for b, n in enumerate(lengths.tolist()):
        if n <= 0:
            continue
        x = q[b: b + 1].double()
        if rotary is not None:
            x = rotate(x, torch.tensor([n - 1], device=q.device), rotary)
        at, off = place(cache, table[b], n)
        k, _, _ = rows(cache, "k", at, off, signs)
        v, _, _ = rows(cache, "v", at, off, signs)
        # keys and queries meet in the model's own coordinates only where dim == padded: use the rotated domain
        _, kl, kn = rows(cache, "k", at, off, signs)
        _, vl, vn = rows(cache, "v", at, off, signs)
        full = torch.zeros(cache.n_kv_heads, group, p, dtype=torch.float64, device=q.device)
        full[..., :dim] = x.view(cache.n_kv_heads, group, dim)
        h = hadamard(p).to(q.device)
        z = (full * signs[:, None]) @ h
        logit = torch.einsum("hgp,thp->hgt", z, kl) * kn.T[:, None] * scale / p
        w = torch.softmax(logit, -1)
        acc = torch.einsum("hgt,thp->hgp", w * vn.T[:, None], vl)
        out[b] = ((acc @ h) * signs[:, None] / p)[..., :dim].reshape(q.shape[1], dim)
    return out


def random_pool(cache, gen, dist="normal"):
    """Fill a cache with codes of normal coordinates and norms around sqrt(dim)."""
    for bits, store, scale in ((cache.k_bits, cache.k_pages, cache.k_scales), (cache.v_bits, cache.v_pages, cache.v_scales)):
        lv = levels(bits).to(store.device)
        u = torch.randn(*store.shape[:3], cache.padded, generator=gen, device=store.device, dtype=torch.float64)
        store.copy_(pack(torch.bucketize(u, (lv[1:] + lv[:-1]) / 2, right=True), bits))
        scale.copy_(math.sqrt(cache.dim) * torch.exp(0.3 * torch.randn(scale.shape, generator=gen, device=store.device)))


def random_table(cache, lengths, gen, extra=1):
    """A block table for sequences of these lengths: pages in random order, -1 behind them."""
    need = [-(-n // cache.page_size) for n in lengths]
    assert sum(need) <= cache.n_pages
    order = torch.randperm(cache.n_pages, generator=gen, device=cache.device).int()
    table = torch.full((len(lengths), max(need) + extra), -1, dtype=torch.int32, device=cache.device)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at: at + m]
        at += m
    return table


def random_signs(heads, p, gen):
    return (torch.randint(0, 2, (heads, p), generator=gen, device=gen.device) * 2 - 1)
