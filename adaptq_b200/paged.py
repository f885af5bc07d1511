"""PagedKVCache: the quantised cache in pages (include/adaptq_paged.h).

Sequences of different lengths share one pool of pages; a sequence is a row of a block table
(page numbers) and a length, both int32 CUDA tensors that the caller keeps.  No call waits,
copies to the host or keeps anything from one call for the next, so every one of them can be
captured into a CUDA graph, and calls on several streams need no more than the pages they share
ordered.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

from . import _lib
from .rotary import TYPES, Rotary, check_written, current_stream, increment_version

_STATUS = ((1, "a block table names a page outside the pool"), (2, "a position or length has no room in its block table"),
           (256, "a device-side index check failed (checked build), the access was skipped"))


def _padded(dim: int) -> int:
    return max(64, 1 << (dim - 1).bit_length())


class PagedKVCache:
    """n_pages pages of page_size tokens, for n_kv_heads heads of `dim` coordinates (33 to 256), keys at k_bits and values
    at v_bits (2, 3 or 4).  `seed` gives the heads the signs of MHAContext(seed=seed); `signs` ([heads, padded] of +1 and
    -1) sets them instead.  One object holds one layer; the layers of a model share the block tables.

    The tensors are public: k_pages, v_pages (uint8 [n_pages, heads, page_size, padded * bits / 8]), k_scales, v_scales
    (float32 [n_pages, heads, page_size])."""

    def __init__(self, n_pages: int, n_kv_heads: int, dim: int, k_bits: int = 4, v_bits: int = 4, page_size: int = 64,
                 seed: int = 42, device=None, signs=None):
        self._check_sizes(n_pages, n_kv_heads, dim, k_bits, v_bits, page_size)
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ValueError(f"PagedKVCache needs a CUDA device, got {device}")
        p = _padded(dim)
        rows = lambda bits: torch.zeros(n_pages, n_kv_heads, page_size, p * bits // 8, dtype=torch.uint8, device=device)  # noqa: E731
        scales = lambda: torch.zeros(n_pages, n_kv_heads, page_size, dtype=torch.float32, device=device)  # noqa: E731
        self._set(rows(k_bits), rows(v_bits), scales(), scales(), dim, k_bits, v_bits, seed, signs)

    @classmethod
    def over(cls, k_pages, v_pages, k_scales, v_scales, dim: int, k_bits: int, v_bits: int, seed: int = 42, signs=None):
        """A cache over tensors that the caller owns (shapes and types as above, contiguous)."""
        self = cls.__new__(cls)
        if k_pages.dim() != 4:
            raise ValueError("k_pages must be (n_pages, heads, page_size, row bytes)")
        cls._check_sizes(*k_pages.shape[:2], dim, k_bits, v_bits, k_pages.shape[2])
        p = _padded(dim)
        for name, t, last, dtype in (("k_pages", k_pages, (p * k_bits // 8,), torch.uint8), ("v_pages", v_pages, (p * v_bits // 8,), torch.uint8),
                                     ("k_scales", k_scales, (), torch.float32), ("v_scales", v_scales, (), torch.float32)):
            want = tuple(k_pages.shape[:3]) + last
            if tuple(t.shape) != want or t.dtype != dtype or not t.is_contiguous() or t.device != k_pages.device:
                raise ValueError(f"{name} must be contiguous {want} {dtype} on {k_pages.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
        if k_pages.device.type != "cuda":
            raise ValueError(f"PagedKVCache needs a CUDA device, got {k_pages.device}")
        self._set(k_pages, v_pages, k_scales, v_scales, dim, k_bits, v_bits, seed, signs)
        return self

    @staticmethod
    def _check_sizes(n_pages, n_kv_heads, dim, k_bits, v_bits, page_size):
        if n_pages <= 0 or n_kv_heads <= 0:
            raise ValueError("n_pages and n_kv_heads must be positive")
        if not 33 <= dim <= 256:
            raise ValueError(f"head dimensions from 33 to 256 are supported, got {dim}")
        if k_bits not in (2, 3, 4) or v_bits not in (2, 3, 4):
            raise ValueError(f"k_bits and v_bits must be 2, 3 or 4, got {k_bits} and {v_bits}")
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError(f"page_size must be 16, 32, 64, 128 or 256, got {page_size}")

    def _set(self, k_pages, v_pages, k_scales, v_scales, dim, k_bits, v_bits, seed, signs):
        self._L = _lib.load()
        self.k_pages, self.v_pages, self.k_scales, self.v_scales = k_pages, v_pages, k_scales, v_scales
        self.n_pages, self.n_kv_heads, self.page_size = (int(s) for s in k_pages.shape[:3])
        self.dim, self.padded, self.k_bits, self.v_bits = int(dim), _padded(dim), int(k_bits), int(v_bits)
        self.device = k_pages.device
        self._index = self.device.index
        words = self.padded // 32
        if signs is None:
            host = torch.zeros(self.n_kv_heads, words, dtype=torch.int32)
            if self._L.adaptq_paged_signs(C.c_uint64(int(seed) & (2**64 - 1)), self.n_kv_heads, self.dim, host.data_ptr()):
                raise RuntimeError(_lib.last_error())
        else:
            s = torch.as_tensor(signs).cpu().numpy()
            if s.shape != (self.n_kv_heads, self.padded) or not (np.abs(s) == 1).all():
                raise ValueError(f"signs must be ({self.n_kv_heads}, {self.padded}) of +1 and -1")
            host = torch.from_numpy(np.packbits(s < 0, axis=1, bitorder="little").view(np.int32))
        self._signs = host.to(self.device)
        self._status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._desc = _lib.Paged(k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                                self._signs.data_ptr(), self._status.data_ptr(), self.n_pages, self.n_kv_heads, self.page_size,
                                self.dim, self.k_bits, self.v_bits, self.device.index)
        self._ref = C.addressof(self._desc)
        self._scale = self.dim ** -0.5
        self._sizes = {}  # bytes of attend's workspace by (sequences, query heads, type)

    # -- arguments ------------------------------------------------------------------------
    def _ints(self, name, t, n):
        if t.dtype is not torch.int32 or t.dim() != 1 or len(t) != n or t.get_device() != self._index:
            raise ValueError(f"{name} must be ({n},) int32 on {self.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
        return t if t.is_contiguous() else t.contiguous()

    def _table(self, t):
        if t.dtype is not torch.int32 or t.dim() != 2 or t.shape[1] == 0 or t.get_device() != self._index:
            raise ValueError(f"block_table must be (sequences, pages > 0) int32 on {self.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
        return t if t.is_contiguous() or t.stride(1) == 1 else t.contiguous()

    def _rows(self, name, t, heads):
        if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != self.dim or t.dtype not in TYPES or t.get_device() != self._index:
            raise ValueError(f"{name} must be (n, {heads}, {self.dim}) float32, float16 or bfloat16 on {self.device}, got {tuple(t.shape)} "
                             f"{t.dtype} on {t.device}")

    def _rotary(self, rotary):
        if rotary is None:
            return None
        if not isinstance(rotary, Rotary) or rotary._index != self._index or rotary.dim > self.dim:
            raise ValueError(f"rotary must be a Rotary of at most {self.dim} coordinates on {self.device}")
        return rotary._ref

    # -- operators ------------------------------------------------------------------------
    def append(self, k, v, block_table, starts, cu_tokens=None, rotary=None):
        """Store tokens.  k, v: (n, heads, dim); block_table (sequences, pages); starts (sequences,): how many tokens each
        sequence holds already, that is the position of its first new one.  cu_tokens (sequences + 1,): sequence b brings
        the rows cu_tokens[b] to cu_tokens[b+1] - 1, rows outside (padding) are left out; without it every sequence brings
        one row.  Keys are rotated by their positions first, if `rotary`.  The pages must be in the block table; a page that
        is written must belong to one sequence."""
        self._append(k, v, block_table, starts, 0, cu_tokens, rotary)

    def _append(self, k, v, block_table, starts, bias, cu_tokens, rotary):
        self._rows("k", k, self.n_kv_heads)
        self._rows("v", v, self.n_kv_heads)
        if k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError(f"k and v must have one shape and type, got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
        k = k if k.stride(2) == 1 else k.contiguous()
        v = v if v.stride(2) == 1 else v.contiguous()
        table = self._table(block_table)
        n_seqs, n = table.shape[0], k.shape[0]
        starts = self._ints("starts", starts, n_seqs)
        if cu_tokens is not None:
            cu_tokens = self._ints("cu_tokens", cu_tokens, n_seqs + 1)
        elif n != n_seqs:
            raise ValueError(f"{n} rows for {n_seqs} sequences: without cu_tokens every sequence brings one")
        ks, vs = k.stride(), v.stride()
        if self._L.adaptq_paged_append(self._ref, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], TYPES[k.dtype], table.data_ptr(),
                                       table.stride(0), table.shape[1], starts.data_ptr(), bias,
                                       None if cu_tokens is None else cu_tokens.data_ptr(), n_seqs, n, self._rotary(rotary), current_stream(self._index)):
            raise RuntimeError(_lib.last_error())

    def attend(self, q, block_table, lengths, rotary=None, scale=None, out=None):
        """Attention of one token per sequence over its first lengths[b] tokens.  q: (sequences, query heads, dim), query head
        j reading KV head j // (query heads / KV heads) -> the same shape and type.  Queries are rotated by position
        lengths[b] - 1 first, if `rotary`.  scale: 1/sqrt(dim) by default.  A sequence of length 0 gives zeros.  `out` may be
        q and is marked as modified; no gradient flows through."""
        return self._attend(*self._attend_arguments(q, block_table, lengths, rotary, scale, out))

    def _attend_arguments(self, q, block_table, lengths, rotary, scale, out):
        if q.dim() != 3 or q.shape[2] != self.dim or q.shape[1] % self.n_kv_heads or not q.shape[1] or q.dtype not in TYPES or q.get_device() != self._index:
            raise ValueError(f"q must be (sequences, a multiple of {self.n_kv_heads} heads, {self.dim}) float32, float16 or bfloat16 on {self.device}, "
                             f"got {tuple(q.shape)} {q.dtype} on {q.device}")
        q = q if q.stride(2) == 1 else q.contiguous()
        n, heads = q.shape[0], q.shape[1]
        table = self._table(block_table)
        if table.shape[0] != n:
            raise ValueError(f"block_table has {table.shape[0]} sequences, q {n}")
        lengths = self._ints("lengths", lengths, n)
        given = out is not None
        if not given:
            out = torch.empty((n, heads, self.dim), dtype=q.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(2) != 1:
            raise ValueError("out must have the shape, type and device of q and contiguous rows")
        else:
            check_written("out", out)
        scale = self._scale if scale is None else C.c_float(scale).value
        if not 0.0 < scale < math.inf:
            raise RuntimeError(f"scale must be positive and finite, got {scale}")
        return q, table, lengths, self._rotary(rotary), scale, out, given

    def _attend(self, q, table, lengths, rotary, scale, out, given):
        n, heads = q.shape[0], q.shape[1]
        kind = TYPES[q.dtype]
        size = self._sizes.get((n, heads, kind))
        if size is None:
            size = self._sizes[n, heads, kind] = self._L.adaptq_paged_attend_workspace(self._ref, n, heads, kind)
        # of this call alone: the allocator hands it on in the order of the stream, also inside a captured graph
        workspace = torch.empty(size, dtype=torch.uint8, device=self.device)
        qs, os = q.stride(), out.stride()
        if self._L.adaptq_paged_attend(self._ref, q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1], kind, table.data_ptr(),
                                       table.stride(0), table.shape[1], lengths.data_ptr(), n, heads,
                                       scale, rotary, workspace.data_ptr(), size, current_stream(self._index)):
            raise RuntimeError(_lib.last_error())
        if given:
            increment_version(out)
        return out

    def step(self, k, v, q, block_table, lengths, rotary=None, scale=None, out=None):
        """One decode step: the new token of every sequence enters as its last (position lengths[b] - 1: lengths count it),
        then its queries attend.  k, v (sequences, heads, dim), q as for attend; a sequence of length 0 takes no part.
        Arguments that are refused leave the cache as it was."""
        arguments = self._attend_arguments(q, block_table, lengths, rotary, scale, out)
        self._append(k, v, block_table, lengths, -1, None, rotary)
        return self._attend(*arguments)

    def read(self, block_table, starts, cu_tokens, total, dtype=torch.bfloat16, out=None):
        """Tokens back as rows: (k, v), each (total, heads, dim) of `dtype`, keys as stored (rotated).  Sequence b gives its
        positions from starts[b] on, to the rows cu_tokens[b] to cu_tokens[b+1] - 1; rows behind them stay as they were
        (with `out` = (k, v), else unspecified), as do rows whose page or position does not exist."""
        table = self._table(block_table)
        n_seqs = table.shape[0]
        starts, cu_tokens = self._ints("starts", starts, n_seqs), self._ints("cu_tokens", cu_tokens, n_seqs + 1)
        if out is None:
            if dtype not in TYPES:
                raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
            k = torch.empty(total, self.n_kv_heads, self.dim, dtype=dtype, device=self.device)
            v = torch.empty_like(k)
        else:
            k, v = out
            self._rows("out[0]", k, self.n_kv_heads)
            self._rows("out[1]", v, self.n_kv_heads)
            if k.shape[0] != total or v.shape != k.shape or v.dtype != k.dtype or k.stride(2) != 1 or v.stride(2) != 1:
                raise ValueError(f"out must be two tensors of {total} rows, of one type, with contiguous rows")
            check_written("out[0]", k)
            check_written("out[1]", v)
            if total and k.data_ptr() == v.data_ptr():
                raise ValueError("out must be two tensors, not one twice")
        ks, vs = k.stride(), v.stride()
        if self._L.adaptq_paged_read(self._ref, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], TYPES[k.dtype], table.data_ptr(),
                                     table.stride(0), table.shape[1], starts.data_ptr(), cu_tokens.data_ptr(), n_seqs, int(total), current_stream(self._index)):
            raise RuntimeError(_lib.last_error())
        if out is not None:
            increment_version((k, v))
        return k, v

    def check(self):
        """Wait for the device -- all of its streams -- and raise RuntimeError if a call since the last check named a page
        outside the pool, or a position or length without room in its block table (those entries were skipped).  Calls that
        other threads make meanwhile report here or at the next check.  Not while a stream is being captured."""
        torch.cuda.synchronize(self.device)
        taken = torch.empty(1, dtype=torch.int32, device=self.device)
        if self._L.adaptq_paged_take_status(self._ref, taken.data_ptr(), current_stream(self._index)):
            raise RuntimeError(_lib.last_error())
        status = int(taken)
        if status:
            raise RuntimeError("PagedKVCache: " + "; ".join(text for bit, text in _STATUS if status & bit))

    @property
    def kv_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_pages, self.v_pages, self.k_scales, self.v_scales))
