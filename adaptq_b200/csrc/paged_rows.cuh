// Rows into the pages and out of them.
//
// One row of P coordinates is held by P/32 lanes, 32 consecutive coordinates each: five of the
// log2 P butterfly stages stay inside a lane, the others are shuffles, and a lane's codes are a
// whole number of words (4, 3 or 2).
#pragma once
#include "paged.cuh"

namespace aq {

constexpr int ROWS_THREADS = 256;
template <int P> constexpr int rows_per_block = ROWS_THREADS / (P / 32);

struct RowsLaunch {
  PagedView c;
  RotaryView r;
  TableView table;
  const int *starts, *cu;
  int start_bias, n_seqs;
  long long n_tokens;
  // the model's rows: keys and values (read by the append, written by the read-back)
  void *k, *v;
  long long k_token, k_head, v_token, v_head;
  int type, k_vec, v_vec; // vec: rows 16-byte aligned, dim a multiple of 8
};

struct TokenPlace { int page, off; long long pos; }; // page < 0: nowhere

// Places of the tokens that this block's rows belong to.
template <int P> __device__ __forceinline__ void find_places(const RowsLaunch &a, long long t0, int nt, TokenPlace *place) {
  for (int i = threadIdx.x; i < nt; i += ROWS_THREADS) {
    const long long t = t0 + i;
    const int b = a.cu ? owner_of(a.cu, a.n_seqs, t) : (t < a.n_seqs ? (int)t : -1);
    TokenPlace p{-1, 0, 0};
    if (b >= 0 && !(a.start_bias < 0 && a.starts[b] == 0)) { // a decode step leaves empty sequences out
      p.pos = (long long)a.starts[b] + a.start_bias + (a.cu ? t - a.cu[b] : 0);
      if (!find_slot(a.c, a.table.entries + b * a.table.stride, a.table.width, p.pos, p.page, p.off)) p.page = -1;
    }
    place[i] = p;
  }
}

// Walsh-Hadamard butterflies over a row: 32 values a lane, P/32 lanes.
template <int P> __device__ __forceinline__ void row_butterflies(float (&x)[32], int lane) {
#pragma unroll
  for (int len = 1; len < 32; len <<= 1) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (!(i & len)) {
        const float a = x[i], b = x[i + len];
        x[i] = a + b;
        x[i + len] = a - b;
      }
  }
#pragma unroll
  for (int m = 1; m < P / 32; m <<= 1) {
    const float sign = (lane & m) ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = fmaf(x[i], sign, __shfl_xor_sync(0xffffffffu, x[i], m));
  }
}

__device__ __forceinline__ void flip_signs(float (&x)[32], uint32_t word) {
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(__float_as_uint(x[i]) ^ ((word << (31 - i)) & 0x80000000u));
}

// 32 codes -> BITS words, most significant bits of each byte first.
template <int BITS> __device__ __forceinline__ void pack_codes(const float (&u)[32], uint32_t (&w)[BITS]) {
  if constexpr (BITS == 3) {
    uint32_t r[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint32_t v = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) v |= (uint32_t)quantize_value<3>(u[8 * g + i]) << (21 - 3 * i);
      r[g] = __byte_perm(v, 0, 0x4012);
    }
    w[0] = r[0] | r[1] << 24;
    w[1] = r[1] >> 8 | r[2] << 16;
    w[2] = r[2] >> 16 | r[3] << 8;
  } else {
    constexpr int PER = 32 / BITS, IN_BYTE = 8 / BITS;
#pragma unroll
    for (int g = 0; g < BITS; ++g) {
      uint32_t v = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        v |= (uint32_t)quantize_value<BITS>(u[PER * g + i]) << (8 * (i / IN_BYTE) + 8 - BITS * (1 + i % IN_BYTE));
      w[g] = v;
    }
  }
}

template <int BITS> __device__ __forceinline__ int code_at(const uint32_t (&w)[BITS], int i) {
  if constexpr (BITS == 3) { // bits 3i, 3i+1, 3i+2 of the row, bytes in memory order
    const int g = i >> 3, at = 24 * g; // group of three bytes
    const uint32_t lo = w[at >> 5] >> (at & 31), hi = (at & 31) ? w[min(2, (at >> 5) + 1)] << (32 - (at & 31)) : 0;
    const uint32_t v = __byte_perm((at & 31) ? lo | hi : lo, 0, 0x4012);
    return (v >> (21 - 3 * (i & 7))) & 7;
  } else {
    constexpr int PER = 32 / BITS, IN_BYTE = 8 / BITS;
    const int j = i % PER;
    return (w[i / PER] >> (8 * (j / IN_BYTE) + 8 - BITS * (1 + j % IN_BYTE))) & ((1 << BITS) - 1);
  }
}

template <int BITS> __device__ __forceinline__ void store_words(uint8_t *p, const uint32_t (&w)[BITS]) {
  if constexpr (BITS == 4) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (BITS == 2) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
  else {
#pragma unroll
    for (int i = 0; i < 3; ++i) reinterpret_cast<uint32_t *>(p)[i] = w[i];
  }
}
template <int BITS> __device__ __forceinline__ void load_words(const uint8_t *p, uint32_t (&w)[BITS]) {
  if constexpr (BITS == 4) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (BITS == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
  }
}

template <int P, int BITS>
__device__ __forceinline__ void append_rows(const RowsLaunch &a, const void *src, long long src_token, long long src_head,
                                            bool vec, uint8_t *pages, float *scales, bool rotate, float2 *turns,
                                            TokenPlace *place) {
  constexpr int LANES = P / 32, ROWS = rows_per_block<P>;
  const int heads = a.c.heads, dim = a.c.dim, half = a.r.dim >> 1;
  const long long n_rows = a.n_tokens * heads, r0 = (long long)blockIdx.x * ROWS;
  const long long t0 = r0 / heads;
  const int nt = (int)(min(n_rows - 1, r0 + ROWS - 1) / heads - t0) + 1;
  const int lane = threadIdx.x & 31, part = lane % LANES, d0 = part * 32;
  long long row = r0 + threadIdx.x / LANES;
  const bool live = row < n_rows;
  if (!live) row = n_rows - 1;
  const long long t = row / heads;
  const int h = (int)(row - t * heads);
  const long long at = t * src_token + h * src_head;

  float x[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = 0.f;
  if (vec) {
#pragma unroll
    for (int i = 0; i < 32; i += 8)
      if (d0 + i < dim) load_eight(src, at + d0 + i, a.type, x + i);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (d0 + i < dim) x[i] = load_one(src, at + d0 + i, a.type);
  }
  const uint32_t signs = a.c.signs[h * LANES + part];

  find_places<P>(a, t0, nt, place);
  __syncthreads();
  if (rotate) {
    for (int i = threadIdx.x; i < nt * half; i += ROWS_THREADS) turns[i] = rotary_turn(a.r, i % half, place[i / half].pos);
    __syncthreads();
    const float2 *cs = turns + (int)(t - t0) * half;
    if (a.r.interleaved) {
#pragma unroll
      for (int i = 0; i < 32; i += 2)
        if (d0 + i < a.r.dim) {
          const float2 k = cs[(d0 + i) >> 1];
          const float u = x[i], v = x[i + 1];
          x[i] = rotary_first(u, v, k);
          x[i + 1] = rotary_second(v, u, k);
        }
    } else {
      // the partner of coordinate i is i +- half: in another lane's same place where half is a
      // multiple of 32, else fetched again (from L1)
      const bool shuffle = (half & 31) == 0;
      const int m = half >> 5, from = part < m ? part + m : part < 2 * m ? part - m : part;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const int d = d0 + i;
        const bool first = d < half, in = d < a.r.dim;
        float other = 0.f;
        if (shuffle) other = __shfl_sync(0xffffffffu, x[i], (lane & ~(LANES - 1)) + from);
        else if (in) other = load_one(src, at + (first ? d + half : d - half), a.type);
        if (in) {
          const float2 k = cs[first ? d : d - half];
          x[i] = first ? rotary_first(x[i], other, k) : rotary_second(x[i], other, k);
        }
      }
    }
  }

  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
  for (int m = 1; m < LANES; m <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  const float norm = sqrtf(sum + 1e-12f), inv = 1.f / norm;
  // the transform first, the norm after it: sums of 16-bit values that are zero (a threshold) stay zero
  flip_signs(x, signs);
  row_butterflies<P>(x, lane);
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] *= inv;
  uint32_t w[BITS];
  pack_codes<BITS>(x, w);

  const TokenPlace p = place[(int)(t - t0)];
  if (live && p.page >= 0) {
    const long long slot = (((long long)p.page * heads + h) << a.c.page_shift) + p.off;
    store_words<BITS>(pages + slot * (P * BITS / 8) + part * (4 * BITS), w);
    if (part == 0) scales[slot] = norm;
  }
}

// blockIdx.y: 0 = keys, 1 = values
template <int P, int KB, int VB> __global__ void __launch_bounds__(ROWS_THREADS) paged_append_kernel(const RowsLaunch a) {
  __shared__ float2 turns[rows_per_block<P> * P / 2];
  __shared__ TokenPlace place[rows_per_block<P>];
  if (blockIdx.y == 0)
    append_rows<P, KB>(a, a.k, a.k_token, a.k_head, a.k_vec, a.c.k_pages, a.c.k_scales, a.r.dim > 0, turns, place);
  else
    append_rows<P, VB>(a, a.v, a.v_token, a.v_head, a.v_vec, a.c.v_pages, a.c.v_scales, false, turns, place);
}

template <int P, int BITS>
__device__ __forceinline__ void read_rows(const RowsLaunch &a, void *dst, long long dst_token, long long dst_head, bool vec,
                                          const uint8_t *pages, const float *scales, float (*level)[32], TokenPlace *place) {
  constexpr int LANES = P / 32, ROWS = rows_per_block<P>;
  const int heads = a.c.heads, dim = a.c.dim;
  const long long n_rows = a.n_tokens * heads, r0 = (long long)blockIdx.x * ROWS;
  const long long t0 = r0 / heads;
  const int nt = (int)(min(n_rows - 1, r0 + ROWS - 1) / heads - t0) + 1;
  const int lane = threadIdx.x & 31, part = lane % LANES, d0 = part * 32;
  long long row = r0 + threadIdx.x / LANES;
  const bool live = row < n_rows;
  if (!live) row = n_rows - 1;
  const long long t = row / heads;
  const int h = (int)(row - t * heads);
  // a copy of the codebook for every lane: 32 reads of any codes hit 32 banks
  for (int i = threadIdx.x; i < (32 << BITS); i += ROWS_THREADS) level[i >> 5][i & 31] = c_cb[BITS - 2][i >> 5];
  find_places<P>(a, t0, nt, place);
  __syncthreads();
  const TokenPlace p = place[(int)(t - t0)];
  const bool found = p.page >= 0;
  uint32_t w[BITS] = {};
  float norm = 0.f;
  if (found) {
    const long long slot = (((long long)p.page * heads + h) << a.c.page_shift) + p.off;
    load_words<BITS>(pages + slot * (P * BITS / 8) + part * (4 * BITS), w);
    norm = scales[slot];
  }
  const uint32_t signs = a.c.signs[h * LANES + part];
  float x[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = level[code_at<BITS>(w, i)][lane];
  row_butterflies<P>(x, lane);
  flip_signs(x, signs);
  const float scale = norm * (1.f / P);
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] *= scale;
  if (!live || !found) return;
  const long long at = t * dst_token + h * dst_head;
  if (vec) {
#pragma unroll
    for (int i = 0; i < 32; i += 8)
      if (d0 + i < dim) store_eight(dst, at + d0 + i, a.type, x + i);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (d0 + i < dim) store_one(dst, at + d0 + i, a.type, x[i]);
  }
}

template <int P, int KB, int VB> __global__ void __launch_bounds__(ROWS_THREADS) paged_read_kernel(const RowsLaunch a) {
  __shared__ float level[16][32];
  __shared__ TokenPlace place[rows_per_block<P>];
  if (blockIdx.y == 0)
    read_rows<P, KB>(a, a.k, a.k_token, a.k_head, a.k_vec, a.c.k_pages, a.c.k_scales, level, place);
  else
    read_rows<P, VB>(a, a.v, a.v_token, a.v_head, a.v_vec, a.c.v_pages, a.c.v_scales, level, place);
}

} // namespace aq
