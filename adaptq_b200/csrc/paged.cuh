// What the kernels of the paged cache share: the pool's geometry, 16- and 32-bit rows in and
// out, rotary phases, and where a token lies.
#pragma once
#include "common.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace aq {

enum { TYPE_F32 = 0, TYPE_F16 = 1, TYPE_BF16 = 2 };
enum { PAGED_BAD_PAGE = 1, PAGED_BAD_POSITION = 2, PAGED_BAD_INDEX = 256 };

// Checked build: an index check in front of an access, which is skipped if it fails, as AQ_CHECK; it leaves a bit in
// the pool's status word.  The constant `true` otherwise.
#ifdef ADAPTQ_CHECKED
#define PAGED_CHECK(status_ptr, cond) ((cond) ? true : (atomicOr((status_ptr), PAGED_BAD_INDEX), false))
#else
#define PAGED_CHECK(status_ptr, cond) (true)
#endif

struct PagedView {
  uint8_t *k_pages, *v_pages;
  float *k_scales, *v_scales;
  const uint32_t *signs;
  int *status;
  long long n_pages;
  int heads, page_size, page_shift, dim;
};

struct RotaryView { // dim == 0: no rotation
  const unsigned long long *turns;
  float factor;
  int dim, interleaved;
};

struct TableView {
  const int *entries;
  long long stride;
  int width;
};

// cos and sin of position * w, times the factor.  The frequency is a 64-bit binary fraction of
// a turn, so the product modulo 2^64 is the phase modulo one turn, exact at every position.
// The nearest quarter turn is taken off in integers: of the eighth of a turn at most that is
// left, rounding to 24 bits takes 2e-8, and nothing that counts next to a zero of either.
__device__ __forceinline__ float2 rotary_turn(const RotaryView &r, int pair, long long pos) {
  const unsigned long long phase = (unsigned long long)pos * r.turns[pair];
  const unsigned quarter = (unsigned)((phase + (1ull << 61)) >> 62);
  float s, c;
  sincospif((float)(long long)(phase - ((unsigned long long)quarter << 62)) * 0x1p-63f, &s, &c); // in half turns, from -1/4 to 1/4
  const float x = (quarter & 1) ? -s : c, y = (quarter & 1) ? c : s;
  return (quarter & 2) ? make_float2(-x * r.factor, -y * r.factor) : make_float2(x * r.factor, y * r.factor);
}

// One element of a rotated pair: mine * cos -+ other * sin (minus for the pair's first element).  One order of
// rounding everywhere, so that a row does not depend on which kernel or layout rotates it.
__device__ __forceinline__ float rotary_first(float mine, float other, float2 k) { return __fmaf_rn(mine, k.x, -__fmul_rn(other, k.y)); }
__device__ __forceinline__ float rotary_second(float mine, float other, float2 k) { return __fmaf_rn(mine, k.x, __fmul_rn(other, k.y)); }

__device__ __forceinline__ float load_one(const void *p, long long i, int type) {
  if (type == TYPE_F32) return static_cast<const float *>(p)[i];
  if (type == TYPE_F16) return __half2float(static_cast<const __half *>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store_one(void *p, long long i, int type, float v) {
  if (type == TYPE_F32) static_cast<float *>(p)[i] = v;
  else if (type == TYPE_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ float2 unpack2(uint32_t w, int type) {
  if (type == TYPE_F16) { __half2 h; memcpy(&h, &w, 4); return __half22float2(h); }
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, int type) {
  uint32_t w;
  if (type == TYPE_F16) { const __half2 h = __floats2half2_rn(a, b); memcpy(&w, &h, 4); }
  else { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); memcpy(&w, &h, 4); }
  return w;
}

// Eight consecutive elements; the address is 16-byte aligned.
template <int TYPE> __device__ __forceinline__ void load_eight(const void *p, long long i, float *v) {
  if constexpr (TYPE == TYPE_F32) {
    const float4 a = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
    const float4 b = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack2(u[j], TYPE);
      v[2 * j] = f.x; v[2 * j + 1] = f.y;
    }
  }
}
template <int TYPE> __device__ __forceinline__ void store_eight(void *p, long long i, const float *v) {
  if constexpr (TYPE == TYPE_F32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(static_cast<float *>(p) + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + i) =
        make_uint4(pack2(v[0], v[1], TYPE), pack2(v[2], v[3], TYPE), pack2(v[4], v[5], TYPE), pack2(v[6], v[7], TYPE));
  }
}
// f(type as a constant): one branch in front of a loop instead of one in it.
template <int TYPE> struct TypeConstant { static constexpr int value = TYPE; };
template <typename F> __device__ __forceinline__ void with_type(int type, F f) {
  if (type == TYPE_BF16) f(TypeConstant<TYPE_BF16>());
  else if (type == TYPE_F16) f(TypeConstant<TYPE_F16>());
  else f(TypeConstant<TYPE_F32>());
}

// Rows of a side of the pool; `n` rows from `row` on lie in it.
__device__ __forceinline__ bool rows_exist(const PagedView &c, long long row, int n) {
  return row >= 0 && row + n <= (c.n_pages * c.heads) << c.page_shift;
}

// Page and place of position `pos` of a sequence whose table row is `row`; false (and a bit
// of the status) if the table or the pool has no such place.
__device__ __forceinline__ bool find_slot(const PagedView &c, const int *row, int width, long long pos, int &page, int &off) {
  if (pos < 0 || (pos >> c.page_shift) >= width) { atomicOr(c.status, PAGED_BAD_POSITION); return false; }
  page = row[pos >> c.page_shift];
  off = (int)(pos & (c.page_size - 1));
  if (page < 0 || page >= c.n_pages) { atomicOr(c.status, PAGED_BAD_PAGE); return false; }
  return true;
}

// The sequence of token t + lane for the whole warp: the last b with cu[b] <= it, or -1 if it lies before the first or
// behind the last.  The warp searches together for token t, 32 probes a step; the others follow from there.
__device__ __forceinline__ int owner_of(const int *cu, int n_seqs, long long t, int lane, int count) {
  int lo = 0, hi = n_seqs; // cu[lo] <= t < cu[hi] if any
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5, at = lo + (lane + 1) * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < hi && cu[at] <= t);
    const int n = __popc(below);
    hi = min(hi, lo + (n + 1) * step);
    lo += n * step;
  }
  if (lane >= count || cu[0] > t + lane || cu[n_seqs] <= t + lane) return -1;
  while (lo + 1 < n_seqs && cu[lo + 1] <= t + lane) ++lo;
  return lo;
}

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void store_32(void *p, const uint32_t (&v)[8]) { // 32 bytes, a whole sector
  asm volatile("st.global.v8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
               "r"(v[6]), "r"(v[7]), "l"(p)
               : "memory");
}
// A load from a table in shared memory that does not change once filled, so that it may move freely.
__device__ __forceinline__ uint32_t table_one(uint32_t at) {
  uint32_t v;
  asm("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}

// N packed bytes of a row -> words (bytes in memory order); the address is a multiple of the largest power of two in N.
template <int N> __device__ __forceinline__ void load_packed(const uint8_t *p, uint32_t *w) {
  if constexpr (N % 16 == 0) {
#pragma unroll
    for (int i = 0; i < N / 16; ++i) {
      const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  } else if constexpr (N % 8 == 0) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      const uint2 v = reinterpret_cast<const uint2 *>(p)[i];
      w[2 * i] = v.x; w[2 * i + 1] = v.y;
    }
  } else if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint32_t h = reinterpret_cast<const uint16_t *>(p)[i];
      if (i & 1) w[i >> 1] |= h << 16; else w[i >> 1] = h;
    }
  } else {
    w[0] = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) w[0] |= (uint32_t)p[i] << (8 * i);
  }
}
// Four fields of six bits -> the lower six bits of four bytes.
__device__ __forceinline__ uint32_t spread6(uint32_t v) {
  v += (v & 0xfff000u) * 15u;      // each half of twelve bits in sixteen
  return v + (v & 0x0fc00fc0u) * 3u; // each field in eight
}
// The g-th group of three bytes as a 24-bit number, first byte on top (3-bit rows).
template <int WORDS> __device__ __forceinline__ uint32_t group24(const uint32_t (&w)[WORDS], int g) {
  const int at = 3 * g, lo = at >> 2, o = at & 3;
  const uint32_t next = lo + 1 < WORDS ? w[lo + 1 < WORDS ? lo + 1 : 0] : 0;
  // bytes o, o+1, o+2 of (w[lo], next), reversed
  return __byte_perm(w[lo], next, (o + 2) | ((o + 1) << 4) | (o << 8) | (o << 12)) & 0xffffffu;
}

} // namespace aq
