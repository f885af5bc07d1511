// Rotary positions: y = R(pos) x over the first coordinates of every head, the rest copied.
//
// Bound by memory: every element is read and written once, a turn costs a pair of elements
// four multiplications, and a turn's sine and cosine are formed once per token and shared by its
// heads.  16384 tokens x 32 heads x 128 in bf16: 46.4 us, 5.8 TB/s, 0.88 of the copy rate.
#pragma once
#include "paged.cuh"

namespace aq {

struct RotaryLaunch {
  RotaryView r;
  const void *x;
  void *y;
  const void *positions;
  long long x_token, x_head, y_token, y_head, n_tokens;
  int heads, dim, type, positions_64, inverse;
  int tokens_per_block, heads_per_block; // whose product with dim stays within 2^30: a block counts in 32 bits
  int vec; // rows are 16-byte aligned and whole eights, and so are the halves
};

constexpr int ROTARY_THREADS = 256;

#ifdef ADAPTQ_CHECKED
__device__ int rotary_status; // this kernel has no pool: adaptq_paged_take_status() adds its failed checks to the next one's
#endif

__global__ void __launch_bounds__(ROTARY_THREADS) rotary_kernel(const RotaryLaunch a) {
  extern __shared__ float2 rotary_turns[]; // [tokens_per_block][r.dim / 2]
  const int half = a.r.dim >> 1;
  const long long t0 = (long long)blockIdx.x * a.tokens_per_block;
  const int nt = (int)min((long long)a.tokens_per_block, a.n_tokens - t0);
  const int h0 = blockIdx.y * a.heads_per_block, heads = min(a.heads_per_block, a.heads - h0);
  for (int i = threadIdx.x; i < nt * half; i += ROTARY_THREADS) {
    const int t = i / half, pair = i - t * half;
    const long long pos = a.positions_64 ? static_cast<const long long *>(a.positions)[t0 + t]
                                         : (long long)static_cast<const int *>(a.positions)[t0 + t];
    float2 cs = rotary_turn(a.r, pair, pos);
    if (a.inverse) cs.y = -cs.y;
    if (PAGED_CHECK(&rotary_status, i >= 0 && i < a.tokens_per_block * half)) rotary_turns[i] = cs;
  }
  __syncthreads();
  if (a.vec) with_type(a.type, [&](auto type) {
    constexpr int TYPE = decltype(type)::value;
    // one thread: eight neighbours and, in the half layout, their eight partners
    const int parts = a.r.interleaved ? a.dim >> 3 : (a.dim - half) >> 3;
    const int n = nt * heads * parts;
    for (int i = threadIdx.x; i < n; i += ROTARY_THREADS) {
      const int part = i % parts, th = i / parts, h = h0 + th % heads, t = th / heads;
      const long long xi = (t0 + t) * a.x_token + h * a.x_head, yi = (t0 + t) * a.y_token + h * a.y_head;
      // the eights of this thread: at 8 part, behind `half` from there in the half layout
      if (!PAGED_CHECK(&rotary_status, part >= 0 && h >= 0 && h < a.heads && t >= 0 && t < nt && 8 * part + (a.r.interleaved ? 8 : half + 8) <= a.dim)) continue;
      const float2 *cs = rotary_turns + t * half;
      float u[8], w[8];
      if (a.r.interleaved) {
        const int d = part << 3;
        load_eight<TYPE>(a.x, xi + d, u);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const bool in = d + j < a.r.dim;
          const float2 k = in ? cs[(d + j) >> 1] : make_float2(1.f, 0.f);
          w[j] = in ? rotary_first(u[j], u[j + 1], k) : u[j];
          w[j + 1] = in ? rotary_second(u[j + 1], u[j], k) : u[j + 1];
        }
        store_eight<TYPE>(a.y, yi + d, w);
      } else if ((part << 3) < half) {
        const int d = part << 3;
        float v[8], z[8];
        load_eight<TYPE>(a.x, xi + d, u);
        load_eight<TYPE>(a.x, xi + d + half, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 k = cs[d + j];
          w[j] = rotary_first(u[j], v[j], k);
          z[j] = rotary_second(v[j], u[j], k);
        }
        store_eight<TYPE>(a.y, yi + d, w);
        store_eight<TYPE>(a.y, yi + d + half, z);
      } else { // behind the rotated part
        const int d = half + (part << 3);
        load_eight<TYPE>(a.x, xi + d, u);
        store_eight<TYPE>(a.y, yi + d, u);
      }
    }
  }); else {
    // one thread: one pair, or one element behind the rotated part
    const int parts = a.dim - half, n = nt * heads * parts;
    for (int i = threadIdx.x; i < n; i += ROTARY_THREADS) {
      const int part = i % parts, th = i / parts, h = h0 + th % heads, t = th / heads;
      const long long xi = (t0 + t) * a.x_token + h * a.x_head, yi = (t0 + t) * a.y_token + h * a.y_head;
      if (!PAGED_CHECK(&rotary_status, part >= 0 && h >= 0 && h < a.heads && t >= 0 && t < nt && half + part < a.dim)) continue;
      if (part < half) {
        const int d = a.r.interleaved ? 2 * part : part, e = a.r.interleaved ? d + 1 : d + half;
        const float2 k = rotary_turns[t * half + part];
        const float u = load_one(a.x, xi + d, a.type), v = load_one(a.x, xi + e, a.type);
        store_one(a.y, yi + d, a.type, rotary_first(u, v, k));
        store_one(a.y, yi + e, a.type, rotary_second(v, u, k));
      } else {
        const int d = half + part;
        store_one(a.y, yi + d, a.type, load_one(a.x, xi + d, a.type));
      }
    }
  }
}

} // namespace aq
