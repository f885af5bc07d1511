// Attention of one token over the pages, in its simplest form: a block per (sequence, query
// head), 128 tokens at a time, one thread per token for the scores and one per coordinate for
// the values, running maximum and sum.
#pragma once
#include "paged.cuh"

namespace aq {

struct AttendLaunch {
  PagedView c;
  RotaryView r;
  TableView table;
  const int *lengths;
  const void *q;
  void *out;
  long long q_seq, q_head, out_seq, out_head;
  int n_seqs, q_heads, group, type;
  float scale;
  float *workspace;
  int q_vec, out_vec;
};

constexpr int ATTEND_THREADS = 128;

__global__ void __launch_bounds__(ATTEND_THREADS) paged_attend_kernel(const AttendLaunch a, int P, int kb, int vb) {
  __shared__ float x[256], acc[256], weight[ATTEND_THREADS], red[8];
  const int b = blockIdx.x / a.q_heads, j = blockIdx.x % a.q_heads, h = j / a.group, tid = threadIdx.x;
  const long long room = (long long)a.table.width << a.c.page_shift;
  long long n = a.lengths[b];
  if (n < 0 || n > room) { if (tid == 0) atomicOr(a.c.status, PAGED_BAD_POSITION); n = n < 0 ? 0 : room; }
  const int dim = a.c.dim, half = a.r.dim >> 1;
  const long long qi = b * a.q_seq + j * a.q_head;
  for (int d = tid; d < P; d += ATTEND_THREADS) {
    float v = d < dim ? load_one(a.q, qi + d, a.type) : 0.f;
    if (d < a.r.dim) {
      const int pair = a.r.interleaved ? d >> 1 : d % half;
      const bool first = a.r.interleaved ? !(d & 1) : d < half;
      const int e = a.r.interleaved ? d ^ 1 : first ? d + half : d - half;
      const float2 k = rotary_turn(a.r, pair, n - 1);
      const float o = load_one(a.q, qi + e, a.type);
      v = first ? rotary_first(v, o, k) : rotary_second(v, o, k);
    }
    x[d] = v * sign_of(a.c.signs + h * (P / 32), d);
    acc[d] = 0.f;
  }
  __syncthreads();
  block_butterflies(x, P);
  float m = -1e30f, l = 0.f;
  const int *row = a.table.entries + b * a.table.stride;
  const int kr = P * kb / 8, vr = P * vb / 8;
  for (long long t0 = 0; t0 < n; t0 += ATTEND_THREADS) {
    int page = 0, off = 0;
    bool ok = t0 + tid < n;
    if (ok) ok = find_slot(a.c, row, a.table.width, t0 + tid, page, off);
    const long long slot = (((long long)page * a.c.heads + h) << a.c.page_shift) + off;
    float s = -INFINITY;
    if (ok) {
      const uint8_t *k = a.c.k_pages + slot * kr;
      float dot = 0.f;
      for (int d = 0; d < P; ++d) dot = fmaf(x[d], c_cb[kb - 2][unpack_at(k, d, kb)], dot);
      s = dot * (a.scale / P) * a.c.k_scales[slot];
    }
    float top = warp_max(s);
    if ((tid & 31) == 0) red[tid >> 5] = top;
    __syncthreads();
    top = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
    const float p = ok ? expf(s - top) : 0.f, old = expf(m - top);
    const float sum = warp_sum(p);
    if ((tid & 31) == 0) red[4 + (tid >> 5)] = sum;
    weight[tid] = ok ? p * a.c.v_scales[slot] : 0.f;
    __syncthreads();
    l = l * old + red[4] + red[5] + red[6] + red[7];
    m = top;
    for (int d = tid; d < P; d += ATTEND_THREADS) {
      float v = acc[d] * old;
      for (int i = 0; i < ATTEND_THREADS && t0 + i < n; ++i) {
        int pg = row[(t0 + i) >> a.c.page_shift];
        if (pg < 0 || pg >= a.c.n_pages) continue;
        const long long at = (((long long)pg * a.c.heads + h) << a.c.page_shift) + ((t0 + i) & (a.c.page_size - 1));
        v = fmaf(weight[i], c_cb[vb - 2][unpack_at(a.c.v_pages + at * vr, d, vb)], v);
      }
      acc[d] = v;
    }
    __syncthreads();
  }
  block_butterflies(acc, P);
  const float inv = n > 0 ? 1.f / (l * P) : 0.f;
  for (int d = tid; d < dim; d += ATTEND_THREADS)
    store_one(a.out, b * a.out_seq + j * a.out_head + d, a.type, n > 0 ? acc[d] * inv * sign_of(a.c.signs + h * (P / 32), d) : 0.f);
}

} // namespace aq
